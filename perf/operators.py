"""Cases and plain forms of the training operators around the U-Net: group normalisation with an activation on
plane-record activations (forward and backward), and AdamW over many tensors with states in 32 or in 8 bits.

A plane-record tensor is ``[N][planes][H][W][record]``: 16 bf16 or 8 fp32 channels per record, channel ``c`` in plane
``c // record``; record slots past the channel count hold zeros.  Per-channel vectors are padded to a multiple of 32.

The 8-bit states are e4m3 codes with one fp32 scale per 256 consecutive elements of a tensor (value = code * scale).  The
scale is the smallest power of two that brings the block's largest magnitude to 448 or below; a magnitude is rounded up or
down at random in proportion (16 bits of a hash of element, step and seed), a second moment above zero keeps at least the
smallest code.
"""
import math
import random

import torch

own = False

EPS = 1e-5
BETA1, BETA2, ADAM_EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-3, 0.01
BLOCK, TOP = 256, 448.0
FIRST_STEP = 100          # the optimizer is met in the middle of a run: its moments are not zero

# the widest listed passes, which no drawn case exceeds
MOST_BYTES = 256 * 32 * 6 * 4096 * 2
MOST_PARAMETERS = 125_000_000

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one small profile through the bottleneck of a two-level net: a call whose launches cost more than its bytes
        {"name": "gn_fwd_f32_small", "op": "gn_fwd", "dtype": "f32", "n": 2, "c": 128, "groups": 8, "h": 5, "w": 64, "act": "relu"},
        # train.py's batch at full scan resolution: groups of 4 channels, four of them in a record
        {"name": "gn_fwd_bf16_batch16", "op": "gn_fwd", "dtype": "bf16", "n": 16, "c": 32, "groups": 8, "h": 5, "w": 4096, "act": "relu"},
        # groups of three channels across piece borders, an odd scan length, six dyes, SiLU
        {"name": "gn_fwd_f32_odd", "op": "gn_fwd", "dtype": "f32", "n": 7, "c": 24, "groups": 8, "h": 6, "w": 333, "act": "silu"},
        # the inference / training batch of the benchmark at level 0, six dyes
        {"name": "gn_fwd_bf16_batch256", "op": "gn_fwd", "dtype": "bf16", "n": 256, "c": 32, "groups": 8, "h": 6, "w": 4096, "act": "relu"},
        # backward of a middle level at train.py's batch
        {"name": "gn_bwd_bf16_batch16", "op": "gn_bwd", "dtype": "bf16", "n": 16, "c": 128, "groups": 8, "h": 5, "w": 1024, "act": "relu"},
        # backward in the reference's precision with a smooth activation, odd sizes
        {"name": "gn_bwd_f32_odd", "op": "gn_bwd", "dtype": "f32", "n": 5, "c": 48, "groups": 6, "h": 5, "w": 517, "act": "silu"},
        # backward of the bottleneck at the benchmark's batch: groups of four whole planes
        {"name": "gn_bwd_bf16_batch256", "op": "gn_bwd", "dtype": "bf16", "n": 256, "c": 512, "groups": 8, "h": 6, "w": 256, "act": "relu"},
        # a two-level net's parameters: a step that is all latency
        {"name": "adamw_f32_small", "op": "adamw", "bits": 32, "p": "f32", "g": "f32", "filters": 8, "depth": 2, "clip": 0.0},
        # the shipped net (depth 4, 32 filters, 3x5), gradients clipped to a global norm
        {"name": "adamw_f32_unet", "op": "adamw", "bits": 32, "p": "f32", "g": "f32", "filters": 32, "depth": 4, "clip": 1.0},
        # a ragged list of bf16 tensors from one element up (vectors, odd matrices)
        {"name": "adamw_bf16_ragged", "op": "adamw", "bits": 32, "p": "bf16", "g": "bf16", "tensors": 150, "largest": 1_500_000, "layout": 3, "clip": 0.0},
        # the shipped net with 8-bit moments and clipping
        {"name": "adamw8_unet", "op": "adamw", "bits": 8, "p": "f32", "g": "f32", "filters": 32, "depth": 4, "clip": 1.0},
        # a net of 104 filters: 128 million parameters, where 8-bit moments are there for the memory
        {"name": "adamw8_wide", "op": "adamw", "bits": 8, "p": "f32", "g": "f32", "filters": 104, "depth": 4, "clip": 0.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.55:
        while True:
            dtype, groups = rng.choice(["f32", "bf16"]), rng.choice([1, 2, 3, 4, 6, 8, 8, 16, 32])
            c = groups * rng.choice([1, 2, 3, 4, 4, 5, 8, 12, 16, 32, 64])
            n, h, w = _log_int(rng, 1, 256), rng.choice([1, 2, 3, 5, 5, 6, 6, 7]), _log_int(rng, 1, 4096)
            size = 4 if dtype == "f32" else 2
            if 64 <= n * c * h * w and n * ((c + 15) // 16 * 16) * h * w * size <= MOST_BYTES and 8 <= c <= 1024:
                break
        return {"op": rng.choice(["gn_fwd", "gn_bwd"]), "dtype": dtype, "n": n, "c": c, "groups": groups,
                "h": h, "w": w, "act": rng.choice(["relu", "relu", "silu", "none"])}
    p = rng.choice(["f32", "f32", "bf16"])
    return {"op": "adamw", "bits": rng.choice([32, 8]), "p": p, "g": rng.choice([p, "f32"]), "tensors": _log_int(rng, 1, 300),
            "largest": _log_int(rng, 100, 2_000_000), "layout": rng.randrange(1 << 30), "clip": rng.choice([0.0, 0.0, 1.0, 100.0])}


# ---- sizes ---------------------------------------------------------------------------------------------------------------

def _planes(case):
    record = 16 if case["dtype"] == "bf16" else 8
    return (case["c"] + record - 1) // record, record


def _tensor_sizes(case):
    """Element counts of the parameter tensors, and the weight decay of each: the weights first, then the vectors and single
    values, which are not decayed."""
    sizes = []
    if "filters" in case:
        f, depth, taps = case["filters"], case["depth"], 15

        def double_conv(cin, cout):
            for ci in (cin, cout):
                sizes.extend([cout * ci * taps, cout, cout, cout])       # weight, bias, scale and offset of the norm

        cin = 1
        for i in range(depth + 1):
            double_conv(cin, f << i)
            cin = f << i
        for i in range(depth):
            cout = f << (depth - 1 - i)
            sizes.extend([cin * cout * 2, cout])                          # transposed convolution
            double_conv(2 * cout, cout)
            cin = cout
        sizes.extend([f, 1])
    else:
        rng = random.Random(case["layout"])
        while len(sizes) < case["tensors"]:
            n = _log_int(rng, 1, case["largest"])
            if sum(sizes) + n <= MOST_PARAMETERS:
                sizes.append(n)
            else:
                break
    weights, vectors = [n for n in sizes if n > 2048], [n for n in sizes if n <= 2048]
    return weights + vectors, [DECAY] * len(weights) + [0.0] * len(vectors)


def _offsets(sizes):
    """Start of every tensor in the flat buffers: multiples of 256 elements, so that a block of the 8-bit states is one row."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return starts, at


def work(case):
    if case["op"] == "adamw":
        n = sum(_tensor_sizes(case)[0])
        p, g = (4 if case["p"] == "f32" else 2), (4 if case["g"] == "f32" else 2)
        state = 8 if case["bits"] == 32 else 2 + 8 / BLOCK
        return {"bytes": n * (2 * p + g + 2 * state), "flops": 15 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    elements = case["n"] * case["c"] * case["h"] * case["w"]
    tensors, flops = (2, 9) if case["op"] == "gn_fwd" else (3, 18)
    vectors = case["n"] * (case["c"] + case["groups"]) * 2 * 4
    return {"bytes": tensors * elements * size + vectors, "flops": flops * elements}


# ---- what a program has in hand --------------------------------------------------------------------------------------------

def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=device)

    if case["op"] == "adamw":
        sizes, decay = _tensor_sizes(case)
        starts, total = _offsets(sizes)
        lengths = torch.tensor([(n + BLOCK - 1) // BLOCK * BLOCK for n in sizes], device=device)
        real = torch.arange(total, device=device) - torch.repeat_interleave(torch.tensor(starts, device=device), lengths, output_size=total)
        real = real < torch.repeat_interleave(torch.tensor(sizes, device=device), lengths, output_size=total)
        # gradients: every tensor has its own magnitude (deep layers' are smaller), elements of a tensor spread by some octaves
        spread = torch.exp(normal(len(sizes)) - 5.0)
        sigma = torch.repeat_interleave(spread, lengths, output_size=total) * torch.exp(0.7 * normal(total)) * real
        s = {"case": dict(case), "sizes": sizes, "starts": starts, "decay": decay, "lengths": lengths,
             "decays": torch.tensor(decay, device=device, dtype=torch.float32), "step": FIRST_STEP, "seed": seed & 0xFFFF, "total": total,
             "p": (0.05 * normal(total) * real).to(TYPES[case["p"]]), "g": (sigma * normal(total)).to(TYPES[case["g"]])}
        m, v = 0.3 * sigma * normal(total), sigma * sigma * (0.3 + uniform(total))
        if case["bits"] == 32:
            s["m"], s["v"] = m, v
        else:
            for name, x in (("m", m.view(-1, BLOCK)), ("v", v.view(-1, BLOCK))):
                scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(1) / TOP)))
                s[name] = (x / scale[:, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(-1)
                s[name + "_scale"] = scale
            positive = (v > 0) & (s["v"].float() == 0)
            s["v"].view(torch.uint8)[positive] = 1
        if own:
            s["optimizer"] = _own_optimizer(s)
        return s

    n, c, h, w, groups = case["n"], case["c"], case["h"], case["w"], case["groups"]
    planes, record = _planes(case)
    channels = torch.arange(planes * record, device=device).view(planes, 1, 1, record) < c
    # a convolution's output on an electropherogram: channels of their own mean and gain, a quiet baseline, a few high peaks
    gain = torch.exp(0.5 * normal(planes, 1, 1, record))
    y = normal(n, planes, h, w, record) * gain + 0.6 * normal(planes, 1, 1, record)
    y += 12.0 * gain * (uniform(n, 1, h, w, 1) < 0.01)
    y = (y * channels).to(TYPES[case["dtype"]])
    del gain
    s = {"case": dict(case), "x": y, "gamma": 1.0 + 0.2 * normal(c), "beta": 0.2 * normal(c)}
    if case["op"] == "gn_bwd":
        s["g"] = (normal(n, planes, h, w, record) * channels * 1e-3).to(TYPES[case["dtype"]])
        # what the forward pass kept: statistics per image and group, the fused scale and shift per image and channel
        mean, second = [], []
        for image in y.split(8):                                          # a few images at a time: the sums are in 64 bits
            xg = image.double().movedim(-1, 2).reshape(image.shape[0], planes * record, h * w)[:, :c].reshape(image.shape[0], groups, -1)
            mean.append(xg.mean(-1))
            second.append(xg.var(-1, unbiased=False))
        mean, rstd = torch.cat(mean).float(), (torch.cat(second) + EPS).rsqrt().float()
        s["mean"], s["rstd"] = mean, rstd
        per = c // groups
        pad = (c + 31) // 32 * 32
        s["scale"], s["shift"] = torch.zeros(n, pad, device=device), torch.zeros(n, pad, device=device)
        s["scale"][:, :c] = s["gamma"] * rstd.repeat_interleave(per, 1)
        s["shift"][:, :c] = s["beta"] - mean.repeat_interleave(per, 1) * s["scale"][:, :c]
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------------

def _own_optimizer(s):
    from dnanet_amd.optim import HipAdamW
    case = s["case"]
    params, grads = ([s[name][at:at + n] for n, at in zip(s["sizes"], s["starts"])] for name in ("p", "g"))
    weights = sum(1 for d in s["decay"] if d)
    groups = [{"params": params[:weights], "weight_decay": DECAY}, {"params": params[weights:], "weight_decay": 0.0}]
    if s["p"].dtype == s["g"].dtype:
        for p, g in zip(params, grads):
            p.grad = g
    else:                                       # torch refuses a .grad of another type: a group's own list
        groups[0]["grads"], groups[1]["grads"] = grads[:weights], grads[weights:]
    opt = HipAdamW([group for group in groups if group["params"]], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                   state_bits=case["bits"], max_grad_norm=case["clip"] or None, seed=s["seed"])
    opt.step_count = FIRST_STEP
    opt.exp_avg.copy_(s["m"])
    opt.exp_avg_sq.copy_(s["v"])
    if case["bits"] == 8:
        opt.exp_avg_scale.copy_(s["m_scale"])
        opt.exp_avg_sq_scale.copy_(s["v_scale"])
    return opt


def _run_own(s):
    case = s["case"]
    if case["op"] == "adamw":
        opt = s["optimizer"]
        opt.step()
        out = {"p": s["p"], "m": opt.exp_avg, "v": opt.exp_avg_sq}
        if case["bits"] == 8:
            out["m_scale"], out["v_scale"] = opt.exp_avg_scale, opt.exp_avg_sq_scale
        if case["clip"]:
            out["norm"] = opt.grad_norm
        return out
    from dnanet_amd.group_norm import GroupNormStats, group_norm_act, group_norm_act_backward
    from dnanet_amd.hip import PlaneBuffer
    x = PlaneBuffer.wrap(s["x"]).ref(case["c"])
    if case["op"] == "gn_fwd":
        a, stats = group_norm_act(x, s["gamma"], s["beta"], case["groups"], eps=EPS, activation=case["act"])
        return {"a": a.data, "mean": stats.mean, "rstd": stats.rstd, "scale": stats.scale, "shift": stats.shift}
    stats = GroupNormStats(s["mean"], s["rstd"], s["scale"], s["shift"], case["groups"], case["act"])
    dx, dgamma, dbeta = group_norm_act_backward(PlaneBuffer.wrap(s["g"]).ref(case["c"]), x, s["gamma"], stats)
    return {"dx": dx.data, "dgamma": dgamma, "dbeta": dbeta}


# ---- the plain forms ---------------------------------------------------------------------------------------------------------

def _channels_first(x, c):
    n, planes, h, w, record = x.shape
    return x.float().permute(0, 1, 4, 2, 3).reshape(n, planes * record, h * w)[:, :c]


def _records(x, like):
    n, planes, h, w, record = like.shape
    full = torch.zeros(n, planes * record, h * w, device=x.device, dtype=torch.float32)
    full[:, :x.shape[1]] = x
    return full.view(n, planes, record, h, w).permute(0, 1, 3, 4, 2).to(like.dtype).contiguous()


def _plain_gn_fwd(s):
    case = s["case"]
    n, c, groups = case["n"], case["c"], case["groups"]
    x = _channels_first(s["x"], c)
    per, pad = c // groups, (c + 31) // 32 * 32
    xg = x.reshape(n, groups, -1)
    mean = xg.mean(-1)
    var = ((xg - mean[..., None]) * (xg - mean[..., None])).mean(-1)
    rstd = 1.0 / torch.sqrt(var + EPS)
    scale, shift = torch.zeros(n, pad, device=x.device), torch.zeros(n, pad, device=x.device)
    scale[:, :c] = s["gamma"] * rstd.repeat_interleave(per, 1)
    shift[:, :c] = s["beta"] - mean.repeat_interleave(per, 1) * scale[:, :c]
    z = x * scale[:, :c, None] + shift[:, :c, None]
    if case["act"] == "relu":
        z = torch.where(z < 0, torch.zeros_like(z), z)
    elif case["act"] == "silu":
        z = z / (1.0 + torch.exp(-z))
    return {"a": _records(z, s["x"]), "mean": mean, "rstd": rstd, "scale": scale, "shift": shift}


def _plain_gn_bwd(s):
    case = s["case"]
    n, c, groups = case["n"], case["c"], case["groups"]
    per = c // groups
    x, g = _channels_first(s["x"], c), _channels_first(s["g"], c)
    scale, shift = s["scale"][:, :c, None], s["shift"][:, :c, None]
    if case["act"] == "relu":
        # the sign of x * scale + shift: in 64 bits, where a value next to the border keeps its side
        dz = torch.where(x.double() * scale + shift <= 0, torch.zeros_like(g), g)
    elif case["act"] == "silu":
        z = x * scale + shift
        sig = 1.0 / (1.0 + torch.exp(-z))
        dz = g * sig * (1.0 + z * (1.0 - sig))
    else:
        dz = g
    mean, rstd = s["mean"].repeat_interleave(per, 1)[..., None], s["rstd"].repeat_interleave(per, 1)[..., None]
    xhat = (x - mean) * rstd
    s1 = dz.sum(-1, dtype=torch.float64)                          # per image and channel
    s2 = (dz * xhat).sum(-1, dtype=torch.float64)
    count = per * x.shape[-1]
    gamma = s["gamma"].double()
    c1 = ((s1 * gamma).view(n, groups, per).sum(-1) / count).float().repeat_interleave(per, 1)[..., None]
    c2 = ((s2 * gamma).view(n, groups, per).sum(-1) / count).float().repeat_interleave(per, 1)[..., None]
    dx = rstd * (s["gamma"][:, None] * dz - c1 - xhat * c2)
    return {"dx": _records(dx, s["x"]), "dgamma": s2.sum(0).float(), "dbeta": s1.sum(0).float()}


def _hash(index, step, seed):
    """32 mixed bits of every element index; whole-number products and shifts of 32 bits, held in 64."""
    x = (index + step * 0x9E3779B9 + seed * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _encode(x, bits, floor):
    """Magnitudes over the block's scale -> e4m3 codes (0..126), rounded up where ``bits`` (16 of them) says so."""
    small = x < 2.0 ** -6
    y = torch.where(small, x + 2.0 ** -6, x)                       # below the smallest normal value the steps are even
    code = ((y.view(torch.int32) + (bits << 4).to(torch.int32)) >> 20) - torch.where(small, 121 * 8, 120 * 8)
    code = code.clamp(max=126)
    return torch.where(floor, code.clamp(min=1), code)


def _plain_adamw(s):
    case = s["case"]
    s["step"] += 1
    t = s["step"]
    p, g = s["p"].float(), s["g"].float()
    out = {}
    if case["clip"]:
        norm = torch.sqrt((g.double() * g.double()).sum())
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0).float()
        out["norm"] = norm.float()
    bc1, bc2 = 1.0 - BETA1 ** t, 1.0 - BETA2 ** t
    if case["bits"] == 32:
        m = BETA1 * s["m"] + (1.0 - BETA1) * g
        v = BETA2 * s["v"] + (1.0 - BETA2) * g * g
        s["m"], s["v"] = m, v
    else:
        # new moments in 64 bits: a magnitude next to a rounding border falls on the same side whoever computes it
        gd = g.double().view(-1, BLOCK)
        if case["clip"]:
            gd = s["g"].double().view(-1, BLOCK) * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0).float().double()
        old_m = s["m"].float().double().view(-1, BLOCK) * s["m_scale"].double()[:, None]
        old_v = s["v"].float().double().view(-1, BLOCK) * s["v_scale"].double()[:, None]
        m = BETA1 * old_m + (1.0 - BETA1) * gd
        v = BETA2 * old_v + (1.0 - BETA2) * gd * gd
        del old_m, old_v, gd
        index = torch.arange(s["total"], device=p.device)
        index = index - torch.repeat_interleave(torch.tensor(s["starts"], device=p.device), s["lengths"], output_size=s["total"])
        number = torch.repeat_interleave(torch.arange(len(s["sizes"]), device=p.device), s["lengths"], output_size=s["total"])
        bits = _hash((index + number * 0xC2B2AE35) & 0xFFFFFFFF, t, s["seed"]).view(-1, BLOCK)
        del index, number
        for name, x, b in (("m", m, bits & 0xFFFF), ("v", v, bits >> 16)):
            y = x.abs().float()
            fraction, exponent = torch.frexp(y.amax(1))            # fraction in [0.5, 1); 448 = 0.875 * 2 ** 9
            exponent = (exponent - torch.where(fraction <= 0.875, 9, 8)).clamp(min=-126)
            scale = torch.where(fraction > 0, torch.ldexp(torch.ones_like(fraction), exponent), torch.zeros_like(fraction))
            y = y * torch.ldexp(torch.ones_like(fraction), -exponent)[:, None]
            code = _encode(y, b, (x > 0) & (scale > 0)[:, None] if name == "v" else torch.zeros_like(x, dtype=torch.bool))
            code = torch.where(x < 0, code + 128, code)
            s[name], s[name + "_scale"] = code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), scale
        m, v = m.float().view(-1), v.float().view(-1)
        out["m_scale"], out["v_scale"] = s["m_scale"], s["v_scale"]
    decay = torch.repeat_interleave(1.0 - LR * s["decays"], s["lengths"], output_size=s["total"])
    p = p * decay - (LR / bc1) * m / (torch.sqrt(v) / math.sqrt(bc2) + ADAM_EPS)
    s["p"].copy_(p)
    return {"p": s["p"], "m": s["m"], "v": s["v"], **out}


def run(s):
    if own:
        return _run_own(s)
    return {"gn_fwd": _plain_gn_fwd, "gn_bwd": _plain_gn_bwd, "adamw": _plain_adamw}[s["case"]["op"]](s)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    c, groups = case["c"], case["groups"]
    parts = []
    for lo in range(0, case["n"], 16):                             # 16 images at a time: 64-bit copies of the largest case are big
        rows = slice(lo, min(lo + 16, case["n"]))
        x = s["x"][rows].double().movedim(-1, 2).flatten(1, 2)[:, :c]          # images, channels, dyes, scans
        if case["op"] == "gn_fwd":
            var, mean = torch.var_mean(x.unflatten(1, (groups, c // groups)), dim=(2, 3, 4), correction=0)
            a = torch.nn.functional.group_norm(x, groups, s["gamma"].double(), s["beta"].double(), EPS)
            a = {"relu": torch.relu, "silu": torch.nn.functional.silu, "none": lambda z: z}[case["act"]](a)
            parts.append((a, mean, (var + EPS) ** -0.5))
        else:
            g = s["g"][rows].double().movedim(-1, 2).flatten(1, 2)[:, :c]
            per = c // groups
            z = x * s["scale"][rows, :c, None, None].double() + s["shift"][rows, :c, None, None].double()
            sig = torch.sigmoid(z)
            slope = {"relu": (z > 0).double(), "silu": sig + z * sig * (1 - sig), "none": torch.ones_like(z)}[case["act"]]
            xhat = ((x.unflatten(1, (groups, per)) - s["mean"][rows].double()[:, :, None, None, None])
                    * s["rstd"][rows].double()[:, :, None, None, None])
            dz = (g * slope).unflatten(1, (groups, per))
            weighted = dz * s["gamma"].double().view(1, groups, per, 1, 1)
            dx = (weighted - weighted.mean((2, 3, 4), keepdim=True) - xhat * (weighted * xhat).mean((2, 3, 4), keepdim=True))
            dx = dx * s["rstd"][rows].double()[:, :, None, None, None]
            parts.append((dx.flatten(1, 2), (dz * xhat).sum((0, 3, 4)).flatten(), dz.sum((0, 3, 4)).flatten()))
    planes, record = _planes(case)
    wide = torch.cat([torch.nn.functional.pad(p[0], (0, 0, 0, 0, 0, planes * record - c)) for p in parts])
    wide = wide.unflatten(1, (planes, record)).movedim(2, -1)
    if case["op"] == "gn_bwd":
        return {"dx": wide, "dgamma": sum(p[1] for p in parts), "dbeta": sum(p[2] for p in parts)}
    mean, rstd = torch.cat([p[1] for p in parts]), torch.cat([p[2] for p in parts])
    pad = (c + 31) // 32 * 32 - c
    scale = s["gamma"].double() * torch.repeat_interleave(rstd, c // groups, 1)
    shift = s["beta"].double() - torch.repeat_interleave(mean, c // groups, 1) * scale
    return {"a": wide, "mean": mean, "rstd": rstd, "scale": torch.nn.functional.pad(scale, (0, pad)),
            "shift": torch.nn.functional.pad(shift, (0, pad))}


def _exact_adamw(s):
    case, t = s["case"], s["step"] + 1
    g = s["g"].double()
    coefficient, norm = 1.0, None
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        coefficient = float(torch.tensor(min(1.0, case["clip"] / (float(norm) + 1e-6)), dtype=torch.float32))
    new_p = torch.zeros_like(g)
    out = {"m": torch.zeros_like(g), "v": torch.zeros_like(g)}
    eight = case["bits"] == 8
    if eight:
        out["m_scale"], out["v_scale"] = torch.zeros_like(s["m_scale"], dtype=torch.float64), torch.zeros_like(s["v_scale"], dtype=torch.float64)
    for k, (n, at) in enumerate(zip(s["sizes"], s["starts"])):     # tensor by tensor
        own_rows = slice(at, at + n)
        moments = {}
        for name, beta, x in (("m", BETA1, g[own_rows] * coefficient), ("v", BETA2, (g[own_rows] * coefficient) ** 2)):
            old = s[name][own_rows].float().double()
            if eight:
                old = old * s[name + "_scale"][at // BLOCK:at // BLOCK + (n + BLOCK - 1) // BLOCK].double().repeat_interleave(BLOCK)[:n]
            moments[name] = old * beta + x * (1.0 - beta)
        if eight:
            key = torch.arange(n, device=g.device) + (k * 0xC2B2AE35 & 0xFFFFFFFF) + t * 0x9E3779B9 + s["seed"] * 0x85EBCA6B
            for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
                key = key % (1 << 32)
                key = (key ^ (key >> shift)) * factor
            key = key % (1 << 32)
            key = key ^ (key >> 16)
            for name, chance in (("m", key % 65536), ("v", key // 65536)):
                x = torch.nn.functional.pad(moments[name], (0, -n % BLOCK)).view(-1, BLOCK)
                biggest = x.abs().max(1).values
                scale = 2.0 ** torch.ceil(torch.log2(biggest / TOP)) * (biggest > 0)
                ratio = (x.abs() / scale.clamp(min=1e-300)[:, None]).flatten()[:n].float().double()
                exponent = torch.floor(torch.log2(ratio.clamp(min=2.0 ** -6)))
                exponent = exponent - (2.0 ** exponent > ratio.clamp(min=2.0 ** -6)).double()
                unit = 2.0 ** (exponent - 3)
                value = torch.floor(ratio / unit + chance.double() / 65536) * unit
                value = value.clamp(max=TOP)
                if name == "v":
                    value = torch.where(moments[name] > 0, value.clamp(min=2.0 ** -9), value)
                out[name][own_rows] = torch.where(moments[name] < 0, -value, value)
                out[name + "_scale"][at // BLOCK:at // BLOCK + scale.numel()] = scale
        else:
            out["m"][own_rows], out["v"][own_rows] = moments["m"], moments["v"]
        step = moments["m"] / (1.0 - BETA1 ** t) / ((moments["v"] / (1.0 - BETA2 ** t)).sqrt() + ADAM_EPS)
        new_p[own_rows] = s["p"][own_rows].double() * (1.0 - LR * s["decay"][k]) - LR * step
    out["p"] = new_p
    if norm is not None:
        out["norm"] = norm
    return out
