"""Error bounds of AdamW with fp32 moments that scale with the values, and mistakes that they find (planted in a plain fp32 form on
the host).  ``test_adamw_bounds_gpu.py`` holds the kernel to them.

Roundings, u = 2^-24, t steps so far, to first order with everything rounded up:

* g' = coef g: the coefficient once, the product once: 2 u.
* m = b1 m + (1 - b1) g': b1, 1 - b1 and the product once each, the sum once: a step adds at most 5 u of
  a = b1 a + (1 - b1) |g'| (the same recursion on magnitudes) to b1 times the error before: 8 t u a holds it.
* v = b2 v + (1 - b2) g'^2: all terms are positive; a new term carries 4 u from g', 3 u of its own products and 1 u of the sum, an old
  one 2 u more per step: 8 t u v.
* a step: m's error over the denominator; the denominator is off by half of v's relative error and 6 u (square root to 2 u, correction,
  sum, reciprocal to 2 u), the products by 3 u: |step| (16 u + 4 t u) + step size * 8 t u a / denominator.
* p: p (1 - lr decay) and the sum: 4 u of the larger of both p, added up over the steps."""
import math

import pytest
import torch

U = 2.0 ** -24
LR, BETAS, EPS, DECAY = 1e-2, (0.9, 0.999), 1e-8, 0.1
SIZES = [1, 3, 255, 256, 257, 4097, 20000, 7, 64]


def gradients(t, clip):
    """Of step ``t``: tensors of their own magnitudes, and the coefficient."""
    gen = torch.Generator().manual_seed(100 + t)
    out = [0.3 * torch.randn(n, generator=gen) * 10.0 ** (k % 3 - 1) for k, n in enumerate(SIZES)]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in out))
    return out, (min(1.0, clip / (norm + 1e-6)) if clip else 1.0), norm


def parameters():
    gen = torch.Generator().manual_seed(7)
    return [0.1 * torch.randn(n, generator=gen) for n in SIZES]


class Bounds:
    """The formulas in 64 bits with their error bounds, step by step."""

    def __init__(self, p):
        self.p = [x.double() for x in p]
        self.m, self.v, self.a, self.tol_p = ([torch.zeros_like(x) for x in self.p] for _ in range(4))
        self.t = 0

    def step(self, grads, coef):
        self.t = t = self.t + 1
        size = LR / (1 - BETAS[0] ** t)
        for k, g in enumerate(grads):
            g = g.double() * coef
            self.m[k] = BETAS[0] * self.m[k] + (1 - BETAS[0]) * g
            self.v[k] = BETAS[1] * self.v[k] + (1 - BETAS[1]) * g * g
            self.a[k] = BETAS[0] * self.a[k] + (1 - BETAS[0]) * g.abs()
            denom = (self.v[k] / (1 - BETAS[1] ** t)).sqrt() + EPS
            step = size * self.m[k] / denom
            new = self.p[k] * (1 - LR * DECAY) - step
            self.tol_p[k] += 4 * U * torch.maximum(self.p[k].abs(), new.abs()) + step.abs() * (16 + 4 * t) * U + size * 8 * t * U * self.a[k] / denom
            self.p[k] = new

    def outside(self, p, m, v):
        """Names of what leaves its bound."""
        wrong = set()
        for k in range(len(self.p)):
            for name, got, want, tol in (("m", m[k], self.m[k], 8 * self.t * U * self.a[k]), ("v", v[k], self.v[k], 8 * self.t * U * self.v[k]),
                                         ("p", p[k], self.p[k], self.tol_p[k])):
                if not bool(((got.double() - want).abs() <= tol + 1e-38).all()):
                    wrong.add(name)
        return wrong


def plain(steps, clip, mistake=""):
    """fp32 on the host, with a mistake."""
    p = parameters()
    m, v = ([torch.zeros_like(x) for x in p] for _ in range(2))
    bounds = Bounds(p)
    for t in range(1, steps + 1):
        grads, coef, _ = gradients(t, clip)
        bounds.step(grads, coef)
        for k, g in enumerate(grads):
            h = g * torch.tensor(coef, dtype=torch.float32)
            m[k] = BETAS[0] * m[k] + (1 - BETAS[0]) * (g if mistake == "m unclipped" else h)
            square = g * h if mistake == "v half clipped" else g * g if mistake == "v unclipped" else h * h
            v[k] = BETAS[1] * v[k] + (1 - BETAS[1]) * square
            if mistake == "v stays zero":
                v[k] = torch.zeros_like(v[k])
            if mistake == "v in 16 bits":
                v[k] = v[k].bfloat16().float()
            if mistake == "m a little off":
                m[k] = m[k] * (1 + 2.0 ** -16)
            correction = 1.0 if mistake == "no correction" and t > 3 else math.sqrt(1 - BETAS[1] ** t)
            step = LR / (1 - BETAS[0] ** t) * m[k] / (v[k].sqrt() / correction + EPS)
            p[k] = p[k] * (1 - (0.0 if mistake == "no decay" else LR * DECAY)) - step
    return bounds.outside(p, m, v)


@pytest.mark.parametrize("clip", [None, 0.5])
def test_plain_fp32_is_within(clip):
    assert plain(6, clip) == set()


@pytest.mark.parametrize("mistake,found", [("m unclipped", "m"), ("v half clipped", "v"), ("v unclipped", "v"), ("v stays zero", "v"),
                                           ("v in 16 bits", "v"), ("m a little off", "m"), ("no correction", "p"), ("no decay", "p")])
def test_mistakes_are_found(mistake, found):
    assert found in plain(6, 0.5, mistake)
