// GroupNorm with an activation on plane-record tensors (see common.h), forward and backward.
//
// Per image n and group g of C / groups channels, over the group's channels and all pixels:
//   mean, var = mean((x - mean)^2), rstd = 1 / sqrt(var + eps)
//   scale[n][c] = gamma[c] * rstd, shift[n][c] = beta[c] - mean * scale[n][c]
//   z = x * scale + shift, a = act(z)
// and for g = dL/da, with dz = g * act'(z) and xhat = (x - mean) * rstd:
//   dbeta[c] = sum dz, dgamma[c] = sum dz * xhat                                     (over images and pixels)
//   dx = rstd * (gamma * dz - mean_group(gamma * dz) - xhat * mean_group(gamma * dz * xhat))
// z comes from the saved scale / shift by one fma, whose sign is that of the exact x * scale + shift: the ReLU mask of the
// backward pass does not depend on who computes it.
//
// A plane of one image is a contiguous run of 16-byte pieces.  It is cut into segments that a block holds in registers, so
// that the variance is taken around the segment's own mean (a sum of squares would cancel where mean^2 >> var); the
// segments' (mean, M2) pairs are joined in fp64.  All sums run in a fixed order: results are bitwise reproducible.
#include <algorithm>
#include "common.h"
#include "dnanet_hip.h"

namespace {

constexpr int GN_THREADS = 256;
constexpr int GN_R = 8;                                   // pieces per thread and segment
constexpr int GN_SEG = GN_THREADS * GN_R;

struct GnShape {
  int N, C, G, P;          // images, channels, groups, planes
  int cpg, cpad;           // channels per group, dn_channel_pad(C)
  int npieces;             // 16-byte pieces of a plane of one image: 2 * H * W
  int nseg, seg_len;       // segments per plane, pieces per segment (even)
};

template <int ACT> __device__ __forceinline__ float gn_act(float z) {
  if constexpr (ACT == DN_ACT_RELU) return z < 0.f ? 0.f : z;            // NaN stays NaN
  if constexpr (ACT == DN_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  return z;
}
template <int ACT> __device__ __forceinline__ float gn_act_grad(float z, float g) {
  if constexpr (ACT == DN_ACT_RELU) return z <= 0.f ? 0.f : g;
  if constexpr (ACT == DN_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return g * s * fmaf(z, 1.f - s, 1.f);
  }
  return g;
}

// Sum of KV x PN per-thread accumulators over the block; threads of even / odd index hold the two halves of the record.
// red: KV * EPR floats per wave.  The result lands in out[c * KV + kv] (LDS), valid after the call's last barrier.
template <int KV, int PN> __device__ __forceinline__ void gn_block_sum(float (&acc)[KV][PN], float* red, float* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int kv = 0; kv < KV; ++kv)
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      float v = acc[kv][j];
#pragma unroll
      for (int m = 2; m < 64; m <<= 1) v += __shfl_xor(v, m);
      if (lane < 2) red[(wave * 2 * PN + lane * PN + j) * KV + kv] = v;
    }
  __syncthreads();
  if ((int)threadIdx.x < 2 * PN * KV) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < GN_THREADS / 64; ++w) s += red[w * 2 * PN * KV + threadIdx.x];
    out[threadIdx.x] = s;
  }
  __syncthreads();
}

__device__ __forceinline__ double gn_block_sum64(double v, double* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < GN_THREADS / 64; ++w) v += red[w];
  return v;
}

struct GnUnit { int seg, plane; long n, cell; int lo, hi; };
__device__ __forceinline__ GnUnit gn_unit(const GnShape& s) {
  GnUnit u;
  const long b = blockIdx.x;
  u.seg = (int)(b % s.nseg);
  const long r = b / s.nseg;
  u.plane = (int)(r % s.P);
  u.n = r / s.P;
  u.cell = b;
  u.lo = u.seg * s.seg_len;
  u.hi = min(s.npieces, u.lo + s.seg_len);
  return u;
}

// part[cell][channel of the plane] = (mean, M2) of the segment
template <typename T>
__global__ __launch_bounds__(GN_THREADS) void gn_stats_kernel(const unsigned char* x, int pt, int p0, GnShape s, float2* part) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  __shared__ float red[GN_THREADS / 64 * EPR], mean[EPR], m2[EPR];
  const GnUnit u = gn_unit(s);
  const unsigned char* base = x + (u.n * pt + p0 + u.plane) * s.npieces * 16;
  uint4 v[GN_R];
#pragma unroll
  for (int k = 0; k < GN_R; ++k) {
    const int i = u.lo + (int)threadIdx.x + k * GN_THREADS;
    v[k] = i < u.hi ? *(const uint4*)(base + (long)i * 16) : make_uint4(0, 0, 0, 0);
  }
  float acc[1][PN] = {};
#pragma unroll
  for (int k = 0; k < GN_R; ++k) {
    float f[PN];
    Piece<T>::unpack(v[k], f);
#pragma unroll
    for (int j = 0; j < PN; ++j) acc[0][j] += f[j];
  }
  gn_block_sum<1, PN>(acc, red, mean);
  const float count = (float)((u.hi - u.lo) / 2);
  const int pc = threadIdx.x & 1;
  float mu[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { mu[j] = mean[pc * PN + j] / count; acc[0][j] = 0.f; }
#pragma unroll
  for (int k = 0; k < GN_R; ++k) {
    if (u.lo + (int)threadIdx.x + k * GN_THREADS >= u.hi) break;
    float f[PN];
    Piece<T>::unpack(v[k], f);
#pragma unroll
    for (int j = 0; j < PN; ++j) acc[0][j] = fmaf(f[j] - mu[j], f[j] - mu[j], acc[0][j]);
  }
  gn_block_sum<1, PN>(acc, red, m2);
  if ((int)threadIdx.x < EPR) part[u.cell * EPR + threadIdx.x] = make_float2(mean[threadIdx.x] / count, m2[threadIdx.x]);
}

// One block per (image, group): joins the group's (mean, M2) pairs,  M2 = sum M2_i + sum n_i (mean_i - mean)^2.
template <int EPR>
__global__ __launch_bounds__(GN_THREADS) void gn_finalize_kernel(const float2* part, GnShape s, const float* gamma, const float* beta,
                                                                 float eps, float* mean_out, float* rstd_out, float* scale, float* shift) {
  __shared__ double red[GN_THREADS / 64];
  const int g = (int)(blockIdx.x % s.G);
  const long n = blockIdx.x / s.G;
  const int cells = s.cpg * s.nseg;
  double sum = 0.0;
  for (int i = threadIdx.x; i < cells; i += GN_THREADS) {
    const int c = g * s.cpg + i / s.nseg, seg = i % s.nseg;
    const int count = (min(s.npieces, (seg + 1) * s.seg_len) - seg * s.seg_len) / 2;
    sum += (double)part[((n * s.P + c / EPR) * s.nseg + seg) * EPR + c % EPR].x * count;
  }
  const double total = (double)s.cpg * (s.npieces / 2), mean = gn_block_sum64(sum, red) / total;
  double m2 = 0.0;
  for (int i = threadIdx.x; i < cells; i += GN_THREADS) {
    const int c = g * s.cpg + i / s.nseg, seg = i % s.nseg;
    const int count = (min(s.npieces, (seg + 1) * s.seg_len) - seg * s.seg_len) / 2;
    const float2 p = part[((n * s.P + c / EPR) * s.nseg + seg) * EPR + c % EPR];
    m2 += (double)p.y + count * (((double)p.x - mean) * ((double)p.x - mean));
  }
  const float rstd = (float)(1.0 / sqrt(gn_block_sum64(m2, red) / total + (double)eps)), mu = (float)mean;
  if (threadIdx.x == 0) { mean_out[n * s.G + g] = mu; rstd_out[n * s.G + g] = rstd; }
  for (int c = g * s.cpg + threadIdx.x; c < (g == s.G - 1 ? s.cpad : (g + 1) * s.cpg); c += GN_THREADS) {
    const float sc = c < s.C ? gamma[c] * rstd : 0.f;
    scale[n * s.cpad + c] = sc;
    shift[n * s.cpad + c] = c < s.C ? fmaf(-mu, sc, beta[c]) : 0.f;
  }
}

template <typename T, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_apply_kernel(const unsigned char* x, int x_pt, int x_p0, unsigned char* a, int a_pt,
                                                              int a_p0, GnShape s, const float* __restrict__ scale,
                                                              const float* __restrict__ shift) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const GnUnit u = gn_unit(s);
  const unsigned char* xb = x + (u.n * x_pt + x_p0 + u.plane) * s.npieces * 16;
  unsigned char* ab = a + (u.n * a_pt + a_p0 + u.plane) * s.npieces * 16;
  const long c0 = u.n * s.cpad + u.plane * EPR + (threadIdx.x & 1) * PN;
  float sc[PN], sh[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; }
  for (int i = u.lo + threadIdx.x; i < u.hi; i += GN_THREADS) {
    float f[PN];
    Piece<T>::unpack(*(const uint4*)(xb + (long)i * 16), f);
#pragma unroll
    for (int j = 0; j < PN; ++j) f[j] = gn_act<ACT>(fmaf(f[j], sc[j], sh[j]));
    *(uint4*)(ab + (long)i * 16) = Piece<T>::pack(f);
  }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// Per-channel constants of a thread's half record: the forward's scale / shift, the group's mean and rstd.
template <int PN> struct GnChannel { float sc[PN], sh[PN], mu[PN], rs[PN]; };
template <int PN>
__device__ __forceinline__ void gn_channel(GnChannel<PN>& k, const GnShape& s, long n, int c0, const float* mean, const float* rstd,
                                           const float* scale, const float* shift) {
#pragma unroll
  for (int j = 0; j < PN; ++j) {
    const int c = c0 + j;
    const bool in = c < s.C;
    k.sc[j] = scale[n * s.cpad + c];
    k.sh[j] = shift[n * s.cpad + c];
    k.mu[j] = in ? mean[n * s.G + c / s.cpg] : 0.f;
    k.rs[j] = in ? rstd[n * s.G + c / s.cpg] : 0.f;
  }
}

// part[cell][channel] = (sum dz, sum dz * xhat) of the segment
template <typename T, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_reduce_kernel(const unsigned char* g, int g_pt, int g_p0, const unsigned char* x,
                                                                   int x_pt, int x_p0, GnShape s, const float* mean, const float* rstd,
                                                                   const float* scale, const float* shift, float2* part) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  __shared__ float red[GN_THREADS / 64 * EPR * 2], sums[EPR * 2];
  const GnUnit u = gn_unit(s);
  const unsigned char* gb = g + (u.n * g_pt + g_p0 + u.plane) * s.npieces * 16;
  const unsigned char* xb = x + (u.n * x_pt + x_p0 + u.plane) * s.npieces * 16;
  GnChannel<PN> k;
  gn_channel<PN>(k, s, u.n, u.plane * EPR + (threadIdx.x & 1) * PN, mean, rstd, scale, shift);
  float acc[2][PN] = {};
  for (int i = u.lo + threadIdx.x; i < u.hi; i += GN_THREADS) {
    float fg[PN], fx[PN];
    Piece<T>::unpack(*(const uint4*)(gb + (long)i * 16), fg);
    Piece<T>::unpack(*(const uint4*)(xb + (long)i * 16), fx);
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      const float dz = gn_act_grad<ACT>(fmaf(fx[j], k.sc[j], k.sh[j]), fg[j]);
      acc[0][j] += dz;
      acc[1][j] = fmaf(dz, (fx[j] - k.mu[j]) * k.rs[j], acc[1][j]);
    }
  }
  gn_block_sum<2, PN>(acc, red, sums);
  if ((int)threadIdx.x < EPR) part[u.cell * EPR + threadIdx.x] = make_float2(sums[2 * threadIdx.x], sums[2 * threadIdx.x + 1]);
}

// One block per (image, group): coef[n][g] = (mean gamma * dz, mean gamma * dz * xhat) over the group
template <int EPR>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_group_kernel(const float2* part, GnShape s, const float* gamma, float2* coef) {
  __shared__ double red[GN_THREADS / 64];
  const int g = (int)(blockIdx.x % s.G);
  const long n = blockIdx.x / s.G;
  double s1 = 0.0, s2 = 0.0;
  for (int i = threadIdx.x; i < s.cpg * s.nseg; i += GN_THREADS) {
    const int c = g * s.cpg + i / s.nseg, seg = i % s.nseg;
    const float2 p = part[((n * s.P + c / EPR) * s.nseg + seg) * EPR + c % EPR];
    s1 += (double)gamma[c] * p.x;
    s2 += (double)gamma[c] * p.y;
  }
  const double total = (double)s.cpg * (s.npieces / 2);
  s1 = gn_block_sum64(s1, red) / total;
  s2 = gn_block_sum64(s2, red) / total;
  if (threadIdx.x == 0) coef[blockIdx.x] = make_float2((float)s1, (float)s2);
}

// One block per channel: dbeta, dgamma = sums over the images and segments
template <int EPR>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_param_kernel(const float2* part, GnShape s, float* dgamma, float* dbeta) {
  __shared__ double red[GN_THREADS / 64];
  const int c = blockIdx.x;
  double s1 = 0.0, s2 = 0.0;
  const long cells = (long)s.N * s.nseg;
  for (long i = threadIdx.x; i < cells; i += GN_THREADS) {
    const float2 p = part[((i / s.nseg * s.P + c / EPR) * s.nseg + i % s.nseg) * EPR + c % EPR];
    s1 += p.x;
    s2 += p.y;
  }
  s1 = gn_block_sum64(s1, red);
  s2 = gn_block_sum64(s2, red);
  if (threadIdx.x == 0) { dbeta[c] = (float)s1; dgamma[c] = (float)s2; }
}

// dx may be g: a thread reads what it writes
template <typename T, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_apply_kernel(const unsigned char* g, int g_pt, int g_p0, const unsigned char* x,
                                                                  int x_pt, int x_p0, unsigned char* dx, int d_pt, int d_p0, GnShape s,
                                                                  const float* mean, const float* rstd, const float* scale,
                                                                  const float* shift, const float* gamma, const float2* coef) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const GnUnit u = gn_unit(s);
  const unsigned char* gb = g + (u.n * g_pt + g_p0 + u.plane) * s.npieces * 16;
  const unsigned char* xb = x + (u.n * x_pt + x_p0 + u.plane) * s.npieces * 16;
  unsigned char* db = dx + (u.n * d_pt + d_p0 + u.plane) * s.npieces * 16;
  const int c0 = u.plane * EPR + (threadIdx.x & 1) * PN;
  GnChannel<PN> k;
  gn_channel<PN>(k, s, u.n, c0, mean, rstd, scale, shift);
  float ga[PN], c1[PN], c2[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) {
    const bool in = c0 + j < s.C;
    const float2 cf = in ? coef[u.n * s.G + (c0 + j) / s.cpg] : make_float2(0.f, 0.f);
    ga[j] = in ? gamma[c0 + j] : 0.f;
    c1[j] = cf.x;
    c2[j] = cf.y;
  }
  for (int i = u.lo + threadIdx.x; i < u.hi; i += GN_THREADS) {
    float fg[PN], fx[PN];
    Piece<T>::unpack(*(const uint4*)(gb + (long)i * 16), fg);
    Piece<T>::unpack(*(const uint4*)(xb + (long)i * 16), fx);
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      const float dz = gn_act_grad<ACT>(fmaf(fx[j], k.sc[j], k.sh[j]), fg[j]);
      const float xhat = (fx[j] - k.mu[j]) * k.rs[j];
      fg[j] = k.rs[j] * (fmaf(ga[j], dz, -c1[j]) - xhat * c2[j]);
    }
    *(uint4*)(db + (long)i * 16) = Piece<T>::pack(fg);
  }
}

int gn_shape(const char* name, dn_tensor x, int N, int H, int W, int groups, int dtype, GnShape* out) {
  DN_CHECK_ARG(dtype == DN_F32 || dtype == DN_BF16, "%s: bad dtype %d", name, dtype);
  DN_CHECK_ARG(N >= 0 && H >= 1 && W >= 1 && (long)H * W <= (1L << 25), "%s: bad size N=%d H=%d W=%d (H * W <= 2^25)", name, N, H, W);
  DN_CHECK_ARG(x.channels >= 1 && groups >= 1 && x.channels % groups == 0, "%s: %d channels do not divide into %d groups", name, x.channels,
               groups);
  GnShape s;
  const int epr = dtype == DN_BF16 ? 16 : 8;
  s.N = N; s.C = x.channels; s.G = groups; s.P = dn_planes(x.channels, dtype);
  s.cpg = x.channels / groups; s.cpad = dn_channel_pad(x.channels);
  s.npieces = 2 * H * W;
  s.nseg = (s.npieces + GN_SEG - 1) / GN_SEG;
  s.seg_len = ((s.npieces / 2 + s.nseg - 1) / s.nseg) * 2;
  s.nseg = (s.npieces + s.seg_len - 1) / s.seg_len;
  DN_CHECK_ARG((long)N * s.P * s.nseg < (1L << 31) && (long)N * s.G < (1L << 31), "%s: too many images x planes", name);
  (void)epr;
  *out = s;
  return DN_OK;
}
int gn_tensor(const char* name, const char* which, dn_tensor t, const GnShape& s) {
  DN_CHECK_ARG(t.base && ((uintptr_t)t.base & 15) == 0, "%s: %s is null or not 16-byte aligned", name, which);
  DN_CHECK_ARG(t.channels == s.C, "%s: %s has %d channels, x has %d", name, which, t.channels, s.C);
  DN_CHECK_ARG(t.plane0 >= 0 && t.plane0 + s.P <= t.planes_total, "%s: planes %d..%d of %s are outside its buffer of %d", name, t.plane0,
               t.plane0 + s.P, which, t.planes_total);
  return DN_OK;
}
long gn_part_bytes(const GnShape& s, int dtype) {
  return (long)s.N * s.P * s.nseg * (dtype == DN_BF16 ? 16 : 8) * (long)sizeof(float2);
}
long gn_workspace(const GnShape& s, int dtype) { return gn_part_bytes(s, dtype) + (long)s.N * s.G * (long)sizeof(float2) + 256; }

template <typename T, int ACT>
void gn_forward_launch(dn_tensor x, dn_tensor a, const GnShape& s, const float* gamma, const float* beta, float eps, float* mean,
                       float* rstd, float* scale, float* shift, float2* part, hipStream_t st) {
  constexpr int EPR = RecTraits<T>::EPR;
  const dim3 grid((unsigned)((long)s.N * s.P * s.nseg));
  hipLaunchKernelGGL((gn_stats_kernel<T>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)x.base, x.planes_total, x.plane0, s, part);
  hipLaunchKernelGGL((gn_finalize_kernel<EPR>), dim3((unsigned)((long)s.N * s.G)), dim3(GN_THREADS), 0, st, part, s, gamma, beta, eps, mean,
                     rstd, scale, shift);
  hipLaunchKernelGGL((gn_apply_kernel<T, ACT>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)x.base, x.planes_total, x.plane0,
                     (unsigned char*)a.base, a.planes_total, a.plane0, s, scale, shift);
}
template <typename T, int ACT>
void gn_backward_launch(dn_tensor g, dn_tensor x, dn_tensor dx, const GnShape& s, const float* gamma, const float* mean, const float* rstd,
                        const float* scale, const float* shift, float* dgamma, float* dbeta, float2* part, float2* coef, hipStream_t st) {
  constexpr int EPR = RecTraits<T>::EPR;
  const dim3 grid((unsigned)((long)s.N * s.P * s.nseg));
  hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, ACT>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)g.base, g.planes_total, g.plane0,
                     (const unsigned char*)x.base, x.planes_total, x.plane0, s, mean, rstd, scale, shift, part);
  hipLaunchKernelGGL((gn_bwd_group_kernel<EPR>), dim3((unsigned)((long)s.N * s.G)), dim3(GN_THREADS), 0, st, part, s, gamma, coef);
  hipLaunchKernelGGL((gn_bwd_param_kernel<EPR>), dim3(s.C), dim3(GN_THREADS), 0, st, part, s, dgamma, dbeta);
  hipLaunchKernelGGL((gn_bwd_apply_kernel<T, ACT>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)g.base, g.planes_total, g.plane0,
                     (const unsigned char*)x.base, x.planes_total, x.plane0, (unsigned char*)dx.base, dx.planes_total, dx.plane0, s, mean,
                     rstd, scale, shift, gamma, coef);
}

}  // namespace

#define GN_DISPATCH(dtype, act, CALL)                                                       \
  if ((dtype) == DN_BF16) {                                                                 \
    if ((act) == DN_ACT_NONE) { CALL(__bf16, DN_ACT_NONE); }                                \
    else if ((act) == DN_ACT_RELU) { CALL(__bf16, DN_ACT_RELU); }                           \
    else { CALL(__bf16, DN_ACT_SILU); }                                                     \
  } else {                                                                                  \
    if ((act) == DN_ACT_NONE) { CALL(float, DN_ACT_NONE); }                                 \
    else if ((act) == DN_ACT_RELU) { CALL(float, DN_ACT_RELU); }                            \
    else { CALL(float, DN_ACT_SILU); }                                                      \
  }

extern "C" {

long dn_group_norm_workspace_bytes(int N, int C, int H, int W, int groups, int dtype) {
  GnShape s;
  dn_tensor t = {nullptr, 0, 0, C};
  if (gn_shape("dn_group_norm_workspace_bytes", t, N, H, W, groups, dtype, &s)) return -1;
  return gn_workspace(s, dtype);
}

int dn_group_norm_act(dn_tensor x, dn_tensor a, int N, int H, int W, int groups, const float* gamma, const float* beta, float eps, int act,
                      float* mean, float* rstd, float* scale, float* shift, void* workspace, long workspace_bytes, int dtype,
                      void* stream) {
  GnShape s;
  int rc = gn_shape("dn_group_norm_act", x, N, H, W, groups, dtype, &s);
  if (rc) return rc;
  if (N == 0) return DN_OK;
  if ((rc = gn_tensor("dn_group_norm_act", "x", x, s)) || (rc = gn_tensor("dn_group_norm_act", "a", a, s))) return rc;
  DN_CHECK_ARG(gamma && beta && mean && rstd && scale && shift, "dn_group_norm_act: null vector");
  DN_CHECK_ARG(eps > 0.f && eps < 1e30f, "dn_group_norm_act: eps must be positive");
  DN_CHECK_ARG(act >= DN_ACT_NONE && act <= DN_ACT_SILU, "dn_group_norm_act: bad activation %d", act);
  DN_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= gn_workspace(s, dtype),
               "dn_group_norm_act: workspace of %ld bytes, %ld needed (16-byte aligned)", workspace_bytes, gn_workspace(s, dtype));
#define GN_CALL(T, A) (gn_forward_launch<T, A>(x, a, s, gamma, beta, eps, mean, rstd, scale, shift, (float2*)workspace, (hipStream_t)stream))
  GN_DISPATCH(dtype, act, GN_CALL)
#undef GN_CALL
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_group_norm_act_backward(dn_tensor g, dn_tensor x, dn_tensor dx, int N, int H, int W, int groups, const float* gamma,
                               const float* mean, const float* rstd, const float* scale, const float* shift, int act, float* dgamma,
                               float* dbeta, void* workspace, long workspace_bytes, int dtype, void* stream) {
  GnShape s;
  int rc = gn_shape("dn_group_norm_act_backward", x, N, H, W, groups, dtype, &s);
  if (rc) return rc;
  DN_CHECK_ARG(N >= 1, "dn_group_norm_act_backward: an empty batch has no gradient");
  if ((rc = gn_tensor("dn_group_norm_act_backward", "x", x, s)) || (rc = gn_tensor("dn_group_norm_act_backward", "g", g, s)) ||
      (rc = gn_tensor("dn_group_norm_act_backward", "dx", dx, s)))
    return rc;
  DN_CHECK_ARG(gamma && mean && rstd && scale && shift && dgamma && dbeta, "dn_group_norm_act_backward: null vector");
  DN_CHECK_ARG(act >= DN_ACT_NONE && act <= DN_ACT_SILU, "dn_group_norm_act_backward: bad activation %d", act);
  DN_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= gn_workspace(s, dtype),
               "dn_group_norm_act_backward: workspace of %ld bytes, %ld needed (16-byte aligned)", workspace_bytes, gn_workspace(s, dtype));
  float2* part = (float2*)workspace;
  float2* coef = (float2*)((char*)workspace + gn_part_bytes(s, dtype));
#define GN_CALL(T, A) (gn_backward_launch<T, A>(g, x, dx, s, gamma, mean, rstd, scale, shift, dgamma, dbeta, part, coef, (hipStream_t)stream))
  GN_DISPATCH(dtype, act, GN_CALL)
#undef GN_CALL
  DN_LAUNCH_CHECK();
  return DN_OK;
}

}  // extern "C"
