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
#include "gn_epoch.h"

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

// Slots past the last channel of a partial plane come out as zero, whatever they hold (0 * NaN would be NaN): the bits of this
// thread's half records that are kept.  Sums need no mask: those of unused slots are their own, and nobody reads them.
template <typename T> __device__ __forceinline__ uint4 gn_kept_bits(const GnShape& s, int plane) {
  constexpr int PN = Piece<T>::N;
  const int left = s.C - plane * RecTraits<T>::EPR - (int)(threadIdx.x & 1) * PN;
  unsigned b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (PN == 4) b[j] = left > j ? ~0u : 0u;
    else b[j] = (left > 2 * j ? 0xFFFFu : 0u) | (left > 2 * j + 1 ? 0xFFFF0000u : 0u);
  }
  return make_uint4(b[0], b[1], b[2], b[3]);
}
__device__ __forceinline__ uint4 gn_and(const uint4& v, const uint4& m) { return make_uint4(v.x & m.x, v.y & m.y, v.z & m.z, v.w & m.w); }

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
  const uint4 kept = gn_kept_bits<T>(s, u.plane);
  for (int i = u.lo + threadIdx.x; i < u.hi; i += GN_THREADS) {
    float f[PN];
    Piece<T>::unpack(gn_and(*(const uint4*)(xb + (long)i * 16), kept), f);
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

// The same for many partials: block (plane, chunk) adds up the rows of its chunk, all channels of the plane side by side, and
// the plane's last block to finish adds the chunks in their order.  `counts` is zero before and after.
int gn_param_chunks(const GnShape& s) {
  const long rows = (long)s.N * s.nseg;
  return (int)std::max(1L, std::min({rows / 64, 64L, 4096L / s.P}));
}
template <int EPR>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_param_chunk_kernel(const float2* part, GnShape s, int chunks, unsigned* counts,
                                                                        double2* sums, float* dgamma, float* dbeta) {
  constexpr int ROWS = GN_THREADS / EPR;
  __shared__ double2 red[GN_THREADS];
  __shared__ bool last;
  const int plane = blockIdx.x, chunk = blockIdx.y, slot = threadIdx.x % EPR, row0 = threadIdx.x / EPR;
  const unsigned rows = (unsigned)s.N * s.nseg, per = (rows + chunks - 1) / chunks, end = min(rows, (chunk + 1) * per);
  double2 v = make_double2(0.0, 0.0);
  auto join = [&]() {                            // v of the threads of a slot, in a fixed order, to the threads of row 0
    red[threadIdx.x] = v;
    __syncthreads();
    if (row0 == 0) {
      v = make_double2(0.0, 0.0);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) { v.x += red[r * EPR + slot].x; v.y += red[r * EPR + slot].y; }
    }
    __syncthreads();
  };
#pragma unroll 4
  for (unsigned r = chunk * per + row0; r < end; r += ROWS) {
    const unsigned n = r / (unsigned)s.nseg;
    const float2 q = part[(((long)n * s.P + plane) * s.nseg + (r - n * s.nseg)) * EPR + slot];
    v.x += q.x;
    v.y += q.y;
  }
  join();
  if (chunks > 1) {
    double2* mine = sums + (long)plane * chunks * EPR;
    if (row0 == 0) {
      mine[chunk * EPR + slot] = v;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    }
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(counts + plane, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)chunks - 1;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) __hip_atomic_store(counts + plane, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    v = make_double2(0.0, 0.0);
#pragma unroll 4
    for (int k = row0; k < chunks; k += ROWS) {
      const double2 q = mine[k * EPR + slot];
      v.x += q.x;
      v.y += q.y;
    }
    join();
  }
  const int c = plane * EPR + slot;
  if (row0 == 0 && c < s.C) { dbeta[c] = (float)v.x; dgamma[c] = (float)v.y; }
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
  const uint4 kept = gn_kept_bits<T>(s, u.plane);
  for (int i = u.lo + threadIdx.x; i < u.hi; i += GN_THREADS) {
    float fg[PN], fx[PN];
    Piece<T>::unpack(gn_and(*(const uint4*)(gb + (long)i * 16), kept), fg);
    Piece<T>::unpack(gn_and(*(const uint4*)(xb + (long)i * 16), kept), fx);
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      const float dz = gn_act_grad<ACT>(fmaf(fx[j], k.sc[j], k.sh[j]), fg[j]);
      const float xhat = (fx[j] - k.mu[j]) * k.rs[j];
      fg[j] = k.rs[j] * (fmaf(ga[j], dz, -c1[j]) - xhat * c2[j]);
    }
    *(uint4*)(db + (long)i * 16) = Piece<T>::pack(fg);
  }
}


// ---- one pass: the blocks of a group hold its values in registers and exchange their sums --------------------------------
// The smallest traffic a group norm can have is one read and one write (backward: two reads and one write); statistics in a launch
// of their own cost a second read of all of it: 234 us forward and 382 us backward for the sizes below.  This form is bound by
// HBM: 256 x 32 x 6 x 4096 bf16 forward 176 us for 0.81 GB (4.6 TB/s, a copy of as many bytes takes 152), 256 x 512 x 6 x 256 backward
// 271 us for 1.21 GB (4.5 TB/s; 228); the vector units are busy for half of that time, and the waits for other blocks are hidden
// behind the other one or two blocks of the CU.  Small calls are bound by the exchange: 2 x 128 x 5 x 64 fp32 8 us on the device.
// Here a block keeps its segment in registers, publishes the segment's sums, waits for those of the other blocks of its
// cluster -- the segments of the planes whose channels form whole groups -- and finishes from registers.
//
// A cluster's blocks are consecutive in the grid.  Where each XCD starts its share of the blocks in their order, the blocks of the
// oldest incomplete cluster are next in line everywhere and only finished clusters lie before them: nobody waits for a block that
// waits for him.  No order is promised, though, so a wait is bounded: a block that gives up has published its own sums; it puts its
// place on a list and exits, which frees its slot on the chip.  The launch's last block finds all sums published and does the
// listed segments over.  So every wait ends and every segment is written, with the same bits, whatever else runs on the GPU.
// (Places drawn from counters when a block starts need no order, but a block's loads wait for them: 182 us instead of 177 for
// 256 x 32 x 6 x 4096 bf16, 12.7 instead of 11.9 for 2 images, and four streams of calls at once took 2.4 to 3.1 instead
// of 1.4 to 2.1 ms a round, blocks of one launch holding the slots that another's needed.  Clusters kept within an XCD: 216 us.)
//
// A published word carries the launch's epoch beside its 32-bit value, so no fence and no clearing is needed: words of earlier
// launches have other epochs (gn_epoch.h).  The launch's last block counts the epoch up and, when it starts again from 0, zeroes
// all words; counters return to zero.
constexpr int GNF_THREADS = 512;
constexpr int GNF_WAVES = GNF_THREADS / 64;
// Blocks of a cluster: 64 KB each, so groups (or sets of planes) up to 12 MB of bf16 or fp32.  bf16, one pass against three launches: 64 x 128
// channels of one group x 6 x 4096 (96 blocks) forward 217 / 240 us, backward 320 / 370; 32 x 256 channels (192 blocks) 226 / 251 and 365 / 376; 32 x 512
// channels (384 blocks) 488 / 488 and 884 / 720: there a CU's two blocks wait for a whole chip of others.  A cluster's cells have to fit
// the LDS as well: at most 1024 / (cells of a plane) blocks, 64 for bf16 groups of an odd number of channels.
constexpr int GNF_MAX_K = 192;
constexpr int GNF_MAX_CELLS = 1024;              // published cells of a cluster
constexpr int GNF_MAX_BLOCKS = 16384;            // blocks of a launch: more images take more launches
constexpr int GNF_POLLS = 4096;                  // looks at a word before a block gives up: about 0.6 ms
constexpr int GNF_SURE = 1 << 16;                // looks at a word that has been stored: about 10 ms
constexpr int GNF_SHARDS = 16;                   // counters of finished clusters
constexpr int GNF_LINE = 32;                     // counters 128 bytes apart: epoch, finished shards, listed, then the shards'
constexpr long GNF_CTRL_BYTES = (3 + GNF_SHARDS) * GNF_LINE * 4L, GNF_DEPART_BYTES = GNF_MAX_BLOCKS * 4L;
constexpr int GNF_MAX_PLANES = 4096;             // of a tensor: 2^15 channels of fp32
constexpr long GNF_PLANES0 = GNF_CTRL_BYTES + GNF_DEPART_BYTES;
constexpr long GNF_LIST0 = GNF_PLANES0 + GNF_MAX_PLANES * 4L;
constexpr long GNF_SLOT0 = GNF_LIST0 + GNF_MAX_BLOCKS * 8L;
constexpr long GNF_END = GNF_SLOT0 + GNF_MAX_BLOCKS * 16L * 16;      // the three-launch form's partials lie behind: no word of theirs
                                                                     // can be taken for a published one
// Division of a small number by one that the host knows: one multiplication (exact while number * divisor < 2^32; divisor 1 has
// mul 0).  A division by a runtime value is some 20 dependent instructions, and a dozen of them lie on a block's critical path.
struct GnDiv {
  unsigned d, mul;
};
__device__ __forceinline__ int gn_div(const GnDiv& v, int n) { return v.mul ? (int)__umulhi((unsigned)n, v.mul) : n; }
__device__ __forceinline__ int gn_mod(const GnDiv& v, int n) { return n - gn_div(v, n) * (int)v.d; }
GnDiv gn_divisor(long d) { return GnDiv{(unsigned)d, d > 1 ? (unsigned)((1ULL << 32) / (unsigned long)d) + 1 : 0}; }

struct GnFused {
  GnShape s;
  int m;                   // channels of a cell: gcd(channels per group, channels per record)
  int ncell;               // cells of a plane
  int ps, nsets;           // planes of a cluster, clusters of an image
  int polls;
  int image0, images;      // this launch's
  GnDiv d_most, d_nsets, d_nseg, d_cpg, d_m;
  double inv_total;        // 1 / values of a group
  unsigned* ctrl;          // counters, GNF_LINE words apart
  unsigned* depart;        // per cluster: blocks that wait no longer
  unsigned* planes;        // per plane: blocks whose partials are there (launches that sum the parameter gradients themselves)
  unsigned long long* list;      // places that were given up, with the epoch
  unsigned long long* slot;
};

// The packed pieces stay in registers and are unpacked anew by each pass over them: kept unpacked, they would fill twice the
// registers and halve the blocks that a CU holds.
template <int R> __device__ __forceinline__ void gnf_keep_packed(uint4 (&v)[R]) {
#pragma unroll
  for (int k = 0; k < R; ++k) asm volatile("" : "+v"(v[k].x), "+v"(v[k].y), "+v"(v[k].z), "+v"(v[k].w));
}

// Four channels of a piece: the passes below take a bf16 piece in two halves, so that the constants of four channels and not of
// eight are held at a time.
template <typename T> __device__ __forceinline__ void gnf_unpack4(const uint4& v, int h, float* f);
template <> __device__ __forceinline__ void gnf_unpack4<float>(const uint4& v, int, float* f) { Piece<float>::unpack(v, f); }
template <> __device__ __forceinline__ void gnf_unpack4<__bf16>(const uint4& v, int h, float* f) {
  const unsigned a = h ? v.z : v.x, b = h ? v.w : v.y;
  f[0] = __uint_as_float(a << 16); f[1] = __uint_as_float(a & 0xffff0000u);
  f[2] = __uint_as_float(b << 16); f[3] = __uint_as_float(b & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ void gnf_pack4(uint4& v, int h, const float* f);
template <> __device__ __forceinline__ void gnf_pack4<float>(uint4& v, int, const float* f) { v = Piece<float>::pack(f); }
template <> __device__ __forceinline__ void gnf_pack4<__bf16>(uint4& v, int h, const float* f) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;           // a pair in one conversion
  unsigned lo = __builtin_bit_cast(unsigned, (bf16x2_t){(__bf16)f[0], (__bf16)f[1]});
  unsigned hi = __builtin_bit_cast(unsigned, (bf16x2_t){(__bf16)f[2], (__bf16)f[3]});
  asm volatile("" : "+v"(lo), "+v"(hi));                                 // packed here and not where it is stored
  if (h) { v.z = lo; v.w = hi; } else { v.x = lo; v.y = hi; }
}

struct GnPlace { int plane, seg, lo, hi, k, set; long n, cluster0, cluster; unsigned place, tag; bool alone; };

__device__ __forceinline__ unsigned gnf_count(unsigned* p) {
  return __hip_atomic_fetch_add(p, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void gnf_reset(unsigned* p) { __hip_atomic_store(p, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// What block `b` is.  Clusters are laid out as if all had f.ps planes: plane >= P is a block with nothing to do (false).
__device__ __forceinline__ bool gnf_locate(const GnFused& f, GnPlace& u, unsigned b) {
  const GnShape& s = f.s;
  u.place = b;
  const int cluster = gn_div(f.d_most, (int)b), member = (int)b - cluster * (int)f.d_most.d, image = gn_div(f.d_nsets, cluster);
  u.cluster = cluster;
  u.set = cluster - image * f.nsets;
  const int plane = gn_div(f.d_nseg, member);
  u.plane = u.set * f.ps + plane;
  u.seg = member - plane * s.nseg;
  u.n = (long)f.image0 + image;
  u.lo = u.seg * s.seg_len;
  u.hi = min(s.npieces, u.lo + s.seg_len);
  u.k = min(f.ps, s.P - u.set * f.ps) * s.nseg;
  u.cluster0 = u.cluster * (long)f.d_most.d;     // the cluster's first block in the slots
  return u.plane < s.P;
}
// This block's place; false: nothing to do.  *missing is zeroed for after the next barrier.
__device__ __forceinline__ bool gnf_place(const GnFused& f, unsigned* missing, GnPlace& u) {
  u.alone = f.d_most.d == 1;                           // every cluster of the launch is one block: nothing is exchanged
  if (threadIdx.x == 0) *missing = 0;
  const unsigned epoch = u.alone ? 0 : __hip_atomic_load(f.ctrl, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  u.tag = gn_epoch_tag(epoch);
  return gnf_locate(f, u, blockIdx.x);
}

// Sums over the wave's 32 lanes of equal record half, of four channels at a time (h: which four of the thread's half record):
// two halving steps leave a channel to a lane, three more add the lanes up.  Lanes 0..7 put them into the wave's row of `red`.
template <int M> __device__ __forceinline__ float gnf_xor(float v) {          // the value of lane ^ M
  if constexpr (M < 32) return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), M << 10 | 0x1F));
  else return __shfl_xor(v, M);
}
template <int WIDTH, int M> __device__ __forceinline__ void gnf_halve(float* acc) {     // 2 * WIDTH values -> WIDTH
  const bool upper = threadIdx.x & M;
#pragma unroll
  for (int j = 0; j < WIDTH; ++j) {
    const float give = upper ? acc[j] : acc[j + WIDTH];
    const float keep = upper ? acc[j + WIDTH] : acc[j];
    acc[j] = keep + gnf_xor<M>(give);
  }
  if constexpr (WIDTH > 1) gnf_halve<WIDTH / 2, M * 2>(acc);
}
template <int PN> __device__ __forceinline__ void gnf_wave_sums(float (&acc)[4], int h, float* red) {
  gnf_halve<2, 2>(acc);
  float v = acc[0];
  v += gnf_xor<8>(v);
  v += gnf_xor<16>(v);
  v += gnf_xor<32>(v);
  const int lane = threadIdx.x & 63;
  if (lane < 8) red[(threadIdx.x >> 6) * 2 * PN + (lane & 1) * PN + 4 * h + (lane & 2) + (lane >> 2)] = v;
}
// After a barrier: the block's sum of channel lane % EPR, in every wave.
template <int PN> __device__ __forceinline__ float gnf_block_sum(const float* red) {
  constexpr int EPR = 2 * PN, ROWS = 64 / EPR;
  const int lane = threadIdx.x & 63;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < GNF_WAVES; w += ROWS) t += red[w * EPR + lane];          // waves w + lane / EPR
  if constexpr (EPR == 8) t += gnf_xor<8>(t);
  t += gnf_xor<16>(t);
  t += gnf_xor<32>(t);
  return t;
}

__device__ __forceinline__ void gnf_publish(const GnFused& f, const GnPlace& u, int cell, float a, float b) {
  unsigned long long* p = f.slot + ((u.cluster0 + (long)(u.plane - u.set * f.ps) * f.s.nseg + u.seg) * f.ncell + cell) * 2;
  const unsigned long long tag = (unsigned long long)u.tag << 32;
  __hip_atomic_store(p, tag | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(p + 1, tag | __float_as_uint(b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// All cells of the cluster into LDS (words 2 * cell, 2 * cell + 1); false: given up, the place is on the list.  Ends with a
// barrier.  *before (thread GNF_COUNTER): blocks of the cluster that waited no longer before this one; the count is under way when
// the call returns, its first use waits for it.  *missing is 0 at the call.
constexpr unsigned GNF_COUNTER = 64;             // not thread 0, which has work to do next
__device__ __forceinline__ bool gnf_collect(const GnFused& f, const GnPlace& u, float* cells, unsigned* missing, unsigned* before) {
  const int words = u.k * f.ncell * 2;
  const unsigned long long* p = f.slot + u.cluster0 * f.ncell * 2;
  for (int w = threadIdx.x; w < words; w += GNF_THREADS) {
    unsigned long long v = __hip_atomic_load(p + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int tries = 0; (unsigned)(v >> 32) != u.tag && tries < f.polls; ++tries) {
      __builtin_amdgcn_s_sleep(1);
      v = __hip_atomic_load(p + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((unsigned)(v >> 32) != u.tag) *missing = 1;
    cells[w] = __uint_as_float((unsigned)v);
  }
  __syncthreads();
  const bool given_up = __builtin_amdgcn_readfirstlane(*missing) != 0;
  if (threadIdx.x == GNF_COUNTER) {
    if (given_up) {
      const unsigned at = gnf_count(f.ctrl + 2 * GNF_LINE);
      if (at < GNF_MAX_BLOCKS)
        __hip_atomic_store(f.list + at, (unsigned long long)u.tag << 32 | u.place, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");                                         // the list before the departure
    }
    *before = gnf_count(f.depart + u.cluster);
  }
  return !given_up;
}
// The launch's last block to wait: all blocks have stored their words, but a word may still be on its way (a block's count of
// departure is not ordered behind the words that another of its waves stored).  One that never comes makes the result NaN.
__device__ __forceinline__ void gnf_collect_again(const GnFused& f, const GnPlace& u, float* cells) {
  const unsigned long long* p = f.slot + u.cluster0 * f.ncell * 2;
  for (int w = threadIdx.x; w < u.k * f.ncell * 2; w += GNF_THREADS) {
    unsigned value = 0;
    const bool there = gn_take(u.tag, GNF_SURE, [&] { return __hip_atomic_load(p + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }, &value);
    cells[w] = there ? __uint_as_float(value) : __builtin_nanf("");
  }
  __syncthreads();
}
// Whether this block is the launch's last to wait (thread GNF_COUNTER; the answer is for after the next barrier).
__device__ __forceinline__ void gnf_last(const GnFused& f, const GnPlace& u, unsigned before, unsigned* last) {
  if (u.alone || threadIdx.x != GNF_COUNTER) return;
  *last = 0;
  if (before != (unsigned)u.k - 1) return;
  gnf_reset(f.depart + u.cluster);                                                             // the cluster's last
  const int shard = (int)u.cluster % GNF_SHARDS, clusters = f.images * f.nsets;
  unsigned* finished = f.ctrl + (3 + shard) * GNF_LINE;
  if (gnf_count(finished) != (unsigned)(clusters - shard + GNF_SHARDS - 1) / GNF_SHARDS - 1) return;
  gnf_reset(finished);                                                                         // the shard's last
  if (gnf_count(f.ctrl + GNF_LINE) != (unsigned)min(GNF_SHARDS, clusters) - 1) return;
  gnf_reset(f.ctrl + GNF_LINE);                                                                // the launch's last
  *last = 1;
}
// The launch's last block, done with everything, after the last tag: all words are zeroed.  All others have read theirs by now.
__device__ __noinline__ void gnf_clear_words(unsigned long long* words) {
  static_assert(GNF_LIST0 + GNF_MAX_BLOCKS * 8L == GNF_SLOT0, "the list and the slots lie together");
  for (long i = threadIdx.x; i < (GNF_END - GNF_LIST0) / 8; i += GNF_THREADS)
    __hip_atomic_store(words + i, 0ULL, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The launch's last block: the next listed place into `u`; false: none is left, and the next launch's epoch is there.
__device__ __forceinline__ bool gnf_next_listed(const GnFused& f, GnPlace& u, unsigned* at, unsigned* next) {
  __syncthreads();
  if (threadIdx.x == 0) {
    if (*at == 0) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    const unsigned listed = min((unsigned)GNF_MAX_BLOCKS, __hip_atomic_load(f.ctrl + 2 * GNF_LINE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    *next = gn_take_listed(
        u.tag, GNF_SURE, listed, at, gridDim.x, [&](unsigned i) { return __hip_atomic_load(f.list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); },
        [&](unsigned place) { GnPlace probe; return place < gridDim.x && gnf_locate(f, probe, place); });
    if (*next == gridDim.x) {
      gnf_reset(f.ctrl + 2 * GNF_LINE);
      __hip_atomic_store(f.ctrl, gn_epoch_after(u.tag), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  const unsigned place = __builtin_amdgcn_readfirstlane(*next);
  return place < gridDim.x && gnf_locate(f, u, place);
}

__device__ __forceinline__ void gnf_wave_sum64(double& a, double& b) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    a += __shfl_xor(a, m);
    b += __shfl_xor(b, m);
  }
}

// the cell (index in LDS) and segment of a group's i-th contribution
__device__ __forceinline__ int gnf_cell(const GnFused& f, const GnPlace& u, int epr, int g, int i, int* seg) {
  const int j = gn_div(f.d_nseg, i);
  *seg = i - j * f.s.nseg;
  const int c = g * f.s.cpg + j * f.m;
  return ((c / epr - u.set * f.ps) * f.s.nseg + *seg) * f.ncell + gn_div(f.d_m, c % epr);
}

template <int EPR> struct GnfShared {
  unsigned missing, next, last, last_plane;

  float red[2][GNF_WAVES * EPR];
  alignas(8) float cells[GNF_MAX_CELLS * 2];
  float gstat[EPR][2], chan[EPR][7];
};

template <int R> __device__ __forceinline__ void gnf_load(uint4 (&v)[R], const void* base, int pt, int p0, const GnShape& s, const GnPlace& u) {
  const unsigned char* b = (const unsigned char*)base + ((u.n * pt + p0 + u.plane) * (long)s.npieces + u.lo) * 16;
  const int len = u.hi - u.lo;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int i = (int)threadIdx.x + k * GNF_THREADS;
    v[k] = i < len ? *(const uint4*)(b + (unsigned)i * 16u) : make_uint4(0, 0, 0, 0);
  }
}

// Stores of a tensor that is larger than what a later reader could find of it in the caches pass them by: 256 x 32 x 6 x 4096 bf16
// forward 190 -> 182 us, backward 307 -> 297, together with a copy of the result 339 -> 336 and 457 -> 450; at 16 images (25 MB) that copy costs
// 28.8 instead of 27.2 us behind such stores, at 32 images 48.8 / 48.2, at 64 (100 MB) 90.3 / 91.8.
constexpr long GNF_STREAM_BYTES = 64L << 20;
__device__ __forceinline__ void gnf_store(void* p, const uint4& v, bool stream) {
  typedef __attribute__((ext_vector_type(4))) unsigned vec_t;
  if (stream) {                                            // kept apart by the comments: merged into one, they lose the hint
    asm volatile("; past the caches");
    __builtin_nontemporal_store((vec_t){v.x, v.y, v.z, v.w}, (vec_t*)p);
    asm volatile("; past the caches");
  } else {
    *(uint4*)p = v;
  }
}

struct GnForward {
  const void* x;
  void* a;
  int x_pt, x_p0, a_pt, a_p0;
  const float *gamma, *beta;
  float eps;
  float *mean, *rstd, *scale, *shift;
  bool stream;             // of the output
};
// From the cluster's cells in LDS to the statistics of this plane's groups, scale and shift of its channels (sh.chan).  Between
// two barriers.  `leave()` runs on the way.
template <int EPR, typename F>
__device__ __forceinline__ void gnf_scales(const GnFused& f, const GnForward& o, const GnPlace& u, GnfShared<EPR>& sh, F leave) {
  const GnShape& s = f.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the groups of this plane's channels, a wave each: M2 = sum M2_i + sum n_i (mean_i - mean)^2
  const int c_lo = u.plane * EPR, c_hi = min(s.C, c_lo + EPR);
  const int g_lo = gn_div(f.d_cpg, c_lo), g_hi = gn_div(f.d_cpg, c_hi - 1);
  const int parts = gn_div(f.d_m, s.cpg) * s.nseg;
  for (int g = g_lo + wave; g <= g_hi; g += GNF_WAVES) {
    // around the first part's mean: M2 = sum (M2_i + n_i d_i^2) - (sum n_i d_i)^2 / n, d_i = mean_i - pivot, in fp64
    int seg;
    const double pivot = (double)sh.cells[2 * gnf_cell(f, u, EPR, g, 0, &seg)];
    double s1 = 0.0, s2 = 0.0;
    for (int i = lane; i < parts; i += 64) {
      const int at = gnf_cell(f, u, EPR, g, i, &seg);
      const double d = (double)sh.cells[2 * at] - pivot;
      const double nd = (double)(f.m * (min(s.npieces, (seg + 1) * s.seg_len) - seg * s.seg_len) / 2) * d;
      s1 += nd;
      s2 += (double)sh.cells[2 * at + 1] + nd * d;
    }
    gnf_wave_sum64(s1, s2);
    const double shift = s1 * f.inv_total;
    const float mean32 = (float)(pivot + shift);
    const float var = (float)((s2 - s1 * shift) * f.inv_total + (double)o.eps);
    float rstd = __builtin_amdgcn_rsqf(var);
    rstd = fmaf(rstd * 0.5f, fmaf(-var * rstd, rstd, 1.f), rstd);                // one Newton step (three launches: a fp64 root)
    if (lane == 0) {
      sh.gstat[g - g_lo][0] = mean32;
      sh.gstat[g - g_lo][1] = rstd;
      if (u.seg == 0 && g * s.cpg >= c_lo) { o.mean[u.n * s.G + g] = mean32; o.rstd[u.n * s.G + g] = rstd; }
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < EPR) {
    const int c = c_lo + threadIdx.x;
    float c_scale = 0.f, c_shift = 0.f;
    if (c < s.C) {
      const int g = gn_div(f.d_cpg, c) - g_lo;
      c_scale = o.gamma[c] * sh.gstat[g][1];
      c_shift = fmaf(-sh.gstat[g][0], c_scale, o.beta[c]);
    }
    sh.chan[threadIdx.x][0] = c_scale;
    sh.chan[threadIdx.x][1] = c_shift;
    if (u.seg == 0) { o.scale[u.n * s.cpad + c] = c_scale; o.shift[u.n * s.cpad + c] = c_shift; }
  } else if (u.seg == 0 && u.plane == s.P - 1) {                               // vector entries past the last plane
    for (int c = s.P * EPR + (int)threadIdx.x - EPR; c < s.cpad; c += GNF_THREADS - EPR) { o.scale[u.n * s.cpad + c] = 0.f; o.shift[u.n * s.cpad + c] = 0.f; }
  }
  leave();
  __syncthreads();
}
// Pieces first, first + GNF_THREADS, ... of the segment: v = act(v * scale + shift), stored.  PARTIAL: channels do not fill the last plane's
// records (an instance of its own: where all instances looked for such planes, a branch that no block took cost 12 us of 276).
template <typename T, int ACT, int R, bool PARTIAL>
__device__ __forceinline__ void gnf_apply(const GnForward& o, const GnShape& s, const GnPlace& u, uint4 (&v)[R], int first,
                                          const GnfShared<RecTraits<T>::EPR>& sh) {
  constexpr int PN = Piece<T>::N;
  const int pc = threadIdx.x & 1, len = u.hi - u.lo;
  unsigned char* ab = (unsigned char*)o.a + ((u.n * o.a_pt + o.a_p0 + u.plane) * (long)s.npieces + u.lo) * 16;
#pragma unroll
  for (int h = 0; h < PN / 4; ++h) {
    float sc[4], sf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { sc[j] = sh.chan[pc * PN + 4 * h + j][0]; sf[j] = sh.chan[pc * PN + 4 * h + j][1]; }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float t[4];
      gnf_unpack4<T>(v[k], h, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = gn_act<ACT>(fmaf(t[j], sc[j], sf[j]));
      gnf_pack4<T>(v[k], h, t);
      const int i = first + k * GNF_THREADS;
      if (h == PN / 4 - 1 && i < len) gnf_store(ab + (unsigned)i * 16u, PARTIAL ? gn_and(v[k], gn_kept_bits<T>(s, u.plane)) : v[k], o.stream);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <typename T, int ACT, int R, bool PARTIAL = false>
__global__ __launch_bounds__(GNF_THREADS, 6) void gn_fused_kernel(GnFused f, GnForward o) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  __shared__ GnfShared<EPR> sh;
  GnPlace u;
  if (!gnf_place(f, &sh.missing, u)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pc = threadIdx.x & 1, len = u.hi - u.lo;
  uint4 v[R];
  gnf_load<R>(v, o.x, o.x_pt, o.x_p0, f.s, u);
#pragma unroll
  for (int h = 0; h < PN / 4; ++h) {
    float acc[4] = {};
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float t[4];
      gnf_unpack4<T>(v[k], h, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += t[j];
      __builtin_amdgcn_sched_barrier(0);                   // piece after piece: interleaved, they would need twice the registers
    }
    gnf_wave_sums<PN>(acc, h, sh.red[0]);
  }
  __syncthreads();
  float sum = gnf_block_sum<PN>(sh.red[0]);
  for (int x2 = 1; x2 < f.m; x2 <<= 1) sum += __shfl_xor(sum, x2);             // over the cell's channels
  const float cmean = sum / (float)(f.m * (len / 2));
  gnf_keep_packed<R>(v);
#pragma unroll
  for (int h = 0; h < PN / 4; ++h) {
    float mu[4], acc[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) mu[j] = __shfl(cmean, pc * PN + 4 * h + j);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if ((int)threadIdx.x + k * GNF_THREADS < len) {
        float t[4];
        gnf_unpack4<T>(v[k], h, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(t[j] - mu[j], t[j] - mu[j], acc[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    gnf_wave_sums<PN>(acc, h, sh.red[1]);
  }
  gnf_keep_packed<R>(v);
  __syncthreads();
  float m2 = gnf_block_sum<PN>(sh.red[1]);
  for (int x2 = 1; x2 < f.m; x2 <<= 1) m2 += __shfl_xor(m2, x2);
  const bool owner = wave == 0 && lane < EPR && gn_mod(f.d_m, lane) == 0;
  bool got = true;
  unsigned before = 0;
  if (!u.alone) {
    if (owner) gnf_publish(f, u, gn_div(f.d_m, lane), cmean, m2);
    got = gnf_collect(f, u, sh.cells, &sh.missing, &before);
  } else {
    if (owner) { sh.cells[2 * (gn_div(f.d_m, lane))] = cmean; sh.cells[2 * (gn_div(f.d_m, lane)) + 1] = m2; }
    __syncthreads();
  }
  if (got) {
    gnf_scales<EPR>(f, o, u, sh, [&] { gnf_last(f, u, before, &sh.last); });
    gnf_apply<T, ACT, R, PARTIAL>(o, f.s, u, v, threadIdx.x, sh);
  } else {
    gnf_last(f, u, before, &sh.last);
    __syncthreads();
  }
  if (u.alone || !sh.last) return;
  for (unsigned listed = 0; gnf_next_listed(f, u, &listed, &sh.next);) {       // the launch's last block: what others gave up
    gnf_collect_again(f, u, sh.cells);
    gnf_scales<EPR>(f, o, u, sh, [] {});
    const unsigned char* xb = (const unsigned char*)o.x + ((u.n * o.x_pt + o.x_p0 + u.plane) * (long)f.s.npieces + u.lo) * 16;
#pragma unroll 1
    for (int i = threadIdx.x; i < u.hi - u.lo; i += GNF_THREADS) {
      uint4 one[1] = {*(const uint4*)(xb + (unsigned)i * 16u)};
      gnf_apply<T, ACT, 1, PARTIAL>(o, f.s, u, one, i, sh);
    }
  }
  if (gn_last_tag(u.tag)) gnf_clear_words(f.list);
}

// backward: part[block][channel] = (sum dz, sum dz * xhat) for the parameter gradients, group sums as above
struct GnBackward {
  const void *g, *x;
  void* dx;
  int g_pt, g_p0, x_pt, x_p0, d_pt, d_p0;
  const float *gamma, *mean, *rstd, *scale, *shift;
  float2* part;
  bool stream;
  float *dgamma, *dbeta;   // null: a launch of their own sums the partials
};
// The parameter gradients of a launch with few partials: a plane's last block to publish its own adds up all of them, in their order.
// Partials are written and read past the caches that other blocks do not share, so that the count alone orders them.  A launch
// of its own costs the host 2.8 us and the device 1 to 3 us more where CUs are idle (4 x 32 x 6 x 4096 fp32: 17.4 against 15.8 us, 16 x 128 x 6 x
// 1024 bf16, 384 blocks: 24.9 / 23.6), but every block waits for its partials: from two blocks a CU on the launch is cheaper (16 x 256 x 6 x 512 bf16,
// 512 blocks: 22.7 / 24.6, 64 x 512 x 6 x 256: 68.2 / 73.6).
constexpr long GNF_OWN_PARAM = 512;              // blocks: fewer sum the parameter gradients themselves
__device__ __forceinline__ unsigned gnf_count_plane(const GnFused& f, const GnBackward& o, const GnPlace& u) {
  if (!o.dgamma || threadIdx.x != GNF_COUNTER) return 0;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // this wave's partials have arrived
  return gnf_count(f.planes + u.plane);
}
__device__ __forceinline__ void gnf_last_plane(const GnFused& f, const GnBackward& o, const GnPlace& u, unsigned before, unsigned* last) {
  if (!o.dgamma || threadIdx.x != GNF_COUNTER) return;
  *last = before == (unsigned)(f.images * f.s.nseg) - 1;
  if (*last) gnf_reset(f.planes + u.plane);
}
template <int EPR> __device__ __forceinline__ void gnf_param(const GnFused& f, const GnBackward& o, const GnPlace& u, GnfShared<EPR>& sh) {
  const GnShape& s = f.s;
  constexpr int ROWS = GNF_THREADS / EPR;
  static_assert(sizeof(sh.cells) >= GNF_WAVES * EPR * 2 * sizeof(double) && GNF_OWN_PARAM <= GNF_MAX_BLOCKS, "the sums fit, and it is one launch");
  const int slot = threadIdx.x % EPR, row0 = threadIdx.x / EPR, rows = f.images * s.nseg;
  double a = 0.0, b = 0.0;
#pragma unroll 1
  for (int r = row0; r < rows; r += ROWS) {
    const int n = gn_div(f.d_nseg, r);
    const unsigned long long v = __hip_atomic_load((const unsigned long long*)(o.part + (((long)n * s.P + u.plane) * s.nseg + (r - n * s.nseg)) * EPR + slot),
                                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a += (double)__uint_as_float((unsigned)v);
    b += (double)__uint_as_float((unsigned)(v >> 32));
  }
#pragma unroll
  for (int m = 32; m >= EPR; m >>= 1) { a += __shfl_xor(a, m); b += __shfl_xor(b, m); }
  double* red = (double*)sh.cells;                         // [wave][slot][2]
  __syncthreads();
  if ((threadIdx.x & 63) < EPR) { red[((threadIdx.x >> 6) * EPR + slot) * 2] = a; red[((threadIdx.x >> 6) * EPR + slot) * 2 + 1] = b; }
  __syncthreads();
  const int c = u.plane * EPR + (int)threadIdx.x;
  if ((int)threadIdx.x < EPR && c < s.C) {
    a = b = 0.0;
#pragma unroll
    for (int w = 0; w < GNF_WAVES; ++w) { a += red[(w * EPR + slot) * 2]; b += red[(w * EPR + slot) * 2 + 1]; }
    o.dbeta[c] = (float)a;
    o.dgamma[c] = (float)b;
  }
}
template <int EPR> __device__ __forceinline__ void gnf_channels(const GnFused& f, const GnBackward& o, const GnPlace& u, GnfShared<EPR>& sh) {
  const GnShape& s = f.s;
  if ((int)threadIdx.x < EPR) {
    const int c = u.plane * EPR + threadIdx.x;
    const bool in = c < s.C;
    float* q = sh.chan[threadIdx.x];
    q[0] = o.scale[u.n * s.cpad + c];
    q[1] = o.shift[u.n * s.cpad + c];
    q[2] = in ? o.mean[u.n * s.G + gn_div(f.d_cpg, c)] : 0.f;
    q[3] = in ? o.rstd[u.n * s.G + gn_div(f.d_cpg, c)] : 0.f;
    q[4] = in ? o.gamma[c] : 0.f;
  }
  __syncthreads();
}
// From the cluster's cells in LDS to the constants of dx (sh.chan).  Between two barriers; `leave()` runs on the way.
template <int EPR, typename F>
__device__ __forceinline__ void gnf_scales_bwd(const GnFused& f, const GnPlace& u, GnfShared<EPR>& sh, F leave) {
  const GnShape& s = f.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c_lo = u.plane * EPR, c_hi = min(s.C, c_lo + EPR);
  const int g_lo = gn_div(f.d_cpg, c_lo), g_hi = gn_div(f.d_cpg, c_hi - 1);
  const int parts = gn_div(f.d_m, s.cpg) * s.nseg;
  for (int gi = g_lo + wave; gi <= g_hi; gi += GNF_WAVES) {
    double p1 = 0.0, p2 = 0.0;
    for (int i = lane; i < parts; i += 64) {
      int seg;
      const int at = gnf_cell(f, u, EPR, gi, i, &seg);
      p1 += (double)sh.cells[2 * at];
      p2 += (double)sh.cells[2 * at + 1];
    }
    gnf_wave_sum64(p1, p2);
    if (lane == 0) { sh.gstat[gi - g_lo][0] = (float)(p1 * f.inv_total); sh.gstat[gi - g_lo][1] = (float)(p2 * f.inv_total); }
  }
  __syncthreads();
  if ((int)threadIdx.x < EPR) {
    const int c = c_lo + threadIdx.x;
    const bool in = c < s.C;
    // dx = rstd (gamma dz - c1 - (x - mean) rstd c2) = k4 dz + (k6 (x - mean) + k5)
    const float r = sh.chan[threadIdx.x][3];
    sh.chan[threadIdx.x][4] *= r;
    sh.chan[threadIdx.x][5] = in ? -r * sh.gstat[gn_div(f.d_cpg, c) - g_lo][0] : 0.f;
    sh.chan[threadIdx.x][6] = in ? -r * r * sh.gstat[gn_div(f.d_cpg, c) - g_lo][1] : 0.f;
  }
  leave();
  __syncthreads();
}
// Whether dz can take the place of g in the registers between the passes, without another rounding: ReLU's is g or 0, fp32 holds any.
// (SiLU's in bf16 is computed twice.)
template <typename T, int ACT> constexpr bool gnf_keeps_dz() { return ACT == DN_ACT_RELU || sizeof(T) == 4; }
// Pieces first, first + GNF_THREADS, ... of the segment: dx, stored.  MASKED: vg holds dz already where it can.
template <typename T, int ACT, int R, bool MASKED, bool PARTIAL>
__device__ __forceinline__ void gnf_apply_bwd(const GnBackward& o, const GnShape& s, const GnPlace& u, uint4 (&vg)[R], uint4 (&vx)[R],
                                              int first, const GnfShared<RecTraits<T>::EPR>& sh) {
  constexpr int PN = Piece<T>::N;
  const int pc = threadIdx.x & 1, len = u.hi - u.lo;
  unsigned char* db = (unsigned char*)o.dx + ((u.n * o.d_pt + o.d_p0 + u.plane) * (long)s.npieces + u.lo) * 16;
#pragma unroll
  for (int h = 0; h < PN / 4; ++h) {
    __builtin_amdgcn_sched_barrier(0);
    float sc[4], sf[4], mu[4], k4[4], k5[4], k6[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* q = sh.chan[pc * PN + 4 * h + j];
      sc[j] = q[0]; sf[j] = q[1]; mu[j] = q[2]; k4[j] = q[4]; k5[j] = q[5]; k6[j] = q[6];
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float fg[4], fx[4];
      gnf_unpack4<T>(vg[k], h, fg);
      gnf_unpack4<T>(vx[k], h, fx);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float dz = MASKED && gnf_keeps_dz<T, ACT>() ? fg[j] : gn_act_grad<ACT>(fmaf(fx[j], sc[j], sf[j]), fg[j]);
        fg[j] = fmaf(k4[j], dz, fmaf(k6[j], fx[j] - mu[j], k5[j]));
      }
      gnf_pack4<T>(vg[k], h, fg);
      const int i = first + k * GNF_THREADS;
      if (h == PN / 4 - 1 && i < len) gnf_store(db + (unsigned)i * 16u, PARTIAL ? gn_and(vg[k], gn_kept_bits<T>(s, u.plane)) : vg[k], o.stream);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <typename T, int ACT, int R, bool PARTIAL = false>
__global__ __launch_bounds__(GNF_THREADS, R <= 4 ? 6 : 4) void gn_fused_bwd_kernel(GnFused f, GnBackward o) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  __shared__ GnfShared<EPR> sh;
  const GnShape& s = f.s;
  GnPlace u;
  if (!gnf_place(f, &sh.missing, u)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pc = threadIdx.x & 1;
  uint4 vg[R], vx[R];
  gnf_load<R>(vg, o.g, o.g_pt, o.g_p0, s, u);
  gnf_load<R>(vx, o.x, o.x_pt, o.x_p0, s, u);
  gnf_channels<EPR>(f, o, u, sh);
#pragma unroll
  for (int h = 0; h < PN / 4; ++h) {
    __builtin_amdgcn_sched_barrier(0);
    float sc[4], sf[4], mu[4], a1[4] = {}, a2[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* q = sh.chan[pc * PN + 4 * h + j];
      sc[j] = q[0]; sf[j] = q[1]; mu[j] = q[2];
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float fg[4], fx[4];
      gnf_unpack4<T>(vg[k], h, fg);
      gnf_unpack4<T>(vx[k], h, fx);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float dz = gn_act_grad<ACT>(fmaf(fx[j], sc[j], sf[j]), fg[j]);   // 0 past the segment's end: fg is
        a1[j] += dz;
        a2[j] = fmaf(dz, fx[j] - mu[j], a2[j]);                                // times rstd below
        fg[j] = dz;
        asm volatile("" : "+v"(a1[j]), "+v"(a2[j]));                           // both here: one put off would keep dz and x alive
      }
      if constexpr (gnf_keeps_dz<T, ACT>()) gnf_pack4<T>(vg[k], h, fg);
      __builtin_amdgcn_sched_barrier(0);
    }
    gnf_wave_sums<PN>(a1, h, sh.red[0]);
    gnf_wave_sums<PN>(a2, h, sh.red[1]);
  }
  gnf_keep_packed<R>(vg);
  gnf_keep_packed<R>(vx);
  __syncthreads();
  float s1 = gnf_block_sum<PN>(sh.red[0]), s2 = gnf_block_sum<PN>(sh.red[1]);
  const int cl = lane % EPR;
  s2 *= sh.chan[cl][3];
  if (wave == (int)GNF_COUNTER / 64 && lane < EPR)
    __hip_atomic_store((unsigned long long*)(o.part + ((u.n * s.P + u.plane) * s.nseg + u.seg) * EPR + lane),
                       (unsigned long long)__float_as_uint(s2) << 32 | __float_as_uint(s1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s1 *= sh.chan[cl][4];
  s2 *= sh.chan[cl][4];
  for (int x2 = 1; x2 < f.m; x2 <<= 1) { s1 += __shfl_xor(s1, x2); s2 += __shfl_xor(s2, x2); }
  const bool owner = wave == 0 && lane < EPR && gn_mod(f.d_m, lane) == 0;
  bool got = true;
  unsigned before = 0;
  if (!u.alone) {
    if (owner) gnf_publish(f, u, gn_div(f.d_m, lane), s1, s2);
    got = gnf_collect(f, u, sh.cells, &sh.missing, &before);
  } else {
    if (owner) { sh.cells[2 * (gn_div(f.d_m, lane))] = s1; sh.cells[2 * (gn_div(f.d_m, lane)) + 1] = s2; }
    __syncthreads();
  }
  const unsigned before_plane = gnf_count_plane(f, o, u);
  if (got) {
    gnf_scales_bwd<EPR>(f, u, sh, [&] { gnf_last(f, u, before, &sh.last); gnf_last_plane(f, o, u, before_plane, &sh.last_plane); });
    gnf_apply_bwd<T, ACT, R, true, PARTIAL>(o, s, u, vg, vx, threadIdx.x, sh);
  } else {
    gnf_last(f, u, before, &sh.last);
    gnf_last_plane(f, o, u, before_plane, &sh.last_plane);
    __syncthreads();
  }
  if (o.dgamma && sh.last_plane) gnf_param<EPR>(f, o, u, sh);
  if (u.alone || !sh.last) return;
  for (unsigned listed = 0; gnf_next_listed(f, u, &listed, &sh.next);) {       // the launch's last block: what others gave up
    gnf_channels<EPR>(f, o, u, sh);
    gnf_collect_again(f, u, sh.cells);
    gnf_scales_bwd<EPR>(f, u, sh, [] {});
    const unsigned char* gb = (const unsigned char*)o.g + ((u.n * o.g_pt + o.g_p0 + u.plane) * (long)s.npieces + u.lo) * 16;
    const unsigned char* xb = (const unsigned char*)o.x + ((u.n * o.x_pt + o.x_p0 + u.plane) * (long)s.npieces + u.lo) * 16;
#pragma unroll 1
    for (int i = threadIdx.x; i < u.hi - u.lo; i += GNF_THREADS) {
      uint4 one_g[1] = {*(const uint4*)(gb + (unsigned)i * 16u)}, one_x[1] = {*(const uint4*)(xb + (unsigned)i * 16u)};
      gnf_apply_bwd<T, ACT, 1, false, PARTIAL>(o, s, u, one_g, one_x, i, sh);
    }
  }
  if (gn_last_tag(u.tag)) gnf_clear_words(f.list);
}

int gn_shape(const char* name, dn_tensor x, int N, int H, int W, int groups, int dtype, GnShape* out) {
  DN_CHECK_ARG(dtype == DN_F32 || dtype == DN_BF16, "%s: bad dtype %d", name, dtype);
  DN_CHECK_ARG(N >= 0 && H >= 1 && W >= 1 && (long)H * W <= (1L << 25), "%s: bad size N=%d H=%d W=%d (H * W <= 2^25)", name, N, H, W);
  DN_CHECK_ARG(x.channels >= 1 && groups >= 1 && x.channels % groups == 0, "%s: %d channels do not divide into %d groups", name, x.channels,
               groups);
  GnShape s;
  s.N = N; s.C = x.channels; s.G = groups; s.P = dn_planes(x.channels, dtype);
  s.cpg = x.channels / groups; s.cpad = dn_channel_pad(x.channels);
  s.npieces = 2 * H * W;
  s.nseg = (s.npieces + GN_SEG - 1) / GN_SEG;
  s.seg_len = ((s.npieces / 2 + s.nseg - 1) / s.nseg) * 2;
  s.nseg = (s.npieces + s.seg_len - 1) / s.seg_len;
  DN_CHECK_ARG((long)N * s.P * s.nseg < (1L << 31) && (long)N * s.G < (1L << 31), "%s: too many images x planes", name);
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
// Whether tensors a and b share memory without being the same planes (the same planes: in place).
bool gn_mixed_up(dn_tensor a, dn_tensor b, const GnShape& s) {
  const long plane = s.npieces * 16L;
  if (a.base == b.base && a.planes_total == b.planes_total) {
    const int apart = a.plane0 > b.plane0 ? a.plane0 - b.plane0 : b.plane0 - a.plane0;
    return apart != 0 && apart < s.P;
  }
  const char *a0 = (const char*)a.base + a.plane0 * plane, *b0 = (const char*)b.base + b.plane0 * plane;
  return a0 < b0 + ((s.N - 1L) * b.planes_total + s.P) * plane && b0 < a0 + ((s.N - 1L) * a.planes_total + s.P) * plane;
}
bool gn_same(dn_tensor a, dn_tensor b) { return a.base == b.base && a.planes_total == b.planes_total && a.plane0 == b.plane0; }
// the three-launch form's blocks: a launch holds less than 2^32 threads
bool gn_launches(const GnShape& s) { return std::max((long)s.N * s.P * s.nseg, (long)s.N * s.G) * GN_THREADS < 1L << 32; }
long gn_part_bytes(const GnShape& s, int dtype) {
  return (long)s.N * s.P * s.nseg * (dtype == DN_BF16 ? 16 : 8) * (long)sizeof(float2);
}
// Whether the one-pass form takes this shape with R pieces per thread, and its plan.
bool gn_fused_plan(const GnShape& s, int dtype, int r, GnFused* f) {
  const int epr = dtype == DN_BF16 ? 16 : 8;
  f->s = s;
  const int seg = GNF_THREADS * r;
  const int nseg = (s.npieces + seg - 1) / seg;
  f->s.seg_len = ((s.npieces / 2 + nseg - 1) / nseg) * 2;
  f->s.nseg = (s.npieces + f->s.seg_len - 1) / f->s.seg_len;
  int a = s.cpg, b = epr;
  while (b) { const int t = a % b; a = b; b = t; }
  f->m = a;
  f->ncell = epr / a;
  f->ps = std::min(s.P, s.cpg / a);              // lcm(cpg, epr) / epr planes
  f->nsets = (s.P + f->ps - 1) / f->ps;
  const long k = (long)f->ps * f->s.nseg;
  f->d_most = gn_divisor(k);
  f->d_nsets = gn_divisor(f->nsets);
  f->d_nseg = gn_divisor(f->s.nseg);
  f->d_cpg = gn_divisor(s.cpg);
  f->d_m = gn_divisor(f->m);
  f->inv_total = 1.0 / ((double)s.cpg * (s.npieces / 2));
  f->polls = dn_tune().gn_polls ? dn_tune().gn_polls - 1 : GNF_POLLS;
  return k <= GNF_MAX_K && k * f->ncell <= GNF_MAX_CELLS && f->nsets * k <= GNF_MAX_BLOCKS && s.C <= 1 << 15;
}
constexpr int GNF_R = 8;                         // 64 KB of a tensor in a block's registers: three blocks on a CU
// Backward holds 64 KB of each of two tensors: two blocks on a CU.  With 32 KB and three blocks, more of them wait for each other:
// 301 us against 281 for 256 x 32 x 6 x 4096 bf16 (302 against 275 for 256 x 512 x 6 x 256, where 64 KB hold whole groups), 29 against 27
// for 16 images; only up to 4 images, which leave CUs without a block, are done sooner (2: 14.0 / 15.7 us).  One size for
// all: an image's results do not depend, not even in their last bits, on how many others are in the batch.
constexpr int GNF_R_BWD = 8;
// counters and published words first, at fixed places whatever the shape; the three-launch form's partials, and the partials of
// the parameter gradients, behind them
long gn_workspace(const GnShape& s, int dtype) {
  GnFused f;
  const bool fused = gn_fused_plan(s, dtype, GNF_R_BWD, &f);
  const long chunks = fused ? (long)s.P * gn_param_chunks(f.s) * (dtype == DN_BF16 ? 16 : 8) * (long)sizeof(double2) : 0;
  const long parts = std::max(gn_part_bytes(s, dtype), fused ? gn_part_bytes(f.s, dtype) + chunks : 0);
  return GNF_END + parts + (long)s.N * s.G * (long)sizeof(float2) + 256;
}
void gn_fused_workspace(GnFused* f, void* workspace) {
  char* w = (char*)workspace;
  f->ctrl = (unsigned*)w;
  f->depart = (unsigned*)(w + GNF_CTRL_BYTES);
  f->planes = (unsigned*)(w + GNF_PLANES0);
  f->list = (unsigned long long*)(w + GNF_LIST0);
  f->slot = (unsigned long long*)(w + GNF_SLOT0);
}
bool gn_streams(const GnShape& s) { return (long)s.N * s.P * s.npieces * 16 >= GNF_STREAM_BYTES; }
// launch(grid) for as many images at a time as a launch takes
template <typename F> void gn_fused_each(GnFused* f, F launch) {
  const long k = (long)f->ps * f->s.nseg;
  const int most = (int)std::min<long>(f->s.N, GNF_MAX_BLOCKS / (f->nsets * k));
  for (f->image0 = 0; f->image0 < f->s.N; f->image0 += most) {
    f->images = std::min(most, f->s.N - f->image0);
    launch(dim3((unsigned)(f->images * f->nsets * k)));
  }
}

template <typename T, int ACT>
void gn_forward_launch(dn_tensor x, dn_tensor a, const GnShape& s, const float* gamma, const float* beta, float eps, float* mean,
                       float* rstd, float* scale, float* shift, void* workspace, int dtype, hipStream_t st) {
  constexpr int EPR = RecTraits<T>::EPR;
  GnFused f;
  if (gn_fused_plan(s, dtype, GNF_R, &f)) {
    gn_fused_workspace(&f, workspace);
    const GnForward o{x.base, a.base, x.planes_total, x.plane0, a.planes_total, a.plane0, gamma, beta, eps, mean, rstd, scale, shift,
                      gn_streams(s)};
    const int rows = (f.s.seg_len + GNF_THREADS - 1) / GNF_THREADS;            // pieces of a thread
    gn_fused_each(&f, [&](dim3 grid) {
      if (s.C % EPR) hipLaunchKernelGGL((gn_fused_kernel<T, ACT, GNF_R, true>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 2) hipLaunchKernelGGL((gn_fused_kernel<T, ACT, 2>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 4) hipLaunchKernelGGL((gn_fused_kernel<T, ACT, 4>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 6) hipLaunchKernelGGL((gn_fused_kernel<T, ACT, 6>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else hipLaunchKernelGGL((gn_fused_kernel<T, ACT, GNF_R>), grid, dim3(GNF_THREADS), 0, st, f, o);
    });
    return;
  }
  float2* part = (float2*)((char*)workspace + GNF_END);
  const dim3 grid((unsigned)((long)s.N * s.P * s.nseg));
  hipLaunchKernelGGL((gn_stats_kernel<T>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)x.base, x.planes_total, x.plane0, s, part);
  hipLaunchKernelGGL((gn_finalize_kernel<EPR>), dim3((unsigned)((long)s.N * s.G)), dim3(GN_THREADS), 0, st, part, s, gamma, beta, eps, mean,
                     rstd, scale, shift);
  hipLaunchKernelGGL((gn_apply_kernel<T, ACT>), grid, dim3(GN_THREADS), 0, st, (const unsigned char*)x.base, x.planes_total, x.plane0,
                     (unsigned char*)a.base, a.planes_total, a.plane0, s, scale, shift);
}
template <typename T, int ACT>
void gn_backward_launch(dn_tensor g, dn_tensor x, dn_tensor dx, const GnShape& s, const float* gamma, const float* mean, const float* rstd,
                        const float* scale, const float* shift, float* dgamma, float* dbeta, void* workspace, int dtype,
                        hipStream_t st) {
  constexpr int EPR = RecTraits<T>::EPR;
  float2* part = (float2*)((char*)workspace + GNF_END);
  GnFused f;
  if (gn_fused_plan(s, dtype, GNF_R_BWD, &f)) {
    gn_fused_workspace(&f, workspace);
    const bool own = (long)s.N * f.nsets * f.d_most.d < GNF_OWN_PARAM;
    const GnBackward o{g.base, x.base, dx.base, g.planes_total, g.plane0, x.planes_total, x.plane0, dx.planes_total, dx.plane0,
                       gamma, mean, rstd, scale, shift, part, gn_streams(s), own ? dgamma : nullptr, own ? dbeta : nullptr};
    const int rows = (f.s.seg_len + GNF_THREADS - 1) / GNF_THREADS;
    gn_fused_each(&f, [&](dim3 grid) {
      if (s.C % EPR) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, GNF_R_BWD, true>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 1) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, 1>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 2) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, 2>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 4) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, 4>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else if (rows <= 6) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, 6>), grid, dim3(GNF_THREADS), 0, st, f, o);
      else hipLaunchKernelGGL((gn_fused_bwd_kernel<T, ACT, GNF_R_BWD>), grid, dim3(GNF_THREADS), 0, st, f, o);
    });
    if (own) return;
    const int chunks = gn_param_chunks(f.s);
    hipLaunchKernelGGL((gn_bwd_param_chunk_kernel<EPR>), dim3(s.P, chunks), dim3(GN_THREADS), 0, st, part, f.s, chunks, f.depart,
                       (double2*)((char*)part + gn_part_bytes(f.s, dtype)), dgamma, dbeta);
    return;
  }
  float2* coef = (float2*)((char*)workspace + GNF_END + gn_part_bytes(s, dtype));
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
  DN_CHECK_ARG(eps >= 1e-30f && eps <= 1e30f, "dn_group_norm_act: eps must be within 1e-30 and 1e30");
  DN_CHECK_ARG(act >= DN_ACT_NONE && act <= DN_ACT_SILU, "dn_group_norm_act: bad activation %d", act);
  GnFused f;
  DN_CHECK_ARG(gn_fused_plan(s, dtype, GNF_R, &f) || gn_launches(s), "dn_group_norm_act: too many images x planes");
  DN_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= gn_workspace(s, dtype),
               "dn_group_norm_act: workspace of %ld bytes, %ld needed (16-byte aligned)", workspace_bytes, gn_workspace(s, dtype));
  DN_CHECK_ARG(!gn_mixed_up(a, x, s), "dn_group_norm_act: a overlaps x and is not x");
#define GN_CALL(T, A) (gn_forward_launch<T, A>(x, a, s, gamma, beta, eps, mean, rstd, scale, shift, workspace, dtype, (hipStream_t)stream))
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
  GnFused f;
  DN_CHECK_ARG(gn_fused_plan(s, dtype, GNF_R_BWD, &f) || gn_launches(s), "dn_group_norm_act_backward: too many images x planes");
  DN_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= gn_workspace(s, dtype),
               "dn_group_norm_act_backward: workspace of %ld bytes, %ld needed (16-byte aligned)", workspace_bytes, gn_workspace(s, dtype));
  DN_CHECK_ARG(!gn_mixed_up(dx, g, s), "dn_group_norm_act_backward: dx overlaps g and is not g");
  DN_CHECK_ARG(!gn_mixed_up(dx, x, s) && !gn_same(dx, x), "dn_group_norm_act_backward: dx overlaps x");
  DN_CHECK_ARG(dgamma + s.C <= dbeta || dbeta + s.C <= dgamma, "dn_group_norm_act_backward: dgamma and dbeta overlap");
#define GN_CALL(T, A) (gn_backward_launch<T, A>(g, x, dx, s, gamma, mean, rstd, scale, shift, dgamma, dbeta, workspace, dtype, (hipStream_t)stream))
  GN_DISPATCH(dtype, act, GN_CALL)
#undef GN_CALL
  DN_LAUNCH_CHECK();
  return DN_OK;
}

}  // extern "C"
