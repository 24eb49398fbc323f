// AdamW over many tensors at once, moments in fp32 or in 8 bits, and the global gradient norm.
//
//   g' = coef * g                      coef = min(1, max_norm / (norm + 1e-6)) of the global norm, or 1
//   m = beta1 m + (1 - beta1) g'       v = beta2 v + (1 - beta2) g'^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// A launch takes up to ADAMW_MAX tensors BY VALUE in its kernel arguments: no table in device memory has to be kept, copied
// or protected from a later call, and a captured launch carries its own.  The moments of all tensors lie in two flat buffers;
// a tensor's start there is a multiple of 256 elements.
//
// 8-bit moments: e4m3 codes and one fp32 scale per 256 consecutive elements of a tensor, the smallest power of two that brings
// the block's largest magnitude to 448 or below (a power of two: dividing by it rounds nothing, so a code depends on the new
// moment alone).  Rounding is stochastic, up with the probability of the remainder, 16 bits of a hash of
// (tensor's number, element in the tensor, step, seed) for each moment: to nearest, a second moment would stand still as soon as
// one step moves it by less than half a code step (2^-4 of its value, where 1 - beta2 is 2^-10).  A second moment above zero keeps at least the smallest code: m / (0 + eps)
// would be a step of any size.  New moments are formed in fp64 before they are rounded to 8 bits, so that which side of a
// code border a value falls on does not depend on how the products were contracted.  A moment that is not finite keeps its
// element to itself: it is left out of the block's scale and stored as NaN.
#include <algorithm>
#include <cmath>
#include "common.h"
#include "dnanet_hip.h"

namespace {

constexpr int ADAMW_MAX = 96;                 // tensors of a launch: their records fill the 4-KiB kernel argument segment
constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_CHUNK = 2048;             // elements of a block, a multiple of the 256-element state blocks: all loads of a wave in
                                              // flight at once; 4096 in two turns: 90 us instead of 88 for 27 M bf16 elements
constexpr unsigned ADAMW_P_BF16 = 1, ADAMW_G_BF16 = 2, ADAMW_VECTOR = 4;
constexpr int ADAMW_NUMBER = 3;               // a tensor's number lies in the flags from this bit on

struct AdamwEntry {                           // 40 bytes
  void* p;
  void* g;
  long n;
  unsigned state;                             // start in the moment buffers / 256
  float decay;
  unsigned block0;                            // first block of this tensor
  unsigned flags;                             // ADAMW_*, and the tensor's number
};
struct AdamwList {
  AdamwEntry e[ADAMW_MAX];
  int count;
};
struct AdamwArgs {
  float beta1, beta2, omb1, omb2, eps;        // omb = 1 - beta, formed in fp64
  double dbeta1, dbeta2, domb1, domb2;
  float lr, step_size, inv_sqrt_bc2;          // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  unsigned step, seed;
  int zero_grad;
  const float* coef;                          // nullable: [1] of {norm, coefficient}
  const float* hyper;                         // nullable: {lr, lr / bc1, 1 / sqrt(bc2)} in device memory
  const long long* step_dev;                  // with hyper
};

// index of the tensor that owns block b (blocks of a tensor are consecutive, block0 ascends): every lane compares two entries,
// one load's latency instead of seven for a binary search
__device__ __forceinline__ int adamw_find(const AdamwList& l, unsigned b) {
  const int lane = threadIdx.x & 63;
  const bool first = lane < l.count && l.e[min(lane, ADAMW_MAX - 1)].block0 <= b;
  const bool second = lane + 64 < l.count && l.e[min(lane + 64, ADAMW_MAX - 1)].block0 <= b;
  return __popcll(__ballot(first)) + __popcll(__ballot(second)) - 1;
}

// 32 mixed bits: two rounds of shift and multiply, shifts and multipliers as C. Wellons published them (2018)
__device__ __forceinline__ unsigned adamw_hash(unsigned x) {
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x = (x ^ (x >> 15)) * 0x846CA68Bu;
  return x ^ (x >> 16);
}

// four elements from index i; where the tensor is not aligned or ends, one by one
template <typename T> __device__ __forceinline__ void adamw_load(const void* base, long i, int count, bool vec, float* f) {
  const T* q = (const T*)base + i;
  if (vec && count == 4) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *(const float4*)q;
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
      const uint2 v = *(const uint2*)q;
      f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
      f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < count ? dn_to_float(q[j]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void adamw_store(void* base, long i, int count, bool vec, const float* f) {
  T* q = (T*)base + i;
  if (vec && count == 4) {
    if constexpr (sizeof(T) == 4) {
      *(float4*)q = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      const __bf16 h[4] = {(__bf16)f[0], (__bf16)f[1], (__bf16)f[2], (__bf16)f[3]};      // to nearest even
      uint2 v;
      v.x = (unsigned)__builtin_bit_cast(unsigned short, h[0]) | ((unsigned)__builtin_bit_cast(unsigned short, h[1]) << 16);
      v.y = (unsigned)__builtin_bit_cast(unsigned short, h[2]) | ((unsigned)__builtin_bit_cast(unsigned short, h[3]) << 16);
      *(uint2*)q = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < count) q[j] = dn_from_float<T>(f[j]);
  }
}
__device__ __forceinline__ void adamw_load_any(const void* base, bool bf16, long i, int count, bool vec, float* f) {
  if (bf16) adamw_load<__bf16>(base, i, count, vec, f); else adamw_load<float>(base, i, count, vec, f);
}
__device__ __forceinline__ void adamw_store_any(void* base, bool bf16, long i, int count, bool vec, const float* f) {
  if (bf16) adamw_store<__bf16>(base, i, count, vec, f); else adamw_store<float>(base, i, count, vec, f);
}

struct AdamwScalars { float lr, step_size, inv_sqrt_bc2, coef; unsigned step; };
__device__ __forceinline__ AdamwScalars adamw_scalars(const AdamwArgs& a) {
  AdamwScalars s{a.lr, a.step_size, a.inv_sqrt_bc2, 1.f, a.step};
  if (a.hyper) { s.lr = a.hyper[0]; s.step_size = a.hyper[1]; s.inv_sqrt_bc2 = a.hyper[2]; s.step = (unsigned)*a.step_dev; }
  if (a.coef) s.coef = a.coef[1];
  return s;
}

// p (1 - lr decay) - step m / (sqrt(v) / sqrt(1 - beta2^t) + eps); square root and reciprocal to 1 ulp.  The square root
// instruction takes a denormal v for zero, which matters where eps is zero: v below 2^-96 is brought up by 2^64.
__device__ __forceinline__ float adamw_update(float p, float m, float v, float keep, const AdamwScalars& s, float eps) {
  const bool tiny = v < 0x1p-96f;
  const float root = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p64f : v);
  const float denom = fmaf(tiny ? root * 0x1p-32f : root, s.inv_sqrt_bc2, eps);
  return fmaf(-s.step_size * m, __builtin_amdgcn_rcpf(denom), p * keep);
}

// A row is 256 elements, four of each lane of a wave; a wave's rows are all in flight at once.
constexpr int ADAMW_ROW = 256, ADAMW_WAVES = ADAMW_THREADS / 64, ADAMW_ROWS = ADAMW_CHUNK / ADAMW_ROW / ADAMW_WAVES;

struct AdamwRow32 { float p[4], g[4], m[4], v[4]; };
__device__ __forceinline__ void adamw_row32(AdamwRow32& r, const AdamwArgs& a, const AdamwScalars& s, float keep) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float g = r.g[j] * s.coef;
    r.m[j] = fmaf(a.beta1, r.m[j], a.omb1 * g);
    r.v[j] = fmaf(a.beta2, r.v[j], a.omb2 * g * g);
    r.p[j] = adamw_update(r.p[j], r.m[j], r.v[j], keep, s, a.eps);
  }
}
// `rows` whole rows of an aligned tensor from element `first` on
template <typename P, typename G>
__device__ __forceinline__ void adamw_rows32(const AdamwEntry& e, long first, int rows, float* m, float* v, const AdamwArgs& a,
                                             const AdamwScalars& s, float keep) {
  const int row = threadIdx.x >> 6;
  AdamwRow32 r[ADAMW_ROWS];
  const long i = first + (long)row * ADAMW_ROW + (threadIdx.x & 63) * 4;
#pragma unroll
  for (int k = 0; k < ADAMW_ROWS; ++k)
    if (row + k * ADAMW_WAVES < rows) {
      const long at = i + (long)k * ADAMW_WAVES * ADAMW_ROW;
      adamw_load<P>(e.p, at, 4, true, r[k].p);
      adamw_load<G>(e.g, at, 4, true, r[k].g);
      adamw_load<float>(m, at, 4, true, r[k].m);
      adamw_load<float>(v, at, 4, true, r[k].v);
    }
#pragma unroll
  for (int k = 0; k < ADAMW_ROWS; ++k)
    if (row + k * ADAMW_WAVES < rows) {
      const long at = i + (long)k * ADAMW_WAVES * ADAMW_ROW;
      adamw_row32(r[k], a, s, keep);
      adamw_store<P>(e.p, at, 4, true, r[k].p);
      adamw_store<float>(m, at, 4, true, r[k].m);
      adamw_store<float>(v, at, 4, true, r[k].v);
      if (a.zero_grad) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        adamw_store<G>(e.g, at, 4, true, zero);
      }
    }
}

// Bound by HBM: 28 bytes an element with fp32 parameters and gradients, 20 with bf16.  128 M fp32 elements 672 us (5.3 TB/s, a copy's
// rate), 12.1 M (a U-Net of four levels of 32 filters) 70 us; 46 k elements 4.2 us, a launch.
__global__ __launch_bounds__(ADAMW_THREADS) void adamw_kernel(AdamwList list, float* exp_avg, float* exp_avg_sq, AdamwArgs a) {
  const AdamwEntry e = list.e[adamw_find(list, blockIdx.x)];
  const AdamwScalars s = adamw_scalars(a);
  const float keep = 1.f - s.lr * e.decay;
  float* m = exp_avg + (long)e.state * 256;
  float* v = exp_avg_sq + (long)e.state * 256;
  const long lo = (long)(blockIdx.x - e.block0) * ADAMW_CHUNK, hi = min(e.n, lo + ADAMW_CHUNK);
  const bool pb = e.flags & ADAMW_P_BF16, gb = e.flags & ADAMW_G_BF16, vec = e.flags & ADAMW_VECTOR;
  const int rows = vec ? (int)((hi - lo) / ADAMW_ROW) : 0;
  if (pb) {
    if (gb) adamw_rows32<__bf16, __bf16>(e, lo, rows, m, v, a, s, keep);
    else adamw_rows32<__bf16, float>(e, lo, rows, m, v, a, s, keep);
  } else {
    if (gb) adamw_rows32<float, __bf16>(e, lo, rows, m, v, a, s, keep);
    else adamw_rows32<float, float>(e, lo, rows, m, v, a, s, keep);
  }
  for (long i = lo + rows * ADAMW_ROW + threadIdx.x * 4; i < hi; i += ADAMW_THREADS * 4) {       // the rest, or an unaligned tensor
    const int count = (int)min(4L, hi - i);
    AdamwRow32 r;
    adamw_load_any(e.p, pb, i, count, vec, r.p);
    adamw_load_any(e.g, gb, i, count, vec, r.g);
    adamw_load<float>(m, i, count, true, r.m);
    adamw_load<float>(v, i, count, true, r.v);
    adamw_row32(r, a, s, keep);
    adamw_store_any(e.p, pb, i, count, vec, r.p);
    adamw_store<float>(m, i, count, true, r.m);
    adamw_store<float>(v, i, count, true, r.v);
    if (a.zero_grad) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      adamw_store_any(e.g, gb, i, count, vec, zero);
    }
  }
}

// Two values over their block's scale -> e4m3 codes in bytes 2 * HALF and up of `codes`.  The conversion adds 20 bits of its
// second operand to the mantissa's 20 bits below a code step (and as far below the even steps under 2^-6) and cuts off: up with the
// probability of the remainder.  Here 16 random bits, from the top.
template <bool HIGH> __device__ __forceinline__ unsigned adamw_encode(unsigned codes, float y0, unsigned bits0, float y1, unsigned bits1) {
  codes = (unsigned)__builtin_amdgcn_cvt_sr_fp8_f32(y0, (int)bits0, (int)codes, HIGH ? 2 : 0);
  return (unsigned)__builtin_amdgcn_cvt_sr_fp8_f32(y1, (int)bits1, (int)codes, HIGH ? 3 : 1);
}

// the block's scale from the bits of its largest finite magnitude, as an exponent: the smallest k with amax <= 448 * 2^k, at
// least -126
__device__ __forceinline__ int adamw_exponent(unsigned amax) {
  return max((int)((amax + 0x1FFFFFu) >> 23) - 127 - 8, -126);
}

// Largest of the lanes' values (bits of magnitudes: they order as the magnitudes do): DPP moves within and across the rows of 16,
// no LDS
__device__ __forceinline__ unsigned adamw_wave_max(unsigned v) {
#define ADAMW_DPP(ctrl) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false))
  ADAMW_DPP(0xB1);       // quad_perm [1,0,3,2]
  ADAMW_DPP(0x4E);       // quad_perm [2,3,0,1]
  ADAMW_DPP(0x124);      // row_ror:4
  ADAMW_DPP(0x128);      // row_ror:8
  ADAMW_DPP(0x142);      // row_bcast:15 -> the next row (rows 1, 3 hold two rows' maximum)
  ADAMW_DPP(0x143);      // row_bcast:31 -> rows 2, 3 (row 3 holds all)
#undef ADAMW_DPP
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// One row of a tensor with 8-bit moments: codes and scales in, codes and scales out.  count: elements of this lane that exist.
struct AdamwRow8 {
  float p[4], g[4];
  unsigned cm, cv;
  float ms, vs;
};
__device__ __forceinline__ void adamw_row8(AdamwRow8& r, int count, unsigned place, const AdamwArgs& a, const AdamwScalars& s, float keep) {
  const double ms = (double)r.ms * a.dbeta1, vs = (double)r.vs * a.dbeta2, coef = (double)s.coef;
  const float om[4] = {__builtin_amdgcn_cvt_f32_fp8(r.cm, 0), __builtin_amdgcn_cvt_f32_fp8(r.cm, 1), __builtin_amdgcn_cvt_f32_fp8(r.cm, 2),
                       __builtin_amdgcn_cvt_f32_fp8(r.cm, 3)};
  const float ov[4] = {__builtin_amdgcn_cvt_f32_fp8(r.cv, 0), __builtin_amdgcn_cvt_f32_fp8(r.cv, 1), __builtin_amdgcn_cvt_f32_fp8(r.cv, 2),
                       __builtin_amdgcn_cvt_f32_fp8(r.cv, 3)};
  float fm[4], fv[4];
  unsigned am = 0, av = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double g = (double)r.g[j] * coef;
    fm[j] = j < count ? (float)fma((double)om[j], ms, a.domb1 * g) : 0.f;
    fv[j] = j < count ? (float)fma((double)ov[j], vs, a.domb2 * g * g) : 0.f;
    const unsigned bm = __float_as_uint(fm[j]) & 0x7FFFFFFFu, bv = __float_as_uint(fv[j]) & 0x7FFFFFFFu;
    am = max(am, bm < 0x7F800000u ? bm : 0u);
    av = max(av, bv < 0x7F800000u ? bv : 0u);
  }
  am = adamw_wave_max(am);
  av = adamw_wave_max(av);
  const int em = adamw_exponent(am), ev = adamw_exponent(av);
  const float im = __uint_as_float((unsigned)(127 - em) << 23), iv = __uint_as_float((unsigned)(127 - ev) << 23);      // 2^-k
  float ym[4], yv[4];
  unsigned h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = adamw_hash(place + j);
    ym[j] = fmaf(fm[j], im, 0.f);                      // the sum makes -0 a +0
    yv[j] = fv[j] > 0.f ? fmaxf(fv[j] * iv, 0x1p-9f) : fv[j];
    r.p[j] = adamw_update(r.p[j], fm[j], fv[j], keep, s, a.eps);
  }
  r.cm = adamw_encode<true>(adamw_encode<false>(0, ym[0], h[0] << 16, ym[1], h[1] << 16), ym[2], h[2] << 16, ym[3], h[3] << 16);
  r.cv = adamw_encode<true>(adamw_encode<false>(0, yv[0], h[0] & 0xFFFF0000u, yv[1], h[1] & 0xFFFF0000u), yv[2], h[2] & 0xFFFF0000u,
                            yv[3], h[3] & 0xFFFF0000u);
  r.ms = am ? __uint_as_float((unsigned)(127 + em) << 23) : 0.f;
  r.vs = av ? __uint_as_float((unsigned)(127 + ev) << 23) : 0.f;
}

struct Adamw8State {
  unsigned char *m, *v;
  float *ms, *vs;
};
template <typename P, typename G>
__device__ __forceinline__ void adamw_rows8(const AdamwEntry& e, long first, int rows, const Adamw8State& o, unsigned key, const AdamwArgs& a,
                                            const AdamwScalars& s, float keep) {
  const int lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  AdamwRow8 r[ADAMW_ROWS];
#pragma unroll
  for (int k = 0; k < ADAMW_ROWS; ++k)
    if (row + k * ADAMW_WAVES < rows) {
      const long base = first + (long)(row + k * ADAMW_WAVES) * ADAMW_ROW, at = base + lane * 4;
      adamw_load<P>(e.p, at, 4, true, r[k].p);
      adamw_load<G>(e.g, at, 4, true, r[k].g);
      r[k].cm = *(const unsigned*)(o.m + at);
      r[k].cv = *(const unsigned*)(o.v + at);
      r[k].ms = o.ms[base >> 8];
      r[k].vs = o.vs[base >> 8];
    }
#pragma unroll
  for (int k = 0; k < ADAMW_ROWS; ++k)
    if (row + k * ADAMW_WAVES < rows) {
      const long base = first + (long)(row + k * ADAMW_WAVES) * ADAMW_ROW, at = base + lane * 4;
      adamw_row8(r[k], 4, (unsigned)at + key, a, s, keep);
      adamw_store<P>(e.p, at, 4, true, r[k].p);
      *(unsigned*)(o.m + at) = r[k].cm;
      *(unsigned*)(o.v + at) = r[k].cv;
      if (lane == 0) { o.ms[base >> 8] = r[k].ms; o.vs[base >> 8] = r[k].vs; }
      if (a.zero_grad) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        adamw_store<G>(e.g, at, 4, true, zero);
      }
    }
}

// 16 bytes an element with fp32 parameters and gradients: bound by HBM, 128 M elements 373 us (5.5 TB/s), 12.1 M 41 us.  With bf16, 10
// bytes: 284 us (4.5 TB/s), the vector units are busy for most of it (61 instructions an element, 10 of them fp64 or conversions to it).
__global__ __launch_bounds__(ADAMW_THREADS) void adamw8_kernel(AdamwList list, unsigned char* exp_avg, unsigned char* exp_avg_sq,
                                                               float* m_scale, float* v_scale, AdamwArgs a) {
  const AdamwEntry e = list.e[adamw_find(list, blockIdx.x)];
  const AdamwScalars s = adamw_scalars(a);
  const float keep = 1.f - s.lr * e.decay;
  const unsigned key = (e.flags >> ADAMW_NUMBER) * 0xC2B2AE35u + s.step * 0x9E3779B9u + a.seed * 0x85EBCA6Bu;
  const Adamw8State o{exp_avg + (long)e.state * 256, exp_avg_sq + (long)e.state * 256, m_scale + e.state, v_scale + e.state};
  const long lo = (long)(blockIdx.x - e.block0) * ADAMW_CHUNK, hi = min(e.n, lo + ADAMW_CHUNK);
  const bool pb = e.flags & ADAMW_P_BF16, gb = e.flags & ADAMW_G_BF16, vec = e.flags & ADAMW_VECTOR;
  const int rows = vec ? (int)((hi - lo) / ADAMW_ROW) : 0;
  if (pb) {
    if (gb) adamw_rows8<__bf16, __bf16>(e, lo, rows, o, key, a, s, keep);
    else adamw_rows8<__bf16, float>(e, lo, rows, o, key, a, s, keep);
  } else {
    if (gb) adamw_rows8<float, __bf16>(e, lo, rows, o, key, a, s, keep);
    else adamw_rows8<float, float>(e, lo, rows, o, key, a, s, keep);
  }
  const int lane = threadIdx.x & 63;
  for (long base = lo + (rows + (threadIdx.x >> 6)) * ADAMW_ROW; base < hi; base += ADAMW_WAVES * ADAMW_ROW) {      // the rest, or an unaligned tensor
    const long at = base + lane * 4;
    const int count = (int)max(0L, min(4L, hi - at));
    AdamwRow8 r;
    adamw_load_any(e.p, pb, at, count, vec, r.p);
    adamw_load_any(e.g, gb, at, count, vec, r.g);
    r.cm = *(const unsigned*)(o.m + at);               // the state buffers hold whole blocks
    r.cv = *(const unsigned*)(o.v + at);
    r.ms = o.ms[base >> 8];
    r.vs = o.vs[base >> 8];
    adamw_row8(r, count, (unsigned)at + key, a, s, keep);
    if (count > 0) {
      adamw_store_any(e.p, pb, at, count, vec, r.p);
      *(unsigned*)(o.m + at) = r.cm;                   // places past the tensor's end are zero and stay zero
      *(unsigned*)(o.v + at) = r.cv;
      if (a.zero_grad) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        adamw_store_any(e.g, gb, at, count, vec, zero);
      }
    }
    if (lane == 0) { o.ms[base >> 8] = r.ms; o.vs[base >> 8] = r.vs; }
  }
}

// step counter and bias corrections in device memory, for a launch sequence that is captured and replayed
__global__ void adamw_hyper_kernel(float* hyper, long long* step, double beta1, double beta2) {
  if (threadIdx.x == 0 && blockIdx.x == 0) {
    const long long t = *step + 1;
    *step = t;
    const double bc1 = 1.0 - pow(beta1, (double)t), bc2 = 1.0 - pow(beta2, (double)t);
    hyper[1] = (float)((double)hyper[0] / bc1);
    hyper[2] = (float)(1.0 / sqrt(bc2));
  }
}

// ---- global gradient norm: squares in fp64 (no overflow, no order that matters beyond 2^-53), fixed order.  One read of the gradients,
// which the step then finds in the last-level cache if they fit there (256 MB): 8 us more for a step over 12.1 M elements, of 70.
template <int WAVES> __device__ __forceinline__ double adamw_block_sum(double v) {
  __shared__ double red[WAVES];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v += red[w];
  return v;
}
constexpr int NORM_CHUNK = 4096, NORM_ROWS = NORM_CHUNK / ADAMW_ROW / ADAMW_WAVES;      // fewer partial sums to join
template <typename G> __device__ __forceinline__ double adamw_rows_norm(const AdamwEntry& e, long first, int rows) {
  const int row = threadIdx.x >> 6;
  const long i = first + (long)row * ADAMW_ROW + (threadIdx.x & 63) * 4;
  float g[NORM_ROWS][4];
#pragma unroll
  for (int k = 0; k < NORM_ROWS; ++k) {
    g[k][0] = g[k][1] = g[k][2] = g[k][3] = 0.f;
    if (row + k * ADAMW_WAVES < rows) adamw_load<G>(e.g, i + (long)k * ADAMW_WAVES * ADAMW_ROW, 4, true, g[k]);
  }
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < NORM_ROWS; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma((double)g[k][j], (double)g[k][j], sum);
  return sum;
}
__global__ __launch_bounds__(ADAMW_THREADS) void grad_norm_kernel(AdamwList list, double* partial) {
  const AdamwEntry e = list.e[adamw_find(list, blockIdx.x)];
  const bool gb = e.flags & ADAMW_G_BF16, vec = e.flags & ADAMW_VECTOR;
  const long lo = (long)(blockIdx.x - e.block0) * NORM_CHUNK, hi = min(e.n, lo + NORM_CHUNK);
  const int rows = vec ? (int)((hi - lo) / ADAMW_ROW) : 0;
  double sum = gb ? adamw_rows_norm<__bf16>(e, lo, rows) : adamw_rows_norm<float>(e, lo, rows);
  for (long i = lo + rows * ADAMW_ROW + threadIdx.x * 4; i < hi; i += ADAMW_THREADS * 4) {       // the rest, or an unaligned tensor
    float fg[4];
    adamw_load_any(e.g, gb, i, (int)min(4L, hi - i), vec, fg);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma((double)fg[j], (double)fg[j], sum);
  }
  sum = adamw_block_sum<ADAMW_WAVES>(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}
constexpr int ADAMW_JOIN = 1024;              // threads that add the partial sums, eight each at a time
__global__ __launch_bounds__(ADAMW_JOIN) void grad_norm_finalize_kernel(const double* partial, long count, float max_norm, float* out) {
  double sum = 0.0;
  for (long i = threadIdx.x; i < count; i += ADAMW_JOIN * 8) {
    double v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + k * ADAMW_JOIN < count ? partial[i + k * ADAMW_JOIN] : 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += v[k];
  }
  sum = adamw_block_sum<ADAMW_JOIN / 64>(sum);
  if (threadIdx.x == 0) {
    const double norm = sqrt(sum), coef = (double)max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = (float)(coef > 1.0 ? 1.0 : coef);         // NaN stays NaN, as the norm
  }
}

long adamw_blocks(long n, int chunk) { return (n + chunk - 1) / chunk; }

int adamw_check(const char* name, const dn_adamw_tensor* t, int count, bool state) {
  DN_CHECK_ARG(count >= 0 && (t || count == 0), "%s: null tensor list", name);
  for (int i = 0; i < count; ++i) {
    DN_CHECK_ARG(t[i].n >= 0 && t[i].n <= (1L << 34), "%s: tensor %d has %ld elements", name, i, t[i].n);
    if (t[i].n == 0) continue;
    DN_CHECK_ARG(t[i].grad && (t[i].param || !state), "%s: tensor %d: null pointer", name, i);
    DN_CHECK_ARG((t[i].param_dtype == DN_F32 || t[i].param_dtype == DN_BF16) && (t[i].grad_dtype == DN_F32 || t[i].grad_dtype == DN_BF16),
                 "%s: tensor %d: bad dtype", name, i);
    const uintptr_t pa = t[i].param_dtype == DN_BF16 ? 1 : 3, ga = t[i].grad_dtype == DN_BF16 ? 1 : 3;
    DN_CHECK_ARG(!((uintptr_t)t[i].grad & ga) && (!state || !((uintptr_t)t[i].param & pa)), "%s: tensor %d: misaligned pointer", name, i);
    DN_CHECK_ARG(!state || (t[i].state >= 0 && t[i].state % 256 == 0 && t[i].state / 256 < (1L << 32)),
                 "%s: tensor %d: state offset %ld is not a multiple of 256", name, i, t[i].state);
    DN_CHECK_ARG(!state || (t[i].number >= 0 && t[i].number < 1 << (32 - ADAMW_NUMBER)), "%s: tensor %d: number %d is not within 0 and 2^29 - 1",
                 name, i, t[i].number);
  }
  return DN_OK;
}

// The next launch's tensors from t[*first] on (empty ones are left out); returns its blocks, 0 when none is left
long adamw_fill(const dn_adamw_tensor* t, int count, int chunk, int* first, AdamwList* l) {
  long blocks = 0;
  l->count = 0;
  while (*first < count && l->count < ADAMW_MAX) {
    const dn_adamw_tensor& x = t[*first];
    const long more = adamw_blocks(x.n, chunk);
    if (blocks && blocks + more >= 1L << 24) break;            // a launch holds less than 2^32 threads
    if (x.n > 0) {
      AdamwEntry& e = l->e[l->count];
      e.p = x.param; e.g = x.grad; e.n = x.n; e.state = (unsigned)(x.state / 256); e.decay = x.weight_decay; e.block0 = (unsigned)blocks;
      const uintptr_t pa = x.param_dtype == DN_BF16 ? 7 : 15, ga = x.grad_dtype == DN_BF16 ? 7 : 15;
      e.flags = (x.param_dtype == DN_BF16 ? ADAMW_P_BF16 : 0) | (x.grad_dtype == DN_BF16 ? ADAMW_G_BF16 : 0) |
                (((uintptr_t)x.param & pa) || ((uintptr_t)x.grad & ga) ? 0 : ADAMW_VECTOR) | (unsigned)x.number << ADAMW_NUMBER;
      ++l->count;
      blocks += more;
    }
    ++*first;
  }
  return blocks;
}

// launch(list, blocks, blocks before) over all tensors, `chunk` elements a block
template <typename F> int adamw_each_launch(const dn_adamw_tensor* t, int count, int chunk, F launch) {
  AdamwList list;
  long before = 0;
  for (int first = 0; first < count;) {
    const long blocks = adamw_fill(t, count, chunk, &first, &list);
    if (!blocks) break;
    launch(list, (unsigned)blocks, before);
    DN_LAUNCH_CHECK();
    before += blocks;
  }
  return DN_OK;
}

int adamw_run(const dn_adamw_tensor* tensors, int count, void* exp_avg, void* exp_avg_sq, float* m_scale, float* v_scale,
              int state_bits, const AdamwArgs& a, hipStream_t st) {
  return adamw_each_launch(tensors, count, ADAMW_CHUNK, [&](const AdamwList& list, unsigned blocks, long) {
    if (state_bits == 8)
      hipLaunchKernelGGL(adamw8_kernel, dim3(blocks), dim3(ADAMW_THREADS), 0, st, list, (unsigned char*)exp_avg, (unsigned char*)exp_avg_sq,
                         m_scale, v_scale, a);
    else
      hipLaunchKernelGGL(adamw_kernel, dim3(blocks), dim3(ADAMW_THREADS), 0, st, list, (float*)exp_avg, (float*)exp_avg_sq, a);
  });
}

int adamw_args(const char* name, const dn_adamw_tensor* tensors, int count, const void* exp_avg, const void* exp_avg_sq,
               const float* m_scale, const float* v_scale, int state_bits, double beta1, double beta2, double eps, unsigned seed,
               const float* clip, int zero_grad, AdamwArgs* a) {
  const int rc = adamw_check(name, tensors, count, true);
  if (rc) return rc;
  DN_CHECK_ARG(state_bits == 32 || state_bits == 8, "%s: state_bits must be 32 or 8, got %d", name, state_bits);
  DN_CHECK_ARG(exp_avg && exp_avg_sq && !((uintptr_t)exp_avg & 15) && !((uintptr_t)exp_avg_sq & 15),
               "%s: moment buffers are null or not 16-byte aligned", name);
  DN_CHECK_ARG(state_bits == 32 || (m_scale && v_scale), "%s: 8-bit moments need their scales", name);
  DN_CHECK_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0, "%s: betas must be in [0, 1), eps must not be negative", name);
  *a = AdamwArgs{};
  a->beta1 = (float)beta1; a->beta2 = (float)beta2; a->omb1 = (float)(1.0 - beta1); a->omb2 = (float)(1.0 - beta2); a->eps = (float)eps;
  a->dbeta1 = beta1; a->dbeta2 = beta2; a->domb1 = 1.0 - beta1; a->domb2 = 1.0 - beta2;
  a->seed = seed; a->zero_grad = zero_grad; a->coef = clip;
  return DN_OK;
}

}  // namespace

extern "C" {

long dn_grad_norm_workspace_bytes(const dn_adamw_tensor* tensors, int count) {
  if (adamw_check("dn_grad_norm_workspace_bytes", tensors, count, false)) return -1;
  long blocks = 1;
  for (int i = 0; i < count; ++i) blocks += adamw_blocks(tensors[i].n, NORM_CHUNK);
  return blocks * (long)sizeof(double);
}

int dn_grad_norm(const dn_adamw_tensor* tensors, int count, float max_norm, float* out, void* workspace, long workspace_bytes, void* stream) {
  const long need = dn_grad_norm_workspace_bytes(tensors, count);
  if (need < 0) return DN_ERR_ARG;
  DN_CHECK_ARG(out && max_norm > 0.f, "dn_grad_norm: null output or max_norm not above zero");
  DN_CHECK_ARG(workspace && !((uintptr_t)workspace & 7) && workspace_bytes >= need,
               "dn_grad_norm: workspace of %ld bytes, %ld needed (8-byte aligned)", workspace_bytes, need);
  double* partial = (double*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  const int rc = adamw_each_launch(tensors, count, NORM_CHUNK, [&](const AdamwList& list, unsigned blocks, long before) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(ADAMW_THREADS), 0, st, list, partial + before);
  });
  if (rc) return rc;
  hipLaunchKernelGGL(grad_norm_finalize_kernel, dim3(1), dim3(ADAMW_JOIN), 0, st, partial, need / (long)sizeof(double) - 1, max_norm, out);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_adamw_step(const dn_adamw_tensor* tensors, int count, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                  float* exp_avg_sq_scale, int state_bits, double lr, double beta1, double beta2, double eps, long step, unsigned seed,
                  const float* clip, int zero_grad, void* stream) {
  AdamwArgs a;
  const int rc = adamw_args("dn_adamw_step", tensors, count, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, state_bits, beta1, beta2,
                            eps, seed, clip, zero_grad, &a);
  if (rc) return rc;
  DN_CHECK_ARG(step >= 1, "dn_adamw_step: step %ld is below 1", step);
  a.lr = (float)lr;
  a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
  a.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  a.step = (unsigned)step;
  return adamw_run(tensors, count, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, state_bits, a, (hipStream_t)stream);
}

int dn_adamw_step_graph(const dn_adamw_tensor* tensors, int count, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                        float* exp_avg_sq_scale, int state_bits, float* hyper, long long* step, double beta1, double beta2, double eps,
                        unsigned seed, const float* clip, int zero_grad, void* stream) {
  AdamwArgs a;
  const int rc = adamw_args("dn_adamw_step_graph", tensors, count, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, state_bits, beta1,
                            beta2, eps, seed, clip, zero_grad, &a);
  if (rc) return rc;
  DN_CHECK_ARG(hyper && step, "dn_adamw_step_graph: null hyper / step");
  a.hyper = hyper;
  a.step_dev = step;
  hipLaunchKernelGGL(adamw_hyper_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, hyper, step, beta1, beta2);
  DN_LAUNCH_CHECK();
  return adamw_run(tensors, count, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, state_bits, a,
                   (hipStream_t)stream);
}

}  // extern "C"
