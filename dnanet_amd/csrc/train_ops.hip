// Memory-bound stages of the training step on plane-record buffers (see common.h):
//   BatchNorm2d statistics / apply+ReLU / backward, MaxPool backward (+ skip-gradient add), 1x1 head
//   backward, ConvTranspose bias gradient, first-convolution weight gradient, Dice loss (+ binary
//   accuracy counts) forward/backward, fused Adam(+L2)+zero_grad.
// Every per-channel reduction is two-stage (per-block partials, then a finalize kernel that sums the
// partials in a fixed order in fp64), so results are bitwise reproducible run to run.
// Reference: unet_architecture.py:17,21 (BatchNorm2d, ReLU), :37 (MaxPool2d), :54-57 (ConvTranspose2d),
// :94-97 (head); loss.py:9-20 (DiceLoss); trainable_unet.py:155-157,343-344 (Adam, zero_grad),
// :295-303,411-415 (BinaryAccuracy).
#include <mutex>
#include "common.h"
#include "ops.h"


// ---- the one entry point that allocates nothing (dn_bn_train_forward_noalloc) -------------------------------------
// Its reduction partials live in this file-scope device array instead of a caller-provided workspace: callers under HIP
// graph capture, or harnesses that forbid hipMalloc, can run a train-mode BatchNorm without owning any scratch memory.
// Every GPU the library runs on holds its own copy (2.02 MiB) until the process ends.  In host code the array's NAME is
// only a stand-in: the per-device address comes from hipGetSymbolAddress, once per device, and only that pointer is
// ever handed to a kernel.
constexpr long DN_NOALLOC_SCRATCH_FLOATS = 512L * DN_NOALLOC_MAX_CHANNELS * 2 + 4096;    // = dn_partial_floats(512)
static __device__ __align__(256) float scratch[DN_NOALLOC_SCRATCH_FLOATS];

namespace {
constexpr int DN_MAX_DEVICES = 64;
std::mutex g_scratch_mutex;
float* g_scratch_ptr[DN_MAX_DEVICES] = {};

// device pointer of `scratch` on the CURRENT device (looked up on the first call on that device)
int noalloc_scratch(float** out) {
  int dev = -1;
  DN_CHECK_HIP(hipGetDevice(&dev));
  if (dev < 0 || dev >= DN_MAX_DEVICES) return dn_set_error(DN_ERR_ARG, "dn_bn_train_forward_noalloc: device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    DN_CHECK_HIP(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
    if (!p) return dn_set_error(DN_ERR_HIP, "dn_bn_train_forward_noalloc: hipGetSymbolAddress returned a null pointer");
    g_scratch_ptr[dev] = (float*)p;
  }
  *out = g_scratch_ptr[dev];
  return DN_OK;
}
}  // namespace

namespace {

constexpr int RED_THREADS = 256;      // 128 pixel lanes x 2 pieces
constexpr int RED_MAX_BLOCKS = 512;

__device__ __forceinline__ long rec_off(int planes_total, int plane, long n, long hw, long HW) {
  return ((n * planes_total + plane) * HW + hw) * 32;
}

// Sum KV x PN per-thread accumulators over the 128 pixel lanes of the block, write partial[blk][c][kv].
template <int KV, int PN>
__device__ __forceinline__ void block_reduce_store(float (&acc)[KV][PN], float* partial, int cpad, int plane, int epr) {
  __shared__ float red[8 * KV * PN];
  // reduce within a wave first over lanes with the same piece parity (xor 2,4,..,32)
#pragma unroll
  for (int kv = 0; kv < KV; ++kv)
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      float v = acc[kv][j];
#pragma unroll
      for (int m = 2; m < 64; m <<= 1) v += __shfl_xor(v, m);
      acc[kv][j] = v;
    }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane < 2) {
#pragma unroll
    for (int kv = 0; kv < KV; ++kv)
#pragma unroll
      for (int j = 0; j < PN; ++j) red[((wave * 2 + lane) * KV + kv) * PN + j] = acc[kv][j];
  }
  __syncthreads();
  const int nout = 2 * KV * PN;   // piece x kv x j
  if ((int)threadIdx.x < nout) {
    const int pc = threadIdx.x / (KV * PN), rem = threadIdx.x % (KV * PN);
    const int kv = rem / PN, j = rem % PN;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < RED_THREADS / 64; ++w) s += red[((w * 2 + pc) * KV + kv) * PN + j];
    const int c = plane * epr + pc * PN + j;
    partial[((long)blockIdx.x * cpad + c) * KV + kv] = s;
  }
}

// One 64-lane wave per channel sums `nblk` partials in fp64 in a fixed order (lane-strided, then a shuffle tree).
__device__ __forceinline__ double wave_sum_partials(const float* partial, int nblk, long stride, long offset) {
  double s = 0;
  for (int b = threadIdx.x; b < nblk; b += 64) s += (double)partial[(long)b * stride + offset];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m);
  return s;
}

// ---- BatchNorm statistics: sum(y), sum(y^2) --------------------------------------------------
// Reduction work split: a plane of one image is a contiguous run of 2*H*W 16-byte pieces; it is cut into segments of
// RED_SEG pieces and the (image, segment) units are dealt round-robin to the blocks of a plane.  A thread reads four
// pieces 256 apart per step (independent loads in flight: a single dependent load per thread left HBM at ~4 TB/s);
// its piece parity, hence its channels, is fixed (threadIdx.x & 1).
#ifndef DN_BWD_ILP
#define DN_BWD_ILP 4
#endif
constexpr int BWD_ILP = DN_BWD_ILP;         // bn_bwd_reduce_kernel: loads of g and of y in flight per thread (2 left HBM at 4.9 TB/s)
constexpr int RED_SEG = 4096;      // pieces per unit at large batch; red_seg() shrinks it when there are few images

template <typename T>
__global__ __launch_bounds__(RED_THREADS) void bn_stats_kernel(const unsigned char* y, int planes_total, int plane0, int N,
                                                                int npieces, int seg_len, float* partial, int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int plane = blockIdx.y;
  float acc[2][PN] = {};
  const int nseg = (npieces + seg_len - 1) / seg_len;
  for (int u = blockIdx.x; u < N * nseg; u += gridDim.x) {
    const int n = u / nseg, seg = u - n * nseg;
    const unsigned char* base = y + ((long)n * planes_total + plane0 + plane) * npieces * 16;
    const int iend = min(npieces, (seg + 1) * seg_len);
    for (int i = seg * seg_len + threadIdx.x; i < iend; i += 4 * RED_THREADS) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int ii = i + k * RED_THREADS;
        v[k] = ii < iend ? *(const uint4*)(base + (long)ii * 16) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[PN];
        Piece<T>::unpack(v[k], f);
#pragma unroll
        for (int j = 0; j < PN; ++j) { acc[0][j] += f[j]; acc[1][j] = fmaf(f[j], f[j], acc[1][j]); }
      }
    }
  }
  block_reduce_store<2, PN>(acc, partial, cpad, plane, EPR);
}

// Sum of the [nblk][cpad] (sum, sum of squares) partial pairs of channel c over a 256-thread block, fixed order, fp64.
// With the statistics fused into the convolution there is one partial per conv tile (thousands): every thread keeps four
// pairs in flight.  The result is valid in thread 0.
constexpr int SUM_THREADS = 1024;   // threads of the kernels that add up per-tile partials: one block per channel
__device__ __forceinline__ void block_sum_pairs(const float* partial, int nblk, int cpad, int c, double& s_out, double& ss_out) {
  const float2* p = (const float2*)partial + c;
  double s = 0.0, ss = 0.0;
  int i = threadIdx.x;
  for (; i + 3 * SUM_THREADS < nblk; i += 4 * SUM_THREADS) {
    const float2 a = p[(long)i * cpad], b = p[(long)(i + SUM_THREADS) * cpad], d = p[(long)(i + 2 * SUM_THREADS) * cpad],
                 e = p[(long)(i + 3 * SUM_THREADS) * cpad];
    s += ((double)a.x + (double)b.x) + ((double)d.x + (double)e.x);
    ss += ((double)a.y + (double)b.y) + ((double)d.y + (double)e.y);
  }
  for (; i < nblk; i += SUM_THREADS) { const float2 a = p[(long)i * cpad]; s += a.x; ss += a.y; }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) { s += __shfl_xor(s, m); ss += __shfl_xor(ss, m); }
  __shared__ double red[SUM_THREADS / 64][2];
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = s; red[threadIdx.x >> 6][1] = ss; }
  __syncthreads();
  s = 0.0; ss = 0.0;
#pragma unroll
  for (int w = 0; w < SUM_THREADS / 64; ++w) { s += red[w][0]; ss += red[w][1]; }   // fixed order
  s_out = s; ss_out = ss;
}

// mean, invstd, running statistics, fused scale / shift of one channel from its totals over `count` values
__device__ __forceinline__ void bn_finalize_channel(int c, double s, double ss, double count, const float* gamma, const float* beta,
                                                    float* running_mean, float* running_var, float momentum, float eps,
                                                    float* mean_out, float* invstd_out, float* scale, float* shift) {
  const double mean = s / count;
  double var = ss / count - mean * mean;
  if (var < 0) var = 0;
  const float invstd = (float)(1.0 / sqrt(var + (double)eps));
  mean_out[c] = (float)mean;
  invstd_out[c] = invstd;
  const float sc = gamma[c] * invstd;
  scale[c] = sc;
  shift[c] = beta[c] - (float)mean * sc;
  if (running_mean) {
    const double unbiased = count > 1 ? var * count / (count - 1) : var;
    {
#pragma clang fp contract(off)      // products and sum rounded separately, whatever instructions the build may use
      const float keep = (1.f - momentum) * running_mean[c];
      const float take = momentum * (float)mean;
      running_mean[c] = keep + take;
    }
    running_var[c] = (1.f - momentum) * running_var[c] + momentum * (float)unbiased;
  }
}

// finalize: mean, invstd, running stats, scale/shift for the apply pass
__global__ void bn_finalize_kernel(const float* partial, int nblk, int cpad, int C, double count, const float* gamma,
                                   const float* beta, float* running_mean, float* running_var, float momentum, float eps,
                                   float* mean_out, float* invstd_out, float* scale, float* shift) {
  const int c = blockIdx.x;       // one SUM_THREADS block per channel
  if (c >= C) { if (threadIdx.x == 0) { scale[c] = 0.f; shift[c] = 0.f; mean_out[c] = 0.f; invstd_out[c] = 0.f; } return; }
  double s, ss;
  block_sum_pairs(partial, nblk, cpad, c, s, ss);
  if (threadIdx.x != 0) return;
  bn_finalize_channel(c, s, ss, count, gamma, beta, running_mean, running_var, momentum, eps, mean_out, invstd_out, scale, shift);
}

// ---- synchronised BatchNorm (data parallel, optional): the same two steps with an all-reduce in between ---------------
// totals[c][2] (fp64) = this rank's sums; the caller sums them over the ranks; the finalize kernels take the global totals
// and the global count.  One rank: bitwise the same as the kernels above (same summation order, same fp64 arithmetic).
__global__ void bn_pair_totals_kernel(const float* partial, int nblk, int cpad, int C, double* totals) {
  const int c = blockIdx.x;
  double s = 0.0, ss = 0.0;
  if (c < C) block_sum_pairs(partial, nblk, cpad, c, s, ss);
  if (threadIdx.x == 0) { totals[2 * c] = s; totals[2 * c + 1] = ss; }
}

__global__ void bn_finalize_totals_kernel(const double* totals, int cpad, int C, double count, const float* gamma, const float* beta,
                                          float* running_mean, float* running_var, float momentum, float eps, float* mean_out,
                                          float* invstd_out, float* scale, float* shift) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cpad) return;
  if (c >= C) { scale[c] = 0.f; shift[c] = 0.f; mean_out[c] = 0.f; invstd_out[c] = 0.f; return; }
  bn_finalize_channel(c, totals[2 * c], totals[2 * c + 1], count, gamma, beta, running_mean, running_var, momentum, eps, mean_out,
                      invstd_out, scale, shift);
}

// a = relu(y * scale + shift).  Grid (x, plane, image): a plane of one image is a contiguous run of 16-byte pieces, so the
// index is 32-bit and there is no division in the loop.
template <typename T>
__global__ __launch_bounds__(256) void bn_apply_relu_kernel(const unsigned char* y, int y_pt, int y_p0, unsigned char* a,
                                                            int a_pt, int a_p0, int npieces,
                                                            const float* __restrict__ scale, const float* __restrict__ shift) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int pl = blockIdx.y, n = blockIdx.z;
  const unsigned char* yp = y + ((long)n * y_pt + y_p0 + pl) * npieces * 16;
  unsigned char* ap = a + ((long)n * a_pt + a_p0 + pl) * npieces * 16;
  // the stride is even, so a thread keeps its piece parity = its channels: coefficients live in registers
  const int c0 = pl * EPR + (threadIdx.x & 1) * PN;
  float sc[PN], sh[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; }
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < npieces; i += gridDim.x * blockDim.x) {
    float f[PN];
    Piece<T>::unpack(*(const uint4*)(yp + (long)i * 16), f);
#pragma unroll
    for (int j = 0; j < PN; ++j) f[j] = fmaxf(fmaf(f[j], sc[j], sh[j]), 0.f);
    *(uint4*)(ap + (long)i * 16) = Piece<T>::pack(f);
  }
}

// The same pass for an encoder block's second unit, with MaxPool2d((1,2)) of the activation written alongside
// (unet_architecture.py:37): a thread handles the same channel piece of the two pixels of a pooling pair.
template <typename T>
__global__ __launch_bounds__(256) void bn_apply_relu_pool_kernel(const unsigned char* y, int y_pt, int y_p0, unsigned char* a,
                                                                 int a_pt, int a_p0, unsigned char* pooled, int p_pt, int p_p0,
                                                                 int npieces, const float* __restrict__ scale,
                                                                 const float* __restrict__ shift) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int pl = blockIdx.y, n = blockIdx.z;
  const unsigned char* yp = y + ((long)n * y_pt + y_p0 + pl) * npieces * 16;
  unsigned char* ap = a + ((long)n * a_pt + a_p0 + pl) * npieces * 16;
  unsigned char* pp = pooled + ((long)n * p_pt + p_p0 + pl) * (npieces / 2) * 16;
  const int c0 = pl * EPR + (threadIdx.x & 1) * PN;       // even stride: the piece parity = the channels stay with the thread
  float sc[PN], sh[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; }
  for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < npieces / 2; k += gridDim.x * blockDim.x) {
    const long i0 = (long)(k >> 1) * 4 + (k & 1);         // pieces of pixel 2j and (i0 + 2) of pixel 2j + 1
    float f0[PN], f1[PN], m[PN];
    Piece<T>::unpack(*(const uint4*)(yp + i0 * 16), f0);
    Piece<T>::unpack(*(const uint4*)(yp + (i0 + 2) * 16), f1);
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      f0[j] = fmaxf(fmaf(f0[j], sc[j], sh[j]), 0.f);
      f1[j] = fmaxf(fmaf(f1[j], sc[j], sh[j]), 0.f);
      m[j] = fmaxf(f0[j], f1[j]);                         // rounding is monotonic: max of the stored values
    }
    *(uint4*)(ap + i0 * 16) = Piece<T>::pack(f0);
    *(uint4*)(ap + (i0 + 2) * 16) = Piece<T>::pack(f1);
    *(uint4*)(pp + (long)k * 16) = Piece<T>::pack(m);
  }
}

// ---- BatchNorm backward ------------------------------------------------------------------------
// reduce: S1 = sum(dz), S2 = sum(dz * xhat), dz = g * (y*scale + shift > 0), xhat = (y - mean) * invstd.
// The ReLU mask is recomputed from y with the forward's fused scale / shift (the same fmaf the apply pass rounded to get
// a), so the activation tensor is not read again: 2 reads here and 2 reads + 1 write in the apply pass.
template <typename T>
__global__ __launch_bounds__(RED_THREADS) void bn_bwd_reduce_kernel(const unsigned char* g, int g_pt, int g_p0,
                                                                     const unsigned char* y, int y_pt, int y_p0,
                                                                     const float* __restrict__ scale,
                                                                     const float* __restrict__ shift, int N, int npieces, int seg_len,
                                                                     const float* __restrict__ mean,
                                                                     const float* __restrict__ invstd, float* partial, int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int plane = blockIdx.y, pc = threadIdx.x & 1;
  const int c0 = plane * EPR + pc * PN;
  float mu[PN], is[PN], sc[PN], sh[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { mu[j] = mean[c0 + j]; is[j] = invstd[c0 + j]; sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; }
  float acc[2][PN] = {};
  const int nseg = (npieces + seg_len - 1) / seg_len;
  for (int u = blockIdx.x; u < N * nseg; u += gridDim.x) {
    const int n = u / nseg, seg = u - n * nseg;
    const unsigned char* gbase = g + ((long)n * g_pt + g_p0 + plane) * npieces * 16;
    const unsigned char* ybase = y + ((long)n * y_pt + y_p0 + plane) * npieces * 16;
    const int iend = min(npieces, (seg + 1) * seg_len);
    for (int i = seg * seg_len + threadIdx.x; i < iend; i += BWD_ILP * RED_THREADS) {
      uint4 vg[BWD_ILP], vy[BWD_ILP];             // BWD_ILP pieces of g and of y in flight per thread
#pragma unroll
      for (int k = 0; k < BWD_ILP; ++k) {
        const int ii = i + k * RED_THREADS;
        const bool in = ii < iend;
        vg[k] = in ? *(const uint4*)(gbase + (long)ii * 16) : make_uint4(0, 0, 0, 0);   // g = 0 adds nothing
        vy[k] = in ? *(const uint4*)(ybase + (long)ii * 16) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < BWD_ILP; ++k) {
        float fg[PN], fy[PN];
        Piece<T>::unpack(vg[k], fg);
        Piece<T>::unpack(vy[k], fy);
#pragma unroll
        for (int j = 0; j < PN; ++j) {
          const float dz = fmaf(fy[j], sc[j], sh[j]) > 0.f ? fg[j] : 0.f;   // the forward's own pre-ReLU value
          acc[0][j] += dz;
          acc[1][j] = fmaf(dz, (fy[j] - mu[j]) * is[j], acc[1][j]);
        }
      }
    }
  }
  block_reduce_store<2, PN>(acc, partial, cpad, plane, EPR);
}

__global__ __launch_bounds__(SUM_THREADS) void bn_bwd_finalize_kernel(const float* partial, int nblk, int cpad, int C, double count,
                                                                      const float* gamma, const float* invstd, float* dgamma,
                                                                      float* dbeta, float* coef /*[3][cpad]*/) {
  const int c = blockIdx.x;       // one block per channel: the partials are per reduction block, or per convolution tile
  if (c >= C) { if (threadIdx.x == 0) { coef[c] = 0.f; coef[cpad + c] = 0.f; coef[2 * cpad + c] = 0.f; } return; }
  double s1, s2;
  block_sum_pairs(partial, nblk, cpad, c, s1, s2);
  if (threadIdx.x != 0) return;
  dbeta[c] = (float)s1;
  dgamma[c] = (float)s2;
  coef[c] = gamma[c] * invstd[c];            // s
  coef[cpad + c] = (float)(s1 / count);      // mean(dz)
  coef[2 * cpad + c] = (float)(s2 / count);  // mean(dz * xhat)
}

// synchronised form: local totals -> (all-reduce by the caller) -> coefficients from the global totals.  dgamma / dbeta stay
// LOCAL sums: the data-parallel gradient all-reduce adds them up like every other parameter gradient.
__global__ __launch_bounds__(SUM_THREADS) void bn_bwd_pair_totals_kernel(const float* partial, int nblk, int cpad, int C, double* totals) {
  const int c = blockIdx.x;
  double s1 = 0.0, s2 = 0.0;
  if (c < C) block_sum_pairs(partial, nblk, cpad, c, s1, s2);
  if (threadIdx.x == 0) { totals[2 * c] = s1; totals[2 * c + 1] = s2; }
}

__global__ void bn_bwd_finalize_totals_kernel(const double* local, const double* global, int cpad, int C, double count,
                                              const float* gamma, const float* invstd, float* dgamma, float* dbeta, float* coef) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cpad) return;
  if (c >= C) { coef[c] = 0.f; coef[cpad + c] = 0.f; coef[2 * cpad + c] = 0.f; return; }
  dbeta[c] = (float)local[2 * c];
  dgamma[c] = (float)local[2 * c + 1];
  coef[c] = gamma[c] * invstd[c];
  coef[cpad + c] = (float)(global[2 * c] / count);
  coef[2 * cpad + c] = (float)(global[2 * c + 1] / count);
}

// apply (in place on g): dy = s * (dz - c1 - xhat * c2).  Grid (x, plane, image) as bn_apply_relu_kernel.
template <typename T>
__global__ __launch_bounds__(256) void bn_bwd_apply_kernel(unsigned char* g, int g_pt, int g_p0, const unsigned char* y, int y_pt,
                                                           int y_p0, const float* __restrict__ scale,
                                                           const float* __restrict__ shift, int npieces,
                                                           const float* __restrict__ mean,
                                                           const float* __restrict__ invstd, const float* __restrict__ coef,
                                                           int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int pl = blockIdx.y, n = blockIdx.z;
  unsigned char* gbase = g + ((long)n * g_pt + g_p0 + pl) * npieces * 16;
  const unsigned char* ybase = y + ((long)n * y_pt + y_p0 + pl) * npieces * 16;
  const int c0 = pl * EPR + (threadIdx.x & 1) * PN;   // fixed per thread (even stride): coefficients in registers
  float sc[PN], sh[PN], mu[PN], is[PN], k0[PN], k1[PN], k2[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) {
    const int c = c0 + j;
    sc[j] = scale[c]; sh[j] = shift[c]; mu[j] = mean[c]; is[j] = invstd[c];
    k0[j] = coef[c]; k1[j] = coef[cpad + c]; k2[j] = coef[2 * cpad + c];
  }
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < npieces; i += gridDim.x * blockDim.x) {
    unsigned char* gp = gbase + (long)i * 16;
    float fg[PN], fy[PN];
    Piece<T>::unpack(*(const uint4*)gp, fg);
    Piece<T>::unpack(*(const uint4*)(ybase + (long)i * 16), fy);
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      const float dz = fmaf(fy[j], sc[j], sh[j]) > 0.f ? fg[j] : 0.f;
      const float xhat = (fy[j] - mu[j]) * is[j];
      fg[j] = k0[j] * (dz - k1[j] - xhat * k2[j]);
    }
    *(uint4*)gp = Piece<T>::pack(fg);
  }
}

// ---- MaxPool backward + skip gradient -----------------------------------------------------------
// g[n,c,h,w] = (dskip ? dskip[n,c,h,w] : 0) + (x[w] is the (first) max of its pair ? dpool[n,c,h,w/2] : 0)
template <typename T>
__global__ __launch_bounds__(256) void pool_bwd_add_kernel(const unsigned char* x, int x_pt, int x_p0, const unsigned char* dpool,
                                                           int dp_pt, int dp_p0, const unsigned char* dskip, int ds_pt, int ds_p0,
                                                           unsigned char* g, int g_pt, int g_p0, int nplanes, long N, int H,
                                                           int Wout) {
  constexpr int PN = Piece<T>::N;
  const long total = N * nplanes * H * Wout * 2;
  const long HW = (long)H * 2 * Wout, HWo = (long)H * Wout;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long)gridDim.x * blockDim.x) {
    const int pc = (int)(i & 1);
    long r = i >> 1;
    const int w = (int)(r % Wout); r /= Wout;
    const int h = (int)(r % H); r /= H;
    const int pl = (int)(r % nplanes);
    const long n = r / nplanes;
    const long hw = (long)h * 2 * Wout + 2 * w;
    const unsigned char* xp = x + rec_off(x_pt, x_p0 + pl, n, hw, HW) + 16 * pc;
    float x0[PN], x1[PN], dp[PN], s0[PN] = {}, s1[PN] = {};
    Piece<T>::unpack(*(const uint4*)xp, x0);
    Piece<T>::unpack(*(const uint4*)(xp + 32), x1);
    Piece<T>::unpack(*(const uint4*)(dpool + rec_off(dp_pt, dp_p0 + pl, n, (long)h * Wout + w, HWo) + 16 * pc), dp);
    if (dskip) {
      const unsigned char* sp = dskip + rec_off(ds_pt, ds_p0 + pl, n, hw, HW) + 16 * pc;
      Piece<T>::unpack(*(const uint4*)sp, s0);
      Piece<T>::unpack(*(const uint4*)(sp + 32), s1);
    }
#pragma unroll
    for (int j = 0; j < PN; ++j) {
      const bool first = x0[j] >= x1[j];       // ties go to the first element (ATen max_pool2d backward)
      s0[j] += first ? dp[j] : 0.f;
      s1[j] += first ? 0.f : dp[j];
    }
    unsigned char* gp = g + rec_off(g_pt, g_p0 + pl, n, hw, HW) + 16 * pc;
    *(uint4*)gp = Piece<T>::pack(s0);
    *(uint4*)(gp + 32) = Piece<T>::pack(s1);
  }
}

// The same with BatchNorm backward's two sums for the unit whose activation x is (the second unit of an encoder block):
// g is that unit's activation gradient, so sum dz and sum dz * xhat are formed here, on the values of g as stored, and
// the unit's reduction pass over g and y is not needed (bn_bwd_reduce_kernel's arithmetic and partial layout; work split
// as there: (image, segment) units of a plane dealt round-robin to the blocks, a thread's piece parity fixed).
// An item = one pooled pixel x one 16-byte piece: two neighbouring full-resolution records.
constexpr int POOL_ILP = 2;          // items in flight per thread of pool_bwd_add_sums_kernel / head_bwd_data_sums_kernel
template <typename T>
__global__ __launch_bounds__(RED_THREADS) void pool_bwd_add_sums_kernel(
    const unsigned char* x, int x_pt, int x_p0, const unsigned char* dpool, int dp_pt, int dp_p0, const unsigned char* dskip,
    int ds_pt, int ds_p0, unsigned char* g, int g_pt, int g_p0, const unsigned char* y, int y_pt, int y_p0,
    const float* __restrict__ scale, const float* __restrict__ shift, const float* __restrict__ mean,
    const float* __restrict__ invstd, int N, int nitems /* 2 * H * Wout */, int seg_len, float* partial, int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int plane = blockIdx.y, pc = threadIdx.x & 1;
  const int c0 = plane * EPR + pc * PN;
  float mu[PN], is[PN], sc[PN], sh[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { mu[j] = mean[c0 + j]; is[j] = invstd[c0 + j]; sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; }
  float acc[2][PN] = {};
  const int nseg = (nitems + seg_len - 1) / seg_len;
  for (int u = blockIdx.x; u < N * nseg; u += gridDim.x) {
    const int n = u / nseg, seg = u - n * nseg;
    // 16-byte pieces of this image's plane: full resolution 2 * nitems of them, pooled nitems
    const unsigned char* xb = x + ((long)n * x_pt + x_p0 + plane) * nitems * 32;
    const unsigned char* yb = y + ((long)n * y_pt + y_p0 + plane) * nitems * 32;
    const unsigned char* sb = dskip ? dskip + ((long)n * ds_pt + ds_p0 + plane) * nitems * 32 : nullptr;
    unsigned char* gb = g + ((long)n * g_pt + g_p0 + plane) * nitems * 32;
    const unsigned char* pb = dpool + ((long)n * dp_pt + dp_p0 + plane) * nitems * 16;
    const int iend = min(nitems, (seg + 1) * seg_len);
    for (int i = seg * seg_len + threadIdx.x; i < iend; i += POOL_ILP * RED_THREADS) {
      // POOL_ILP items' loads (7 pieces each) are issued before the first is used
      uint4 vx0[POOL_ILP], vx1[POOL_ILP], vdp[POOL_ILP], vy0[POOL_ILP], vy1[POOL_ILP], vs0[POOL_ILP], vs1[POOL_ILP];
#pragma unroll
      for (int k = 0; k < POOL_ILP; ++k) {
        const int ii = i + k * RED_THREADS < iend ? i + k * RED_THREADS : i;   // past the end: item i again (loaded, not used)
        const long full = (long)(ii >> 1) * 64 + 16 * pc;      // byte offset of the even column's piece; the odd one is 32 further
        vx0[k] = *(const uint4*)(xb + full); vx1[k] = *(const uint4*)(xb + full + 32);
        vdp[k] = *(const uint4*)(pb + (long)ii * 16);
        vy0[k] = *(const uint4*)(yb + full); vy1[k] = *(const uint4*)(yb + full + 32);
        vs0[k] = sb ? *(const uint4*)(sb + full) : make_uint4(0, 0, 0, 0);
        vs1[k] = sb ? *(const uint4*)(sb + full + 32) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < POOL_ILP; ++k) {
        const int ii = i + k * RED_THREADS;
        if (ii < iend) {
          const long full = (long)(ii >> 1) * 64 + 16 * pc;
          float x0[PN], x1[PN], dp[PN], s0[PN], s1[PN], y0[PN], y1[PN];
          Piece<T>::unpack(vs0[k], s0); Piece<T>::unpack(vs1[k], s1);       // (all-zero bits are 0.0 in both storage types)
          Piece<T>::unpack(vx0[k], x0); Piece<T>::unpack(vx1[k], x1); Piece<T>::unpack(vdp[k], dp);
          Piece<T>::unpack(vy0[k], y0); Piece<T>::unpack(vy1[k], y1);
#pragma unroll
          for (int j = 0; j < PN; ++j) {
            const bool first = x0[j] >= x1[j];       // ties go to the first element (ATen max_pool2d backward)
            s0[j] += first ? dp[j] : 0.f;
            s1[j] += first ? 0.f : dp[j];
          }
          const uint4 g0 = Piece<T>::pack(s0), g1 = Piece<T>::pack(s1);
          *(uint4*)(gb + full) = g0;
          *(uint4*)(gb + full + 32) = g1;
          Piece<T>::unpack(g0, s0); Piece<T>::unpack(g1, s1);          // the gradient as stored
#pragma unroll
          for (int j = 0; j < PN; ++j) {
            const float dz0 = fmaf(y0[j], sc[j], sh[j]) > 0.f ? s0[j] : 0.f;
            const float dz1 = fmaf(y1[j], sc[j], sh[j]) > 0.f ? s1[j] : 0.f;
            acc[0][j] += dz0 + dz1;
            acc[1][j] = fmaf(dz1, (y1[j] - mu[j]) * is[j], fmaf(dz0, (y0[j] - mu[j]) * is[j], acc[1][j]));
          }
        }
      }
    }
  }
  block_reduce_store<2, PN>(acc, partial, cpad, plane, EPR);
}

// ---- head backward ---------------------------------------------------------------------------------
// g[n,c,h,w] = dlogit[n,h,w] * w[c]
template <typename T>
__global__ __launch_bounds__(256) void head_bwd_data_kernel(const float* __restrict__ dlogit, const float* __restrict__ w,
                                                            unsigned char* g, int g_pt, int g_p0, int nplanes, long N, long HW) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const long total = N * nplanes * HW * 2;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long)gridDim.x * blockDim.x) {
    const int pc = (int)(i & 1);
    long r = i >> 1;
    const long hw = r % HW; r /= HW;
    const int pl = (int)(r % nplanes);
    const long n = r / nplanes;
    const float d = dlogit[n * HW + hw];
    float f[PN];
#pragma unroll
    for (int j = 0; j < PN; ++j) f[j] = d * w[pl * EPR + pc * PN + j];
    *(uint4*)(g + rec_off(g_pt, g_p0 + pl, n, hw, HW) + 16 * pc) = Piece<T>::pack(f);
  }
}

// The same with BatchNorm backward's two sums of the unit whose activation the head reads (the last DoubleConv's second
// unit): g is its activation gradient.  Work split and partial layout as bn_bwd_reduce_kernel.
template <typename T>
__global__ __launch_bounds__(RED_THREADS) void head_bwd_data_sums_kernel(
    const float* __restrict__ dlogit, const float* __restrict__ w, unsigned char* g, int g_pt, int g_p0, const unsigned char* y,
    int y_pt, int y_p0, const float* __restrict__ scale, const float* __restrict__ shift, const float* __restrict__ mean,
    const float* __restrict__ invstd, int N, int npieces /* 2 * H * W */, int seg_len, float* partial, int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int plane = blockIdx.y, pc = threadIdx.x & 1;
  const int c0 = plane * EPR + pc * PN;
  float mu[PN], is[PN], sc[PN], sh[PN], wv[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) { mu[j] = mean[c0 + j]; is[j] = invstd[c0 + j]; sc[j] = scale[c0 + j]; sh[j] = shift[c0 + j]; wv[j] = w[c0 + j]; }
  float acc[2][PN] = {};
  const int nseg = (npieces + seg_len - 1) / seg_len;
  for (int u = blockIdx.x; u < N * nseg; u += gridDim.x) {
    const int n = u / nseg, seg = u - n * nseg;
    unsigned char* gb = g + ((long)n * g_pt + g_p0 + plane) * npieces * 16;
    const unsigned char* yb = y + ((long)n * y_pt + y_p0 + plane) * npieces * 16;
    const float* dl = dlogit + (long)n * (npieces >> 1);
    const int iend = min(npieces, (seg + 1) * seg_len);
    for (int i = seg * seg_len + threadIdx.x; i < iend; i += POOL_ILP * RED_THREADS) {
      uint4 vy[POOL_ILP]; float d[POOL_ILP];
#pragma unroll
      for (int k = 0; k < POOL_ILP; ++k) {
        const int ii = i + k * RED_THREADS;
        const bool in = ii < iend;
        vy[k] = in ? *(const uint4*)(yb + (long)ii * 16) : make_uint4(0, 0, 0, 0);
        d[k] = in ? dl[ii >> 1] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < POOL_ILP; ++k) {
        const int ii = i + k * RED_THREADS;
        if (ii < iend) {
          float f[PN], fy[PN];
          Piece<T>::unpack(vy[k], fy);
#pragma unroll
          for (int j = 0; j < PN; ++j) f[j] = d[k] * wv[j];
          const uint4 gv = Piece<T>::pack(f);
          *(uint4*)(gb + (long)ii * 16) = gv;
          Piece<T>::unpack(gv, f);                                       // the gradient as stored
#pragma unroll
          for (int j = 0; j < PN; ++j) {
            const float dz = fmaf(fy[j], sc[j], sh[j]) > 0.f ? f[j] : 0.f;
            acc[0][j] += dz;
            acc[1][j] = fmaf(dz, (fy[j] - mu[j]) * is[j], acc[1][j]);
          }
        }
      }
    }
  }
  block_reduce_store<2, PN>(acc, partial, cpad, plane, EPR);
}

// per-channel sum over pixels of x * (scale ? scale[pixel] : 1):  head weight gradient (scale = dlogit),
// ConvTranspose bias gradient (scale = null).  Work split as bn_stats_kernel: (image, segment) units of a plane's contiguous
// 16-byte pieces dealt round-robin to the blocks, four pieces in flight per thread, no division in the loop (the first
// version walked pixels with a wrap-around loop that spun 40 times per step on the 256-column planes: 2.6 TB/s).
template <typename T>
__global__ __launch_bounds__(RED_THREADS) void channel_sum_kernel(const unsigned char* x, int x_pt, int x_p0, int N, int npieces,
                                                                   int seg_len, const float* __restrict__ pixscale, float* partial,
                                                                   int cpad) {
  constexpr int PN = Piece<T>::N, EPR = RecTraits<T>::EPR;
  const int plane = blockIdx.y;
  float acc[1][PN] = {};
  const int nseg = (npieces + seg_len - 1) / seg_len;
  for (int u = blockIdx.x; u < N * nseg; u += gridDim.x) {
    const int n = u / nseg, seg = u - n * nseg;
    const unsigned char* base = x + ((long)n * x_pt + x_p0 + plane) * npieces * 16;
    const float* ps = pixscale ? pixscale + (long)n * (npieces >> 1) : nullptr;
    const int iend = min(npieces, (seg + 1) * seg_len);
    for (int i = seg * seg_len + threadIdx.x; i < iend; i += 4 * RED_THREADS) {
      uint4 v[4];
      float sc[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int ii = i + k * RED_THREADS;
        v[k] = ii < iend ? *(const uint4*)(base + (long)ii * 16) : make_uint4(0, 0, 0, 0);
        sc[k] = (ps && ii < iend) ? ps[ii >> 1] : 1.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[PN];
        Piece<T>::unpack(v[k], f);
#pragma unroll
        for (int j = 0; j < PN; ++j) acc[0][j] = fmaf(f[j], sc[k], acc[0][j]);
      }
    }
  }
  block_reduce_store<1, PN>(acc, partial, cpad, plane, EPR);
}

__global__ void channel_sum_finalize_kernel(const float* partial, int nblk, int cpad, int C, float* out) {
  const int c = blockIdx.x;       // one wave per channel
  if (c >= C) return;
  const double s = wave_sum_partials(partial, nblk, cpad, c);
  if (threadIdx.x == 0) out[c] = (float)s;
}

// ---- first-convolution weight gradient: dW[co][tap] = sum_pix dy[pix][co] * x[pix + tap] ------------
// A thread owns one 16-byte piece (8 bf16 / 4 fp32 channels) of one pixel per step and all TAPS accumulators for it:
// dy is read exactly once (16 B per lane, coalesced), the KH*KW neighbours of x come from L1 (fp32: raw RFU does not
// fit bf16), 8*TAPS FMAs per load.  Per-block partial[blk][c][tap] via the common wave/LDS reduction.
template <typename T, int KH, int KW>
__global__ __launch_bounds__(RED_THREADS) void conv_first_wgrad_kernel(const float* __restrict__ x, const unsigned char* dy,
                                                                        int dy_pt, int dy_p0, int N, int H, int W,
                                                                        float* partial, int cpad) {
  constexpr int EPR = RecTraits<T>::EPR, PN = Piece<T>::N, TAPS = KH * KW, PH = KH / 2, PW = KW / 2;
  const int plane = blockIdx.y, pc = threadIdx.x & 1;
  float acc[TAPS][PN] = {};
  const unsigned HW = (unsigned)H * W, total = (unsigned)N * HW;
  for (unsigned i = blockIdx.x * 128u + (threadIdx.x >> 1); i < total; i += gridDim.x * 128u) {
    const unsigned n = i / HW, hw = i - n * HW;
    const int h = (int)(hw / (unsigned)W), w = (int)(hw - (unsigned)h * W);
    float f[PN];
    Piece<T>::unpack(*(const uint4*)(dy + rec_off(dy_pt, dy_p0 + plane, n, hw, HW) + 16 * pc), f);
    const float* xrow = x + (long)n * HW;
#pragma unroll
    for (int kh = 0; kh < KH; ++kh) {
      const int hh = h + kh - PH;
      const bool row_ok = hh >= 0 && hh < H;
#pragma unroll
      for (int kw = 0; kw < KW; ++kw) {
        const int ww = w + kw - PW;
        const float xv = (row_ok && ww >= 0 && ww < W) ? xrow[hh * W + ww] : 0.f;
#pragma unroll
        for (int j = 0; j < PN; ++j) acc[kh * KW + kw][j] = fmaf(xv, f[j], acc[kh * KW + kw][j]);
      }
    }
  }
  block_reduce_store<TAPS, PN>(acc, partial, cpad, plane, EPR);
}

__global__ void conv_first_wgrad_finalize_kernel(const float* partial, int nblk, int taps, int cpad, int C, float* dw /*[C][taps]*/) {
  const int i = blockIdx.x;       // one wave per (channel, tap)
  if (i >= C * taps) return;
  const int c = i / taps, t = i % taps;
  const double s = wave_sum_partials(partial, nblk, (long)taps * cpad, (long)c * taps + t);
  if (threadIdx.x == 0) dw[i] = (float)s;
}

// ---- Dice loss ------------------------------------------------------------------------------------------
// partial[blk][4] = { sum p*t, sum p, sum t, #correct }, p = sigmoid(z)
__global__ __launch_bounds__(256) void dice_fwd_kernel(const float* __restrict__ z, const signed char* __restrict__ t, long n,
                                                       float* partial) {
  float acc[4] = {};
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
    const float p = 1.f / (1.f + expf(-z[i]));
    const float tv = (float)t[i];
    acc[0] = fmaf(p, tv, acc[0]);
    acc[1] += p;
    acc[2] += tv;
    acc[3] += ((p >= 0.5f) == (t[i] != 0)) ? 1.f : 0.f;
  }
  __shared__ float red[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) acc[k] += __shfl_xor(acc[k], m);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) { for (int k = 0; k < 4; ++k) red[wave][k] = acc[k]; }
  __syncthreads();
  if (threadIdx.x < 4) partial[(long)blockIdx.x * 4 + threadIdx.x] = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
}

// sums[0..3] = I, P, T, correct (fp32, fp64-accumulated); sums[4] = loss of THESE sums (local batch)
__global__ void dice_finalize_kernel(const float* partial, int nblk, float* sums, float smooth) {
  double s[4];
  for (int k = 0; k < 4; ++k) s[k] = wave_sum_partials(partial, nblk, 4, k);
  if (threadIdx.x != 0) return;
  for (int k = 0; k < 4; ++k) sums[k] = (float)s[k];
  sums[4] = (float)(1.0 - (2.0 * s[0] + smooth) / (s[1] + s[2] + smooth));
}

// dz = -[2 t D - (2 I + smooth)] / D^2 * p (1 - p),  D = P + T + smooth; sums may have been all-reduced
__global__ __launch_bounds__(256) void dice_bwd_kernel(const float* __restrict__ z, const signed char* __restrict__ t, long n,
                                                       const float* __restrict__ sums, float smooth, float* dz) {
  const float I = sums[0], D = sums[1] + sums[2] + smooth;
  const float num = 2.f * I + smooth, invD2 = 1.f / (D * D);
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
    const float p = 1.f / (1.f + expf(-z[i]));
    dz[i] = -(2.f * (float)t[i] * D - num) * invD2 * p * (1.f - p);
  }
}

// ---- Adam (coupled L2) + zero_grad ---------------------------------------------------------------------
__global__ __launch_bounds__(256) void adam_kernel(float* __restrict__ p, float* __restrict__ g, float* __restrict__ m,
                                                   float* __restrict__ v, long n, float lr_over_bc1, float inv_sqrt_bc2,
                                                   float beta1, float beta2, float eps, float wd, float gscale, int zero_grad,
                                                   const float* __restrict__ hyper) {
  if (hyper) { lr_over_bc1 = hyper[1]; inv_sqrt_bc2 = hyper[2]; }   // graph replay: the step-dependent scalars live in HBM
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) {
    const float pv = p[i];
    const float gv = fmaf(wd, pv, g[i] * gscale);
    const float mv = fmaf(beta1, m[i], (1.f - beta1) * gv);
    const float vv = fmaf(beta2, v[i], (1.f - beta2) * gv * gv);
    m[i] = mv;
    v[i] = vv;
    float denom;
    {
#pragma clang fp contract(off)      // product and sum rounded separately, whatever instructions the build may use
      denom = sqrtf(vv) * inv_sqrt_bc2;
      denom = denom + eps;
    }
    p[i] = pv - lr_over_bc1 * mv / denom;
    if (zero_grad) g[i] = 0.f;
  }
}

// Step counter and bias corrections on the device, so that a captured launch sequence (HIP graph) can be replayed:
// hyper = [lr (written by the host when it changes), lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)], t = ++*step.
__global__ void adam_hyper_kernel(float* hyper, long long* step, float beta1, float beta2) {
  if (threadIdx.x == 0 && blockIdx.x == 0) {
    const long long t = *step + 1;
    *step = t;
    const double bc1 = 1.0 - pow((double)beta1, (double)t), bc2 = 1.0 - pow((double)beta2, (double)t);
    hyper[1] = (float)((double)hyper[0] / bc1);
    hyper[2] = (float)(1.0 / sqrt(bc2));
  }
}

// raw int16 RFU (H,W per image, already channel-first) -> fp32 (trainable_unet.py:70-72)
__global__ __launch_bounds__(256) void i16_to_f32_kernel(const short* __restrict__ in, float* __restrict__ out, long n) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) out[i] = (float)in[i];
}

// plain sum of an fp32 array (head bias gradient): partials then fixed-order fp64 finalize
__global__ __launch_bounds__(256) void sum_partial_kernel(const float* __restrict__ x, long n, float* partial) {
  float acc = 0.f;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x) acc += x[i];
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) acc += __shfl_xor(acc, m);
  __shared__ float red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}
__global__ void sum_finalize_kernel(const float* partial, int nblk, float* out) {
  const double s = wave_sum_partials(partial, nblk, 1, 0);
  if (threadIdx.x == 0) out[0] = (float)s;
}

inline unsigned ew_grid(long total) { return (unsigned)std::min<long>((total + 255) / 256, 8192); }
// segment length of the plane reductions: RED_SEG pieces, halved while the launch would leave CUs without work
inline int red_seg(int N, int nplanes, int npieces) {
  int seg = RED_SEG;
  while (seg > 1024 && (long)N * nplanes * ((npieces + seg - 1) / seg) < 2048) seg >>= 1;
  return seg;
}
inline int red_blocks(long pixels) { return (int)std::max<long>(1, std::min<long>((pixels + 127) / 128, RED_MAX_BLOCKS)); }

}  // namespace

#define DN_DISPATCH_T(dtype, CALL_BF16, CALL_F32, NAME)            \
  if ((dtype) == DN_BF16) { CALL_BF16; }                           \
  else if ((dtype) == DN_F32) { CALL_F32; }                        \
  else return dn_set_error(DN_ERR_ARG, NAME ": bad dtype %d", (dtype));

extern "C" {

int dn_reduce_blocks(long pixels) { return red_blocks(pixels); }

static int bn_train_forward_impl(dn_tensor y, dn_tensor a, int N, int H, int W, const float* gamma, const float* beta,
                                 float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                                 float* scale, float* shift, float* partial, int given_nblk, int dtype, void* stream,
                                 const dn_tensor* pooled = nullptr, const double* totals = nullptr, double total_count = 0);

int dn_bn_train_forward(dn_tensor y, dn_tensor a, int N, int H, int W, const float* gamma, const float* beta,
                        float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                        float* scale, float* shift, float* partial, int dtype, void* stream) {
  return bn_train_forward_impl(y, a, N, H, W, gamma, beta, running_mean, running_var, momentum, eps, mean, invstd, scale, shift,
                               partial, 0, dtype, stream);
}

int dn_bn_train_forward_noalloc(dn_tensor y, dn_tensor a, int N, int H, int W, const float* gamma, const float* beta,
                                float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                                float* scale, float* shift, int dtype, void* stream) {
  DN_CHECK_ARG(y.channels > 0 && y.channels <= DN_NOALLOC_MAX_CHANNELS,
               "dn_bn_train_forward_noalloc: %d channels, the built-in scratch holds the partials of at most %d "
               "(use dn_bn_train_forward with a workspace of dn_partial_floats(C) floats)", y.channels, DN_NOALLOC_MAX_CHANNELS);
  float* partial = nullptr;
  const int rc = noalloc_scratch(&partial);
  if (rc != DN_OK) return rc;
  // every partial the finalize kernel reads is written by this call's statistics kernel first: nothing to clear
  return bn_train_forward_impl(y, a, N, H, W, gamma, beta, running_mean, running_var, momentum, eps, mean, invstd, scale, shift,
                               partial, 0, dtype, stream);
}

int dn_bn_train_apply(dn_tensor y, dn_tensor a, int N, int H, int W, const float* gamma, const float* beta,
                      float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                      float* scale, float* shift, const float* partial, int ntiles, int dtype, void* stream) {
  DN_CHECK_ARG(ntiles > 0, "dn_bn_train_apply: no partial statistics");
  return bn_train_forward_impl(y, a, N, H, W, gamma, beta, running_mean, running_var, momentum, eps, mean, invstd, scale, shift,
                               (float*)partial, ntiles, dtype, stream);
}

int dn_bn_train_apply_pool(dn_tensor y, dn_tensor a, dn_tensor pooled, int N, int H, int W, const float* gamma, const float* beta,
                           float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                           float* scale, float* shift, const float* partial, int ntiles, int dtype, void* stream) {
  DN_CHECK_ARG(ntiles > 0, "dn_bn_train_apply_pool: no partial statistics");
  return bn_train_forward_impl(y, a, N, H, W, gamma, beta, running_mean, running_var, momentum, eps, mean, invstd, scale, shift,
                               (float*)partial, ntiles, dtype, stream, &pooled);
}

// given_nblk > 0: `partial` already holds [given_nblk][cpad][2] sums (dn_conv2d_stats), the statistics pass is skipped
static int bn_train_forward_impl(dn_tensor y, dn_tensor a, int N, int H, int W, const float* gamma, const float* beta,
                                 float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                                 float* scale, float* shift, float* partial, int given_nblk, int dtype, void* stream,
                                 const dn_tensor* pooled, const double* totals, double total_count) {
  DN_CHECK_ARG(y.base && a.base && gamma && beta && mean && invstd && scale && shift && (partial || totals), "dn_bn_train_forward: null pointer");
  DN_CHECK_ARG(y.channels == a.channels && N > 0 && H > 0 && W > 0, "dn_bn_train_forward: bad shape");
  const int C = y.channels, cpad = dn_channel_pad(C), nplanes = dn_planes(C, dtype);
  const long HW = (long)H * W;
  DN_CHECK_ARG(HW * 2 < (1L << 31) && N < 65536 && nplanes < 65536, "dn_bn_train_forward: plane too large for the launch grid");
  const int nblk = given_nblk > 0 ? given_nblk : red_blocks((long)N * HW);
  hipStream_t s = (hipStream_t)stream;
  if (totals) {
    // statistics already summed (over every rank of a data-parallel group): finalize from the global totals and count
    hipLaunchKernelGGL(bn_finalize_totals_kernel, dim3((cpad + 63) / 64), dim3(64), 0, s, totals, cpad, C, total_count, gamma, beta,
                       running_mean, running_var, momentum, eps, mean, invstd, scale, shift);
  } else {
  if (given_nblk <= 0) {
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(bn_stats_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)y.base, y.planes_total, y.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), partial, cpad),
    hipLaunchKernelGGL(bn_stats_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)y.base, y.planes_total, y.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), partial, cpad),
    "dn_bn_train_forward");
  }
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(bn_finalize_kernel, dim3(cpad), dim3(SUM_THREADS), 0, s, partial, nblk, cpad, C, (double)N * HW, gamma, beta,
                     running_mean, running_var, momentum, eps, mean, invstd, scale, shift);
  }
  DN_LAUNCH_CHECK();
  const int npieces = (int)(HW * 2);
  const dim3 egrid(std::min((npieces + 1023) / 1024, 64), nplanes, N);   // ~4 pieces per thread
  if (pooled) {
    DN_CHECK_ARG(W % 2 == 0 && pooled->base && pooled->channels == C && pooled->plane0 >= 0 &&
                 pooled->plane0 + nplanes <= pooled->planes_total, "dn_bn_train_apply_pool: bad pooled tensor (W must be even)");
#define ARGS_P (const unsigned char*)y.base, y.planes_total, y.plane0, (unsigned char*)a.base, a.planes_total, a.plane0, \
               (unsigned char*)pooled->base, pooled->planes_total, pooled->plane0, npieces, scale, shift
    DN_DISPATCH_T(dtype,
      hipLaunchKernelGGL(bn_apply_relu_pool_kernel<__bf16>, egrid, dim3(256), 0, s, ARGS_P),
      hipLaunchKernelGGL(bn_apply_relu_pool_kernel<float>, egrid, dim3(256), 0, s, ARGS_P),
      "dn_bn_train_apply_pool");
#undef ARGS_P
    DN_LAUNCH_CHECK();
    return DN_OK;
  }
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(bn_apply_relu_kernel<__bf16>, egrid, dim3(256), 0, s, (const unsigned char*)y.base, y.planes_total, y.plane0, (unsigned char*)a.base, a.planes_total, a.plane0, npieces, scale, shift),
    hipLaunchKernelGGL(bn_apply_relu_kernel<float>, egrid, dim3(256), 0, s, (const unsigned char*)y.base, y.planes_total, y.plane0, (unsigned char*)a.base, a.planes_total, a.plane0, npieces, scale, shift),
    "dn_bn_train_forward");
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_bn_partial_totals(const float* partial, int ntiles, int C, double* totals, void* stream) {
  DN_CHECK_ARG(partial && totals && ntiles > 0 && C > 0, "dn_bn_partial_totals: bad argument");
  const int cpad = dn_channel_pad(C);
  hipLaunchKernelGGL(bn_pair_totals_kernel, dim3(cpad), dim3(SUM_THREADS), 0, (hipStream_t)stream, partial, ntiles, cpad, C, totals);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_bn_train_apply_totals(dn_tensor y, dn_tensor a, dn_tensor pooled, int N, int H, int W, const float* gamma, const float* beta,
                             float* running_mean, float* running_var, float momentum, float eps, float* mean, float* invstd,
                             float* scale, float* shift, const double* totals, double count, int dtype, void* stream) {
  DN_CHECK_ARG(totals && count >= 1, "dn_bn_train_apply_totals: no totals / bad count");
  return bn_train_forward_impl(y, a, N, H, W, gamma, beta, running_mean, running_var, momentum, eps, mean, invstd, scale, shift,
                               nullptr, 0, dtype, stream, pooled.base ? &pooled : nullptr, totals, count);
}

static int bn_train_backward_impl(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                                  const float* gamma, const float* mean, const float* invstd, float* dgamma, float* dbeta, float* coef,
                                  float* partial, int dtype, void* stream, int phase, double* local_totals,
                                  const double* global_totals, double count, int given_nblk = 0);

int dn_bn_train_backward(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                         const float* gamma, const float* mean, const float* invstd, float* dgamma, float* dbeta, float* coef,
                         float* partial, int dtype, void* stream) {
  return bn_train_backward_impl(g, y, scale, shift, N, H, W, gamma, mean, invstd, dgamma, dbeta, coef, partial, dtype, stream, 0,
                                nullptr, nullptr, 0);
}

int dn_bn_train_backward_sums(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                              const float* gamma, const float* mean, const float* invstd, float* dgamma, float* dbeta, float* coef,
                              const float* sums, int ntiles, int dtype, void* stream) {
  DN_CHECK_ARG(sums && ntiles > 0, "dn_bn_train_backward_sums: no sums");
  return bn_train_backward_impl(g, y, scale, shift, N, H, W, gamma, mean, invstd, dgamma, dbeta, coef, (float*)sums, dtype, stream, 0,
                                nullptr, nullptr, 0, ntiles);
}

int dn_bn_backward_sums_totals(const float* sums, int ntiles, int channels, double* totals, void* stream) {
  DN_CHECK_ARG(sums && totals && ntiles > 0 && channels > 0, "dn_bn_backward_sums_totals: bad argument");
  const int cpad = dn_channel_pad(channels);
  hipLaunchKernelGGL(bn_bwd_pair_totals_kernel, dim3(cpad), dim3(SUM_THREADS), 0, (hipStream_t)stream, sums, ntiles, cpad, channels, totals);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_bn_train_backward_totals(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                                const float* mean, const float* invstd, float* partial, double* totals, int dtype, void* stream) {
  DN_CHECK_ARG(totals, "dn_bn_train_backward_totals: null pointer");
  return bn_train_backward_impl(g, y, scale, shift, N, H, W, nullptr, mean, invstd, nullptr, nullptr, nullptr, partial, dtype, stream,
                                1, totals, nullptr, 0);
}

int dn_bn_train_backward_apply_totals(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                                      const float* gamma, const float* mean, const float* invstd, const double* local_totals,
                                      const double* global_totals, double count, float* dgamma, float* dbeta, float* coef,
                                      int dtype, void* stream) {
  DN_CHECK_ARG(local_totals && global_totals && count >= 1, "dn_bn_train_backward_apply_totals: no totals / bad count");
  return bn_train_backward_impl(g, y, scale, shift, N, H, W, gamma, mean, invstd, dgamma, dbeta, coef, nullptr, dtype, stream, 2,
                                (double*)local_totals, global_totals, count);
}

// phase 0: reduce + finalize + apply (one device).  phase 1: reduce + per-channel totals only.  phase 2: finalize from
// (local, global) totals + apply.
static int bn_train_backward_impl(dn_tensor g, dn_tensor y, const float* scale, const float* shift, int N, int H, int W,
                                  const float* gamma, const float* mean, const float* invstd, float* dgamma, float* dbeta, float* coef,
                                  float* partial, int dtype, void* stream, int phase, double* local_totals,
                                  const double* global_totals, double count, int given_nblk) {
  // given_nblk > 0: `partial` already holds [given_nblk][cpad][2] sums (dn_conv2d_dgrad_bn_sums), the reduction pass is skipped
  DN_CHECK_ARG(g.base && y.base && scale && shift && mean && invstd, "dn_bn_train_backward: null pointer");
  DN_CHECK_ARG(phase == 2 || partial, "dn_bn_train_backward: no partial workspace");
  DN_CHECK_ARG(phase == 1 || (gamma && dgamma && dbeta && coef), "dn_bn_train_backward: null pointer");
  DN_CHECK_ARG(g.channels == y.channels && N > 0 && H > 0 && W > 0, "dn_bn_train_backward: bad shape");
  const int C = y.channels, cpad = dn_channel_pad(C), nplanes = dn_planes(C, dtype);
  const long HW = (long)H * W;
  DN_CHECK_ARG(HW * 2 < (1L << 31) && N < 65536 && nplanes < 65536, "dn_bn_train_backward: plane too large for the launch grid");
  const int nblk = given_nblk > 0 ? given_nblk : red_blocks((long)N * HW);
  hipStream_t s = (hipStream_t)stream;
  if (phase != 2 && given_nblk <= 0) {
#define ARGS_R (const unsigned char*)g.base, g.planes_total, g.plane0, (const unsigned char*)y.base, y.planes_total, y.plane0, \
               scale, shift, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), mean, invstd, partial, cpad
    DN_DISPATCH_T(dtype,
      hipLaunchKernelGGL(bn_bwd_reduce_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, ARGS_R),
      hipLaunchKernelGGL(bn_bwd_reduce_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, ARGS_R),
      "dn_bn_train_backward");
#undef ARGS_R
    DN_LAUNCH_CHECK();
  }
  if (phase == 1) {
    hipLaunchKernelGGL(bn_bwd_pair_totals_kernel, dim3(cpad), dim3(SUM_THREADS), 0, s, partial, nblk, cpad, C, local_totals);
    DN_LAUNCH_CHECK();
    return DN_OK;
  }
  if (phase == 2)
    hipLaunchKernelGGL(bn_bwd_finalize_totals_kernel, dim3((cpad + 63) / 64), dim3(64), 0, s, local_totals, global_totals, cpad, C,
                       count, gamma, invstd, dgamma, dbeta, coef);
  else
    hipLaunchKernelGGL(bn_bwd_finalize_kernel, dim3(cpad), dim3(SUM_THREADS), 0, s, partial, nblk, cpad, C, (double)N * HW, gamma,
                       invstd, dgamma, dbeta, coef);
  DN_LAUNCH_CHECK();
  const int npieces = (int)(HW * 2);
  const dim3 egrid(std::min((npieces + 1023) / 1024, 64), nplanes, N);
#define ARGS_A (unsigned char*)g.base, g.planes_total, g.plane0, (const unsigned char*)y.base, y.planes_total, y.plane0, \
               scale, shift, npieces, mean, invstd, coef, cpad
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(bn_bwd_apply_kernel<__bf16>, egrid, dim3(256), 0, s, ARGS_A),
    hipLaunchKernelGGL(bn_bwd_apply_kernel<float>, egrid, dim3(256), 0, s, ARGS_A),
    "dn_bn_train_backward");
#undef ARGS_A
  DN_LAUNCH_CHECK();
  return DN_OK;
}

// the BatchNorm unit whose activation gradient a producer writes: saved convolution output and per-channel vectors
struct BnUnit { dn_tensor y; const float *scale, *shift, *mean, *invstd; float* sums; long sums_floats; int* nblk; };

static int bn_unit_check(const BnUnit& bn, int channels, int dtype, long pixels, const char* who) {
  DN_CHECK_ARG(bn.y.base && bn.scale && bn.shift && bn.mean && bn.invstd && bn.sums && bn.nblk, "%s: null pointer", who);
  DN_CHECK_ARG(bn.y.channels == channels, "%s: bn_y has %d channels, g %d", who, bn.y.channels, channels);
  const int bp = dn_planes(channels, dtype);
  DN_CHECK_ARG(bn.y.plane0 >= 0 && bn.y.plane0 + bp <= bn.y.planes_total, "%s: bn_y planes [%d,%d) outside buffer of %d", who,
               bn.y.plane0, bn.y.plane0 + bp, bn.y.planes_total);
  const long need = (long)red_blocks(pixels) * dn_channel_pad(channels) * 2;
  DN_CHECK_ARG(need <= bn.sums_floats, "%s: sums buffer of %ld floats, need %ld", who, bn.sums_floats, need);
  return DN_OK;
}

static int maxpool_backward_impl(dn_tensor x, dn_tensor dpool, dn_tensor dskip, dn_tensor g, int N, int H, int Wout, int dtype,
                                 void* stream, const BnUnit* bn) {
  DN_CHECK_ARG(x.base && dpool.base && g.base, "dn_maxpool_1x2_backward: null pointer");
  DN_CHECK_ARG(x.channels == dpool.channels && x.channels == g.channels && (!dskip.base || dskip.channels == x.channels),
               "dn_maxpool_1x2_backward: channel mismatch");
  DN_CHECK_ARG(dtype == DN_BF16 || dtype == DN_F32, "dn_maxpool_1x2_backward: bad dtype %d", dtype);
  const int nplanes = dn_planes(x.channels, dtype);
  if (bn) {
    const long pix = (long)N * H * Wout * 2;
    if (int rc = bn_unit_check(*bn, x.channels, dtype, pix, "dn_maxpool_1x2_backward_bn_sums")) return rc;
    DN_CHECK_ARG((long)H * Wout * 4 < (1L << 31) && nplanes < 65536, "dn_maxpool_1x2_backward_bn_sums: plane too large for the launch grid");
    const int nblk = red_blocks(pix), nitems = 2 * H * Wout, cpad = dn_channel_pad(x.channels);
#define ARGS_S (const unsigned char*)x.base, x.planes_total, x.plane0, (const unsigned char*)dpool.base, dpool.planes_total, dpool.plane0, \
               (const unsigned char*)dskip.base, dskip.planes_total, dskip.plane0, (unsigned char*)g.base, g.planes_total, g.plane0, \
               (const unsigned char*)bn->y.base, bn->y.planes_total, bn->y.plane0, bn->scale, bn->shift, bn->mean, bn->invstd, N, \
               nitems, red_seg(N, nplanes, nitems), bn->sums, cpad
    DN_DISPATCH_T(dtype,
      hipLaunchKernelGGL(pool_bwd_add_sums_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, (hipStream_t)stream, ARGS_S),
      hipLaunchKernelGGL(pool_bwd_add_sums_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, (hipStream_t)stream, ARGS_S),
      "dn_maxpool_1x2_backward_bn_sums");
#undef ARGS_S
    DN_LAUNCH_CHECK();
    *bn->nblk = nblk;
    return DN_OK;
  }
  const long total = (long)N * nplanes * H * Wout * 2;
#define ARGS (const unsigned char*)x.base, x.planes_total, x.plane0, (const unsigned char*)dpool.base, dpool.planes_total, dpool.plane0, \
             (const unsigned char*)dskip.base, dskip.planes_total, dskip.plane0, (unsigned char*)g.base, g.planes_total, g.plane0, \
             nplanes, (long)N, H, Wout
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(pool_bwd_add_kernel<__bf16>, dim3(ew_grid(total)), dim3(256), 0, (hipStream_t)stream, ARGS),
    hipLaunchKernelGGL(pool_bwd_add_kernel<float>, dim3(ew_grid(total)), dim3(256), 0, (hipStream_t)stream, ARGS),
    "dn_maxpool_1x2_backward");
#undef ARGS
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_maxpool_1x2_backward(dn_tensor x, dn_tensor dpool, dn_tensor dskip, dn_tensor g, int N, int H, int Wout, int dtype,
                            void* stream) {
  return maxpool_backward_impl(x, dpool, dskip, g, N, H, Wout, dtype, stream, nullptr);
}

int dn_maxpool_1x2_backward_bn_sums(dn_tensor x, dn_tensor dpool, dn_tensor dskip, dn_tensor g, dn_tensor bn_y, const float* scale,
                                    const float* shift, const float* mean, const float* invstd, int N, int H, int Wout, int dtype,
                                    float* sums, long sums_floats, int* nblk, void* stream) {
  const BnUnit bn{bn_y, scale, shift, mean, invstd, sums, sums_floats, nblk};
  return maxpool_backward_impl(x, dpool, dskip, g, N, H, Wout, dtype, stream, &bn);
}

static int head_backward_impl(const float* dlogits, dn_tensor x, const float* w, dn_tensor g, float* dw, float* db, float* partial,
                              int N, int H, int W, int dtype, void* stream, const BnUnit* bn);

int dn_head_1x1_backward(const float* dlogits, dn_tensor x, const float* w, dn_tensor g, float* dw, float* db, float* partial,
                         int N, int H, int W, int dtype, void* stream) {
  return head_backward_impl(dlogits, x, w, g, dw, db, partial, N, H, W, dtype, stream, nullptr);
}

int dn_head_1x1_backward_bn_sums(const float* dlogits, dn_tensor x, const float* w, dn_tensor g, float* dw, float* db, float* partial,
                                 dn_tensor bn_y, const float* scale, const float* shift, const float* mean, const float* invstd,
                                 int N, int H, int W, int dtype, float* sums, long sums_floats, int* nblk, void* stream) {
  const BnUnit bn{bn_y, scale, shift, mean, invstd, sums, sums_floats, nblk};
  return head_backward_impl(dlogits, x, w, g, dw, db, partial, N, H, W, dtype, stream, &bn);
}

static int head_backward_impl(const float* dlogits, dn_tensor x, const float* w, dn_tensor g, float* dw, float* db, float* partial,
                              int N, int H, int W, int dtype, void* stream, const BnUnit* bn) {
  DN_CHECK_ARG(dlogits && x.base && w && g.base && dw && db && partial, "dn_head_1x1_backward: null pointer");
  DN_CHECK_ARG(x.channels == g.channels, "dn_head_1x1_backward: channel mismatch");
  DN_CHECK_ARG(N > 0 && (long)H * W > 0 && (long)H * W * 2 < (1L << 31), "dn_head_1x1_backward: bad shape / plane too large");
  const int C = x.channels, cpad = dn_channel_pad(C), nplanes = dn_planes(C, dtype);
  const long HW = (long)H * W;
  hipStream_t s = (hipStream_t)stream;
  const long total = (long)N * nplanes * HW * 2;
  const int nblk = red_blocks((long)N * HW);
  if (bn) {
    if (int rc = bn_unit_check(*bn, x.channels, dtype, (long)N * HW, "dn_head_1x1_backward_bn_sums")) return rc;
    DN_CHECK_ARG(nplanes < 65536, "dn_head_1x1_backward_bn_sums: too many planes for the launch grid");
#define ARGS_H dlogits, w, (unsigned char*)g.base, g.planes_total, g.plane0, (const unsigned char*)bn->y.base, bn->y.planes_total, \
               bn->y.plane0, bn->scale, bn->shift, bn->mean, bn->invstd, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), bn->sums, cpad
    DN_DISPATCH_T(dtype,
      hipLaunchKernelGGL(head_bwd_data_sums_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, ARGS_H),
      hipLaunchKernelGGL(head_bwd_data_sums_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, ARGS_H),
      "dn_head_1x1_backward_bn_sums");
#undef ARGS_H
    *bn->nblk = nblk;
  } else {
    DN_DISPATCH_T(dtype,
      hipLaunchKernelGGL(head_bwd_data_kernel<__bf16>, dim3(ew_grid(total)), dim3(256), 0, s, dlogits, w, (unsigned char*)g.base, g.planes_total, g.plane0, nplanes, (long)N, HW),
      hipLaunchKernelGGL(head_bwd_data_kernel<float>, dim3(ew_grid(total)), dim3(256), 0, s, dlogits, w, (unsigned char*)g.base, g.planes_total, g.plane0, nplanes, (long)N, HW),
      "dn_head_1x1_backward");
  }
  DN_LAUNCH_CHECK();
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(channel_sum_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)x.base, x.planes_total, x.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), dlogits, partial, cpad),
    hipLaunchKernelGGL(channel_sum_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)x.base, x.planes_total, x.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), dlogits, partial, cpad),
    "dn_head_1x1_backward");
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(channel_sum_finalize_kernel, dim3(C), dim3(64), 0, s, partial, nblk, cpad, C, dw);
  DN_LAUNCH_CHECK();
  // bias gradient = sum(dlogits): reuse the Dice reduction shape via a 1-plane trick is overkill; a tiny kernel does it
  float* p2 = partial + (long)nblk * cpad;
  const int nb2 = (int)std::min<long>(((long)N * HW + 255) / 256, 512);
  hipLaunchKernelGGL(sum_partial_kernel, dim3(nb2), dim3(256), 0, s, dlogits, (long)N * HW, p2);
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(sum_finalize_kernel, dim3(1), dim3(64), 0, s, p2, nb2, db);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_channel_sum(dn_tensor x, float* out, float* partial, int N, int H, int W, int dtype, void* stream) {
  DN_CHECK_ARG(x.base && out && partial, "dn_channel_sum: null pointer");
  const int C = x.channels, cpad = dn_channel_pad(C), nplanes = dn_planes(C, dtype);
  const long HW = (long)H * W;
  DN_CHECK_ARG(N > 0 && HW > 0 && HW * 2 < (1L << 31) && nplanes < 65536, "dn_channel_sum: bad shape / plane too large for the launch grid");
  const int nblk = red_blocks((long)N * HW);
  hipStream_t s = (hipStream_t)stream;
  DN_DISPATCH_T(dtype,
    hipLaunchKernelGGL(channel_sum_kernel<__bf16>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)x.base, x.planes_total, x.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), (const float*)nullptr, partial, cpad),
    hipLaunchKernelGGL(channel_sum_kernel<float>, dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, (const unsigned char*)x.base, x.planes_total, x.plane0, N, (int)(HW * 2), red_seg(N, nplanes, (int)(HW * 2)), (const float*)nullptr, partial, cpad),
    "dn_channel_sum");
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(channel_sum_finalize_kernel, dim3(C), dim3(64), 0, s, partial, nblk, cpad, C, out);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_conv_first_wgrad(const float* x, dn_tensor dy, float* dw, float* partial, long partial_floats, int N, int H, int W, int kh,
                        int kw, int dtype, void* stream) {
  DN_CHECK_ARG(x && dy.base && dw && partial, "dn_conv_first_wgrad: null pointer");
  DN_CHECK_ARG(N > 0 && H > 0 && W > 0 && kh > 0 && kw > 0 && dy.channels > 0, "dn_conv_first_wgrad: bad shape");
  const int C = dy.channels, cpad = dn_channel_pad(C), nplanes = dn_planes(C, dtype), taps = kh * kw;
  const int nblk = dn_conv_first_wgrad_blocks(N, H, W);
  DN_CHECK_ARG((long)nblk * taps * cpad <= partial_floats, "dn_conv_first_wgrad: partial buffer of %ld floats, need %ld",
               partial_floats, (long)nblk * taps * cpad);
  hipStream_t s = (hipStream_t)stream;
  DN_CHECK_ARG((long)N * H * W < (1L << 31), "dn_conv_first_wgrad: more than 2^31 pixels");
#define LAUNCH(TT, KH, KW) hipLaunchKernelGGL((conv_first_wgrad_kernel<TT, KH, KW>), dim3(nblk, nplanes), dim3(RED_THREADS), 0, s, x, \
    (const unsigned char*)dy.base, dy.planes_total, dy.plane0, N, H, W, partial, cpad)
  if (kh == 3 && kw == 5) { DN_DISPATCH_T(dtype, LAUNCH(__bf16, 3, 5), LAUNCH(float, 3, 5), "dn_conv_first_wgrad"); }
  else if (kh == 1 && kw == 3) { DN_DISPATCH_T(dtype, LAUNCH(__bf16, 1, 3), LAUNCH(float, 1, 3), "dn_conv_first_wgrad"); }
  else if (kh == 1 && kw == 1) { DN_DISPATCH_T(dtype, LAUNCH(__bf16, 1, 1), LAUNCH(float, 1, 1), "dn_conv_first_wgrad"); }
  else return dn_set_error(DN_ERR_UNSUPPORTED, "dn_conv_first_wgrad: kernel size (%d,%d) not built", kh, kw);
#undef LAUNCH
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(conv_first_wgrad_finalize_kernel, dim3(C * taps), dim3(64), 0, s, partial, nblk, taps, cpad, C, dw);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_conv_first_wgrad_blocks(int N, int H, int W) {
  return (int)std::max<long>(1, std::min<long>(((long)N * H * W + 127) / 128, 512));
}

int dn_dice_forward(const float* logits, const signed char* targets, long n, float* sums, float* partial, void* stream) {
  DN_CHECK_ARG(logits && targets && sums && partial && n > 0, "dn_dice_forward: bad argument");
  const int nblk = (int)std::min<long>((n + 255) / 256, 1024);
  hipLaunchKernelGGL(dice_fwd_kernel, dim3(nblk), dim3(256), 0, (hipStream_t)stream, logits, targets, n, partial);
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(dice_finalize_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, partial, nblk, sums, 1.0f);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_dice_backward(const float* logits, const signed char* targets, long n, const float* sums, float* dlogits, void* stream) {
  DN_CHECK_ARG(logits && targets && sums && dlogits && n > 0, "dn_dice_backward: bad argument");
  hipLaunchKernelGGL(dice_bwd_kernel, dim3(ew_grid(n)), dim3(256), 0, (hipStream_t)stream, logits, targets, n, sums, 1.0f, dlogits);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_adam_step(float* params, float* grads, float* exp_avg, float* exp_avg_sq, long n, float lr, float beta1, float beta2,
                 float eps, float weight_decay, long step, float grad_scale, int zero_grad, void* stream) {
  DN_CHECK_ARG(params && grads && exp_avg && exp_avg_sq && n > 0 && step >= 1, "dn_adam_step: bad argument");
  const double bc1 = 1.0 - pow((double)beta1, (double)step), bc2 = 1.0 - pow((double)beta2, (double)step);
  hipLaunchKernelGGL(adam_kernel, dim3(ew_grid(n)), dim3(256), 0, (hipStream_t)stream, params, grads, exp_avg, exp_avg_sq, n,
                     (float)(lr / bc1), (float)(1.0 / sqrt(bc2)), beta1, beta2, eps, weight_decay, grad_scale, zero_grad,
                     (const float*)nullptr);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_adam_step_graph(float* params, float* grads, float* exp_avg, float* exp_avg_sq, long n, float* hyper, long long* step,
                       float beta1, float beta2, float eps, float weight_decay, float grad_scale, int zero_grad, void* stream) {
  DN_CHECK_ARG(params && grads && exp_avg && exp_avg_sq && hyper && step && n > 0, "dn_adam_step_graph: bad argument");
  hipLaunchKernelGGL(adam_hyper_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, hyper, step, beta1, beta2);
  DN_LAUNCH_CHECK();
  hipLaunchKernelGGL(adam_kernel, dim3(ew_grid(n)), dim3(256), 0, (hipStream_t)stream, params, grads, exp_avg, exp_avg_sq, n,
                     0.f, 0.f, beta1, beta2, eps, weight_decay, grad_scale, zero_grad, (const float*)hyper);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

int dn_i16_to_f32(const short* in, float* out, long n, void* stream) {
  DN_CHECK_ARG(in && out && n > 0, "dn_i16_to_f32: bad argument");
  hipLaunchKernelGGL(i16_to_f32_kernel, dim3(ew_grid(n)), dim3(256), 0, (hipStream_t)stream, in, out, n);
  DN_LAUNCH_CHECK();
  return DN_OK;
}

}  // extern "C"
