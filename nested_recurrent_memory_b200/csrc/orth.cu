// Newton-Schulz orthogonalisation of weight updates: X_0 = G / (|G|_F + eps),
// then X <- (a I + b A + c A A) X with A = X X^T, on the smaller side of G (a
// tall G is worked on transposed: X is m x n with m <= n).
//
// Precision. A step stretches what lies along small singular values by up to
// a = 3.4, so five steps stretch a rounding next to a large singular value
// by up to 485: single 16-bit operands leave errors of 1e-3 (full-rank
// Gaussian updates, fp16) to 3e-1 (a strong direction over a weak remainder,
// bf16). So every operand is held as two fp16 planes, hi + lo (22 bits; X,
// A and B scaled to the middle of fp16's range), and a product is three MMAs,
// hi hi + hi lo + lo hi, summed in fp32 in tensor memory: the accuracy of fp32
// arithmetic (about 1e-6 .. 1e-5 on the same updates) at a third of the
// tensor cores' rate. A 16-bit update fits its hi plane, so the first step
// needs one product for A and two for X.
//
// Kernels: the squared norm (partial sums in 64 bits), the conversion to
// planes, then per step three products: A = X X^T, B = a I + b A + c A A
// (both symmetric: tiles on and above the diagonal only, written twice) and
// X' = B X, which reads X as it lies, rows along the reduction.
//
// Products: a pair of CTAs computes 256 x 256 tiles (tcgen05, cta_group::2; each
// CTA holds its 128 rows of the left operand and half of the right one), fed
// by a thread that issues TMA loads three 64-deep stages ahead, with two
// accumulators in tensor memory so that one tile's results are written while
// the next is multiplied. The pair tile halves what each multiprocessor must
// read: 64 KB a stage for 12 MMAs.

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "launch.cuh"
#include "tc_ptx.cuh"

using namespace ngdn2;
using namespace ngdn2::tc;

namespace {

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

// Planes hold kScale times the values of X (after the first step), A and B.
constexpr float kScale = 1024.f;
// |a + b s^2 + c s^4| and singular values s stay below these (checked on the
// host), so that the planes stay within fp16.
constexpr double kMaxFactor = 60.0, kMaxSigma = 4.0;

__device__ __forceinline__ void split(float x, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn(x - __half2float(hi));
}

// ---------------------------------------------------------------------------
// Norm and conversion
// ---------------------------------------------------------------------------

constexpr int kPrepThreads = 256, kNormParts = 64;

struct PrepArgs {
  const void* g;
  int dtype;
  int64_t batch, m, n;     // X is m x n
  int64_t sb, sr, sc;      // element strides of the update by matrix, row and column of X
  float eps;
  double* part;            // [batch][kNormParts]
  float* sigma;            // [batch]: X_0 = sigma * planes
  __half* x;               // [batch][2][m][ld]
  int64_t ld;
};

// Squares are summed in 64 bits, so neither large nor small updates leave
// the range.
__global__ void __launch_bounds__(kPrepThreads) orth_norm_kernel(const __grid_constant__ PrepArgs p) {
  __shared__ double red[kPrepThreads / 32];
  const int64_t b = blockIdx.x / kNormParts, part = blockIdx.x % kNormParts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Lanes along the dimension with the smaller stride.
  const bool along_c = p.sc <= p.sr;
  const int64_t outer = along_c ? p.m : p.n, inner = along_c ? p.n : p.m;
  const int64_t so = along_c ? p.sr : p.sc, si = along_c ? p.sc : p.sr;
  double s = 0.0;
  for (int64_t r = part * (kPrepThreads / 32) + warp; r < outer; r += int64_t(kNormParts) * (kPrepThreads / 32)) {
    const int64_t base = b * p.sb + r * so;
    double row = 0.0;
#pragma unroll 8
    for (int64_t c = lane; c < inner; c += 32) {
      const double x = load_elem(p.g, base + c * si, p.dtype);
      row = fma(x, x, row);
    }
    s += row;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) s += red[w];
    p.part[b * kNormParts + part] = s;
  }
  let_next_start();
}

// The power of two that brings the norm into [2^11, 2^12), and sigma.
__device__ __forceinline__ void norm_scale(const PrepArgs& p, int64_t b, int* k, float* sigma) {
  double s = p.part[b * kNormParts + (threadIdx.x & 31)] + p.part[b * kNormParts + 32 + (threadIdx.x & 31)];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const double norm = sqrt(s);
  int e = 0;
  if (norm > 0.0 && norm < 1e300) frexp(norm, &e);
  *k = (norm > 0.0 && norm < 1e300) ? 12 - e : 0;
  *sigma = float(1.0 / (norm + double(p.eps)) / scalbn(1.0, *k));
}

constexpr int kConvTile = 64;

__global__ void __launch_bounds__(kPrepThreads) orth_convert_kernel(const __grid_constant__ PrepArgs p) {
  __shared__ float tile[kConvTile][kConvTile + 1];
  after_previous();
  const int64_t tc = (p.n + kConvTile - 1) / kConvTile, tr = (p.m + kConvTile - 1) / kConvTile;
  const int64_t b = blockIdx.x / (tc * tr), q = blockIdx.x % (tc * tr);
  const int64_t r0 = q / tc * kConvTile, c0 = q % tc * kConvTile;
  int k;
  float sigma;
  norm_scale(p, b, &k, &sigma);
  if (q == 0 && threadIdx.x == 0) p.sigma[b] = sigma;
  const float s1 = scalbnf(1.f, k / 2), s2 = scalbnf(1.f, k - k / 2);
  const bool along_c = p.sc <= p.sr;
#pragma unroll 4
  for (int e = threadIdx.x; e < kConvTile * kConvTile; e += kPrepThreads) {
    const int i = e / kConvTile, j = e % kConvTile;
    const int r = along_c ? i : j, c = along_c ? j : i;
    float x = 0.f;
    if (r0 + r < p.m && c0 + c < p.n)
      x = load_elem(p.g, b * p.sb + (r0 + r) * p.sr + (c0 + c) * p.sc, p.dtype) * s1 * s2;
    tile[r][c] = x;
  }
  __syncthreads();
  __half* hi = p.x + b * 2 * p.m * p.ld;
  __half* lo = hi + p.m * p.ld;
  for (int e = threadIdx.x; e < kConvTile * kConvTile / 4; e += kPrepThreads) {
    const int r = e / (kConvTile / 4), c = e % (kConvTile / 4) * 4;
    if (r0 + r >= p.m || c0 + c >= p.ld) continue;  // (ld is a multiple of 8)
    __half h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split(tile[r][c + i], h[i], l[i]);
    const int64_t o = (r0 + r) * p.ld + c0 + c;
    *reinterpret_cast<uint2*>(hi + o) = *reinterpret_cast<const uint2*>(h);
    *reinterpret_cast<uint2*>(lo + o) = *reinterpret_cast<const uint2*>(l);
  }
  let_next_start();
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

enum { kGram = 0, kPoly = 1, kApply = 2 };  // A = X X^T; B = a I + b A + c A A; X' = B X

constexpr int kTile = 256;            // rows and columns of a pair's tile
constexpr int kDepth = 64;            // reduction elements of a stage
constexpr int kPlane = 128 * kDepth * 2;  // bytes of one operand's plane in one CTA, a stage
constexpr int kStages = 3, kStageBytes = 4 * kPlane;
constexpr int kMulThreads = 384;      // load, multiply, 2 idle warps, 8 that write results
constexpr int kWriters = 8;
constexpr int kSmem = kStages * kStageBytes + 1024 + 256;

struct MulArgs {
  int64_t batch, m, n;   // X is m x n
  int64_t depth;         // of the reduction
  int64_t nt, tiles_n, per;  // row tiles, column tiles, tiles of a matrix
  bool lo_left, lo_right;    // whether the operands' lo planes are read
  float a, b, c;
  const float* sigma;    // [batch], or NULL for 1 / kScale
  const __half* old;     // kPoly: the planes of A
  __half* out;           // [batch][2][m][ld], or
  void* final_out;       // the result (kApply)
  int out_dtype, transposed;
  int64_t ld;
  int32_t* status;
};

struct Barriers {
  uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int dead;
};

// Tile number t of a matrix: all of them, or those on and above the diagonal.
template <int MODE>
__device__ __forceinline__ void tile_at(const MulArgs& p, int64_t t, int64_t* b, int64_t* tm, int64_t* tn) {
  *b = t / p.per;
  int64_t q = t % p.per;
  if (MODE == kApply) {
    *tm = q / p.tiles_n;
    *tn = q % p.tiles_n;
  } else {
    int64_t r = 0, len = p.nt;
    while (q >= len) {
      q -= len;
      --len;
      ++r;
    }
    *tm = r;
    *tn = r + q;
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of the pair's first CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t in_first(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One box into this CTA, its bytes counted by the first CTA's barrier.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Arrives at this barrier of both CTAs when the MMAs so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// Descriptor of a right operand that lies rows along the reduction: blocks of 64
// columns (8 KB: 64 rows of 128 bytes, 128-byte swizzle), 8-row groups of 1 KB.
__device__ __forceinline__ uint64_t desc_sw128_mn(uint32_t saddr) {
  return (desc_sw128(saddr, 1024) & ~(uint64_t(0x3FFF) << 16)) | uint64_t(8192 >> 4) << 16;
}

// A bounded wait that gives up for the whole CTA.
__device__ __forceinline__ bool wait_or_die(Barriers* s, uint64_t* bar, uint32_t phase, int32_t* status) {
  for (uint32_t i = 0; i < (1u << 20); ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (*reinterpret_cast<volatile int*>(&s->dead)) return false;
  }
  s->dead = 1;
  atomicOr(status, NGDN2_STATUS_WAIT_TIMEOUT);
  return false;
}

// 32 neighbouring results of one row, from the accumulator's values v.
template <int MODE>
__device__ __forceinline__ void write32(const MulArgs& p, int64_t b, int64_t r, int64_t c, bool mirror,
                                        float sigma, const float* v) {
  const int64_t cols = MODE == kApply ? p.n : p.m;
  const int left = int(cols - c < 32 ? cols - c : 32);
  if (MODE == kApply && p.final_out) {
    const float s = sigma / kScale;
    if (p.transposed) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < left) store_elem(p.final_out, (b * p.n + c + i) * p.m + r, s * v[i], p.out_dtype);
    } else {
      const int64_t o = (b * p.m + r) * p.n + c;
      const int el = p.out_dtype == NGDN2_F32 ? 4 : 2;
      char* to = static_cast<char*>(p.final_out) + o * el;
      if (left == 32 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          alignas(16) unsigned char w[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) store_elem(w, j, s * v[i + j], p.out_dtype);
          reinterpret_cast<uint4*>(to)[i * el / 16] = *reinterpret_cast<const uint4*>(w);
          if (el == 4) reinterpret_cast<uint4*>(to)[i * el / 16 + 1] = *reinterpret_cast<const uint4*>(w + 16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < left) store_elem(p.final_out, o + i, s * v[i], p.out_dtype);
      }
    }
    return;
  }
  const int64_t rows = p.m, plane = rows * p.ld, at = r * p.ld + c;
  const __half* old = p.old + b * 2 * plane;
  __half* out = p.out + b * 2 * plane;
#pragma unroll
  for (int i0 = 0; i0 < 32; i0 += 8) {
    alignas(16) __half h[8], l[8], oh[8], ol[8];
    const bool whole = i0 + 8 <= left;  // (rows are multiples of 8 apart)
    if (MODE == kPoly) {
      if (i0 < left) {  // (what lies past the row's end is not used)
        *reinterpret_cast<uint4*>(oh) = *reinterpret_cast<const uint4*>(old + at + i0);
        *reinterpret_cast<uint4*>(ol) = *reinterpret_cast<const uint4*>(old + plane + at + i0);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x;
      if (MODE == kGram) {
        x = v[i0 + j] * sigma * sigma * kScale;
      } else if (MODE == kPoly) {
        x = p.c * (v[i0 + j] / kScale) + p.b * (__half2float(oh[j]) + __half2float(ol[j])) +
            (c + i0 + j == r ? p.a * kScale : 0.f);
      } else {
        x = v[i0 + j] * sigma;  // sigma X^ B^ / kScale, times kScale
      }
      split(x, h[j], l[j]);
    }
    if (whole) {
      *reinterpret_cast<uint4*>(out + at + i0) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(out + plane + at + i0) = *reinterpret_cast<const uint4*>(l);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < left) {
          out[at + i0 + j] = h[j];
          out[plane + at + i0 + j] = l[j];
        }
    }
    if (MODE != kApply && mirror) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < left) {
          out[(c + i0 + j) * p.ld + r] = h[j];
          out[plane + (c + i0 + j) * p.ld + r] = l[j];
        }
    }
  }
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMulThreads, 1)
orth_mul_kernel(const __grid_constant__ MulArgs p, const __grid_constant__ CUtensorMap left,
                const __grid_constant__ CUtensorMap right) {
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  Barriers* s = reinterpret_cast<Barriers*>(raw + (base - smem_u32(raw)) + kStages * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int64_t first = blockIdx.x / 2, step = gridDim.x / 2, total = p.batch * p.per;
  const int blocks = int((p.depth + kDepth - 1) / kDepth);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s->acc_full[i], 1);
      mbar_init(&s->acc_empty[i], 2 * kWriters);
    }
    s->dead = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s->tmem)),
                 "r"(2 * kTile)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_barrier();
  fence_after_sync();
  const uint32_t tmem = s->tmem;
  after_previous();
  let_next_start();

  if (warp == 0 && lane == 0) {
    // Loads of this CTA's halves: 128 rows of the left operand, 128 rows (or
    // columns, kApply) of the right one, hi and lo.
    uint32_t st = 0, phase = 0;
    const uint32_t bytes = 2 * kPlane * (2 + (p.lo_left ? 1 : 0) + (p.lo_right ? 1 : 0));
    for (int64_t t = first; t < total; t += step) {
      int64_t b, tm, tn;
      tile_at<MODE>(p, t, &b, &tm, &tn);
      const int row = int(tm * kTile + rank * 128), col = int(tn * kTile + rank * 128), z = int(b * 2);
      for (int k = 0; k < blocks; ++k) {
        if (!wait_or_die(s, &s->empty[st], phase ^ 1, p.status)) goto done;
        const uint32_t at = base + st * kStageBytes, bar = in_first(&s->full[st]);
        if (rank == 0) mbar_arrive_expect_tx(&s->full[st], bytes);
        for (int pl = 0; pl < 2; ++pl) {
          if (pl == 0 || p.lo_left) load_box(at + pl * kPlane, &left, k * kDepth, row, z + pl, bar);
          if (pl == 0 || p.lo_right) {
            const uint32_t to = at + (2 + pl) * kPlane;
            if (MODE == kApply) {
              load_box(to, &right, col, k * kDepth, z + pl, bar);
              load_box(to + kPlane / 2, &right, col + 64, k * kDepth, z + pl, bar);
            } else {
              load_box(to, &right, k * kDepth, col, z + pl, bar);
            }
          }
        }
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // Until the last MMAs have signalled here, this CTA's memory is needed.
    for (int i = 0; i < kStages; ++i) {
      if (!wait_or_die(s, &s->empty[st], phase ^ 1, p.status)) goto done;
      if (++st == kStages) {
        st = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t idesc = idesc_f16(256, kTile, false, false, MODE == kApply);
    uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
    for (int64_t t = first; t < total; t += step) {
      if (!wait_or_die(s, &s->acc_empty[buf], acc_phase ^ 1, p.status)) goto done;
      const uint32_t d = tmem + buf * kTile;
      for (int k = 0; k < blocks; ++k) {
        if (!wait_or_die(s, &s->full[st], phase, p.status)) goto done;
        fence_after_sync();
        const uint32_t at = base + st * kStageBytes;
#pragma unroll
        for (int kk = 0; kk < kDepth / 16; ++kk) {
          auto L = [&](int pl) { return desc_sw128(at + pl * kPlane + kk * 32, 1024); };
          auto R = [&](int pl) {
            const uint32_t r = at + (2 + pl) * kPlane;
            return MODE == kApply ? desc_sw128_mn(r + kk * 2048) : desc_sw128(r + kk * 32, 1024);
          };
          mma_pair(d, L(0), R(0), idesc, (k | kk) != 0);
          if (p.lo_right) mma_pair(d, L(0), R(1), idesc, 1);
          if (p.lo_left) mma_pair(d, L(1), R(0), idesc, 1);
        }
        commit_pair(&s->empty[st]);
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
      commit_pair(&s->acc_full[buf]);
      buf ^= 1;
      if (buf == 0) acc_phase ^= 1;
    }
  } else if (warp >= 4) {
    uint32_t buf = 0, acc_phase = 0;
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    for (int64_t t = first; t < total; t += step) {
      int64_t b, tm, tn;
      tile_at<MODE>(p, t, &b, &tm, &tn);
      if (!wait_or_die(s, &s->acc_full[buf], acc_phase, p.status)) break;
      __syncwarp();
      fence_after_sync();
      const float sigma = p.sigma ? p.sigma[b] : 1.f / kScale;
      const int64_t r = tm * kTile + rank * 128 + quarter * 32 + lane;
      const int64_t cols = MODE == kApply ? p.n : p.m;
#pragma unroll 1
      for (int c0 = half * (kTile / 2); c0 < (half + 1) * (kTile / 2); c0 += 32) {
        const int64_t c = tn * kTile + c0;
        if (c >= cols) break;
        float v[32];
        tmem_ld32(taddr(tmem, quarter * 32, buf * kTile + c0), v);
        if (r < p.m) write32<MODE>(p, b, r, c, tm != tn, sigma, v);
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(in_first(&s->acc_empty[buf]));
      buf ^= 1;
      if (buf == 0) acc_phase ^= 1;
    }
  }
done:
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  cluster_barrier();
  if (warp == 2) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kTile) : "memory");
  }
}

// steps = 0: the normalised update itself.
__global__ void __launch_bounds__(kPrepThreads)
orth_scale_kernel(const __grid_constant__ PrepArgs p, void* out, int out_dtype, int transposed) {
  after_previous();
  const int64_t i = int64_t(blockIdx.x) * kPrepThreads + threadIdx.x;
  if (i >= p.batch * p.m * p.n) return;
  const int64_t b = i / (p.m * p.n), r = i / p.n % p.m, c = i % p.n;
  const __half* hi = p.x + b * 2 * p.m * p.ld + r * p.ld + c;
  const float x = (__half2float(hi[0]) + __half2float(hi[p.m * p.ld])) * p.sigma[b];
  store_elem(out, b * p.m * p.n + (transposed ? c * p.m + r : r * p.n + c), x, out_dtype);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct OrthLayout {
  int64_t m, n, ldx, lda;
  size_t x, y, A, B, part, sigma, total;
};

OrthLayout layout(const ngdn2_orth_args* a) {
  OrthLayout L;
  L.m = a->rows < a->cols ? a->rows : a->cols;
  L.n = a->rows < a->cols ? a->cols : a->rows;
  L.ldx = (L.n + 7) / 8 * 8;
  L.lda = (L.m + 7) / 8 * 8;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~size_t(255);
    return o;
  };
  L.x = take(size_t(a->batch) * 2 * L.m * L.ldx * 2);
  L.y = take(size_t(a->batch) * 2 * L.m * L.ldx * 2);
  L.A = take(size_t(a->batch) * 2 * L.m * L.lda * 2);
  L.B = take(size_t(a->batch) * 2 * L.m * L.lda * 2);
  L.part = take(size_t(a->batch) * kNormParts * sizeof(double));
  L.sigma = take(size_t(a->batch) * sizeof(float));
  L.total = at + 256;
  return L;
}

PFN_cuTensorMapEncodeTiled encoder() {
  static PFN_cuTensorMapEncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled>(f);
  }();
  return fn;
}

// Planes [batch][2][rows][ld] as boxes of 64 columns by ``box`` rows, 128-byte
// swizzled; zeros outside [rows, cols].
bool make_map(CUtensorMap* map, const __half* p, int64_t batch, int64_t rows, int64_t cols, int64_t ld, int box) {
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch) * 2};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(rows) * ld * 2};
  const cuuint32_t boxes[3] = {kDepth, cuuint32_t(box), 1}, ones[3] = {1, 1, 1};
  return encoder() &&
         encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(p), dims, strides, boxes, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE>
cudaError_t multiply(MulArgs p, const CUtensorMap& left, const CUtensorMap& right, int sms, cudaStream_t st) {
  p.nt = (p.m + kTile - 1) / kTile;
  p.tiles_n = MODE == kApply ? (p.n + kTile - 1) / kTile : p.nt;
  p.per = MODE == kApply ? p.nt * p.tiles_n : p.nt * (p.nt + 1) / 2;
  const cudaError_t e = cudaFuncSetAttribute(orth_mul_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  const int64_t total = p.batch * p.per, pairs = sms / 2;
  return launch_next(orth_mul_kernel<MODE>, dim3(unsigned(2 * (total < pairs ? total : pairs))), dim3(kMulThreads),
                     kSmem, st, true, p, left, right);
}

// The scalar iteration s <- s (a + b s^2 + c s^4) from every start in [0, 1]
// (a grid) has to stay within kMaxSigma, its factor within kMaxFactor.
bool coefficients_ok(const ngdn2_orth_args* a) {
  for (int i = 0; i <= 1024; ++i) {
    double s = i / 1024.0;
    for (int k = 0; k < a->steps; ++k) {
      const double q = s * s, f = a->coef[0] + q * (a->coef[1] + q * a->coef[2]);
      s *= f;
      if (!(fabs(f) <= kMaxFactor && fabs(s) <= kMaxSigma)) return false;
    }
  }
  return true;
}

int validate_orth(const ngdn2_orth_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype)) return NGDN2_ERR_DTYPE;
  if (a->batch < 1 || a->rows < 1 || a->cols < 1 || a->batch > (1 << 20) || a->rows > (1 << 20) ||
      a->cols > (1 << 20) || a->steps < 0 || a->steps > 64 || !(a->eps >= 0.f))
    return NGDN2_ERR_SHAPE;
  if (!coefficients_ok(a)) return NGDN2_ERR_COEFFICIENTS;
  if (!a->update || !a->out || !a->status) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

}  // namespace

extern "C" {

NGDN2_API size_t ngdn2_sizeof_orth_args(void) { return sizeof(ngdn2_orth_args); }

NGDN2_API int ngdn2_orth_workspace_size(const ngdn2_orth_args* a, size_t* bytes) {
  const int rc = validate_orth(a);
  if (rc != NGDN2_OK) return rc;
  if (!bytes) return NGDN2_ERR_NULL;
  *bytes = layout(a).total;
  return NGDN2_OK;
}

NGDN2_API int ngdn2_orth(const ngdn2_orth_args* a, void* stream) {
  const int rc = validate_orth(a);
  if (rc != NGDN2_OK) return rc;
  const OrthLayout L = layout(a);
  if (!a->workspace || a->workspace_bytes < L.total) return NGDN2_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(a->workspace) + 255) & ~uintptr_t(255));
  __half *x = reinterpret_cast<__half*>(ws + L.x), *y = reinterpret_cast<__half*>(ws + L.y);
  __half *A = reinterpret_cast<__half*>(ws + L.A), *B = reinterpret_cast<__half*>(ws + L.B);
  const bool tall = a->rows > a->cols;
  PrepArgs pr;
  pr.g = a->update;
  pr.dtype = a->dtype;
  pr.batch = a->batch;
  pr.m = L.m;
  pr.n = L.n;
  pr.sb = a->update_stride[0];
  pr.sr = a->update_stride[tall ? 2 : 1];
  pr.sc = a->update_stride[tall ? 1 : 2];
  pr.eps = a->eps;
  pr.part = reinterpret_cast<double*>(ws + L.part);
  pr.sigma = reinterpret_cast<float*>(ws + L.sigma);
  pr.x = x;
  pr.ld = L.ldx;
  const int64_t conv = a->batch * ((L.m + kConvTile - 1) / kConvTile) * ((L.n + kConvTile - 1) / kConvTile);
  if (conv >= (int64_t(1) << 31)) return NGDN2_ERR_SHAPE;
  cudaError_t e = launch_next(orth_norm_kernel, dim3(unsigned(a->batch * kNormParts)), dim3(kPrepThreads), 0, st, false, pr);
  if (e == cudaSuccess)
    e = launch_next(orth_convert_kernel, dim3(unsigned(conv)), dim3(kPrepThreads), 0, st, true, pr);
  if (e != cudaSuccess) return NGDN2_ERR_CUDA;
  if (a->steps == 0) {
    const int64_t n = (a->batch * L.m * L.n + kPrepThreads - 1) / kPrepThreads;
    e = launch_next(orth_scale_kernel, dim3(unsigned(n)), dim3(kPrepThreads), 0, st, true, pr, a->out,
                    a->out_dtype, int(tall));
    return e == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
  }
  // Operands: rows of X, A or B (128 rows a box), and X rows along the reduction (64).
  CUtensorMap mx[2], mxr[2], mA, mB;
  if (!make_map(&mx[0], x, a->batch, L.m, L.n, L.ldx, 128) || !make_map(&mx[1], y, a->batch, L.m, L.n, L.ldx, 128) ||
      !make_map(&mxr[0], x, a->batch, L.m, L.n, L.ldx, 64) || !make_map(&mxr[1], y, a->batch, L.m, L.n, L.ldx, 64) ||
      !make_map(&mA, A, a->batch, L.m, L.m, L.lda, 128) || !make_map(&mB, B, a->batch, L.m, L.m, L.lda, 128))
    return NGDN2_ERR_CUDA;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return NGDN2_ERR_CUDA;
  MulArgs p{};
  p.batch = a->batch;
  p.m = L.m;
  p.n = L.n;
  p.a = a->coef[0];
  p.b = a->coef[1];
  p.c = a->coef[2];
  p.out_dtype = a->out_dtype;
  p.transposed = tall;
  p.status = a->status;
  for (int k = 0; k < a->steps && e == cudaSuccess; ++k) {
    const int in = k & 1;
    const bool lo = k > 0 || a->dtype == NGDN2_F32;  // whether X has a lo plane
    p.sigma = k == 0 ? pr.sigma : nullptr;
    p.old = nullptr;
    p.final_out = nullptr;
    p.depth = L.n;
    p.lo_left = p.lo_right = lo;
    p.out = A;
    p.ld = L.lda;
    e = multiply<kGram>(p, mx[in], mx[in], sms, st);
    if (e != cudaSuccess) break;
    p.depth = L.m;
    p.lo_left = p.lo_right = true;
    p.old = A;
    p.out = B;
    e = multiply<kPoly>(p, mA, mA, sms, st);
    if (e != cudaSuccess) break;
    p.old = nullptr;
    p.lo_right = lo;
    p.out = in ? x : y;
    p.ld = L.ldx;
    p.final_out = k + 1 == a->steps ? a->out : nullptr;
    e = multiply<kApply>(p, mB, mxr[in], sms, st);
  }
  return e == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
