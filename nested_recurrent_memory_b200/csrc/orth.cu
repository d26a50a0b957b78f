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
// hi hi + hi lo + lo hi, summed in fp32 (in tensor memory, and in registers from
// 512 terms on): the error of fp32 arithmetic within a factor of ten (4e-6 .. 3e-5
// after five steps, whatever the size) at a third of the tensor cores' rate. A 16-bit
// update fits its hi plane, so the first step needs one product for A and two for X.
// The last step is computed like the others whatever the result's type: a 16-bit
// result is the fp32 one rounded once. (Its hi planes alone would take 13/15 of the
// MMAs, and change bf16 results by as much as their rounding does.)
//
// Matrices of up to 128 rows and about 1500 columns (more for fewer rows) take one
// launch, a CTA or a cluster each (orth_small_kernel). Larger ones: the squared
// norm (partial sums in 64 bits), the conversion to planes, and the products of all
// steps: A = X X^T, B = a I + b A + c A A (both symmetric: the tiles on and above the
// diagonal, written twice) and X' = B X, which reads X as it lies, rows along the
// reduction. The products are cut into tiles, handed out by a counter. For large batches one
// launch does them all, in an order in which every tile's operands come from
// tiles before it: a tile waits until those of its matrix are done, so one
// matrix's next product starts while others' last one still runs. Every wait
// is bounded.
//
// A pair of CTAs computes tiles of 256 rows by 256, 128 or 64 columns (tcgen05,
// cta_group::2; each CTA holds its 128 rows of the left operand and half of
// the right one), fed by a thread that issues TMA loads of 64-deep stages
// ahead, with two accumulators in tensor memory so that one tile's results are
// written while the next is multiplied. The pair tile halves what each
// multiprocessor must read: 64 KB a stage for 12 MMAs of 256 columns. The
// narrower tiles read more for each MMA, but few tiles finish sooner. All
// sum in the same order, so a matrix has the same bits in any batch.

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "tc_ptx.cuh"

using namespace ngdn2;
using namespace ngdn2::tc;

namespace {

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

// Planes hold kScale times the values of A and B, and of X (after the first step)
// where X may reach 1/2. Where it cannot, because |G|_F is far below eps or the
// coefficients shrink it, they hold as many powers of two more: at a fixed scale its
// digits fell below fp16's smallest number (|G|_F = 1e-14, eps = 1e-7: off by 1 %).
constexpr float kScale = 1024.f;

// A bound on a step's X: its Frobenius norm, grown by |a| + |b| s^2 + |c| s^4 a step.
__device__ __forceinline__ float grown(float u, float a, float b, float c) {
  const float q = u * u;
  return u * (fabsf(a) + q * (fabsf(b) + q * fabsf(c)));
}

// The power of two that brings a bound below 1/2 into [1/2, 1), 2^112 at most; 1 for others.
__device__ __forceinline__ float room(float u) {
  const int e = 126 - int(__float_as_uint(u) >> 23);
  return __uint_as_float(uint32_t(127 + (e < 0 ? 0 : e > 112 ? 112 : e)) << 23);
}
// |a + b s^2 + c s^4| and singular values s stay below these (checked on the
// host), so that the planes stay within fp16.
constexpr double kMaxFactor = 60.0, kMaxSigma = 4.0;

// Neighbouring values as words of the two planes.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The sum of both planes.
__device__ __forceinline__ float2 join(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2(h.x + l.x, h.y + l.y);
}

// ---------------------------------------------------------------------------
// Norm and conversion
// ---------------------------------------------------------------------------

// What the CTAs of a launch tell each other, zero at its start.
struct Sync {
  uint32_t units;    // handed out so far
  uint32_t stop;     // a wait gave up
  uint64_t done[1];  // of each matrix: the writing warps' finished units
};
constexpr int kSyncWords = (sizeof(Sync) - 8) / 8;  // before ``done``

constexpr int kPrepThreads = 256, kNormParts = 128;

struct PrepArgs {
  const void* g;
  int64_t batch, m, n;     // X is m x n
  int64_t sb, sr, sc;      // element strides of the update by matrix, row and column of X
  float eps;
  int parts;               // of a matrix's sum of squares, a multiple of 32
  double* part;            // [batch][parts]
  float2* scale;           // [batch][steps] (one at least): X = x * planes, and B X * y gives
                           // the next step's planes, or the result
  int steps;
  float ca, cb, cc;        // coefficients
  __half* x;               // [batch][2][m][ld]; the lo plane only where lo is set
  int64_t ld;
  bool lo;
  uint64_t* sync;          // the products' Sync, cleared here
};

// Sixteen bytes as fp32.
template <int DT>
__device__ __forceinline__ void unpack16(const uint4& t, float* v) {
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == NGDN2_F32) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = DT == NGDN2_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]))
                                        : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// Squares are summed in 64 bits, so neither large nor small updates leave
// the range. FLAT: each matrix lies in one piece on 16-byte boundaries.
template <int DT, bool FLAT>
__global__ void __launch_bounds__(kPrepThreads) orth_norm_kernel(const __grid_constant__ PrepArgs p) {
  __shared__ double red[kPrepThreads / 32];
  const int64_t b = blockIdx.x / p.parts;
  const int part = int(blockIdx.x % p.parts), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0 && part == 0) p.sync[kSyncWords + b] = 0;
  if (threadIdx.x < kSyncWords && blockIdx.x == 0) p.sync[threadIdx.x] = 0;
  double s = 0.0;
  if constexpr (FLAT) {
    constexpr int kPer = DT == NGDN2_F32 ? 4 : 8;
    const int64_t pieces = p.m * p.n / kPer;
    const char* g = static_cast<const char*>(p.g) + b * p.sb * (16 / kPer);
    const int64_t hop = int64_t(p.parts) * kPrepThreads;
#pragma unroll 4
    for (int64_t i = int64_t(part) * kPrepThreads + threadIdx.x; i < pieces; i += hop) {
      float v[8];
      unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(g) + i), v);
#pragma unroll
      for (int j = 0; j < kPer; ++j) s = fma(double(v[j]), double(v[j]), s);
    }
    for (int64_t i = pieces * kPer + threadIdx.x; part == 0 && i < p.m * p.n; i += kPrepThreads) {
      const double x = load_typed<DT>(g, i);
      s = fma(x, x, s);
    }
  } else {
    // Lanes along the dimension with the smaller stride.
    const bool along_c = p.sc <= p.sr;
    const int64_t outer = along_c ? p.m : p.n, inner = along_c ? p.n : p.m;
    const int64_t so = along_c ? p.sr : p.sc, si = along_c ? p.sc : p.sr;
    constexpr int kWarps = kPrepThreads / 32;
    for (int64_t r = int64_t(part) * kWarps + warp; r < outer; r += int64_t(p.parts) * kWarps) {
      const int64_t base = b * p.sb + r * so;
#pragma unroll 8
      for (int64_t c = lane; c < inner; c += 32) {
        const double x = load_typed<DT>(p.g, base + c * si);
        s = fma(x, x, s);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPrepThreads / 32; ++w) s += red[w];
    p.part[b * p.parts + part] = s;
  }
  let_next_start();
}

// What a CTA scales an update by, computed by one of its threads (64-bit square
// roots and divisions by all of them queue up for the few 64-bit units):
// x * s1 * s2, by a power of two that brings the norm into [2^11, 2^12), are the
// planes' values, and sigma times them X_0, whose norm is u. (2^140 at most: it brings
// even the smallest fp32 number into fp16's range, and sigma stays a normal number.)
struct Scale {
  float s1, s2, sigma, u;
  __device__ __forceinline__ void set(double sum, float eps) {
    const double norm = sqrt(sum);
    const bool finite = norm > 0.0 && norm < 1e300;
    int e = 12;
    if (finite) frexp(norm, &e);
    const int k = 12 - e < 140 ? 12 - e : 140;
    s1 = scalbnf(1.f, k / 2);
    s2 = scalbnf(1.f, k - k / 2);
    const double per = 1.0 / (norm + double(eps));
    sigma = float(per / scalbn(1.0, k));
    u = finite ? float(norm * per) : 1.f;
  }
};

__device__ __forceinline__ void norm_scale(const PrepArgs& p, int64_t b, Scale* shared) {
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < p.parts; i += 32) s += p.part[b * p.parts + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) shared->set(s, p.eps);
  }
  __syncthreads();
}

// The planes of X_0 / sigma. ROWS: X's rows lie on 16-byte boundaries in the
// update, and a CTA takes kConvRows of them in pieces of eight; otherwise it
// takes a tile, read along the update's dimension with the smaller stride.
constexpr int kConvTile = 64, kConvRows = 4;

template <int DT, bool ROWS>
__global__ void __launch_bounds__(kPrepThreads) orth_convert_kernel(const __grid_constant__ PrepArgs p) {
  __shared__ float tile[ROWS ? 1 : kConvTile][kConvTile + 1];
  after_previous();
  const int64_t tc = ROWS ? 1 : (p.n + kConvTile - 1) / kConvTile;
  const int64_t tr = ROWS ? (p.m + kConvRows - 1) / kConvRows : (p.m + kConvTile - 1) / kConvTile;
  const int64_t b = blockIdx.x / (tc * tr), q = blockIdx.x % (tc * tr);
  __shared__ Scale scale;
  norm_scale(p, b, &scale);
  if (q == 0 && threadIdx.x == 0) {
    float x = scale.sigma, u = scale.u;
    float2* to = p.scale + b * (p.steps > 0 ? p.steps : 1);
    to[0].x = x;
    for (int k = 0; k < p.steps; ++k) {
      u = grown(u, p.ca, p.cb, p.cc);
      const float more = room(u);
      to[k] = make_float2(x, k + 1 < p.steps ? x * more : x / kScale);
      x = 1.f / (kScale * more);
    }
  }
  const float s1 = scale.s1, s2 = scale.s2;
  __half* hi = p.x + b * 2 * p.m * p.ld;
  __half* lo = hi + p.m * p.ld;
  if constexpr (ROWS) {
    const int64_t r0 = q * kConvRows;
    const int per = int(p.n / 8), rows = int(p.m - r0 < kConvRows ? p.m - r0 : kConvRows);
#pragma unroll 2
    for (int e = threadIdx.x; e < rows * per; e += kPrepThreads) {
      const int r = e / per, c = e % per * 8;
      const int64_t at = b * p.sb + (r0 + r) * p.sr + c;
      float v[8];
      if constexpr (DT == NGDN2_F32) {
        const uint4* g = reinterpret_cast<const uint4*>(static_cast<const float*>(p.g) + at);
        const uint4 t0 = __ldg(g), t1 = __ldg(g + 1);
        unpack16<DT>(t0, v);
        unpack16<DT>(t1, v + 4);
      } else {
        unpack16<DT>(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.g) + at)), v);
      }
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split(v[2 * i] * s1 * s2, v[2 * i + 1] * s1 * s2, h[i], l[i]);
      const int64_t o = (r0 + r) * p.ld + c;
      *reinterpret_cast<uint4*>(hi + o) = make_uint4(h[0], h[1], h[2], h[3]);
      if (p.lo) *reinterpret_cast<uint4*>(lo + o) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  } else {
    const int64_t r0 = q / tc * kConvTile, c0 = q % tc * kConvTile;
    const bool along_c = p.sc <= p.sr;
#pragma unroll 8
    for (int e = threadIdx.x; e < kConvTile * kConvTile; e += kPrepThreads) {
      const int i = e / kConvTile, j = e % kConvTile;
      const int r = along_c ? i : j, c = along_c ? j : i;
      float x = 0.f;
      if (r0 + r < p.m && c0 + c < p.n)
        x = load_typed<DT>(p.g, b * p.sb + (r0 + r) * p.sr + (c0 + c) * p.sc);
      tile[r][c] = x;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kConvTile * kConvTile / 4; e += kPrepThreads) {
      const int r = e / (kConvTile / 4), c = e % (kConvTile / 4) * 4;
      if (r0 + r >= p.m || c0 + c >= p.ld) continue;  // (ld is a multiple of 8)
      uint32_t h[2], l[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) split(tile[r][c + 2 * i] * s1 * s2, tile[r][c + 2 * i + 1] * s1 * s2, h[i], l[i]);
      const int64_t o = (r0 + r) * p.ld + c0 + c;
      *reinterpret_cast<uint2*>(hi + o) = make_uint2(h[0], h[1]);
      if (p.lo) *reinterpret_cast<uint2*>(lo + o) = make_uint2(l[0], l[1]);
    }
  }
  let_next_start();
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

enum { kGram = 0, kPoly = 1, kApply = 2 };  // A = X X^T; B = a I + b A + c A A; X' = B X

constexpr int kRows = 256;            // of a pair's tile
constexpr int kDepth = 64;            // reduction elements of a stage
// Stages whose sum stays in the tensor core's accumulator, which cuts every addition
// off instead of rounding it, so that the error grows with their number; longer sums are
// added up in fp32 registers. (Relative error of a 4096 x 4096 fp32 result: one sum 7.6e-5,
// sums of 16, 8 and 4 stages 2.6e-5, 1.4e-5 and 7.2e-6, fp32 arithmetic 6.5e-6. us a call
// in a row, one sum and sums of 8 stages: 1001 x 345 174 and 177, 1024 x 2816 340 and 354,
// 12 x 1024 x 2816 1757 and 1773.)
constexpr int kRun = 8;
constexpr int kLeft = 128 * kDepth * 2;  // bytes of the left operand's plane in one CTA, a stage

// Tiles of BN columns: a stage holds both operands' planes; as many stages as
// fit beside the results' stage (four at most). The right operand comes in boxes
// of kBoxCols of its columns.
template <int BN>
struct Shape {
  static constexpr int kBoxCols = BN / 2 < 64 ? BN / 2 : 64, kBoxes = BN / 2 / kBoxCols;
  static constexpr int kBox = kBoxCols * kDepth * 2;
  static constexpr int kRight = kBoxes * kBox;
  static constexpr int kStage = 2 * (kLeft + kRight);
  static constexpr int kStages = BN == 256 ? 3 : 4;
};
constexpr int kStagesMost = 4;
constexpr int kMulThreads = 384;      // load, multiply, 2 idle warps, 8 that write results
constexpr int kWriters = 8;
// A writing warp's stage: 32 x 32 results, hi and lo, rows of 64 bytes (64-byte
// swizzle), stored by TMA, which leaves out what lies past the matrix.
constexpr int kOutPlane = 32 * 64, kOutBytes = kWriters * 2 * kOutPlane;
constexpr int kSmem = 3 * 65536 + kOutBytes + 1024 + 256;
static_assert(Shape<256>::kStages * Shape<256>::kStage == 3 * 65536, "");
static_assert(Shape<128>::kStages * Shape<128>::kStage == 3 * 65536, "");
static_assert(Shape<64>::kStages * Shape<64>::kStage <= 3 * 65536, "");

struct MulArgs {
  int64_t batch, m, n;   // X is m x n
  int steps;
  float a, b, c;
  const float2* scale;   // [batch][steps], as PrepArgs has it
  bool x_lo;             // whether the first step's X has a lo plane
  __half *A, *B;         // their planes, rows ld apart
  int64_t ld;
  void* final_out;       // [batch][m][n], or transposed
  int out_dtype, transposed;
  uint32_t first, end;   // the launch's units
  bool wait;             // whether their operands may come from the same launch
  Sync* sync;
  int32_t* status;
};

// X and X' change places every step.
struct Maps {
  CUtensorMap x_left[2], x_right[2], x_out[2], a_left, a_right, a_out, b_left, b_out;
};

struct Barriers {
  uint64_t full[kStagesMost], empty[kStagesMost], acc_full[2], acc_empty[2];
  uint64_t unit_full[2], unit_empty[2];
  uint32_t unit[2];
  uint32_t tmem;
  int dead;
};

// The work of the whole iteration in units, each a tile of one product of one
// matrix; their order is one in which every unit's operands come from units
// before it: by steps, then products, then matrices.
template <int BN>
struct Plan {
  uint32_t sym, app;  // tiles of A or B (those that reach the diagonal or lie above it), and of X'
  uint32_t cols_s, cols_a, per_step, total;
  explicit Plan(const MulArgs& p) {
    const uint32_t rows = uint32_t((p.m + kRows - 1) / kRows);
    cols_s = uint32_t((p.m + BN - 1) / BN);
    cols_a = uint32_t((p.n + BN - 1) / BN);
    sym = rows * cols_s - rows * (rows - 1) / 2 * (kRows / BN);
    app = rows * cols_a;
    per_step = uint32_t(p.batch) * (2 * sym + app);
    total = per_step * uint32_t(p.steps);
  }
};

struct Unit {
  int step, mode;
  int64_t b, tm, tn;
  int blocks;           // of the reduction
  bool lo_left, lo_right;
  bool last;
  uint64_t need;        // of the matrix's finished warps' units, before this one may start
};

template <int BN>
__device__ __forceinline__ Unit unit_at(const MulArgs& p, const Plan<BN>& plan, uint32_t t) {
  Unit u;
  u.step = int(t / plan.per_step);
  uint32_t r = t % plan.per_step;
  const uint32_t s = uint32_t(p.batch) * plan.sym;
  u.mode = r < s ? kGram : r < 2 * s ? kPoly : kApply;
  r -= u.mode * s;
  const uint32_t per = u.mode == kApply ? plan.app : plan.sym;
  u.b = r / per;
  uint32_t q = r % per;
  if (u.mode == kApply) {
    u.tm = q / plan.cols_a;
    u.tn = q % plan.cols_a;
  } else {
    uint32_t row = 0, len = plan.cols_s;
    while (q >= len) {
      q -= len;
      len -= kRows / BN;
      ++row;
    }
    u.tm = row;
    u.tn = row * (kRows / BN) + q;
  }
  u.last = u.step + 1 == p.steps;
  const bool x_lo = u.step > 0 || p.x_lo;
  u.blocks = int(((u.mode == kGram ? p.n : p.m) + kDepth - 1) / kDepth);
  u.lo_left = u.mode != kGram || x_lo;
  u.lo_right = u.mode == kPoly || x_lo;
  u.need = (uint64_t(u.step) * (2 * plan.sym + plan.app) + u.mode * plan.sym) * (2 * kWriters);
  return u;
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
// Descriptor of a right operand that lies rows along the reduction: blocks of
// COLS columns (64: rows of 128 bytes, 128-byte swizzle; 32: half of both)
// ``block`` bytes apart, in groups of 8 rows.
template <int COLS = 64>
__device__ __forceinline__ uint64_t desc_down(uint32_t saddr, uint32_t block) {
  static_assert(COLS == 64 || COLS == 32, "");
  const uint64_t d = desc_sw128(saddr, COLS * 16) & ~(uint64_t(0x3FFF) << 16) & ~(uint64_t(7) << 61);
  return d | uint64_t(block >> 4) << 16 | uint64_t(COLS == 64 ? 2 : 4) << 61;
}

constexpr uint32_t kNone = 0xffffffffu;

// Waits are bounded. One that gives up does so for its CTA, and tells the others.
constexpr uint32_t kPolls = 1u << 23;

__device__ __forceinline__ void give_up(Barriers* s, const MulArgs& p) {
  s->dead = 1;
  atomicExch(&p.sync->stop, 1u);
  atomicOr(p.status, NGDN2_STATUS_WAIT_TIMEOUT);
}

__device__ __forceinline__ bool gone(Barriers* s, const MulArgs& p, uint32_t poll) {
  if (*reinterpret_cast<volatile int*>(&s->dead)) return true;
  if ((poll & 1023) == 1023 && *reinterpret_cast<volatile uint32_t*>(&p.sync->stop)) {
    s->dead = 1;
    return true;
  }
  return false;
}

__device__ __forceinline__ bool wait_or_die(Barriers* s, uint64_t* bar, uint32_t phase, const MulArgs& p) {
  for (uint32_t i = 0; i < kPolls; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (gone(s, p, i)) return false;
  }
  give_up(s, p);
  return false;
}

// For a barrier at which another CTA arrives with data.
__device__ __forceinline__ bool wait_cluster_or_die(Barriers* s, uint64_t* bar, uint32_t phase, const MulArgs& p) {
  for (uint32_t i = 0; i < kPolls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P1;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P1, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, P1;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase)
        : "memory");
    if (ok) return true;
    if (gone(s, p, i)) return false;
  }
  give_up(s, p);
  return false;
}

// What is still under way when a CTA leaves early, waited for with a limit of its own.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t phase, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i)
    if (mbar_try_wait(bar, phase)) return;
}

// Until the matrix's operands of a unit are written; what follows, by whichever
// path it reads, comes after.
__device__ __forceinline__ bool wait_operands(Barriers* s, const MulArgs& p, const Unit& u) {
  const uint64_t* done = p.sync->done + u.b;
  for (uint32_t i = 0; i < kPolls; ++i) {
    uint64_t v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(done) : "memory");
    if (v >= u.need) {
      asm volatile("fence.proxy.async;" ::: "memory");
      return true;
    }
    if (gone(s, p, i)) return false;
  }
  give_up(s, p);
  return false;
}

// The next unit's number: in turn, where no unit waits for another, else from
// the ring that the pair's first CTA fills.
__device__ __forceinline__ bool next_unit(Barriers* s, const MulArgs& p, uint32_t* slot, uint32_t* phase,
                                          uint32_t* t) {
  if (!p.wait) {
    *t = *t == kNone ? p.first + blockIdx.x / 2 : *t + gridDim.x / 2;
    return true;
  }
  if (!wait_cluster_or_die(s, &s->unit_full[*slot], *phase, p)) return false;
  *t = *reinterpret_cast<volatile uint32_t*>(&s->unit[*slot]);
  arrive_at(in_first(&s->unit_empty[*slot]));
  *slot ^= 1;
  if (*slot == 0) *phase ^= 1;
  return true;
}

// Up to eight neighbouring values of one row of the result, ``left`` of them there.
__device__ __forceinline__ void write_final(const MulArgs& p, int64_t b, int64_t r, int64_t c, float s,
                                            const float* v, int left) {
  if (p.transposed) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) store_elem(p.final_out, (b * p.n + c + i) * p.m + r, s * v[i], p.out_dtype);
    return;
  }
  const int64_t o = (b * p.m + r) * p.n + c;
  const int el = p.out_dtype == NGDN2_F32 ? 4 : 2;
  char* to = static_cast<char*>(p.final_out) + o * el;
  if (left >= 8 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
    alignas(16) unsigned char w[32];
#pragma unroll
    for (int j = 0; j < 8; ++j) store_elem(w, j, s * v[j], p.out_dtype);
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(w);
    if (el == 4) reinterpret_cast<uint4*>(to)[1] = *reinterpret_cast<const uint4*>(w + 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) store_elem(p.final_out, o + i, s * v[i], p.out_dtype);
  }
}

// Byte of element (row, col) in a writing warp's stage plane.
__device__ __forceinline__ uint32_t out_at(int row, int col) {
  return row * 64 + (((col >> 3) ^ (row >> 1 & 3)) << 4) + (col & 7) * 2;
}

__device__ __forceinline__ void store_box(const CUtensorMap* map, int c0, int c1, int c2, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(src)
               : "memory");
}

// The stage's planes to the matrix, from row r0 and column c0 on.
__device__ __forceinline__ void store_stage(const CUtensorMap* map, int c0, int r0, int z, uint32_t stage) {
  fence_proxy_async();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    store_box(map, c0, r0, z, stage);
    store_box(map, c0, r0, z + 1, stage + kOutPlane);
    bulk_commit();
  }
}

// Before the stage is written again.
__device__ __forceinline__ void stage_free() {
  if ((threadIdx.x & 31) == 0) bulk_wait_read0();
  __syncwarp();
}

// A unit whose reduction is longer than kRun stages comes in parts, by turns in both
// accumulators. A writing warp adds them up in registers and leaves the sum in
// the last one's place.
template <int BN>
__device__ __forceinline__ bool add_parts(Barriers* s, const MulArgs& p, int parts, uint32_t tmem, uint32_t* buf,
                                          uint32_t* phase) {
  const int quarter = threadIdx.x >> 5 & 3, half = (threadIdx.x >> 7) - 1;
  float sum[BN / 2] = {};
  for (;;) {
    if (!__all_sync(0xffffffffu, wait_or_die(s, &s->acc_full[*buf], *phase, p))) return false;
    fence_after_sync();
    const uint32_t at = taddr(tmem + *buf * BN, quarter * 32, half * (BN / 2));
#pragma unroll
    for (int i = 0; i < BN / 2; i += 16) {
      float v[16];
      tmem_ld16(at + i, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[i + j] += v[j];
    }
    if (--parts == 0) {
#pragma unroll
      for (int i = 0; i < BN / 2; i += 16) tmem_st16(at + i, sum + i);
      tmem_wait_st();
      return true;
    }
    fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) arrive_at(in_first(&s->acc_empty[*buf]));
    *buf ^= 1;
    if (*buf == 0) *phase ^= 1;
  }
}

// A writing warp's part of a unit: 32 rows by BN / 2 columns, sixteen columns at a
// time in a loop that is not unrolled: a launch that writes few tiles finds its
// code cold, and 32 columns spelled out took 15000 cycles of a product's 26000
// (1001 x 345) to be fetched.
template <int MODE, int BN>
__device__ __forceinline__ bool write_unit(Barriers* s, const MulArgs& p, const Unit& u, const CUtensorMap* out,
                                           unsigned char* mem, uint32_t rank, uint32_t tmem, uint32_t* buf,
                                           uint32_t* phase) {
  const int lane = threadIdx.x & 31, quarter = threadIdx.x >> 5 & 3, half = (threadIdx.x >> 7) - 1;
  const int m = int(p.m), cols = int(MODE == kApply ? p.n : p.m), z = int(u.b * 2);
  const int r0 = int(u.tm * kRows + rank * 128 + quarter * 32), r = r0 + lane, c1 = int(u.tn * BN + half * (BN / 2));
  const bool mirror = MODE != kApply && u.tn / (kRows / BN) != u.tm;
  float2 scale = p.scale[u.b * p.steps + u.step];
  // Once a wait of this call has given up, in this launch or an earlier one, operands
  // may be unfinished: nothing made of them passes as a result.
  if (MODE == kApply && u.last && *reinterpret_cast<volatile uint32_t*>(&p.sync->stop))
    scale.y = __int_as_float(0x7fc00000);
  // A's own values for sixteen columns from c on, asked for one turn ahead.
  const __half* old = p.A + (int64_t(z) * m + r) * p.ld;
  uint4 oh[2] = {}, ol[2] = {};
  auto ask = [&](int c) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (r < m && c + 8 * k < m) {  // (a row has room for a multiple of 8)
        oh[k] = __ldcg(reinterpret_cast<const uint4*>(old + c + 8 * k));
        ol[k] = __ldcg(reinterpret_cast<const uint4*>(old + int64_t(m) * p.ld + c + 8 * k));
      }
  };
  const bool early = BN < 256 && !p.wait;  // (else the registers are for the sum)
  if (MODE == kPoly && early) ask(c1);
  const int parts = (u.blocks + kRun - 1) / kRun;
  bool ok = parts > 1 ? add_parts<BN>(s, p, parts, tmem, buf, phase) : wait_or_die(s, &s->acc_full[*buf], *phase, p);
  const uint32_t acc = tmem + *buf * BN;
  // (The product is there, so A is. Only now: eight warps of every CTA that
  // polled for it would hold up those that announce it.)
  if (MODE == kPoly && p.wait && lane == 0) ok = ok && wait_operands(s, p, u);
  if (!__all_sync(0xffffffffu, ok)) return false;
  __syncwarp();
  fence_after_sync();
  if (MODE == kPoly && !early) ask(c1);
  // Below the diagonal lanes are neighbours: two lanes swap values so that each
  // stores two of them, of every other column. (Through the stage as well,
  // each store would wait for the one before.)
  const int odd = lane & 1, even = r - odd;
  __half* below = (MODE == kGram ? p.A : p.B) + (int64_t(z) * m + c1 + odd) * p.ld + even;
  auto swap = [&](uint32_t w) {
    return __byte_perm(w, __shfl_xor_sync(0xffffffffu, w, 1), odd ? 0x3276 : 0x5410);
  };
#pragma unroll 1
  for (int i = 0; i < BN / 2; i += 16) {
    const int c = c1 + i;
    if (c >= cols || r0 >= m) break;
    float v[16];
    __syncwarp();
    tmem_ld16(taddr(acc, quarter * 32, half * (BN / 2) + i), v);
    if (MODE == kApply && u.last) {
      if (r < m) {
        write_final(p, u.b, r, c, scale.y, v, cols - c);
        if (c + 8 < cols) write_final(p, u.b, r, c + 8, scale.y, v + 8, cols - c - 8);
      }
      continue;
    }
    uint32_t h[8], l[8];
    const uint4 ph[2] = {oh[0], oh[1]}, pl[2] = {ol[0], ol[1]};
    if (MODE == kPoly) ask(c + 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x[2] = {v[2 * j], v[2 * j + 1]};
      if (MODE == kGram) {
#pragma unroll
        for (int k = 0; k < 2; ++k) x[k] = x[k] * scale.x * scale.x * kScale;
      } else if (MODE == kPoly) {
        const float2 o = join(reinterpret_cast<const uint32_t*>(ph)[j], reinterpret_cast<const uint32_t*>(pl)[j]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          x[k] = p.c * (x[k] / kScale) + p.b * (k ? o.y : o.x) + (c + 2 * j + k == r ? p.a * kScale : 0.f);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) x[k] *= scale.y;
      }
      split(x[0], x[1], h[j], l[j]);
    }
    if ((i & 31) == 0) stage_free();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t at = out_at(lane, (i & 31) + 8 * j);
      *reinterpret_cast<uint4*>(mem + at) = make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
      *reinterpret_cast<uint4*>(mem + kOutPlane + at) = make_uint4(l[4 * j], l[4 * j + 1], l[4 * j + 2], l[4 * j + 3]);
    }
    if ((i & 31) == 16 || c + 16 >= cols) store_stage(out, c & ~31, r0, z, smem_u32(mem));
    if (mirror) {
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const uint32_t hv = swap(h[j / 2]), lv = swap(l[j / 2]);
        if (even < m && c + j + odd < cols) {  // (a row has room for an even number)
          __half* to = below + int64_t(i + j) * p.ld;
          *reinterpret_cast<uint32_t*>(to) = hv;
          *reinterpret_cast<uint32_t*>(to + int64_t(m) * p.ld) = lv;
        }
      }
    }
  }
  return true;
}

// Pairs of CTAs take units as they come free, one's results written while the
// next is multiplied. In each CTA a thread issues the loads (the first CTA's
// also fetches unit numbers for both) and eight warps write; in the first CTA a
// thread issues the MMAs for both.
// SYM, APP: whether the launch has units of A or B, and of X' (a kernel for all
// takes longer to start: a call of 512 x 4096 321 us with it, 313 with one for each).
template <int BN, bool SYM, bool APP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMulThreads, 1)
orth_steps_kernel(const __grid_constant__ MulArgs p, const __grid_constant__ Plan<BN> plan,
                  const __grid_constant__ Maps maps) {
  constexpr int kStages = Shape<BN>::kStages, kStage = Shape<BN>::kStage, kRight = Shape<BN>::kRight;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* const smem = raw + (base - smem_u32(raw));
  Barriers* s = reinterpret_cast<Barriers*>(smem + kStages * kStage + kOutBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s->acc_full[i], 1);
      mbar_init(&s->acc_empty[i], 2 * kWriters);
      mbar_init(&s->unit_full[i], 1);
      mbar_init(&s->unit_empty[i], 2 + 2 * kWriters);  // multiply, load (second CTA), write
    }
    s->dead = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s->tmem)),
                 "r"(2 * BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_barrier();
  fence_after_sync();
  const uint32_t tmem = s->tmem;
  let_next_start();
  // (Each thread that reads or writes global memory waits for the launches
  // before this one when it comes to that.)
  uint32_t slot = 0, unit_phase = 0, t = kNone;

  if (warp == 0 && lane == 0) {
    // Loads of this CTA's halves: 128 rows of the left operand, BN / 2 rows (or
    // columns, kApply) of the right one, hi and lo. The first CTA's thread also
    // fetches the next unit's number, with its last load of a unit: earlier,
    // and units would wait here while other pairs go idle (2048 x 2048 in one
    // launch took 1.6 times as long with two units fetched ahead).
    uint32_t st = 0, phase = 0;
    auto fetch = [&](uint32_t* next) {
      *next = atomicAdd(&p.sync->units, 1u);
      if (!wait_cluster_or_die(s, &s->unit_empty[slot], unit_phase ^ 1, p)) return false;
      for (uint32_t r = 0; r < 2; ++r) {
        uint32_t at, bar;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&s->unit[slot])), "r"(r));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&s->unit_full[slot])), "r"(r));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(*next) : "memory");
        arrive_at(bar);
      }
      slot ^= 1;
      if (slot == 0) unit_phase ^= 1;
      return true;
    };
    uint32_t next = 0, filled = 0;  // (stages, kStages at most)
    const bool fetches = rank == 0 && p.wait;
    if (p.wait) after_previous();
    bool ok = !fetches || fetch(&next);
    while (ok) {
      if (fetches) t = next;
      else if (!next_unit(s, p, &slot, &unit_phase, &t)) ok = false;
      if (!ok || t >= p.end) break;
      const Unit u = unit_at<BN>(p, plan, t);
      const CUtensorMap* left = u.mode == kGram ? &maps.x_left[u.step & 1] : u.mode == kPoly ? &maps.a_left : &maps.b_left;
      const CUtensorMap* right = u.mode == kPoly ? &maps.a_right : &maps.x_right[u.step & 1];
      const int row = int(u.tm * kRows + rank * 128), col = int(u.tn * BN + rank * (BN / 2)), z = int(u.b * 2);
      const uint32_t bytes = 2 * (kLeft * (u.lo_left ? 2 : 1) + kRight * (u.lo_right ? 2 : 1));
      if (!p.wait) after_previous();
      else ok = wait_operands(s, p, u);
      for (int k = 0; ok && k < u.blocks; ++k) {
        if (fetches && k + 1 == u.blocks) ok = fetch(&next);
        ok = ok && wait_or_die(s, &s->empty[st], phase ^ 1, p);
        if (!ok) break;
        const uint32_t at = base + st * kStage, bar = in_first(&s->full[st]);
        if (rank == 0) mbar_arrive_expect_tx(&s->full[st], bytes);
        for (int pl = 0; pl < 2; ++pl) {
          if (pl == 0 || u.lo_left) load_box(at + pl * kLeft, left, k * kDepth, row, z + pl, bar);
          if (pl == 0 || u.lo_right)
#pragma unroll
            for (int i = 0; i < Shape<BN>::kBoxes; ++i) {
              const uint32_t to = at + 2 * kLeft + pl * kRight + i * Shape<BN>::kBox;
              const int c = col + i * Shape<BN>::kBoxCols;
              if (APP && (!SYM || u.mode == kApply)) load_box(to, right, c, k * kDepth, z + pl, bar);
              else load_box(to, right, k * kDepth, c, z + pl, bar);
            }
        }
        filled += filled < kStages;
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // Until the last MMAs have signalled here, this CTA's memory is needed.
    uint32_t end = st, end_phase = phase;
    for (int i = 0; ok && i < kStages; ++i) {
      ok = wait_or_die(s, &s->empty[end], end_phase ^ 1, p);
      if (++end == kStages) {
        end = 0;
        end_phase ^= 1;
      }
    }
    // Left early: the loads under way, as far as both CTAs' parts of a stage are
    // counted here.
    for (; !ok && rank == 0 && filled > 0; --filled) {
      if (st == 0) {
        st = kStages;
        phase ^= 1;
      }
      drain(&s->full[--st], phase, 1u << 16);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
    uint64_t* last = nullptr;  // signalled by the latest MMAs, in phase last_phase
    uint32_t last_phase = 0;
    bool ok = true;
    for (;;) {
      if (!next_unit(s, p, &slot, &unit_phase, &t) || t >= p.end) break;
      const Unit u = unit_at<BN>(p, plan, t);
      const bool down = APP && (!SYM || u.mode == kApply);
      const uint32_t idesc = idesc_f16(kRows, BN, false, false, down);
      const uint64_t left_desc = desc_sw128(base, 1024), right_step = (down ? Shape<BN>::kBoxCols * 32 : 32) >> 4;
      const uint64_t right_desc = down ? desc_down<Shape<BN>::kBoxCols>(base + 2 * kLeft, Shape<BN>::kBox)
                                       : desc_sw128(base + 2 * kLeft, 1024);
      for (int left = u.blocks; ok && left > 0; left -= kRun) {
        ok = wait_or_die(s, &s->acc_empty[buf], acc_phase ^ 1, p);
        const uint32_t d = tmem + buf * BN;
        const int stages = left < kRun ? left : kRun;
        for (int k = 0; ok && k < stages; ++k) {
          ok = wait_or_die(s, &s->full[st], phase, p);
          if (!ok) break;
          fence_after_sync();
          // Descriptors count 16 bytes: the lo planes and the next 16 of the
          // reduction (32 bytes of a row, or 16 rows) are additions away. One thread
          // issues everything, so what it computes for an MMA must not take
          // longer than the MMA (64 cycles for 128 columns).
          uint64_t dl = left_desc + ((st * kStage) >> 4), dr = right_desc + ((st * kStage) >> 4);
#pragma unroll
          for (int kk = 0; kk < kDepth / 16; ++kk) {
            mma_pair(d, dl, dr, idesc, (k | kk) != 0);
            if (u.lo_right) mma_pair(d, dl, dr + (kRight >> 4), idesc, 1);
            if (u.lo_left) mma_pair(d, dl + (kLeft >> 4), dr, idesc, 1);
            dl += 32 >> 4;
            dr += right_step;
          }
          commit_pair(&s->empty[st]);
          last = &s->empty[st];
          last_phase = phase;
          if (++st == kStages) {
            st = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        commit_pair(&s->acc_full[buf]);
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
      if (!ok) break;
    }
    // (The loads' thread waits for the same, unless it has left early.)
    if (last) drain(last, last_phase, kPolls);
  } else if (warp >= 4) {
    uint32_t buf = 0, acc_phase = 0;
    unsigned char* const mem = smem + kStages * kStage + (warp - 4) * 2 * kOutPlane;
    for (;;) {
      bool ok = true;
      if (lane == 0) ok = next_unit(s, p, &slot, &unit_phase, &t);
      if (!__all_sync(0xffffffffu, ok)) break;
      t = __shfl_sync(0xffffffffu, t, 0);
      if (t >= p.end) break;
      const Unit u = unit_at<BN>(p, plan, t);
      after_previous();
      auto write = [&](auto mode, const CUtensorMap* out) {
        return write_unit<decltype(mode)::value, BN>(s, p, u, out, mem, rank, tmem, &buf, &acc_phase);
      };
      if constexpr (SYM)
        if (u.mode == kGram) ok = write(std::integral_constant<int, kGram>{}, &maps.a_out);
        else if (u.mode == kPoly) ok = write(std::integral_constant<int, kPoly>{}, &maps.b_out);
      if constexpr (APP)
        if (u.mode == kApply) ok = write(std::integral_constant<int, kApply>{}, &maps.x_out[~u.step & 1]);
      if (!__all_sync(0xffffffffu, ok)) break;
      fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        arrive_at(in_first(&s->acc_empty[buf]));
        // All of the warp's results are in memory before the unit counts: its
        // bulk stores are waited for, the others come before the release.
        if (p.wait) bulk_wait0();
        if (p.wait) asm volatile("red.release.gpu.global.add.u64 [%0], %1;" ::"l"(p.sync->done + u.b), "l"(uint64_t(1)) : "memory");
      }
      buf ^= 1;
      if (buf == 0) acc_phase ^= 1;
    }
  }
  if (warp >= 4 && lane == 0) bulk_wait0();
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  // The second CTA's loads signal in the first, which may have left before it
  // counted them: a copy takes microseconds, and this CTA's memory stays that long.
  if (s->dead)
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  cluster_barrier();
  if (warp == 2) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
  }
  if (s->dead) {  // (its units may not have been written at all)
    for (int64_t e = threadIdx.x; e < p.batch * p.m * p.n; e += kMulThreads)
      store_elem(p.final_out, e, __int_as_float(0x7fc00000), p.out_dtype);
  }
}

// ---------------------------------------------------------------------------
// Matrices of m <= 128 and few enough columns: the whole iteration in one launch,
// a cluster of CTAs a matrix, each with a slice of X's columns. X's slice and A
// (then B in its place) stay in shared memory as hi and lo planes in blocks of
// 64 columns, rows of 128 bytes, 128-byte swizzled: as they lie they are left
// and right operands with the reduction along the rows, and X is the right
// operand with the reduction down the columns. A's slices are summed through
// distributed shared memory: every CTA adds up a part of A's rows and gives its
// planes to all. What bounds it is the chain of a step's three
// products, 2.7 us each (16 matrices 128 x 128: 43 us a call in a row), most of it not the
// MMAs but getting the results out of tensor memory and back as operands.
// ---------------------------------------------------------------------------

constexpr int kSmallM = 128, kSmallSlice = 256, kSmallThreads = 512, kSmallCtas = 8;
constexpr int kSmallMost = 227 * 1024 - 512;  // bytes of shared memory

struct SmallArgs {
  PrepArgs in;
  MulArgs out;
  int ctas, slice;  // of a matrix; columns of X a CTA, a multiple of 16
  int rows;         // m up to a multiple of 16
  int part;         // rows of A that a CTA adds up, a multiple of 8
};

// Bytes of a plane's block of 64 columns, of X's and A's planes, of the sums.
struct SmallLayout {
  int block, x_plane, a_plane, sums, total;
  __host__ __device__ explicit SmallLayout(const SmallArgs& q) {
    block = q.rows * 128;
    x_plane = block * ((q.slice + 63) / 64);
    a_plane = block * ((q.rows + 63) / 64);
    sums = q.ctas > 1 ? q.ctas * (q.rows / 4) * (q.part + 1) * 16 : 0;
    // An MMA reads 128 rows, whatever lies there: the last block's reach.
    total = 2 * (x_plane + a_plane) + sums + (128 * 128 - block) + 1024;
  }
};

// As few CTAs as hold the matrix; false where kSmallCtas do not.
bool fits_small(SmallArgs* q, int64_t m, int64_t n) {
  if (m > kSmallM) return false;
  q->rows = int(m + 15) / 16 * 16;
  for (q->ctas = 1; q->ctas <= kSmallCtas; q->ctas *= 2) {
    const int64_t slice = ((n + q->ctas - 1) / q->ctas + 15) / 16 * 16;
    if (slice > kSmallSlice) continue;
    q->slice = int(slice);
    q->part = ((q->rows + q->ctas - 1) / q->ctas + 7) / 8 * 8;
    if (SmallLayout(*q).total <= kSmallMost) return true;
  }
  return false;
}

// Byte of element (r, c) in a plane.
__device__ __forceinline__ uint32_t block_at(int block, int r, int c) {
  return (c >> 6) * block + (r >> 3) * 1024 + (r & 7) * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
}

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}

// Four neighbours that lie on a multiple of four elements.
template <int DT>
__device__ __forceinline__ void load4(const void* p, int64_t at, float* v) {
  if constexpr (DT == NGDN2_F32) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + at));
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
    const uint2 t = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at));
    const uint16_t w[4] = {uint16_t(t.x), uint16_t(t.x >> 16), uint16_t(t.y), uint16_t(t.y >> 16)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load_typed<DT>(w, i);
  }
}

template <int DT>
__global__ void __launch_bounds__(kSmallThreads, 1) orth_small_kernel(const __grid_constant__ SmallArgs q) {
  extern __shared__ unsigned char raw[];
  __shared__ double red[kSmallThreads / 32], slices[kSmallCtas];
  __shared__ Scale scale;
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_at;
  __shared__ int lost;  // a CTA of the cluster gave up
  const PrepArgs& p = q.in;
  const SmallLayout lay(q);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int m = int(p.m), ctas = q.ctas, rank = ctas > 1 ? int(cluster_rank()) : 0;
  const int64_t b = blockIdx.x / ctas, col0 = int64_t(rank) * q.slice;
  const int n = int(p.n - col0 < 0 ? 0 : p.n - col0 < q.slice ? p.n - col0 : q.slice);  // columns here
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* mem = raw + (base - smem_u32(raw));
  const int xp = lay.x_plane, ap = lay.a_plane, block = lay.block;
  unsigned char *mx = mem, *ma = mem + 2 * xp, *ms = ma + 2 * ap;
  const uint32_t ax = base, aa = base + 2 * xp, as = aa + 2 * ap;
  if (tid == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
    lost = 0;
  }
  if (warp == 0) tmem_alloc(&tmem_at, 256);
  for (int i = tid * 16; i < 2 * (xp + ap); i += kSmallThreads * 16)
    *reinterpret_cast<uint4*>(mem + i) = make_uint4(0, 0, 0, 0);
  // The slice, in registers: four neighbours along the dimension with the
  // smaller stride are a piece, all pieces' loads are in flight together (16
  // matrices 128 x 128: 5 us more where the planes' values were read again after
  // the norm).
  const bool along_c = p.sc <= p.sr;
  const int outer = along_c ? m : n, inner = along_c ? n : m;
  const int64_t so = along_c ? p.sr : p.sc, si = along_c ? p.sc : p.sr;
  const int64_t origin = b * p.sb + col0 * p.sc;
  const int log = inner <= 4 ? 0 : 32 - __clz((inner - 1) / 4);  // pieces a row, as a power of two
  constexpr int kPieces = kSmallM * kSmallSlice / 4 / kSmallThreads;
  float x[kPieces][4];
  const bool quads = si == 1 && (so | origin | inner) % 4 == 0 &&
                     reinterpret_cast<uintptr_t>(p.g) % (DT == NGDN2_F32 ? 16 : 8) == 0;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int e = tid + k * kSmallThreads, i = e >> log, j = (e & ((1 << log) - 1)) * 4;
    const int64_t at = origin + i * so + j * si;
    const int left = i < outer ? inner - j : 0;
    if (quads) {
      if (left > 0) load4<DT>(p.g, at, x[k]);
      else x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.f;
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) x[k][u] = u < left ? load_typed<DT>(p.g, at + u * si) : 0.f;
    }
  }
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kPieces; ++k)
#pragma unroll
    for (int u = 0; u < 4; ++u) sum = fma(double(x[k][u]), double(x[k][u]), sum);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  if (ctas > 1) {
    sum = 0.0;
    for (int w = 0; w < kSmallThreads / 32; ++w) sum += red[w];
    if (tid < ctas)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_cta(smem_u32(&slices[rank]), tid)), "d"(sum) : "memory");
    cluster_barrier();
  }
  if (tid == 0) {
    const int parts = ctas > 1 ? ctas : kSmallThreads / 32;
    sum = 0.0;
    for (int i = 0; i < parts; ++i) sum += ctas > 1 ? slices[i] : red[i];
    scale.set(sum, p.eps);
  }
  __syncthreads();
  float sigma = scale.sigma, bound = scale.u;
  const float s1 = scale.s1, s2 = scale.s2;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int e = tid + k * kSmallThreads, i = e >> log, j = (e & ((1 << log) - 1)) * 4;
    const int left = i < outer ? inner - j : 0;
    if (left <= 0) continue;
    uint32_t h[2], l[2];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[k][u] = u < left ? x[k][u] * s1 * s2 : 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) split(x[k][2 * u], x[k][2 * u + 1], h[u], l[u]);
    if (along_c) {
      *reinterpret_cast<uint2*>(mx + block_at(block, i, j)) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2*>(mx + xp + block_at(block, i, j)) = make_uint2(l[0], l[1]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t at = block_at(block, j + u, i);
        *reinterpret_cast<uint16_t*>(mx + at) = uint16_t(h[u / 2] >> (u & 1) * 16);
        *reinterpret_cast<uint16_t*>(mx + xp + at) = uint16_t(l[u / 2] >> (u & 1) * 16);
      }
    }
  }
  const uint32_t tmem = tmem_at;
  const int quarter = warp & 3, c1 = (warp >> 2) * 32, row = quarter * 32 + lane;
  uint32_t phase = 0;
  bool alive = true;

  // D[128 x cols] = L R, reduction over ``depth`` (multiples of 16). After a wait
  // that gave up nothing is multiplied any more, but the cluster goes on
  // together, and learns of it when A's slices are exchanged.
  auto product = [&](uint32_t L, int lp, uint32_t R, int rp, int depth, int cols, bool down) {
    fence_proxy_async();
    fence_before_sync();
    __syncthreads();
    if (!alive) return;
    if (tid == 0) {
      fence_after_sync();
      const uint32_t idesc = idesc_f16(128, cols, false, false, down);
      for (int kk = 0; kk < depth / 16; ++kk) {
        const uint64_t dl = desc_sw128(L + (kk >> 2) * block + (kk & 3) * 32, 1024);
        const uint64_t dr = down ? desc_down(R + kk * 2048, block)
                                 : desc_sw128(R + (kk >> 2) * block + (kk & 3) * 32, 1024);
        mma_f16(tmem, dl, dr, idesc, kk > 0);
        mma_f16(tmem, dl, dr + (rp >> 4), idesc, 1);
        mma_f16(tmem, dl + (lp >> 4), dr, idesc, 1);
      }
      mma_commit(&bar);
    }
    const bool ok = mbar_wait(&bar, phase, 1u << 20);
    phase ^= 1;
    fence_after_sync();
    if (!ok) {
      atomicOr(q.out.status, NGDN2_STATUS_WAIT_TIMEOUT);
      mbar_wait(&bar, phase ^ 1, 1u << 20);  // (once more: nothing is under way when the CTA leaves)
    }
    alive = !__syncthreads_or(!ok);
  };
  // Eight results as planes.
  auto put8 = [&](unsigned char* to, int plane, int c, const float* x) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split(x[2 * j], x[2 * j + 1], h[j], l[j]);
    *reinterpret_cast<uint4*>(to + block_at(block, row, c)) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(to + plane + block_at(block, row, c)) = make_uint4(l[0], l[1], l[2], l[3]);
  };

  const int rows = q.rows, cols = (n + 15) & ~15;
  for (int step = 0; step < q.out.steps; ++step) {
    bound = grown(bound, q.out.a, q.out.b, q.out.c);
    const float more = room(bound);
    float v[32];
    product(ax, xp, ax, xp, cols, rows, false);
    if (ctas == 1) {
      for (int c = c1; c < m; c += 128) {
        tmem_ld32(taddr(tmem, quarter * 32, c), v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c + i < m ? v[i] * sigma * sigma * kScale : 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          if (row < rows && c + i < rows) put8(ma, ap, c + i, v + i);
      }
    } else {
      // By source, four columns of a CTA's rows lie together (and a gap, for the
      // banks): neighbouring lanes send to neighbouring places.
      const int groups = rows / 4, gap = q.part + 1;
      if (c1 < rows) {
        tmem_ld32(taddr(tmem, quarter * 32, c1), v);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = cols > 0 ? v[i] : 0.f;  // (no columns here: nothing was multiplied)
        const uint32_t to = in_cta(as + ((rank * groups + c1 / 4) * gap + row % q.part) * 16, row / q.part);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          if (c1 + i < rows && row < rows)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + i / 4 * gap * 16), "f"(v[i]),
                         "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3])
                         : "memory");
      }
      if (!alive && tid < ctas)
        asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(in_cta(smem_u32(&lost), tid)) : "memory");
      cluster_barrier();
      alive = alive && !*reinterpret_cast<volatile int*>(&lost);
      // Eight columns of a row a thread; eight neighbours' results are 128 bytes.
      for (int e = tid; e < q.part * (rows / 8); e += kSmallThreads) {
        const int g = e % (rows / 8), r = rank * q.part + e / (rows / 8);
        if (r >= rows) break;
        float w[8] = {};
        for (int j = 0; j < ctas; ++j) {
          const unsigned char* f = ms + ((j * groups + 2 * g) * gap + e / (rows / 8)) * 16;
          const float4 f0 = *reinterpret_cast<const float4*>(f), f1 = *reinterpret_cast<const float4*>(f + gap * 16);
          w[0] += f0.x; w[1] += f0.y; w[2] += f0.z; w[3] += f0.w;
          w[4] += f1.x; w[5] += f1.y; w[6] += f1.z; w[7] += f1.w;
        }
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 8 * g + i < m ? w[i] * sigma * sigma * kScale : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) split(w[2 * i], w[2 * i + 1], h[i], l[i]);
        const uint4 hv = make_uint4(h[0], h[1], h[2], h[3]), lv = make_uint4(l[0], l[1], l[2], l[3]);
        const uint32_t at = aa + block_at(block, r, 8 * g);
        for (int j = 0; j < ctas; ++j) {
          const uint32_t to = in_cta(at, j);
          asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(hv.x), "r"(hv.y), "r"(hv.z),
                       "r"(hv.w)
                       : "memory");
          asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + ap), "r"(lv.x), "r"(lv.y),
                       "r"(lv.z), "r"(lv.w)
                       : "memory");
        }
      }
      cluster_barrier();
    }
    product(aa, ap, aa, ap, rows, rows, false);
    for (int c = c1; c < m; c += 128) {
      tmem_ld32(taddr(tmem, quarter * 32, c), v);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        if (row >= rows || c + i >= rows) continue;
        const uint4 h = *reinterpret_cast<const uint4*>(ma + block_at(block, row, c + i));
        const uint4 l = *reinterpret_cast<const uint4*>(ma + ap + block_at(block, row, c + i));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 o = join(reinterpret_cast<const uint32_t*>(&h)[j / 2], reinterpret_cast<const uint32_t*>(&l)[j / 2]);
          v[i + j] = c + i + j < m ? q.out.c * (v[i + j] / kScale) + q.out.b * (j & 1 ? o.y : o.x) +
                                         (c + i + j == row ? q.out.a * kScale : 0.f)
                                   : 0.f;
        }
        put8(ma, ap, c + i, v + i);
      }
    }
    if (cols > 0) product(aa, ap, ax, xp, rows, cols, true);
    // Nothing that was not computed passes as a result. (A CTA that gave up since A was
    // summed has spoilt only its own columns.)
    const float last = alive ? sigma / kScale : __int_as_float(0x7fc00000), next = sigma * more;
    sigma = 1.f / (kScale * more);
    for (int c = c1; c < n; c += 128) {
      tmem_ld32(taddr(tmem, quarter * 32, c), v);
      if (step + 1 == q.out.steps) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          if (row < m && c + i < n) write_final(q.out, b, row, col0 + c + i, last, v + i, n - c - i);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c + i < n ? v[i] * next : 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          if (row < rows && c + i < q.slice) put8(mx, xp, c + i, v + i);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    fence_after_sync();
    tmem_dealloc(tmem, 256);
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
  const float x = (__half2float(hi[0]) + (p.lo ? __half2float(hi[p.m * p.ld]) : 0.f)) * p.scale[b].x;
  store_elem(out, b * p.m * p.n + (transposed ? c * p.m + r : r * p.n + c), x, out_dtype);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

template <class F>
cudaError_t by_type(int dt, F&& f) {
  switch (dt) {
    case NGDN2_BF16: return f(std::integral_constant<int, NGDN2_BF16>{});
    case NGDN2_F16: return f(std::integral_constant<int, NGDN2_F16>{});
    default: return f(std::integral_constant<int, NGDN2_F32>{});
  }
}

struct OrthLayout {
  int64_t m, n, ldx, lda;
  int parts;
  size_t x, y, A, B, part, scale, sync, total;
};

OrthLayout layout(const ngdn2_orth_args* a) {
  OrthLayout L;
  L.m = a->rows < a->cols ? a->rows : a->cols;
  L.n = a->rows < a->cols ? a->cols : a->rows;
  L.ldx = (L.n + 7) / 8 * 8;
  L.lda = (L.m + 7) / 8 * 8;
  L.parts = kNormParts;
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
  L.part = take(size_t(a->batch) * L.parts * sizeof(double));
  L.scale = take(size_t(a->batch) * (a->steps > 0 ? a->steps : 1) * sizeof(float2));
  L.sync = take((kSyncWords + size_t(a->batch)) * sizeof(uint64_t));
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

// Planes [batch][2][rows][ld] as boxes of ``width`` columns by ``box`` rows,
// swizzled over the box's rows (64 columns: 128 bytes, 32: 64); zeros outside
// [rows, cols].
bool make_map(CUtensorMap* map, const __half* p, int64_t batch, int64_t rows, int64_t cols, int64_t ld, int box,
              int width = kDepth) {
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch) * 2};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(rows) * ld * 2};
  const cuuint32_t boxes[3] = {cuuint32_t(width), cuuint32_t(box), 1}, ones[3] = {1, 1, 1};
  return encoder() &&
         encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(p), dims, strides, boxes, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE,
                   width == kDepth ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool SYM, bool APP>
cudaError_t launch_units(MulArgs p, const Maps& maps, uint32_t first, uint32_t n, uint32_t pairs, cudaStream_t st) {
  auto* kernel = orth_steps_kernel<BN, SYM, APP>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  p.first = first;
  p.end = first + n;
  return launch_next(kernel, dim3(2 * (n < pairs ? n : pairs)), dim3(kMulThreads), kSmem, st, true, p, Plan<BN>(p), maps);
}

// The units of one product (of all matrices) of one step.
template <int BN>
cudaError_t launch_product(const MulArgs& p, const Maps& maps, int step, int mode, uint32_t pairs, cudaStream_t st) {
  const Plan<BN> plan(p);
  const uint32_t sym = uint32_t(p.batch) * plan.sym, app = uint32_t(p.batch) * plan.app;
  const uint32_t first = step * plan.per_step + mode * sym;
  return mode == kApply ? launch_units<BN, false, true>(p, maps, first, app, pairs, st)
                        : launch_units<BN, true, false>(p, maps, first, sym, pairs, st);
}

// The tiles' width goes by the rounds that the pairs of CTAs take: one of 128
// columns takes 0.6 of the time of one of 256, one of 64 0.5 (us a call, calls in a
// row, with tiles of 64 columns and without: 1001 x 345 176 and 199, 256 x 512 130 and 149,
// 8 x 256 x 512 141 and 158, 1024 x 2816 355 and 384). An element's sum has the same
// order in all.
constexpr double kTime128 = 0.6, kTime64 = 0.5;

// One launch for all steps where a product of all matrices fills the pairs more
// than once, so that there is always a unit whose operands are ready; otherwise
// a launch for each product, whose start costs less than the signals between
// units (us a call, calls in a row, one launch against one a product: 12 x 1024 x 1024 741
// and 881, 80 x 200 x 264 301 and 372, 26 x 300 x 400 240 and 258; 1024 x 2816 396 and 355,
// 1001 x 345 210 and 176).
cudaError_t launch_steps(MulArgs p, const Maps& maps, const Maps& thin_rows, const Maps& thin_down, uint32_t pairs,
                         cudaStream_t st) {
  const Plan<256> wide(p);
  const Plan<128> narrow(p);
  const Plan<64> thin(p);
  auto rounds = [&](uint32_t tiles) { return double((uint64_t(p.batch) * tiles + pairs - 1) / pairs); };
  p.wait = p.batch > 1 && p.batch * wide.sym > pairs;
  if (p.wait) {
    auto all = [&](uint32_t sym, uint32_t app) { return rounds(sym) * (p.n + p.m) + rounds(app) * p.m; };
    return kTime128 * all(narrow.sym, narrow.app) < all(wide.sym, wide.app)
               ? launch_units<128, true, true>(p, maps, 0, narrow.total, pairs, st)
               : launch_units<256, true, true>(p, maps, 0, wide.total, pairs, st);
  }
  auto product = [&](int step, int mode) {
    const bool app = mode == kApply;
    const double t256 = rounds(app ? wide.app : wide.sym), t128 = kTime128 * rounds(app ? narrow.app : narrow.sym);
    if (kTime64 * rounds(app ? thin.app : thin.sym) < fmin(t128, t256))
      return launch_product<64>(p, app ? thin_down : thin_rows, step, mode, pairs, st);
    return t128 < t256 ? launch_product<128>(p, maps, step, mode, pairs, st)
                       : launch_product<256>(p, maps, step, mode, pairs, st);
  };
  cudaError_t e = cudaSuccess;
  for (int step = 0; step < p.steps; ++step)
    for (int mode = kGram; mode <= kApply && e == cudaSuccess; ++mode) e = product(step, mode);
  return e;
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
  pr.batch = a->batch;
  pr.m = L.m;
  pr.n = L.n;
  pr.sb = a->update_stride[0];
  pr.sr = a->update_stride[tall ? 2 : 1];
  pr.sc = a->update_stride[tall ? 1 : 2];
  pr.eps = a->eps;
  pr.part = reinterpret_cast<double*>(ws + L.part);
  pr.scale = reinterpret_cast<float2*>(ws + L.scale);
  pr.steps = a->steps;
  pr.ca = a->coef[0];
  pr.cb = a->coef[1];
  pr.cc = a->coef[2];
  pr.x = x;
  pr.ld = L.ldx;
  pr.parts = L.parts;
  pr.sync = reinterpret_cast<uint64_t*>(ws + L.sync);
  pr.lo = a->dtype == NGDN2_F32;  // 16-bit updates fit their hi plane
  SmallArgs q{};
  if (a->steps > 0 && fits_small(&q, L.m, L.n)) {
    q.in = pr;
    q.out.m = L.m;
    q.out.n = L.n;
    q.out.steps = a->steps;
    q.out.a = a->coef[0];
    q.out.b = a->coef[1];
    q.out.c = a->coef[2];
    q.out.final_out = a->out;
    q.out.out_dtype = a->out_dtype;
    q.out.transposed = tall;
    q.out.status = a->status;
    const int smem = SmallLayout(q).total;
    const cudaError_t e = by_type(a->dtype, [&](auto T) {
      auto* kernel = orth_small_kernel<decltype(T)::value>;
      const cudaError_t f = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      return f != cudaSuccess ? f
                              : launch_clusters(kernel, dim3(unsigned(a->batch * q.ctas)), dim3(kSmallThreads), smem,
                                                st, q.ctas, q);
    });
    return e == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
  }
  const int64_t el = a->dtype == NGDN2_F32 ? 4 : 2;
  const bool on16 = reinterpret_cast<uintptr_t>(a->update) % 16 == 0 && pr.sb * el % 16 == 0;
  const bool flat = on16 && a->update_stride[2] == 1 && a->update_stride[1] == a->cols;
  const bool rows = on16 && pr.sc == 1 && pr.sr * el % 16 == 0 && L.n % 8 == 0;
  const int64_t conv = a->batch * (rows ? (L.m + kConvRows - 1) / kConvRows
                                        : (L.m + kConvTile - 1) / kConvTile * ((L.n + kConvTile - 1) / kConvTile));
  if (conv >= (int64_t(1) << 31)) return NGDN2_ERR_SHAPE;
  cudaError_t e = by_type(a->dtype, [&](auto T) {
    constexpr int DT = decltype(T)::value;
    const dim3 grid(unsigned(a->batch * L.parts)), block(kPrepThreads);
    const cudaError_t f = launch_next(flat ? orth_norm_kernel<DT, true> : orth_norm_kernel<DT, false>, grid, block, 0, st, false, pr);
    return f != cudaSuccess ? f
                            : launch_next(rows ? orth_convert_kernel<DT, true> : orth_convert_kernel<DT, false>,
                                          dim3(unsigned(conv)), block, 0, st, true, pr);
  });
  if (e != cudaSuccess) return NGDN2_ERR_CUDA;
  if (a->steps == 0) {
    const int64_t n = (a->batch * L.m * L.n + kPrepThreads - 1) / kPrepThreads;
    e = launch_next(orth_scale_kernel, dim3(unsigned(n)), dim3(kPrepThreads), 0, st, true, pr, a->out,
                    a->out_dtype, int(tall));
    return e == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
  }
  // Left operands (128 rows a box), right ones (64, or 32 for thin tiles),
  // results (32 x 32).
  Maps maps;
  const auto of_x = [&](CUtensorMap* map, const __half* q, int box, int width) {
    return make_map(map, q, a->batch, L.m, L.n, L.ldx, box, width);
  };
  const auto of_a = [&](CUtensorMap* map, const __half* q, int box, int width) {
    return make_map(map, q, a->batch, L.m, L.m, L.lda, box, width);
  };
  for (int i = 0; i < 2; ++i)
    if (!of_x(&maps.x_left[i], i ? y : x, 128, kDepth) ||
        !of_x(&maps.x_right[i], i ? y : x, Shape<128>::kBoxCols, kDepth) || !of_x(&maps.x_out[i], i ? y : x, 32, 32))
      return NGDN2_ERR_CUDA;
  if (!of_a(&maps.a_left, A, 128, kDepth) || !of_a(&maps.a_right, A, Shape<128>::kBoxCols, kDepth) ||
      !of_a(&maps.a_out, A, 32, 32) || !of_a(&maps.b_left, B, 128, kDepth) || !of_a(&maps.b_out, B, 32, 32))
    return NGDN2_ERR_CUDA;
  Maps thin_rows = maps, thin_down = maps;  // (for tiles of 64 columns, 32 in each CTA)
  for (int i = 0; i < 2; ++i)
    if (!of_x(&thin_rows.x_right[i], i ? y : x, Shape<64>::kBoxCols, kDepth) ||
        !of_x(&thin_down.x_right[i], i ? y : x, kDepth, Shape<64>::kBoxCols))
      return NGDN2_ERR_CUDA;
  if (!of_a(&thin_rows.a_right, A, Shape<64>::kBoxCols, kDepth)) return NGDN2_ERR_CUDA;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return NGDN2_ERR_CUDA;
  MulArgs p{};
  p.batch = a->batch;
  p.m = L.m;
  p.n = L.n;
  p.steps = a->steps;
  p.a = a->coef[0];
  p.b = a->coef[1];
  p.c = a->coef[2];
  p.scale = pr.scale;
  p.x_lo = pr.lo;
  p.A = A;
  p.B = B;
  p.ld = L.lda;
  p.final_out = a->out;
  p.out_dtype = a->out_dtype;
  p.transposed = tall;
  p.sync = reinterpret_cast<Sync*>(pr.sync);
  p.status = a->status;
  if (double(a->batch) * a->steps * (double(L.m) / 128 + 1) * (double(L.n + L.m) / 64 + 2) >= double(1u << 31))
    return NGDN2_ERR_SHAPE;  // units are counted in 32 bits
  e = launch_steps(p, maps, thin_rows, thin_down, uint32_t(sms / 2), st);
  return e == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
