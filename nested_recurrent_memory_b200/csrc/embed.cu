// Scaled embedding lookup and its gradient:
//   out[n]     = scale * weight[ids[n]]
//   dweight[v] = scale * sum over {n : ids[n] = v} of d_out[n]
// Products and sums in fp32, rounded once to the output's type. Both are bound
// by memory: the lookup reads the rows and writes out; the gradient reads
// d_out once and writes every row of dweight once.
//
// The gradient sorts (token, position) pairs by token with a stable radix
// sort, so that a row's terms are added in the order of their positions and
// the result is reproducible. The sorted list is then cut into chunks of
// equal length, however often a token occurs: a CTA adds up the runs of
// equal tokens in its chunk; a run that lies within the chunk is its row's
// gradient, the parts of one that crosses into other chunks are left in
// fp32 and joined in order afterwards. Rows without a token are zeroed by
// CTAs of the same launch.

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"

using namespace ngdn2;

namespace {

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

__device__ __forceinline__ int64_t load_id(const void* ids, int i32, int64_t n) {
  return i32 ? int64_t(reinterpret_cast<const int32_t*>(ids)[n])
             : reinterpret_cast<const int64_t*>(ids)[n];
}

// W elements of type DT as one access (16 bytes, or a single element).
template <int DT, int W>
struct Pack {
  static constexpr int kEl = DT == NGDN2_F32 ? 4 : 2;
  using T = typename std::conditional<W * kEl == 16, uint4,
                                      typename std::conditional<kEl == 4, uint32_t, uint16_t>::type>::type;
  static __device__ __forceinline__ void unpack(const T& t, float* v) {
    if constexpr (W == 1) {
      v[0] = load_typed<DT>(&t, 0);
    } else if constexpr (DT == NGDN2_F32) {
      v[0] = __uint_as_float(t.x); v[1] = __uint_as_float(t.y);
      v[2] = __uint_as_float(t.z); v[3] = __uint_as_float(t.w);
    } else {
      const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = DT == NGDN2_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]))
                                          : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  static __device__ __forceinline__ T pack(const float* v) {
    T t;
    if constexpr (W == 1) {
      store_elem(&t, 0, v[0], DT);
    } else if constexpr (DT == NGDN2_F32) {
      t = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                     __float_as_uint(v[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == NGDN2_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      t = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return t;
  }
};

// ---------------------------------------------------------------------------
// Lookup
// ---------------------------------------------------------------------------

constexpr int kLookupThreads = 256, kLookupEach = 4;

// A CTA takes ``rows`` tokens as one range of W-element pieces, each thread
// kLookupEach of them at a time with their loads in flight together. A token
// outside [0, V) reads nothing: its row is NaN, so that it cannot pass as a
// result, and the status word says why.
template <int DT, int W>
__global__ void __launch_bounds__(kLookupThreads)
embed_kernel(const __grid_constant__ ngdn2_embed_args a, int rows) {
  using P = Pack<DT, W>;
  using T = typename P::T;
  const uint32_t per = uint32_t(a.D / W);
  const T* weight = static_cast<const T*>(a.weight);
  const int64_t ws = a.weight_stride / W;
  for (int64_t n0 = int64_t(blockIdx.x) * rows; n0 < a.N; n0 += int64_t(gridDim.x) * rows) {
    const uint32_t here = uint32_t(a.N - n0 < rows ? a.N - n0 : rows) * per;
    T* out = static_cast<T*>(a.out) + n0 * per;
    for (uint32_t q0 = threadIdx.x; q0 < here; q0 += kLookupThreads * kLookupEach) {
      T t[kLookupEach];
      bool ok[kLookupEach];
#pragma unroll
      for (int k = 0; k < kLookupEach; ++k) {
        const uint32_t q = q0 + k * kLookupThreads;
        ok[k] = false;
        if (q < here) {
          const uint32_t r = q / per, c = q % per;
          const int64_t v = load_id(a.ids, a.ids_i32, n0 + r);
          ok[k] = v >= 0 && v < a.V;
          if (ok[k]) t[k] = __ldg(weight + v * ws + c);
          else if (c == 0) atomicOr(a.status, NGDN2_STATUS_BAD_INDEX);
        }
      }
#pragma unroll
      for (int k = 0; k < kLookupEach; ++k) {
        const uint32_t q = q0 + k * kLookupThreads;
        float v[W];
        if (ok[k]) P::unpack(t[k], v);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = ok[k] ? a.scale * v[i] : __int_as_float(0x7fc00000);
        if (q < here) out[q] = P::pack(v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Sort of (token, position) by token: stable, kDigitMost bits or fewer a pass,
// the fewest passes and then the fewest bits. Tokens that get no gradient
// (padding, foreign ones) take the value V and come last.
// ---------------------------------------------------------------------------

constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr int kSortEach = 8, kTile = kSortThreads * kSortEach;
constexpr int kDigitMost = 9, kBinsMost = 1 << kDigitMost;

struct SortArgs {
  const void* ids;
  int ids_i32, bits;     // bits of a digit
  int64_t N, V, pad, tiles;
  uint2 *a, *b;          // pairs: sorted ones end in a
  uint32_t* count;       // [tiles][bins]
  uint8_t* present;      // [V + 1]: the token occurs
  int32_t* status;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& s, int64_t n) {
  const int64_t v = load_id(s.ids, s.ids_i32, n);
  if (v < 0 || v >= s.V) {
    atomicOr(s.status, NGDN2_STATUS_BAD_INDEX);
    return uint32_t(s.V);
  }
  return uint32_t(v == s.pad ? s.V : v);
}

// A thread's pairs of tile ``tile``: warp w has 256 in a row, 32 at a time,
// so that rank order is position order.
__device__ __forceinline__ int64_t pair_index(int64_t tile, int k) {
  return tile * kTile + (threadIdx.x >> 5) * (32 * kSortEach) + k * 32 + (threadIdx.x & 31);
}

template <bool FIRST>
__device__ __forceinline__ uint2 load_pair(const SortArgs& s, const uint2* src, int64_t n) {
  if (FIRST) return make_uint2(sort_key(s, n), uint32_t(n));
  return src[n];
}

// Digit counts of every tile; the first pass also clears ``present``.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const __grid_constant__ SortArgs s, const uint2* src, int shift) {
  __shared__ uint32_t bins[kBinsMost];
  const int nb = 1 << s.bits, tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < nb; i += kSortThreads) bins[i] = 0;
  if (!FIRST) after_previous();
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t n = pair_index(blockIdx.x, k);
    const uint32_t d = n < s.N ? load_pair<FIRST>(s, src, n).x >> shift & (nb - 1) : uint32_t(nb);
    const unsigned same = __match_any_sync(0xffffffffu, d);
    if (d < uint32_t(nb) && (same & ((1u << lane) - 1)) == 0) atomicAdd(bins + d, __popc(same));
  }
  __syncthreads();
  for (int i = tid; i < nb; i += kSortThreads) s.count[int64_t(blockIdx.x) * nb + i] = bins[i];
  if (FIRST)
    for (int64_t v = int64_t(blockIdx.x) * kSortThreads + tid; v <= s.V; v += int64_t(gridDim.x) * kSortThreads)
      s.present[v] = 0;
  let_next_start();
}

// Where each of this thread's pairs goes among the tile's pairs of its digit:
// at[k] counts the equal digits before it in its warp; warp_bins[w][d] becomes
// the count of digit d in the warps before w.
__device__ __forceinline__ void rank_pairs(int nb, const uint32_t* digit, uint32_t* at,
                                           uint32_t (*warp_bins)[kBinsMost]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = lane; i < nb; i += 32) warp_bins[warp][i] = 0;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const uint32_t d = digit[k];
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const unsigned before = same & ((1u << lane) - 1);
    uint32_t base = 0;
    if (d < uint32_t(nb)) base = warp_bins[warp][d];
    __syncwarp();
    if (d < uint32_t(nb) && before == 0) warp_bins[warp][d] = base + __popc(same);
    __syncwarp();
    at[k] = base + __popc(before);
  }
  __syncthreads();
  for (int d = tid; d < nb; d += kSortThreads) {
    uint32_t sum = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = warp_bins[w][d];
      warp_bins[w][d] = sum;
      sum += c;
    }
  }
}

// Exclusive prefix of v over the CTA's threads.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < kSortWarps; ++w) before += w < warp ? part[w] : 0;
  return before + x - v;
}

template <bool FIRST, bool LAST>
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const __grid_constant__ SortArgs s, const uint2* src, uint2* dst, int shift) {
  __shared__ uint32_t warp_bins[kSortWarps][kBinsMost];
  __shared__ uint32_t total[kSortThreads], before[kSortThreads], part[kSortWarps], base[kBinsMost];
  const int nb = 1 << s.bits, tid = threadIdx.x;
  after_previous();
  uint2 p[kSortEach];
  uint32_t digit[kSortEach], at[kSortEach];
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t n = pair_index(blockIdx.x, k);
    p[k] = n < s.N ? load_pair<FIRST>(s, src, n) : make_uint2(0, 0);
    digit[k] = n < s.N ? p[k].x >> shift & (nb - 1) : uint32_t(nb);
  }
  // Pairs of smaller digits, and of this digit in earlier tiles: threads of
  // one digit share the tiles.
  const int d = tid & (nb - 1), share = kSortThreads / nb, first = tid / nb;
  uint32_t all = 0, earlier = 0;
#pragma unroll 8
  for (int64_t t = first; t < s.tiles; t += share) {
    const uint32_t c = s.count[t * nb + d];
    all += c;
    earlier += t < blockIdx.x ? c : 0;
  }
  total[tid] = all;
  before[tid] = earlier;
  rank_pairs(nb, digit, at, warp_bins);
  __syncthreads();
  all = earlier = 0;
  if (tid < nb)
    for (int i = 0; i < share; ++i) {
      all += total[tid + i * nb];
      earlier += before[tid + i * nb];
    }
  const uint32_t smaller = block_prefix(tid < nb ? all : 0, part);
  if (tid < nb) base[tid] = smaller + earlier;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortEach; ++k)
    if (digit[k] < uint32_t(nb)) {
      dst[base[digit[k]] + warp_bins[tid >> 5][digit[k]] + at[k]] = p[k];
      if (LAST) s.present[p[k].x] = 1;
    }
  let_next_start();
}

// All passes for up to one tile of pairs, in one CTA.
__global__ void __launch_bounds__(kSortThreads)
sort_small_kernel(const __grid_constant__ SortArgs s, int passes) {
  extern __shared__ __align__(16) unsigned char sort_smem[];
  uint32_t(*warp_bins)[kBinsMost] = reinterpret_cast<uint32_t(*)[kBinsMost]>(sort_smem);
  uint2* pairs = reinterpret_cast<uint2*>(sort_smem + sizeof(uint32_t) * kSortWarps * kBinsMost);
  __shared__ uint32_t part[kSortWarps], base[kBinsMost];
  const int nb = 1 << s.bits, tid = threadIdx.x;
  for (int64_t v = tid; v <= s.V; v += kSortThreads) s.present[v] = 0;
  uint2 p[kSortEach];
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t n = pair_index(0, k);
    p[k] = n < s.N ? load_pair<true>(s, nullptr, n) : make_uint2(0, 0);
  }
  for (int pass = 0; pass < passes; ++pass) {
    uint32_t digit[kSortEach], at[kSortEach];
#pragma unroll
    for (int k = 0; k < kSortEach; ++k)
      digit[k] = pair_index(0, k) < s.N ? p[k].x >> (pass * s.bits) & (nb - 1) : uint32_t(nb);
    rank_pairs(nb, digit, at, warp_bins);
    // The last warp's pairs add to the counts before it: the digit's total.
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; ++k) at[k] += digit[k] < uint32_t(nb) ? warp_bins[tid >> 5][digit[k]] : 0;
    __syncthreads();
    for (int i = tid; i < nb; i += kSortThreads) base[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; ++k)
      if (digit[k] < uint32_t(nb)) atomicMax(base + digit[k], at[k] + 1);
    __syncthreads();
    const uint32_t count = tid < nb ? base[tid] : 0;
    const uint32_t smaller = block_prefix(count, part);
    if (tid < nb) base[tid] = smaller;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; ++k)
      if (digit[k] < uint32_t(nb)) pairs[base[digit[k]] + at[k]] = p[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortEach; ++k) {
      const int64_t n = pair_index(0, k);
      if (n < s.N) p[k] = pairs[n];
    }
  }
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t n = pair_index(0, k);
    if (n < s.N) {
      s.a[n] = p[k];
      s.present[p[k].x] = 1;
    }
  }
  let_next_start();
}

// ---------------------------------------------------------------------------
// Sums over the sorted list
// ---------------------------------------------------------------------------

constexpr int kSumThreads = 128, kSumAhead = 8;
constexpr int kChunkMost = 64, kZeroRows = 16;

struct SumArgs {
  const uint2* pairs;
  const uint8_t* present;
  const void* d_out;
  void* dweight;
  float* part;          // [chunks][2][D]: a chunk's part of the run that came in, of the one that goes on
  int64_t N, V, D, d_stride, chunks;
  int chunk;
  float scale;
};

// Column blocks of kSumThreads * W in grid.y; in grid.x the chunks, then the
// rows to be zeroed.
template <int DT, int OT, int W>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const __grid_constant__ SumArgs s) {
  using P = Pack<DT, W>;
  using PO = Pack<OT, W>;
  constexpr bool kPackOut = W == 1 || DT == OT;  // else element by element
  __shared__ uint2 list[kChunkMost + 2];
  const int tid = threadIdx.x;
  const int64_t col = (int64_t(blockIdx.y) * kSumThreads + tid) * W;
  auto write = [&](int64_t v, const float* x) {
    if constexpr (kPackOut) {
      reinterpret_cast<typename PO::T*>(s.dweight)[(v * s.D + col) / W] = PO::pack(x);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) store_elem(s.dweight, v * s.D + col + i, x[i], OT);
    }
  };
  after_previous();
  if (blockIdx.x >= s.chunks) {
    const int64_t v0 = (int64_t(blockIdx.x) - s.chunks) * kZeroRows;
    if (col < s.D) {
      float zero[W] = {};
      for (int r = 0; r < kZeroRows; ++r)
        if (v0 + r < s.V && !s.present[v0 + r]) write(v0 + r, zero);
    }
    let_next_start();
    return;
  }
  const int64_t i0 = int64_t(blockIdx.x) * s.chunk;
  const int len = int(s.N - i0 < s.chunk ? s.N - i0 : s.chunk);
  const uint32_t none = 0xffffffffu;
  // list[1 ..]: the chunk, with its neighbours on both sides.
  for (int i = tid; i < len + 2; i += kSumThreads) {
    const int64_t n = i0 + i - 1;
    list[i] = n >= 0 && n < s.N ? s.pairs[n] : make_uint2(none, 0);
  }
  __syncthreads();
  let_next_start();
  if (col >= s.D) return;
  const typename P::T* d_out = static_cast<const typename P::T*>(s.d_out) + col / W;
  const int64_t ds = s.d_stride / W;
  float acc[W] = {};
  bool came_in = list[0].x == list[1].x;
  for (int j0 = 0; j0 < len; j0 += kSumAhead) {
    typename P::T t[kSumAhead];
#pragma unroll
    for (int j = 0; j < kSumAhead; ++j)
      if (j0 + j < len && list[1 + j0 + j].x < uint32_t(s.V))
        t[j] = __ldg(d_out + list[1 + j0 + j].y * ds);
#pragma unroll
    for (int j = 0; j < kSumAhead; ++j) {
      if (j0 + j >= len) break;
      const uint32_t v = list[1 + j0 + j].x, after = list[2 + j0 + j].x;
      if (v >= uint32_t(s.V)) return;  // only tokens without a gradient from here on
      float x[W];
      P::unpack(t[j], x);
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] += x[i];
      const bool last = j0 + j + 1 == len;
      if (after != v || last) {
        const bool goes_on = after == v;
        if (came_in || goes_on) {
          float* to = s.part + (int64_t(blockIdx.x) * 2 + (came_in ? 0 : 1)) * s.D + col;
#pragma unroll
          for (int i = 0; i < W; ++i) to[i] = acc[i];
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) acc[i] *= s.scale;
          write(v, acc);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = 0.f;
        came_in = false;
      }
    }
  }
}

// The rows whose runs cross chunks: the CTA of the chunk in which a run
// starts adds up its parts, eight warps every eighth chunk, and then the
// warps' sums, in order. 32 columns a CTA.
constexpr int kJoinWarps = 8;

template <int OT>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ SumArgs s) {
  __shared__ float sums[kJoinWarps][32];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x, i0 = c * s.chunk, i1 = i0 + s.chunk;
  if (i1 >= s.N) return;
  const uint32_t v = s.pairs[i1 - 1].x;
  if (v >= uint32_t(s.V) || s.pairs[i1].x != v) return;
  if (s.pairs[i0].x == v && i0 > 0 && s.pairs[i0 - 1].x == v) return;  // it started earlier
  // How many further chunks it reaches.
  int64_t more = 0;
  for (;;) {
    const int64_t at = (c + 1 + more + threadIdx.x) * s.chunk;
    const int n = __syncthreads_count(at < s.N && s.pairs[at].x == v);
    more += n;
    if (n < int(blockDim.x)) break;
  }
  for (int64_t d0 = int64_t(blockIdx.y) * 32; d0 < s.D; d0 += int64_t(gridDim.y) * 32) {
    const int64_t d = d0 + lane;
    float x = 0.f;
    if (d < s.D) {
#pragma unroll 8
      for (int64_t k = warp; k <= more; k += kJoinWarps)
        x += s.part[((c + k) * 2 + (k == 0 ? 1 : 0)) * s.D + d];
    }
    sums[warp][lane] = x;
    __syncthreads();
    if (warp == 0 && d < s.D) {
      x = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) x += sums[w][lane];
      store_elem(s.dweight, v * s.D + d, s.scale * x, OT);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

int validate_embed(const ngdn2_embed_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype)) return NGDN2_ERR_DTYPE;
  if (a->N < 0 || a->V < 1 || a->D < 1 || a->N >= (int64_t(1) << 31) ||
      a->V >= (int64_t(1) << 31) - 1 || a->D >= (int64_t(1) << 24) || a->weight_stride < 0)
    return NGDN2_ERR_SHAPE;
  if (!a->weight || !a->status || (a->N > 0 && (!a->ids || !a->out))) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

int validate_embed_bwd(const ngdn2_embed_bwd_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype)) return NGDN2_ERR_DTYPE;
  if (a->N < 0 || a->V < 1 || a->D < 1 || a->N >= (int64_t(1) << 31) ||
      a->V >= (int64_t(1) << 31) - 1 || a->D >= (int64_t(1) << 22) || a->d_stride < 0)
    return NGDN2_ERR_SHAPE;
  if (!a->dweight || !a->status || (a->N > 0 && (!a->ids || !a->d_out))) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

struct BwdPlan {
  int bits, passes, chunk;
  int64_t tiles, chunks;
  size_t a, b, count, present, part, total;
};

BwdPlan plan_bwd(const ngdn2_embed_bwd_args* a) {
  BwdPlan p{};
  int bits = 1;
  while ((a->V >> bits) > 0) ++bits;  // of the values 0 .. V
  p.passes = (bits + kDigitMost - 1) / kDigitMost;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tiles = (a->N + kTile - 1) / kTile;
  // Chunks short enough for a few CTAs a multiprocessor, long enough to leave
  // few parts of hot tokens.
  p.chunk = a->N <= 16384 ? 16 : kChunkMost;
  p.chunks = (a->N + p.chunk - 1) / p.chunk;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~size_t(255);
    return o;
  };
  p.a = take(size_t(a->N) * 8);
  p.b = take(p.tiles > 1 ? size_t(a->N) * 8 : 0);
  p.count = take(p.tiles > 1 ? size_t(p.tiles) << p.bits << 2 : 0);
  p.present = take(size_t(a->V) + 1);
  p.part = take(size_t(p.chunks) * 2 * size_t(a->D) * 4);
  p.total = at + 256;
  return p;
}

cudaError_t sort_pairs(const SortArgs& s, int passes, cudaStream_t st) {
  if (s.tiles <= 1) {
    constexpr size_t smem = sizeof(uint32_t) * kSortWarps * kBinsMost + sizeof(uint2) * kTile;
    const cudaError_t e = cudaFuncSetAttribute(sort_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    return launch_next(sort_small_kernel, dim3(1), dim3(kSortThreads), smem, st, false, s, passes);
  }
  const dim3 grid(unsigned(s.tiles)), block(kSortThreads);
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < passes && e == cudaSuccess; ++pass) {
    // The last pass writes to a.
    uint2* dst = (passes - 1 - pass) % 2 == 0 ? s.a : s.b;
    const uint2* src = dst == s.a ? s.b : s.a;
    const int shift = pass * s.bits;
    const bool last = pass + 1 == passes;
    e = pass == 0 ? launch_next(sort_count_kernel<true>, grid, block, 0, st, false, s, src, shift)
                  : launch_next(sort_count_kernel<false>, grid, block, 0, st, true, s, src, shift);
    if (e != cudaSuccess) break;
    if (pass == 0)
      e = last ? launch_next(sort_place_kernel<true, true>, grid, block, 0, st, true, s, src, dst, shift)
               : launch_next(sort_place_kernel<true, false>, grid, block, 0, st, true, s, src, dst, shift);
    else
      e = last ? launch_next(sort_place_kernel<false, true>, grid, block, 0, st, true, s, src, dst, shift)
               : launch_next(sort_place_kernel<false, false>, grid, block, 0, st, true, s, src, dst, shift);
  }
  return e;
}

template <class F>
cudaError_t by_type(int dt, F&& f) {
  switch (dt) {
    case NGDN2_BF16: return f(std::integral_constant<int, NGDN2_BF16>{});
    case NGDN2_F16: return f(std::integral_constant<int, NGDN2_F16>{});
    default: return f(std::integral_constant<int, NGDN2_F32>{});
  }
}

// Whether rows of D elements at this pointer and row stride can be moved 16 bytes at a time.
bool rows16(const void* p, int dt, int64_t stride, int64_t D) {
  const int64_t el = dt == NGDN2_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * el % 16 == 0 && D * el % 16 == 0;
}

}  // namespace

extern "C" {

NGDN2_API size_t ngdn2_sizeof_embed_args(void) { return sizeof(ngdn2_embed_args); }
NGDN2_API size_t ngdn2_sizeof_embed_bwd_args(void) { return sizeof(ngdn2_embed_bwd_args); }

NGDN2_API int ngdn2_embed(const ngdn2_embed_args* a, void* stream) {
  const int rc = validate_embed(a);
  if (rc != NGDN2_OK) return rc;
  if (a->N == 0) return NGDN2_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = rows16(a->weight, a->dtype, a->weight_stride, a->D) &&
                    rows16(a->out, a->dtype, a->D, a->D);
  const cudaError_t err = by_type(a->dtype, [&](auto T) {
    constexpr int DT = decltype(T)::value, W = DT == NGDN2_F32 ? 4 : 8;
    const int64_t per = wide ? a->D / W : a->D;
    // As many rows a CTA as fill its threads' pieces, but few enough that a
    // small batch spreads over the GPU.
    int64_t rows = (kLookupThreads * kLookupEach + per - 1) / per;
    while (rows > 1 && a->N / rows < 296) rows = (rows + 1) / 2;
    const int64_t ctas = (a->N + rows - 1) / rows;
    const dim3 grid(unsigned(ctas < (1 << 24) ? ctas : (1 << 24)));
    return wide ? launch_next(embed_kernel<DT, W>, grid, dim3(kLookupThreads), 0, st, false, *a, int(rows))
                : launch_next(embed_kernel<DT, 1>, grid, dim3(kLookupThreads), 0, st, false, *a, int(rows));
  });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_embed_bwd_workspace_size(const ngdn2_embed_bwd_args* a, size_t* bytes) {
  const int rc = validate_embed_bwd(a);
  if (rc != NGDN2_OK) return rc;
  if (!bytes) return NGDN2_ERR_NULL;
  *bytes = a->N == 0 ? 0 : plan_bwd(a).total;
  return NGDN2_OK;
}

NGDN2_API int ngdn2_embed_bwd(const ngdn2_embed_bwd_args* a, void* stream) {
  const int rc = validate_embed_bwd(a);
  if (rc != NGDN2_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->N == 0) {
    const size_t bytes = size_t(a->V) * size_t(a->D) * (a->out_dtype == NGDN2_F32 ? 4 : 2);
    return cudaMemsetAsync(a->dweight, 0, bytes, st) == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
  }
  const BwdPlan p = plan_bwd(a);
  if (!a->workspace || a->workspace_bytes < p.total) return NGDN2_ERR_WORKSPACE;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(a->workspace) + 255) & ~uintptr_t(255));
  SortArgs so;
  so.ids = a->ids;
  so.ids_i32 = a->ids_i32;
  so.bits = p.bits;
  so.N = a->N;
  so.V = a->V;
  so.pad = a->padding_idx;
  so.tiles = p.tiles;
  so.a = reinterpret_cast<uint2*>(ws + p.a);
  so.b = reinterpret_cast<uint2*>(ws + p.b);
  so.count = reinterpret_cast<uint32_t*>(ws + p.count);
  so.present = reinterpret_cast<uint8_t*>(ws + p.present);
  so.status = a->status;
  SumArgs su;
  su.pairs = so.a;
  su.present = so.present;
  su.d_out = a->d_out;
  su.dweight = a->dweight;
  su.part = reinterpret_cast<float*>(ws + p.part);
  su.N = a->N;
  su.V = a->V;
  su.D = a->D;
  su.d_stride = a->d_stride;
  su.chunks = p.chunks;
  su.chunk = p.chunk;
  su.scale = a->scale;
  const int64_t ctas = p.chunks + (a->V + kZeroRows - 1) / kZeroRows;
  if (ctas >= (int64_t(1) << 31)) return NGDN2_ERR_SHAPE;
  cudaError_t err = sort_pairs(so, p.passes, st);
  if (err != cudaSuccess) return NGDN2_ERR_CUDA;
  const bool wide = rows16(a->d_out, a->dtype, a->d_stride, a->D) &&
                    (a->dtype != a->out_dtype || rows16(a->dweight, a->out_dtype, a->D, a->D));
  err = by_type(a->dtype, [&](auto T) {
    return by_type(a->out_dtype, [&](auto O) {
      constexpr int DT = decltype(T)::value, OT = decltype(O)::value, W = DT == NGDN2_F32 ? 4 : 8;
      const int64_t block = int64_t(kSumThreads) * (wide ? W : 1);
      const dim3 grid(unsigned(ctas), unsigned((a->D + block - 1) / block));
      return wide ? launch_next(sum_kernel<DT, OT, W>, grid, dim3(kSumThreads), 0, st, true, su)
                  : launch_next(sum_kernel<DT, OT, 1>, grid, dim3(kSumThreads), 0, st, true, su);
    });
  });
  if (err != cudaSuccess) return NGDN2_ERR_CUDA;
  if (p.chunks > 1)
    err = by_type(a->out_dtype, [&](auto O) {
      const int64_t cols = (a->D + 31) / 32;
      return launch_next(join_kernel<decltype(O)::value>, dim3(unsigned(p.chunks - 1), unsigned(cols < 64 ? cols : 64)),
                         dim3(32 * kJoinWarps), 0, st, true, su);
    });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
