// Scaled embedding lookup and its gradient:
//   out[n]     = scale * weight[ids[n]]
//   dweight[v] = scale * sum over {n : ids[n] = v} of d_out[n]
// Products and sums in fp32, rounded once to the output's type. Both are bound
// by memory: the lookup reads the rows and writes out; the gradient reads
// d_out once and writes every row of dweight once.
//
// The gradient sorts (token, position) pairs by token with a stable radix
// sort (in one launch by a cluster up to 16384 tokens), so that a row's terms lie
// in the order of their positions. The sorted list is then cut into chunks of
// equal length, however often a token occurs: a CTA adds up the runs of
// equal tokens in its chunk, in order; a run that lies within the chunk is its row's
// gradient, the parts of one that crosses into other chunks are left in
// fp32 and joined afterwards: every fourth part by one of four warps, then the
// warps' sums. So the order of a row's additions follows from the tokens and N alone,
// and the result is reproducible. A short list's sort keeps few multiprocessors
// busy; the others meanwhile zero dweight's last rows, whether they have
// tokens or not, as far as its time goes. Other rows without a token are
// zeroed by CTAs of the launch that sums.

#include <cooperative_groups.h>

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

// Stores that leave L2 to the table.
template <class T>
__device__ __forceinline__ void store_stream(T* p, const T& t) { __stcs(p, t); }
__device__ __forceinline__ void store_stream(uint16_t* p, const uint16_t& t) {
  __stcs(reinterpret_cast<unsigned short*>(p), t);
}

constexpr int kLookupThreads = 256, kLookupEach = 2;

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
        if (q < here) store_stream(out + q, P::pack(v));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Sort of (token, position) by token: stable, kDigitMost bits or fewer a pass,
// the fewest passes and then the fewest bits. Tokens that get no gradient
// (padding, foreign ones) take the value V and come last.
// ---------------------------------------------------------------------------

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
// Pairs a thread has of its tile. One up to kFewTokens: small tiles spread the
// scattered stores over the GPU; beyond, eight keep the tiles' counts few.
constexpr int kManyEach = 8;
constexpr int64_t kFewTokens = 256 * kSortThreads;
constexpr int kDigitMost = 9, kBinsMost = 1 << kDigitMost;

struct SortArgs {
  const void* ids;
  int ids_i32, bits;     // bits of a digit
  int64_t N, V, pad, tiles;
  uint2 *a, *b;          // pairs: sorted ones end in a
  uint32_t* count;       // [bins][tiles], then [bins]: the tiles' digit counts, all tiles'
  uint32_t* crossing;    // how many runs cross chunks, then their first chunks
  char* zero;            // the part of dweight to be zeroed beside the sort
  int64_t zero_bytes;
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

// A thread's pairs of tile ``tile``: a warp has 32 * EACH in a row, 32 at a
// time, so that rank order is position order.
template <int EACH>
__device__ __forceinline__ int64_t pair_index(int64_t tile, int k) {
  return tile * (kSortThreads * EACH) + (threadIdx.x >> 5) * (32 * EACH) + k * 32 + (threadIdx.x & 31);
}

template <bool FIRST>
__device__ __forceinline__ uint2 load_pair(const SortArgs& s, const uint2* src, int64_t n) {
  if (FIRST) return make_uint2(sort_key(s, n), uint32_t(n));
  return src[n];
}

// Digit counts of every tile.
template <bool FIRST, int EACH>
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const __grid_constant__ SortArgs s, const uint2* src, int shift) {
  __shared__ uint32_t bins[kBinsMost];
  const int nb = 1 << s.bits, tid = threadIdx.x;
  for (int i = tid; i < nb; i += kSortThreads) bins[i] = 0;
  if (!FIRST) after_previous();
  __syncthreads();
  uint32_t d[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t n = pair_index<EACH>(blockIdx.x, k);
    d[k] = n < s.N ? load_pair<FIRST>(s, src, n).x >> shift & (nb - 1) : uint32_t(nb);
  }
#pragma unroll
  for (int k = 0; k < EACH; ++k)
    if (d[k] < uint32_t(nb)) atomicAdd(bins + d[k], 1u);
  __syncthreads();
  for (int i = tid; i < nb; i += kSortThreads) s.count[int64_t(i) * s.tiles + blockIdx.x] = bins[i];
  if (FIRST && blockIdx.x == 0 && tid == 0) s.crossing[0] = 0;
  let_next_start();
}

// Each digit's counts become the counts of the tiles before; a warp a digit.
constexpr int kPrefixThreads = 128;

__global__ void __launch_bounds__(kPrefixThreads) sort_prefix_kernel(const __grid_constant__ SortArgs s) {
  const int lane = threadIdx.x & 31, d = blockIdx.x * (kPrefixThreads / 32) + (threadIdx.x >> 5);
  const int nb = 1 << s.bits;
  after_previous();
  let_next_start();
  if (d >= nb) return;
  uint32_t* row = s.count + int64_t(d) * s.tiles;
  uint32_t sum = 0;
  for (int64_t t0 = 0; t0 < s.tiles; t0 += 128) {
    uint32_t c[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = x[i] = t0 + 32 * i + lane < s.tiles ? row[t0 + 32 * i + lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x[i], o);
        if (lane >= o) x[i] += y;
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t0 + 32 * i + lane < s.tiles) row[t0 + 32 * i + lane] = sum + x[i] - c[i];
      sum += __shfl_sync(0xffffffffu, x[i], 31);
    }
  }
  if (lane == 0) s.count[nb * s.tiles + d] = sum;
}

// The lanes whose digit equals this lane's: one vote a bit.
__device__ __forceinline__ unsigned equal_lanes(uint32_t d, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b <= bits; ++b) {  // bit ``bits`` marks pairs past the end
    const unsigned v = __ballot_sync(0xffffffffu, d >> b & 1);
    same &= d >> b & 1 ? v : ~v;
  }
  return same;
}

// Where each of this thread's pairs goes among the tile's pairs of its digit:
// at[k] counts the equal digits before it in its warp; bins[w][d] becomes the
// count of digit d in the warps before w, totals[d] that in all (unless NULL).
template <int EACH>
__device__ __forceinline__ void rank_pairs(int bits, const uint32_t* digit, uint32_t* at,
                                           uint16_t (*bins)[kBinsMost], uint32_t* totals) {
  const int nb = 1 << bits, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = lane; i < nb; i += 32) bins[warp][i] = 0;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const uint32_t d = digit[k];
    const unsigned same = equal_lanes(d, bits), before = same & ((1u << lane) - 1);
    uint32_t base = 0;
    if (d < uint32_t(nb)) base = bins[warp][d];
    __syncwarp();
    if (d < uint32_t(nb) && before == 0) bins[warp][d] = uint16_t(base + __popc(same));
    __syncwarp();
    at[k] = base + __popc(before);
  }
  __syncthreads();
  for (int d = tid; d < nb; d += kSortThreads) {
    uint32_t c[kSortWarps], sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) c[w] = bins[w][d];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      bins[w][d] = uint16_t(sum);
      sum += c[w];
    }
    if (totals) totals[d] = sum;
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
  // The warps' sums: every warp adds up those before it.
  uint32_t before = lane < warp ? part[lane] : 0;
  static_assert(kSortWarps <= 32, "");
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  return before + x - v;
}

template <bool FIRST, int EACH>
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const __grid_constant__ SortArgs s, const uint2* src, uint2* dst, int shift) {
  __shared__ uint16_t warp_bins[kSortWarps][kBinsMost];
  __shared__ uint32_t part[kSortWarps], base[kBinsMost];
  const int nb = 1 << s.bits, tid = threadIdx.x;
  after_previous();
  uint2 p[EACH];
  uint32_t digit[EACH], at[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t n = pair_index<EACH>(blockIdx.x, k);
    p[k] = n < s.N ? load_pair<FIRST>(s, src, n) : make_uint2(0, 0);
    digit[k] = n < s.N ? p[k].x >> shift & (nb - 1) : uint32_t(nb);
  }
  // Pairs of smaller digits, and of this digit in earlier tiles.
  const uint32_t all = tid < nb ? s.count[nb * s.tiles + tid] : 0;
  const uint32_t earlier = tid < nb ? s.count[tid * s.tiles + blockIdx.x] : 0;
  rank_pairs<EACH>(s.bits, digit, at, warp_bins, nullptr);
  const uint32_t smaller = block_prefix(all, part);
  if (tid < nb) base[tid] = smaller + earlier;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < EACH; ++k)
    if (digit[k] < uint32_t(nb))
      dst[base[digit[k]] + warp_bins[tid >> 5][digit[k]] + at[k]] = p[k];
  let_next_start();
}

// All passes in one launch for up to 8192 EACH pairs: a cluster of eight CTAs
// exchanges the digits' totals and the pairs themselves through distributed
// shared memory. (With EACH = 16, for 131072 pairs, its scattered stores took
// 68 us.) The CTAs after the cluster zero their part of dweight.
constexpr int kCluster = 8, kClusterEach = 2;
constexpr int64_t kClusterTokens = kCluster * kSortThreads * kClusterEach;

template <int EACH>
constexpr size_t cluster_smem() {
  return sizeof(uint16_t) * kSortWarps * kBinsMost + sizeof(uint2) * kSortThreads * EACH;
}

template <int EACH>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSortThreads)
sort_cluster_kernel(const __grid_constant__ SortArgs s, int passes) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char sort_smem[];
  uint16_t(*warp_bins)[kBinsMost] = reinterpret_cast<uint16_t(*)[kBinsMost]>(sort_smem);
  uint2* buf = reinterpret_cast<uint2*>(sort_smem + sizeof(uint16_t) * kSortWarps * kBinsMost);
  __shared__ uint32_t totals[kBinsMost], part[kSortWarps], base[kBinsMost];
  __shared__ uint32_t total[kSortThreads], before[kSortThreads];
  const int nb = 1 << s.bits, tid = threadIdx.x, warp = tid >> 5;
  if (blockIdx.x >= kCluster) {
    let_next_start();
    const int64_t pieces = s.zero_bytes / 16, step = int64_t(gridDim.x - kCluster) * kSortThreads;
    for (int64_t i = int64_t(blockIdx.x - kCluster) * kSortThreads + tid; i < pieces; i += step)
      reinterpret_cast<uint4*>(s.zero)[i] = make_uint4(0, 0, 0, 0);
    if (blockIdx.x == kCluster && tid < s.zero_bytes % 16) s.zero[pieces * 16 + tid] = 0;
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t mine = blockIdx.x;  // (one cluster)
  if (mine == 0 && tid == 0) s.crossing[0] = 0;
  constexpr uint32_t kRoom = kSortThreads * EACH;
  uint2 p[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t n = pair_index<EACH>(mine, k);
    p[k] = n < s.N ? load_pair<true>(s, nullptr, n) : make_uint2(0, 0);
  }
  for (int pass = 0; pass < passes; ++pass) {
    uint32_t digit[EACH], at[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      digit[k] = pair_index<EACH>(mine, k) < s.N ? p[k].x >> (pass * s.bits) & (nb - 1) : uint32_t(nb);
    rank_pairs<EACH>(s.bits, digit, at, warp_bins, totals);
    cluster.sync();  // all totals are there, and all pairs in registers
    const int d = tid & (nb - 1), share = kSortThreads / nb;
    uint32_t all = 0, earlier = 0;
    for (uint32_t c = tid / nb; c < kCluster; c += share) {
      const uint32_t x = *cluster.map_shared_rank(totals + d, c);
      all += x;
      earlier += c < mine ? x : 0;
    }
    total[tid] = all;
    before[tid] = earlier;
    __syncthreads();
    all = earlier = 0;
    if (tid < nb)
      for (int i = 0; i < share && i < kCluster; ++i) {
        all += total[tid + i * nb];
        earlier += before[tid + i * nb];
      }
    const uint32_t smaller = block_prefix(tid < nb ? all : 0, part);
    if (tid < nb) base[tid] = smaller + earlier;
    __syncthreads();
    const bool last = pass + 1 == passes;
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (digit[k] < uint32_t(nb)) {
        const uint32_t to = base[digit[k]] + warp_bins[warp][digit[k]] + at[k];
        if (last) s.a[to] = p[k];
        else *cluster.map_shared_rank(buf + to % kRoom, to / kRoom) = p[k];
      }
    if (last) let_next_start();
    cluster.sync();  // the pairs have arrived; nobody reads these totals any more
    if (!last)
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const int64_t n = pair_index<EACH>(mine, k);
        if (n < s.N) p[k] = buf[n - int64_t(mine) * kRoom];
      }
  }
}

// ---------------------------------------------------------------------------
// Sums over the sorted list
// ---------------------------------------------------------------------------

constexpr int kSumThreads = 128, kSumAhead = 8;
constexpr int kChunkMost = 128, kZeroRows = 64, kLookThrough = 2048;

struct SumArgs {
  const uint2* pairs;
  const void* d_out;
  void* dweight;
  uint32_t* crossing;
  float* part;          // [chunks][2][D]: a chunk's part of the run that came in, of the one that goes on
  int64_t N, V, D, d_stride, chunks;
  int64_t zero_rows;    // rows to be zeroed here if they have no token: the first ones
  int chunk;
  float scale;
};

// The first of the sorted pairs [lo, hi) that is not less than v, left in lo,
// for M values at once. One whole warp.
template <int M>
__device__ __forceinline__ void lower_bounds(const uint2* pairs, int64_t* lo, int64_t* hi, const uint32_t* v) {
  const int lane = threadIdx.x & 31;
  for (int64_t span = hi[0] - lo[0]; span > 0; span = span > 1 ? (span + 31) / 32 : 0) {
    const int64_t step = (span + 31) / 32;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int64_t at = lo[m] + lane * step;
      const bool less = at < hi[m] && pairs[at].x < v[m];
      const int n = __popc(__ballot_sync(0xffffffffu, less));
      // It lies after the last probe that was less and not after the next one.
      hi[m] = lo[m] + n * step < hi[m] ? lo[m] + n * step : hi[m];
      lo[m] = n == 0 ? lo[m] : lo[m] + (n - 1) * step + 1;
    }
  }
}

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
    // Which of kZeroRows rows have a token: the rows' part of the sorted list is
    // searched for, 32 ways a step, and then looked through, or searched row by
    // row where it is long.
    const int64_t v0 = (int64_t(blockIdx.x) - s.chunks) * kZeroRows;
    const int lane = tid & 31;
    int64_t lo[2] = {0, 0}, hi[2] = {s.N, s.N};
    const uint32_t ends[2] = {uint32_t(v0), uint32_t(v0 + kZeroRows)};
    lower_bounds<2>(s.pairs, lo, hi, ends);
    if (tid < kZeroRows) list[tid].x = 0;
    __syncthreads();
    if (lo[1] - lo[0] <= kLookThrough) {
      for (int64_t i = lo[0] + tid; i < lo[1]; i += kSumThreads) list[s.pairs[i].x - ends[0]].x = 1;
    } else {
      for (int r = tid / 32; r < kZeroRows; r += kSumThreads / 32) {
        int64_t l = lo[0], h = lo[1];
        const uint32_t v = uint32_t(v0 + r);
        lower_bounds<1>(s.pairs, &l, &h, &v);
        if (lane == 0 && l < s.N && s.pairs[l].x == v) list[r].x = 1;
      }
    }
    __syncthreads();
    let_next_start();
    if (col < s.D) {
      float zero[W] = {};
      for (int r = 0; r < kZeroRows; ++r)
        if (v0 + r < s.zero_rows && !list[r].x) write(v0 + r, zero);
    }
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
          if (!came_in && tid == 0 && blockIdx.y == 0)
            s.crossing[1 + atomicAdd(s.crossing, 1u)] = blockIdx.x;
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

// The rows whose runs cross chunks, from the list of the chunks in which such
// runs start (in whatever order: each row is summed by itself). A run's parts
// are added by kJoinWarps warps, every kJoinWarps-th part each, and then the
// warps' sums, in order. 128 columns at a time, column blocks in grid.y.
constexpr int kJoinWarps = 4;

template <int OT>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ SumArgs s) {
  __shared__ float4 sums[kJoinWarps][32];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t count = s.crossing[0];
  for (uint32_t i = blockIdx.x; i < count; i += gridDim.x) {
    const int64_t c = s.crossing[1 + i];
    const uint32_t v = s.pairs[(c + 1) * s.chunk].x;
    int64_t more = 0;  // how many further chunks the run reaches
    for (;;) {
      const int64_t at = (c + 1 + more + threadIdx.x) * s.chunk;
      const int n = __syncthreads_count(at < s.N && s.pairs[at].x == v);
      more += n;
      if (n < int(blockDim.x)) break;
    }
    for (int64_t d0 = int64_t(blockIdx.y) * 128; d0 < s.D; d0 += int64_t(gridDim.y) * 128) {
      const int64_t d = d0 + 4 * lane;
      float x[4] = {};
      const float* part = s.part + c * 2 * s.D + d;
      if (s.D % 4 == 0 && d < s.D) {
#pragma unroll 8
        for (int64_t k = warp; k <= more; k += kJoinWarps) {
          const float4 f = *reinterpret_cast<const float4*>(part + (k * 2 + (k == 0 ? 1 : 0)) * s.D);
          x[0] += f.x;
          x[1] += f.y;
          x[2] += f.z;
          x[3] += f.w;
        }
      } else {
#pragma unroll 2
        for (int64_t k = warp; k <= more; k += kJoinWarps)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d + j < s.D) x[j] += part[(k * 2 + (k == 0 ? 1 : 0)) * s.D + j];
      }
      sums[warp][lane] = make_float4(x[0], x[1], x[2], x[3]);
      __syncthreads();
      if (threadIdx.x < 128) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) y += reinterpret_cast<const float*>(sums[w])[threadIdx.x];
        if (d0 + threadIdx.x < s.D) store_elem(s.dweight, v * s.D + d0 + threadIdx.x, s.scale * y, OT);
      }
      __syncthreads();
    }
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

// How much of dweight the multiprocessors without a part in a cluster's sort can
// zero in its time, and by how many CTAs. (More, or beside the sort of a
// longer list, takes longer than zeroing only rows without a token: 131072
// tokens, 32000 x 1024 bf16, 101 against 94 us.)
constexpr int kZeroCtas = 35 * kCluster;
constexpr int64_t kZeroBytes = int64_t(64) << 20;

struct BwdPlan {
  int bits, passes, chunk;
  int64_t tiles, chunks;
  size_t a, b, count, crossing, part, total;
};

BwdPlan plan_bwd(const ngdn2_embed_bwd_args* a) {
  BwdPlan p{};
  int bits = 1;
  while ((a->V >> bits) > 0) ++bits;  // of the values 0 .. V
  p.passes = (bits + kDigitMost - 1) / kDigitMost;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t tile = kSortThreads * (a->N <= kFewTokens ? 1 : kManyEach);
  p.tiles = (a->N + tile - 1) / tile;
  // Chunks short enough for a few CTAs a multiprocessor, long enough to leave
  // few parts of hot tokens.
  p.chunk = 8;
  while (p.chunk < kChunkMost && a->N / p.chunk > 1024) p.chunk *= 2;
  p.chunks = (a->N + p.chunk - 1) / p.chunk;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~size_t(255);
    return o;
  };
  p.a = take(size_t(a->N) * 8);
  const bool clustered = a->N <= kClusterTokens;
  p.b = take(clustered ? 0 : size_t(a->N) * 8);
  p.count = take(clustered ? 0 : size_t(p.tiles + 1) << p.bits << 2);
  p.crossing = take(size_t(p.chunks + 1) * 4);
  p.part = take(size_t(p.chunks) * 2 * size_t(a->D) * 4);
  p.total = at + 256;
  return p;
}

template <int EACH>
cudaError_t sort_in_tiles(const SortArgs& s, int passes, cudaStream_t st) {
  const dim3 grid(unsigned(s.tiles)), block(kSortThreads);
  cudaError_t e = cudaSuccess;
  for (int pass = 0; pass < passes && e == cudaSuccess; ++pass) {
    // The last pass writes to a.
    uint2* dst = (passes - 1 - pass) % 2 == 0 ? s.a : s.b;
    const uint2* src = dst == s.a ? s.b : s.a;
    const int shift = pass * s.bits;
    e = pass == 0 ? launch_next(sort_count_kernel<true, EACH>, grid, block, 0, st, false, s, src, shift)
                  : launch_next(sort_count_kernel<false, EACH>, grid, block, 0, st, true, s, src, shift);
    if (e != cudaSuccess) break;
    constexpr int kDigits = kPrefixThreads / 32;
    e = launch_next(sort_prefix_kernel, dim3(((1u << s.bits) + kDigits - 1) / kDigits), dim3(kPrefixThreads), 0,
                    st, true, s);
    if (e != cudaSuccess) break;
    auto* place = pass == 0 ? sort_place_kernel<true, EACH> : sort_place_kernel<false, EACH>;
    e = launch_next(place, grid, block, 0, st, true, s, src, dst, shift);
  }
  return e;
}

template <int EACH>
cudaError_t sort_in_cluster(const SortArgs& s, int passes, cudaStream_t st) {
  constexpr size_t smem = cluster_smem<EACH>();
  const cudaError_t e = cudaFuncSetAttribute(sort_cluster_kernel<EACH>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e != cudaSuccess) return e;
  return launch_next(sort_cluster_kernel<EACH>, dim3(kCluster + (s.zero_bytes ? kZeroCtas : 0)),
                     dim3(kSortThreads), smem, st, false, s, passes);
}

cudaError_t sort_pairs(const SortArgs& s, int passes, cudaStream_t st) {
  if (s.N <= kCluster * kSortThreads) return sort_in_cluster<1>(s, passes, st);
  if (s.N <= kClusterTokens) return sort_in_cluster<kClusterEach>(s, passes, st);
  return s.N <= kFewTokens ? sort_in_tiles<1>(s, passes, st) : sort_in_tiles<kManyEach>(s, passes, st);
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
  so.crossing = reinterpret_cast<uint32_t*>(ws + p.crossing);
  so.status = a->status;
  SumArgs su;
  su.pairs = so.a;
  su.d_out = a->d_out;
  su.dweight = a->dweight;
  su.crossing = so.crossing;
  su.part = reinterpret_cast<float*>(ws + p.part);
  su.N = a->N;
  su.V = a->V;
  su.D = a->D;
  su.d_stride = a->d_stride;
  su.chunks = p.chunks;
  su.chunk = p.chunk;
  su.scale = a->scale;
  const int64_t row = a->D * (a->out_dtype == NGDN2_F32 ? 4 : 2);
  const int64_t budget = a->N <= kClusterTokens ? kZeroBytes / row : 0;
  // A row number of which 16 is a factor starts on a 16-byte boundary.
  su.zero_rows = reinterpret_cast<uintptr_t>(a->dweight) % 16 ? a->V
                 : a->V > budget ? (a->V - budget + 15) / 16 * 16 < a->V ? (a->V - budget + 15) / 16 * 16 : a->V
                                 : 0;
  so.zero = static_cast<char*>(a->dweight) + su.zero_rows * row;
  so.zero_bytes = (a->V - su.zero_rows) * row;
  const int64_t ctas = p.chunks + (su.zero_rows + kZeroRows - 1) / kZeroRows;
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
      const int64_t cols = (a->D + 127) / 128, items = p.chunks - 1;
      return launch_next(join_kernel<decltype(O)::value>,
                         dim3(unsigned(items < 256 ? items : 256), unsigned(cols < 8 ? cols : 8)),
                         dim3(32 * kJoinWarps), 0, st, true, su);
    });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
