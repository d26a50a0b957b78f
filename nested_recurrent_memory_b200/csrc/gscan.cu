// Gated linear recurrence, per (batch row, channel):
//   h_t = e^{g_t} h_{t-1} + x_t
// and its backward
//   u_t = dh_t + e^{g_{t+1}} u_{t+1},  dx = u,  dg_t = u_t e^{g_t} h_{t-1},  dh_0 = e^{g_1} u_1.
// Written with c_t = e^{g_t} u_t the backward is itself such a recurrence, from
// the end: c_t = e^{g_t} (dh_t + c_{t+1}), c_{T+1} = d_final. States are fp32.
//
// Both are bound by memory: forward x, g -> h, backward x, g, dh -> dx, dg,
// each byte moved once. A CTA takes a tile of steps x channels into shared
// memory, every thread a run of R steps of four channels. A run maps the
// state that enters it to the one that leaves, s -> A s + H; runs are joined
// within the warp by shuffles, across warps through shared memory, and
// across tiles by a chain in global memory: a tile posts its (A, H), looks
// back for the nearest tile whose leaving state is there, applies the (A, H) of
// those in between in order, and posts its own leaving state. That is
// the same sequence of operations however far it has to look, so the result
// does not depend on timing. Tiles are handed out in chain order by a
// counter, so a tile only waits for tiles that already run; the wait is
// bounded, and one that gives up poisons its outputs with NaN and sets
// NGDN2_STATUS_WAIT_TIMEOUT.

#include <math.h>

#include <type_traits>

#include "common.cuh"

using namespace ngdn2;

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr unsigned kAll = 0xffffffffu;

// CTAs a multiprocessor: 64 registers a thread forward, 80 (16-bit x) or 128
// backward.
constexpr int kFwdCtas = 8;
constexpr int bwd_ctas(int x_dtype) { return x_dtype == NGDN2_F32 ? 4 : 6; }

constexpr uint32_t kPollLimit = 1u << 21;

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

// ---------------------------------------------------------------------------
// The chain of tiles. A tile is CL lanes of four channels by 128 / CL runs of R
// steps.
// ---------------------------------------------------------------------------

// Per-tile records of the chain, [strip][position][channel] in chain order: a
// tile's map (A, H) and the state that leaves it. All bits set means "not
// there yet": the arithmetic that makes these values never does. So each value
// tells by itself whether it is there, and needs no flag and no fence.
constexpr int kChainCh = 32;
constexpr uint32_t kNotYet = 0xffffffffu;

struct Chain {
  uint64_t* map;
  uint32_t* state;
  uint32_t* ticket;  // one more than the tiles handed out, so that it starts as kNotYet
  int64_t strips;
  int tiles;
};

size_t chain_words(int64_t strips, int64_t tiles) { return size_t(strips) * tiles * kChainCh; }

size_t chain_bytes(int64_t strips, int64_t tiles) {
  return tiles < 2 ? 0 : 16 + chain_words(strips, tiles) * 12 + 4;
}

Chain make_chain(void* ws, int64_t strips, int64_t tiles) {
  Chain c{};
  c.strips = strips;
  c.tiles = int(tiles);
  if (tiles < 2) return c;
  c.map = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(ws) + 15) & ~uintptr_t(15));
  c.state = reinterpret_cast<uint32_t*>(c.map + chain_words(strips, tiles));
  c.ticket = c.state + chain_words(strips, tiles);
  return c;
}

__device__ __forceinline__ uint32_t peek(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t peek(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void post(uint32_t* p, float v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(__float_as_uint(v)) : "memory");
}
__device__ __forceinline__ void post(uint64_t* p, float A, float H) {
  const uint64_t v = uint64_t(__float_as_uint(H)) << 32 | __float_as_uint(A);
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// Tiles are handed out in chain order, positions of all strips in turn, to
// CTAs that stay. A CTA asks for its next tile when the state entering this
// one is known: earlier, and the tile would hold up its chain until this one
// is done (1 x 65536 x 1024: 199 us when asked for right after the loads). A lone
// position needs no counter: its tiles go round.
__device__ __forceinline__ uint32_t ask_tile(const Chain& ch, uint32_t last) {
  return ch.tiles < 2 ? last + gridDim.x : atomicAdd(ch.ticket, 1u) + 1u;
}

// The state entering tile ``pos`` > 0 for the lane's channel, whose own map is
// (A, H). One whole warp. The nearest of the kBack tiles before this one whose
// leaving state is there, and the maps of those in between, in order.
constexpr int kBack = 8;

__device__ __forceinline__ float chain_state(const Chain& ch, int64_t at, int pos, float A, float H,
                                             int32_t* status) {
  const int lane = threadIdx.x & 31;
  const uint64_t* map = ch.map + at * kChainCh + lane;
  const uint32_t* state = ch.state + at * kChainCh + lane;
  for (uint32_t poll = 0; poll < kPollLimit; ++poll) {
    uint32_t st[kBack];
    uint64_t mp[kBack];
#pragma unroll
    for (int k = 0; k < kBack; ++k) {
      st[k] = k < pos ? peek(state - (k + 1) * kChainCh) : kNotYet;
      mp[k] = k + 1 < pos && k + 1 < kBack ? peek(map - (k + 1) * kChainCh) : ~uint64_t(0);
    }
    if (poll == 0) post(ch.map + at * kChainCh + lane, A, H);
    int back = -1;
    bool joined = true;
#pragma unroll
    for (int k = 0; k < kBack; ++k) {
      if (back < 0 && joined && st[k] != kNotYet) back = k;
      joined = joined && uint32_t(mp[k]) != kNotYet && uint32_t(mp[k] >> 32) != kNotYet;
    }
    if (__all_sync(kAll, back >= 0)) {
      float s = 0.f;
#pragma unroll
      for (int k = kBack - 1; k >= 0; --k) {
        if (k == back) s = __uint_as_float(st[k]);
        if (k < back) s = fmaf(__uint_as_float(uint32_t(mp[k])), s, __uint_as_float(uint32_t(mp[k] >> 32)));
      }
      return s;
    }
  }
  if (lane == 0) atomicOr(status, NGDN2_STATUS_WAIT_TIMEOUT);
  return __int_as_float(0x7fc00000);
}

// ---------------------------------------------------------------------------
// A tile of one tensor in shared memory, in its own type: runs of R rows (steps)
// of the tile's channels. Runs are padded apart where rows are half of the
// 128 bytes that the banks span, so that the two runs of a half warp's 8-byte
// reads fall on different banks.
// ---------------------------------------------------------------------------

template <int DT, int CL, int R>
struct Stage {
  static constexpr int kEl = DT == NGDN2_F32 ? 4 : 2;
  static constexpr int kRow = 4 * CL * kEl;
  static constexpr int kRun = R * kRow + (kRow == 64 ? 64 : 0);
  static constexpr int kSteps = kThreads / CL * R;
  static constexpr int kBytes = kThreads / CL * kRun;
  static __device__ __forceinline__ int at(int t) { return t / R * kRun + t % R * kRow; }
};

// Copies of G bytes at a time without registers in between (G = 16 or 4), zeros
// for what lies outside [T, D]; G = 0 moves single elements of any stride.
template <int G>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool ok) {
  const uint32_t n = ok ? G : 0;
  if constexpr (G == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

template <int DT, int CL, int R, int G>
__device__ __forceinline__ void fill(unsigned char* sm, const void* p, const int64_t* st, int64_t b,
                                     int64_t t0, int64_t d0, int64_t T, int64_t D) {
  using S = Stage<DT, CL, R>;
  const int64_t base = b * st[0] + t0 * st[1] + d0 * st[2];
  if constexpr (G > 0) {
    // A thread keeps its columns and steps down the rows.
    constexpr int kPer = S::kRow / G, kHop = kThreads / kPer;
    static_assert(kThreads % kPer == 0 && S::kSteps % kHop == 0 && (kHop % R == 0 || R % kHop == 0), "");
    const int t = threadIdx.x / kPer, c = threadIdx.x % kPer * G;
    const bool in = d0 + c / S::kEl < D;
    const char* src = static_cast<const char*>(p) + (base + t * st[1]) * S::kEl + c;
    const int64_t hop = kHop * st[1] * S::kEl;
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(sm)) + c;
    const int64_t left = T - t0 - t;
#pragma unroll 8
    for (int j = 0; j < S::kSteps / kHop; ++j) {
      const bool ok = in && j * kHop < left;
      const uint32_t to = kHop % R == 0 ? S::at(t) + j * (kHop / R) * S::kRun : S::at(t + j * kHop);
      copy_async<G>(dst + to, ok ? src : p, ok);
      src += hop;
    }
  } else {
    using E = typename std::conditional<S::kEl == 4, uint32_t, uint16_t>::type;
    const E* src = static_cast<const E*>(p) + base;
#pragma unroll 8
    for (int q = threadIdx.x; q < S::kSteps * 4 * CL; q += kThreads) {
      const int t = q / (4 * CL), c = q % (4 * CL);
      const bool ok = t0 + t < T && d0 + c < D;
      *reinterpret_cast<E*>(sm + S::at(t) + c * S::kEl) = ok ? src[t * st[1] + c * st[2]] : E(0);
    }
  }
}

__device__ __forceinline__ void fill_done() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  __syncthreads();
}

// Four neighbouring elements as fp32, and back (rounded once).
template <int DT>
__device__ __forceinline__ void get4(const void* p, float* v) {
  if constexpr (DT == NGDN2_F32) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    float2 a, b;
    if constexpr (DT == NGDN2_BF16) {
      a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.x));
      b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.y));
    } else {
      a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
      b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    }
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
}

template <int DT>
__device__ __forceinline__ void put4(void* p, const float* v) {
  if constexpr (DT == NGDN2_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint2 r;
    if constexpr (DT == NGDN2_BF16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      r.x = *reinterpret_cast<const uint32_t*>(&a);
      r.y = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
      r.x = *reinterpret_cast<const uint32_t*>(&a);
      r.y = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint2*>(p) = r;
  }
}

// A tile's rows from shared memory to a contiguous [B, T, D] output, element
// by element with neighbouring threads on neighbouring channels: for widths
// whose rows four-channel accesses cannot follow.
template <int DT, int CL, int R>
__device__ __forceinline__ void drain(const unsigned char* sm, void* out, int64_t b, int64_t t0,
                                      int64_t d0, int64_t T, int64_t D) {
  using S = Stage<DT, CL, R>;
  using E = typename std::conditional<S::kEl == 4, uint32_t, uint16_t>::type;
  E* dst = static_cast<E*>(out) + (b * T + t0) * D + d0;
#pragma unroll 8
  for (int q = threadIdx.x; q < S::kSteps * 4 * CL; q += kThreads) {
    const int t = q / (4 * CL), c = q % (4 * CL);
    if (t0 + t < T && d0 + c < D)
      dst[t * D + c] = *reinterpret_cast<const E*>(sm + S::at(t) + c * S::kEl);
  }
}

// Decays of a run's step: e^g, kept in g's place once computed where g is fp32.
template <int GT>
__device__ __forceinline__ void decay4(const void* p, bool first, float* e) {
  get4<GT>(p, e);
  if (first || GT != NGDN2_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = expf(e[i]);
  }
}

// ---------------------------------------------------------------------------
// Forward. G is the copy size of the fills (see fill); with G = 16 the outputs
// go straight to memory, four channels at a time, else through the stage.
// ---------------------------------------------------------------------------

template <int XT, int GT, int CL, int R>
constexpr int fwd_smem() {
  return Stage<XT, CL, R>::kBytes + Stage<GT, CL, R>::kBytes;
}

template <int XT, int GT, int G, int CL, int R>
__global__ void __launch_bounds__(kThreads, kFwdCtas)
scan_kernel(const __grid_constant__ ngdn2_scan_args a, Chain chain, int row_strips) {
  constexpr int kCh = 4 * CL, NV = kCh / 32, kSteps = kThreads / CL * R;
  using SX = Stage<XT, CL, R>;
  using SG = Stage<GT, CL, R>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float2 part[kWarps][kCh];  // the warps' maps
  __shared__ float enter[kWarps][kCh];  // the state entering each warp's runs
  __shared__ uint32_t ticket;
  const uint32_t total = uint32_t(chain.strips * chain.tiles);
  unsigned char *sx = smem, *sg = smem + SX::kBytes;
  if (threadIdx.x == 0) ticket = ask_tile(chain, blockIdx.x - gridDim.x);
  __syncthreads();
  for (uint32_t mine = ticket; mine < total; mine = ticket) {
  const int strip = int(mine % uint32_t(chain.strips)), pos = int(mine / uint32_t(chain.strips));
  const int64_t b = strip / row_strips, d0 = int64_t(strip % row_strips) * kCh;
  const int64_t t0 = int64_t(pos) * kSteps;
  fill<XT, CL, R, G>(sx, a.x, a.x_stride, b, t0, d0, a.T, a.D);
  fill<GT, CL, R, G>(sg, a.g, a.g_stride, b, t0, d0, a.T, a.D);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = 4 * (lane % CL), run = threadIdx.x / CL;
  unsigned char *mx = sx + run * SX::kRun + c * SX::kEl, *mg = sg + run * SG::kRun + c * SG::kEl;
  uint32_t next = 0;
  fill_done();

  // The run's map. Past the end x = g = 0: the identity.
  float A[4] = {1.f, 1.f, 1.f, 1.f}, H[4] = {};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float x[4], e[4];
    get4<XT>(mx + r * SX::kRow, x);
    decay4<GT>(mg + r * SG::kRow, true, e);
    if (GT == NGDN2_F32) put4<NGDN2_F32>(mg + r * SG::kRow, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      A[i] *= e[i];
      H[i] = fmaf(e[i], H[i], x[i]);
    }
  }
  // Within the warp: the maps of all runs up to this one, then up to the
  // one before.
#pragma unroll
  for (int o = CL; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float pa = __shfl_up_sync(kAll, A[i], o), ph = __shfl_up_sync(kAll, H[i], o);
      if (lane >= o) {
        H[i] = fmaf(A[i], ph, H[i]);
        A[i] *= pa;
      }
    }
  if (lane >= 32 - CL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][c + i] = make_float2(A[i], H[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float pa = CL < 32 ? __shfl_up_sync(kAll, A[i], CL & 31) : 1.f;
    const float ph = CL < 32 ? __shfl_up_sync(kAll, H[i], CL & 31) : 0.f;
    A[i] = lane >= CL ? pa : 1.f;
    H[i] = lane >= CL ? ph : 0.f;
  }
  __syncthreads();
  if (warp == 0) {
    float ta[NV], th[NV], s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = lane + 32 * i;
      ta[i] = 1.f;
      th[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 m = part[w][ch];
        th[i] = fmaf(m.x, th[i], m.y);
        ta[i] *= m.x;
      }
      s[i] = pos == 0 && a.initial_state && d0 + ch < a.D ? a.initial_state[b * a.D + d0 + ch] : 0.f;
    }
    const int64_t at = int64_t(strip) * chain.tiles + pos;
    if (CL == 8 && pos > 0) s[0] = chain_state(chain, at, pos, ta[0], th[0], a.status);
    if (CL == 8 && pos + 1 < chain.tiles)  // the same by whichever way s came
      post(chain.state + at * kChainCh + lane, fmaf(ta[0], s[0], th[0]));
    if (lane == 0) next = ask_tile(chain, mine);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = lane + 32 * i;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        enter[w][ch] = s[i];
        s[i] = fmaf(part[w][ch].x, s[i], part[w][ch].y);
      }
      if (a.final_state && t0 + kSteps >= a.T && d0 + ch < a.D)
        a.final_state[b * a.D + d0 + ch] = s[i];
    }
  }
  __syncthreads();
  float h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = fmaf(A[i], enter[warp][c + i], H[i]);
  const int64_t t1 = t0 + run * R, d = d0 + c;
  if (a.carries && t1 % NGDN2_SCAN_CHUNK == 0 && t1 < a.T) {
    const int64_t NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
    float* to = a.carries + (b * NC + t1 / NGDN2_SCAN_CHUNK) * a.D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < a.D) to[i] = h[i];
  }
  unsigned char* out = static_cast<unsigned char*>(a.h) + ((b * a.T + t1) * a.D + d) * SX::kEl;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float x[4], e[4];
    get4<XT>(mx + r * SX::kRow, x);
    decay4<GT>(mg + r * SG::kRow, false, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmaf(e[i], h[i], x[i]);
    if (G != 16) put4<XT>(mx + r * SX::kRow, h);
    else if (t1 + r < a.T && d < a.D) put4<XT>(out + r * a.D * SX::kEl, h);
  }
  if (threadIdx.x == 0) ticket = next;
  __syncthreads();
  if (G != 16) {
    drain<XT, CL, R>(sx, a.h, b, t0, d0, a.T, a.D);
    __syncthreads();
  }
  }
}

// ---------------------------------------------------------------------------
// Backward: a tile's states from the one that the forward left at its start,
// the gradients from the chain that runs from the end.
// ---------------------------------------------------------------------------

template <int XT, int GT, int CL, int R>
constexpr int bwd_smem() {
  return 2 * Stage<XT, CL, R>::kBytes + Stage<GT, CL, R>::kBytes;
}

template <int XT, int GT, int G, int CL, int R>
__global__ void __launch_bounds__(kThreads, bwd_ctas(XT))
scan_bwd_kernel(const __grid_constant__ ngdn2_scan_bwd_args p, Chain chain, int row_strips) {
  constexpr int kCh = 4 * CL, NV = kCh / 32, kSteps = kThreads / CL * R;
  static_assert(NGDN2_SCAN_CHUNK % kSteps == 0, "a tile starts at a state that the forward left, or within its chunk as the only tile");
  using SX = Stage<XT, CL, R>;
  using SG = Stage<GT, CL, R>;
  const ngdn2_scan_args& a = p.fwd;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float2 part_h[kWarps][kCh], part_c[kWarps][kCh];
  __shared__ float enter_h[kWarps][kCh], enter_c[kWarps][kCh];
  __shared__ uint32_t ticket;
  const uint32_t total = uint32_t(chain.strips * chain.tiles);
  unsigned char *sx = smem, *sd = smem + SX::kBytes, *sg = smem + 2 * SX::kBytes;
  if (threadIdx.x == 0) ticket = ask_tile(chain, blockIdx.x - gridDim.x);
  __syncthreads();
  for (uint32_t mine = ticket; mine < total; mine = ticket) {
  const int strip = int(mine % uint32_t(chain.strips)), pos = int(mine / uint32_t(chain.strips));
  const int64_t b = strip / row_strips, d0 = int64_t(strip % row_strips) * kCh;
  const int64_t tile = chain.tiles - 1 - pos, t0 = tile * kSteps;
  fill<XT, CL, R, G>(sx, a.x, a.x_stride, b, t0, d0, a.T, a.D);
  fill<GT, CL, R, G>(sg, a.g, a.g_stride, b, t0, d0, a.T, a.D);
  fill<XT, CL, R, G>(sd, p.d_h, p.d_h_stride, b, t0, d0, a.T, a.D);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = 4 * (lane % CL), run = threadIdx.x / CL;
  unsigned char *mx = sx + run * SX::kRun + c * SX::kEl, *md = sd + run * SX::kRun + c * SX::kEl,
                *mg = sg + run * SG::kRun + c * SG::kEl;
  uint32_t next = 0;
  fill_done();

  float Ah[4] = {1.f, 1.f, 1.f, 1.f}, H[4] = {}, Ac[4], C[4] = {};
  {
    float e[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x[4];
      get4<XT>(mx + r * SX::kRow, x);
      decay4<GT>(mg + r * SG::kRow, true, e[r]);
      if (GT == NGDN2_F32) put4<NGDN2_F32>(mg + r * SG::kRow, e[r]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Ah[i] *= e[r][i];
        H[i] = fmaf(e[r][i], H[i], x[i]);
      }
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float dh[4];
      get4<XT>(md + r * SX::kRow, dh);
#pragma unroll
      for (int i = 0; i < 4; ++i) C[i] = e[r][i] * (dh[i] + C[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) Ac[i] = Ah[i];
#pragma unroll
  for (int o = CL; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float pa = __shfl_up_sync(kAll, Ah[i], o), ph = __shfl_up_sync(kAll, H[i], o);
      if (lane >= o) {
        H[i] = fmaf(Ah[i], ph, H[i]);
        Ah[i] *= pa;
      }
      const float na = __shfl_down_sync(kAll, Ac[i], o), nc = __shfl_down_sync(kAll, C[i], o);
      if (lane + o < 32) {
        C[i] = fmaf(Ac[i], nc, C[i]);
        Ac[i] *= na;
      }
    }
  if (lane >= 32 - CL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part_h[warp][c + i] = make_float2(Ah[i], H[i]);
  }
  if (lane < CL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part_c[warp][c + i] = make_float2(Ac[i], C[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float pa = CL < 32 ? __shfl_up_sync(kAll, Ah[i], CL & 31) : 1.f;
    const float ph = CL < 32 ? __shfl_up_sync(kAll, H[i], CL & 31) : 0.f;
    Ah[i] = lane >= CL ? pa : 1.f;
    H[i] = lane >= CL ? ph : 0.f;
    const float na = CL < 32 ? __shfl_down_sync(kAll, Ac[i], CL & 31) : 1.f;
    const float nc = CL < 32 ? __shfl_down_sync(kAll, C[i], CL & 31) : 0.f;
    Ac[i] = lane + CL < 32 ? na : 1.f;
    C[i] = lane + CL < 32 ? nc : 0.f;
  }
  __syncthreads();
  if (warp == 0) {
    float ta[NV], tc[NV], s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = lane + 32 * i;
      ta[i] = 1.f;
      tc[i] = 0.f;
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        const float2 m = part_c[w][ch];
        tc[i] = fmaf(m.x, tc[i], m.y);
        ta[i] *= m.x;
      }
      s[i] = pos == 0 && p.d_final && d0 + ch < a.D ? p.d_final[b * a.D + d0 + ch] : 0.f;
    }
    const int64_t at = int64_t(strip) * chain.tiles + pos;
    if (CL == 8 && pos > 0) s[0] = chain_state(chain, at, pos, ta[0], tc[0], p.status);
    if (CL == 8 && pos + 1 < chain.tiles)
      post(chain.state + at * kChainCh + lane, fmaf(ta[0], s[0], tc[0]));
    if (lane == 0) next = ask_tile(chain, mine);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = lane + 32 * i;
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        enter_c[w][ch] = s[i];
        s[i] = fmaf(part_c[w][ch].x, s[i], part_c[w][ch].y);
      }
      if (p.d_initial && tile == 0 && d0 + ch < a.D) p.d_initial[b * a.D + d0 + ch] = s[i];
    }
  } else if (warp == 1) {
    const int64_t NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int ch = lane + 32 * i;
      float s = d0 + ch < a.D ? a.carries[(b * NC + t0 / NGDN2_SCAN_CHUNK) * a.D + d0 + ch] : 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        enter_h[w][ch] = s;
        s = fmaf(part_h[w][ch].x, s, part_h[w][ch].y);
      }
    }
  }
  __syncthreads();
  float h[R][4], cc[4];  // h[r]: the state before step r
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[0][i] = fmaf(Ah[i], enter_h[warp][c + i], H[i]);
    cc[i] = fmaf(Ac[i], enter_c[warp][c + i], C[i]);
  }
#pragma unroll
  for (int r = 0; r + 1 < R; ++r) {
    float x[4], e[4];
    get4<XT>(mx + r * SX::kRow, x);
    decay4<GT>(mg + r * SG::kRow, false, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[r + 1][i] = fmaf(e[i], h[r][i], x[i]);
  }
  const int64_t t1 = t0 + run * R, d = d0 + c, o = (b * a.T + t1) * a.D + d;
  unsigned char *ox = static_cast<unsigned char*>(p.dx) + o * SX::kEl,
                *og = static_cast<unsigned char*>(p.dg) + o * SG::kEl;
#pragma unroll
  for (int r = R - 1; r >= 0; --r) {
    float u[4], e[4], dg[4];
    get4<XT>(md + r * SX::kRow, u);
    decay4<GT>(mg + r * SG::kRow, false, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] += cc[i];
      cc[i] = e[i] * u[i];
      dg[i] = cc[i] * h[r][i];
    }
    if (G != 16) {
      put4<XT>(md + r * SX::kRow, u);
      put4<GT>(mg + r * SG::kRow, dg);
    } else if (t1 + r < a.T && d < a.D) {
      put4<XT>(ox + r * a.D * SX::kEl, u);
      put4<GT>(og + r * a.D * SG::kEl, dg);
    }
  }
  if (threadIdx.x == 0) ticket = next;
  __syncthreads();
  if (G != 16) {
    drain<XT, CL, R>(sd, p.dx, b, t0, d0, a.T, a.D);
    drain<GT, CL, R>(sg, p.dg, b, t0, d0, a.T, a.D);
    __syncthreads();
  }
  }
}

__global__ void __launch_bounds__(128) scan_step_kernel(ngdn2_scan_step_args a) {
  const int64_t i = int64_t(blockIdx.x) * 128 + threadIdx.x;
  if (i >= int64_t(a.B) * a.D) return;
  const int64_t b = i / a.D, d = i % a.D;
  const float x = load_elem(a.x, b * a.x_stride[0] + d * a.x_stride[1], a.x_dtype);
  const float g = load_elem(a.g, b * a.g_stride[0] + d * a.g_stride[1], a.g_dtype);
  const float h = fmaf(expf(g), a.state_in[i], x);
  a.state_out[i] = h;
  store_elem(a.h, i, h, a.x_dtype);
}

// ---------------------------------------------------------------------------
// Choice of tile and launch
// ---------------------------------------------------------------------------

// The largest copy that every row of a [B, T, D] view allows: 16 or 4 bytes,
// or 0 for element by element.
int granule(const void* p, int dt, const int64_t* st, int64_t D) {
  const int64_t el = dt == NGDN2_F32 ? 4 : 2;
  if (st[2] != 1) return 0;
  const uintptr_t all = reinterpret_cast<uintptr_t>(p) | uintptr_t(st[0] * el) | uintptr_t(st[1] * el) |
                        uintptr_t(D * el);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 0;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ``per_sm`` CTAs a multiprocessor at most (what the registers allow; where
// shared memory holds fewer, the others find no tile left).
template <class K, class... Args>
cudaError_t launch(K kernel, int64_t tiles, int per_sm, int smem, cudaStream_t st, const Args&... args) {
  cudaError_t e = cudaSuccess;
  if (smem > 32 * 1024)  // (with the static part it may pass what needs no asking)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int dev = 0, sms = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  const int64_t fit = int64_t(sms) * per_sm;
  kernel<<<unsigned(tiles < fit ? tiles : fit), kThreads, smem, st>>>(args...);
  return cudaGetLastError();
}

template <class F>
cudaError_t by_types(int xt, int gt, F&& f) {
  auto g = [&](auto X) {
    switch (gt) {
      case NGDN2_BF16: return f(X, std::integral_constant<int, NGDN2_BF16>{});
      case NGDN2_F16: return f(X, std::integral_constant<int, NGDN2_F16>{});
      default: return f(X, std::integral_constant<int, NGDN2_F32>{});
    }
  };
  switch (xt) {
    case NGDN2_BF16: return g(std::integral_constant<int, NGDN2_BF16>{});
    case NGDN2_F16: return g(std::integral_constant<int, NGDN2_F16>{});
    default: return g(std::integral_constant<int, NGDN2_F32>{});
  }
}

// The narrow tile (32 channels) leaves the long axis in few, long tiles, so
// that the chain is short; the wide one (128 channels) is for sequences of
// at most its 32 steps, whose narrow tiles would be mostly empty.
constexpr int kNarrowR = 8, kNarrowSteps = kThreads / 8 * kNarrowR;
constexpr int kWideR = 8, kWideSteps = kThreads / 32 * kWideR;

template <class F>
cudaError_t by_tile(int channels, int granule, F&& f) {
  auto g = [&](auto CL, auto R) {
    switch (granule) {
      case 16: return f(std::integral_constant<int, 16>{}, CL, R);
      case 4: return f(std::integral_constant<int, 4>{}, CL, R);
      default: return f(std::integral_constant<int, 0>{}, CL, R);
    }
  };
  return channels == 128
             ? g(std::integral_constant<int, 32>{}, std::integral_constant<int, kWideR>{})
             : g(std::integral_constant<int, 8>{}, std::integral_constant<int, kNarrowR>{});
}

struct Shape {
  int row_strips, channels;
  int64_t strips, tiles;
};

Shape shape_of(const ngdn2_scan_args* a) {
  Shape s;
  s.channels = a->T <= kWideSteps ? 128 : 32;
  s.row_strips = int((a->D + s.channels - 1) / s.channels);
  s.strips = int64_t(a->B) * s.row_strips;
  s.tiles = a->T <= kWideSteps ? 1 : (a->T + kNarrowSteps - 1) / kNarrowSteps;
  return s;
}

int validate_scan(const ngdn2_scan_args* a, bool outputs) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->g_dtype)) return NGDN2_ERR_DTYPE;
  // The strips of all tiles are counted in 31 bits.
  if (a->B < 1 || a->T < 1 || a->D < 1 || a->T >= (int64_t(1) << 31) ||
      a->D >= (int64_t(1) << 31) ||
      (a->D + 31) / 32 * ((a->T + kNarrowSteps - 1) / kNarrowSteps) > ((int64_t(1) << 31) - 1) / a->B)
    return NGDN2_ERR_SHAPE;
  if (!a->x || !a->g || (outputs && (!a->h || !a->status))) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

int validate_scan_bwd(const ngdn2_scan_bwd_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  const int rc = validate_scan(&a->fwd, false);
  if (rc != NGDN2_OK) return rc;
  if (a->d_h_dtype != a->fwd.x_dtype) return NGDN2_ERR_DTYPE;
  if (!a->fwd.carries || !a->d_h || !a->dx || !a->dg || !a->status) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

// The chain of one launch, with nothing there yet.
int start_chain(const Shape& s, void* ws, size_t ws_bytes, cudaStream_t st, Chain* c) {
  const size_t need = chain_bytes(s.strips, s.tiles);
  if (need && (!ws || ws_bytes < need)) return NGDN2_ERR_WORKSPACE;
  *c = make_chain(ws, s.strips, s.tiles);
  if (need && cudaMemsetAsync(c->map, 0xff, need - 16, st) != cudaSuccess)
    return NGDN2_ERR_CUDA;
  return NGDN2_OK;
}

}  // namespace

extern "C" {

NGDN2_API size_t ngdn2_sizeof_scan_args(void) { return sizeof(ngdn2_scan_args); }
NGDN2_API size_t ngdn2_sizeof_scan_bwd_args(void) { return sizeof(ngdn2_scan_bwd_args); }
NGDN2_API size_t ngdn2_sizeof_scan_step_args(void) { return sizeof(ngdn2_scan_step_args); }

NGDN2_API int ngdn2_scan_workspace_size(const ngdn2_scan_args* a, size_t* bytes) {
  const int rc = validate_scan(a, false);
  if (rc != NGDN2_OK) return rc;
  if (!bytes) return NGDN2_ERR_NULL;
  const Shape s = shape_of(a);
  *bytes = chain_bytes(s.strips, s.tiles);
  return NGDN2_OK;
}

NGDN2_API int ngdn2_scan(const ngdn2_scan_args* a, void* stream) {
  int rc = validate_scan(a, true);
  if (rc != NGDN2_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Shape s = shape_of(a);
  Chain chain;
  rc = start_chain(s, a->workspace, a->workspace_bytes, st, &chain);
  if (rc != NGDN2_OK) return rc;
  int g = granule(a->x, a->x_dtype, a->x_stride, a->D);
  const int g2 = granule(a->g, a->g_dtype, a->g_stride, a->D);
  g = g2 < g ? g2 : g;
  if (g == 16 && !aligned16(a->h)) g = 4;
  const cudaError_t err = by_types(a->x_dtype, a->g_dtype, [&](auto X, auto Gt) {
    constexpr int XT = decltype(X)::value, GT = decltype(Gt)::value;
    return by_tile(s.channels, g, [&](auto GR, auto CLc, auto Rc) {
      constexpr int G = decltype(GR)::value, CL = decltype(CLc)::value, R = decltype(Rc)::value;
      return launch(scan_kernel<XT, GT, G, CL, R>, s.strips * s.tiles, kFwdCtas, fwd_smem<XT, GT, CL, R>(), st,
                    *a, chain, s.row_strips);
    });
  });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_scan_bwd(const ngdn2_scan_bwd_args* p, void* stream) {
  int rc = validate_scan_bwd(p);
  if (rc != NGDN2_OK) return rc;
  const ngdn2_scan_args* a = &p->fwd;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Shape s = shape_of(a);
  Chain chain;
  rc = start_chain(s, p->workspace, p->workspace_bytes, st, &chain);
  if (rc != NGDN2_OK) return rc;
  int g = granule(a->x, a->x_dtype, a->x_stride, a->D);
  for (const int o : {granule(a->g, a->g_dtype, a->g_stride, a->D),
                      granule(p->d_h, p->d_h_dtype, p->d_h_stride, a->D)})
    g = o < g ? o : g;
  if (g == 16 && (!aligned16(p->dx) || !aligned16(p->dg))) g = 4;
  const cudaError_t err = by_types(a->x_dtype, a->g_dtype, [&](auto X, auto Gt) {
    constexpr int XT = decltype(X)::value, GT = decltype(Gt)::value;
    return by_tile(s.channels, g, [&](auto GR, auto CLc, auto Rc) {
      constexpr int G = decltype(GR)::value, CL = decltype(CLc)::value, R = decltype(Rc)::value;
      return launch(scan_bwd_kernel<XT, GT, G, CL, R>, s.strips * s.tiles, bwd_ctas(XT),
                    bwd_smem<XT, GT, CL, R>(), st, *p, chain, s.row_strips);
    });
  });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_scan_step(const ngdn2_scan_step_args* a, void* stream) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->g_dtype)) return NGDN2_ERR_DTYPE;
  const int64_t n = int64_t(a->B) * a->D;
  if (a->B < 1 || a->D < 1 || a->D >= (int64_t(1) << 31) || n >= (int64_t(1) << 36))
    return NGDN2_ERR_SHAPE;
  if (!a->x || !a->g || !a->state_in || !a->state_out || !a->h) return NGDN2_ERR_NULL;
  scan_step_kernel<<<unsigned((n + 127) / 128), 128, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
