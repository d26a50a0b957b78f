// Gated linear recurrence, per (batch row, channel):
//   h_t = e^{g_t} h_{t-1} + x_t
// and its backward
//   u_t = dh_t + e^{g_{t+1}} u_{t+1},  dx = u,  dg_t = u_t e^{g_t} h_{t-1},  dh_0 = e^{g_1} u_1.
// Written with c_t = e^{g_t} u_t the backward is itself such a recurrence, from
// the end: c_t = e^{g_t} (dh_t + c_{t+1}), c_{T+1} = d_final. States are fp32.
//
// Both are bound by memory: forward x, g -> h, backward x, g, dh -> dx, dg,
// each byte moved once. A CTA takes a tile of steps x channels: every thread
// a run of R steps of four channels, which it keeps in registers. A run maps the
// state that enters it to the one that leaves, s -> A s + H; runs are joined
// within the warp by shuffles, across warps through shared memory, and
// across tiles by a chain in global memory: a tile publishes its (A, H) as
// soon as it has them, then looks back for the nearest tile whose leaving
// state is known and applies the (A, H) of those in between in order. That is
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

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr unsigned kAll = 0xffffffffu;
constexpr uint32_t kPollLimit = 1u << 21;

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

// ---------------------------------------------------------------------------
// Tiles: CL lanes of four channels by 256 / CL runs of R steps.
// ---------------------------------------------------------------------------

template <int CL, int R>
struct Tile {
  static constexpr int kChannels = 4 * CL;
  static constexpr int kSteps = kThreads / CL * R;
};

// Per-tile records of the chain, [strip][position] in chain order: a state
// word (0 nothing, 1 (A, H) is there, 2 the leaving state too) and the
// values for the tile's channels.
struct Chain {
  uint32_t* ticket;
  uint32_t* flag;
  float2* agg;
  float* inc;
  int64_t strips;
  int tiles;
};

size_t chain_flag_bytes(int64_t strips, int64_t tiles) {
  return size_t((strips * tiles + 1) * 4 + 255) & ~size_t(255);
}

size_t chain_bytes(int64_t strips, int64_t tiles, int channels) {
  return tiles < 2 ? 0 : 256 + chain_flag_bytes(strips, tiles) +
                             size_t(strips) * tiles * channels * (sizeof(float2) + sizeof(float));
}

Chain make_chain(void* ws, int64_t strips, int64_t tiles, int channels) {
  Chain c{};
  c.strips = strips;
  c.tiles = int(tiles);
  if (tiles < 2) return c;
  char* p = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(ws) + 255) & ~uintptr_t(255));
  c.ticket = reinterpret_cast<uint32_t*>(p);
  c.flag = c.ticket + 1;
  p += chain_flag_bytes(strips, tiles);
  c.agg = reinterpret_cast<float2*>(p);
  c.inc = reinterpret_cast<float*>(p + size_t(strips) * tiles * channels * sizeof(float2));
  return c;
}

__device__ __forceinline__ uint32_t load_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(uint32_t* p, uint32_t v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// Which tile this CTA takes: position in its chain and strip of channels.
// Positions of all strips in turn, by the counter (a lone position needs none).
__device__ __forceinline__ void take_tile(const Chain& ch, int* strip, int* pos) {
  __shared__ uint32_t ticket;
  if (ch.tiles < 2) {
    *strip = int(blockIdx.x);
    *pos = 0;
    return;
  }
  if (threadIdx.x == 0) ticket = atomicAdd(ch.ticket, 1u);
  __syncthreads();
  *strip = int(ticket % uint32_t(ch.strips));
  *pos = int(ticket / uint32_t(ch.strips));
}

// The state entering tile ``pos`` for NV channels a lane (channel lane +
// 32 i), whose own map is (A, H); publishes the map and the leaving state.
// ``first`` is the state that enters position 0. One whole warp.
template <int NV>
__device__ __forceinline__ void chain_state(const Chain& ch, int strip, int pos, const float* A,
                                            const float* H, const float* first, float* s,
                                            int32_t* status) {
  constexpr int kCh = 32 * NV;
  const int lane = threadIdx.x & 31;
  const int64_t at = int64_t(strip) * ch.tiles + pos;
  if (pos == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = first[i];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      ch.agg[at * kCh + lane + 32 * i] = make_float2(A[i], H[i]);
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      store_release(ch.flag + at, 1u);
    }
    int back = -1;  // how many tiles lie between this one and the known state
    for (uint32_t poll = 0; poll < kPollLimit; ++poll) {
      const uint32_t f = lane < pos ? load_acquire(ch.flag + at - 1 - lane) : 0u;
      const unsigned known = __ballot_sync(kAll, f == 2u), there = __ballot_sync(kAll, f >= 1u);
      const int p = __ffs(known) - 1;
      const unsigned between = p >= 0 ? (1u << p) - 1u : 0u;
      if (p >= 0 && (there & between) == between) {
        back = p;
        break;
      }
    }
    __syncwarp();
    if (back < 0) {
      if (lane == 0) atomicOr(status, NGDN2_STATUS_WAIT_TIMEOUT);
#pragma unroll
      for (int i = 0; i < NV; ++i) s[i] = __int_as_float(0x7fc00000);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) s[i] = __ldcg(ch.inc + (at - 1 - back) * kCh + lane + 32 * i);
#pragma unroll 8
      for (int k = back; k > 0; --k)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float2 m = __ldcg(ch.agg + (at - k) * kCh + lane + 32 * i);
          s[i] = fmaf(m.x, s[i], m.y);
        }
    }
  }
  if (pos + 1 < ch.tiles) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      ch.inc[at * kCh + lane + 32 * i] = fmaf(A[i], s[i], H[i]);
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      store_release(ch.flag + at, 2u);
    }
  }
}

// ---------------------------------------------------------------------------
// Four channels of one step. VEC: neighbouring, unit stride and aligned, one
// vector access. Otherwise CL apart (so a warp's accesses stay together), each
// by its own strides.
// ---------------------------------------------------------------------------

template <int DT, bool VEC, int CL>
__device__ __forceinline__ void load4(const void* p, int64_t o, int64_t sd, int left, float* v) {
  if constexpr (VEC) {
    if (left <= 0) {
      v[0] = v[1] = v[2] = v[3] = 0.f;
    } else if constexpr (DT == NGDN2_F32) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + o));
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + o));
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
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = CL * i < left ? load_typed<DT>(p, o + CL * i * sd) : 0.f;
  }
}

template <int DT, bool VEC, int CL>
__device__ __forceinline__ void store4(void* p, int64_t o, int left, const float* v) {
  if constexpr (VEC) {
    if (left <= 0) return;
    if constexpr (DT == NGDN2_F32) {
      __stcs(reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + o),
             make_float4(v[0], v[1], v[2], v[3]));
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
      __stcs(reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + o), r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (CL * i < left) store_elem(p, o + CL * i, v[i], DT);
  }
}

// A thread's place in its tile: lane of channels, run of steps, its first
// channel d and how many of the row's channels lie from there on, the
// spacing of its four channels.
template <int CL, bool VEC>
struct Place {
  int cl, run;
  int64_t d;
  int left;
  static constexpr int kGap = VEC ? 1 : CL;
  __device__ Place(int64_t d0, int64_t D) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    cl = lane % CL;
    run = warp * (32 / CL) + lane / CL;
    d = d0 + (VEC ? 4 * cl : cl);
    left = D - d > 4 * CL ? 4 * CL : int(D - d);
  }
  // Tile-local index of channel i.
  __device__ int ch(int i) const { return (VEC ? 4 * cl : cl) + kGap * i; }
};

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------

template <int XT, int GT, bool VEC, int CL, int R>
__global__ void __launch_bounds__(kThreads) scan_kernel(ngdn2_scan_args a, Chain chain, int row_strips) {
  using TL = Tile<CL, R>;
  constexpr int kCh = TL::kChannels, NV = kCh / 32;
  __shared__ float2 part[kWarps][kCh];  // the warps' maps
  __shared__ float enter[kWarps][kCh];  // the state entering each warp's runs
  int strip, pos;
  take_tile(chain, &strip, &pos);
  const int64_t b = strip / row_strips, d0 = int64_t(strip % row_strips) * kCh;
  const Place<CL, VEC> me(d0, a.D);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t0 = int64_t(pos) * TL::kSteps + me.run * R;

  float x[R][4], e[R][4];
  const int64_t xo = b * a.x_stride[0] + t0 * a.x_stride[1] + me.d * a.x_stride[2];
  const int64_t go = b * a.g_stride[0] + t0 * a.g_stride[1] + me.d * a.g_stride[2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int left = t0 + r < a.T ? me.left : 0;
    load4<XT, VEC, CL>(a.x, xo + r * a.x_stride[1], a.x_stride[2], left, x[r]);
    load4<GT, VEC, CL>(a.g, go + r * a.g_stride[1], a.g_stride[2], left, e[r]);
  }
  // Past the end x = g = 0: the identity.
  float A[4] = {1.f, 1.f, 1.f, 1.f}, H[4] = {};
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[r][i] = expf(e[r][i]);
      A[i] *= e[r][i];
      H[i] = fmaf(e[r][i], H[i], x[r][i]);
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
    for (int i = 0; i < 4; ++i) part[warp][me.ch(i)] = make_float2(A[i], H[i]);
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
    float ta[NV], th[NV], first[NV], s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      first[i] = a.initial_state && d0 + c < a.D ? a.initial_state[b * a.D + d0 + c] : 0.f;
      ta[i] = 1.f;
      th[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 m = part[w][c];
        th[i] = fmaf(m.x, th[i], m.y);
        ta[i] *= m.x;
      }
    }
    chain_state<NV>(chain, strip, pos, ta, th, first, s, a.status);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        enter[w][c] = s[i];
        s[i] = fmaf(part[w][c].x, s[i], part[w][c].y);
      }
      if (a.final_state && (int64_t(pos) + 1) * TL::kSteps >= a.T && d0 + c < a.D)
        a.final_state[b * a.D + d0 + c] = s[i];
    }
  }
  __syncthreads();
  float h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = fmaf(A[i], enter[warp][me.ch(i)], H[i]);
  if (a.carries && t0 % NGDN2_SCAN_CHUNK == 0 && t0 < a.T) {
    const int64_t NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
    store4<NGDN2_F32, VEC, CL>(a.carries, (b * NC + t0 / NGDN2_SCAN_CHUNK) * a.D + me.d, me.left, h);
  }
  const int64_t ho = (b * a.T + t0) * a.D + me.d;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmaf(e[r][i], h[i], x[r][i]);
    if (t0 + r < a.T) store4<XT, VEC, CL>(a.h, ho + r * a.D, me.left, h);
  }
}

// ---------------------------------------------------------------------------
// Backward: a tile's states from the one that the forward left at its start,
// the gradients from the chain that runs from the end.
// ---------------------------------------------------------------------------

template <int XT, int GT, bool VEC, int CL, int R>
__global__ void __launch_bounds__(kThreads)
scan_bwd_kernel(ngdn2_scan_bwd_args p, Chain chain, int row_strips) {
  using TL = Tile<CL, R>;
  constexpr int kCh = TL::kChannels, NV = kCh / 32;
  static_assert(TL::kSteps <= NGDN2_SCAN_CHUNK && NGDN2_SCAN_CHUNK % TL::kSteps == 0, "");
  const ngdn2_scan_args& a = p.fwd;
  __shared__ float2 part_h[kWarps][kCh], part_c[kWarps][kCh];
  __shared__ float enter_h[kWarps][kCh], enter_c[kWarps][kCh];
  int strip, pos;
  take_tile(chain, &strip, &pos);
  const int64_t b = strip / row_strips, d0 = int64_t(strip % row_strips) * kCh;
  const int64_t tile = chain.tiles - 1 - pos;
  const Place<CL, VEC> me(d0, a.D);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t0 = tile * TL::kSteps + me.run * R;

  float x[R][4], e[R][4], dh[R][4];
  const int64_t xo = b * a.x_stride[0] + t0 * a.x_stride[1] + me.d * a.x_stride[2];
  const int64_t go = b * a.g_stride[0] + t0 * a.g_stride[1] + me.d * a.g_stride[2];
  const int64_t dho = b * p.d_h_stride[0] + t0 * p.d_h_stride[1] + me.d * p.d_h_stride[2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int left = t0 + r < a.T ? me.left : 0;
    load4<XT, VEC, CL>(a.x, xo + r * a.x_stride[1], a.x_stride[2], left, x[r]);
    load4<GT, VEC, CL>(a.g, go + r * a.g_stride[1], a.g_stride[2], left, e[r]);
    load4<XT, VEC, CL>(p.d_h, dho + r * p.d_h_stride[1], p.d_h_stride[2], left, dh[r]);
  }
  float Ah[4] = {1.f, 1.f, 1.f, 1.f}, H[4] = {}, Ac[4], C[4] = {};
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[r][i] = expf(e[r][i]);
      Ah[i] *= e[r][i];
      H[i] = fmaf(e[r][i], H[i], x[r][i]);
    }
#pragma unroll
  for (int r = R - 1; r >= 0; --r)
#pragma unroll
    for (int i = 0; i < 4; ++i) C[i] = e[r][i] * (dh[r][i] + C[i]);
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
    for (int i = 0; i < 4; ++i) part_h[warp][me.ch(i)] = make_float2(Ah[i], H[i]);
  }
  if (lane < CL) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part_c[warp][me.ch(i)] = make_float2(Ac[i], C[i]);
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
    float ta[NV], tc[NV], first[NV], s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      first[i] = p.d_final && d0 + c < a.D ? p.d_final[b * a.D + d0 + c] : 0.f;
      ta[i] = 1.f;
      tc[i] = 0.f;
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        const float2 m = part_c[w][c];
        tc[i] = fmaf(m.x, tc[i], m.y);
        ta[i] *= m.x;
      }
    }
    chain_state<NV>(chain, strip, pos, ta, tc, first, s, p.status);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
#pragma unroll
      for (int w = kWarps - 1; w >= 0; --w) {
        enter_c[w][c] = s[i];
        s[i] = fmaf(part_c[w][c].x, s[i], part_c[w][c].y);
      }
      if (p.d_initial && tile == 0 && d0 + c < a.D) p.d_initial[b * a.D + d0 + c] = s[i];
    }
  } else if (warp == 1) {
    const int64_t NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
    const int64_t chunk = tile * TL::kSteps / NGDN2_SCAN_CHUNK;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      float s = d0 + c < a.D ? a.carries[(b * NC + chunk) * a.D + d0 + c] : 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        enter_h[w][c] = s;
        s = fmaf(part_h[w][c].x, s, part_h[w][c].y);
      }
    }
  }
  __syncthreads();
  float h[4], c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = fmaf(Ah[i], enter_h[warp][me.ch(i)], H[i]);
    c[i] = fmaf(Ac[i], enter_c[warp][me.ch(i)], C[i]);
  }
  // x[r] becomes the state before step r.
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float next = fmaf(e[r][i], h[i], x[r][i]);
      x[r][i] = h[i];
      h[i] = next;
    }
  const int64_t o = (b * a.T + t0) * a.D + me.d;
#pragma unroll
  for (int r = R - 1; r >= 0; --r) {
    float u[4], dg[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = dh[r][i] + c[i];
      c[i] = e[r][i] * u[i];
      dg[i] = c[i] * x[r][i];
    }
    if (t0 + r < a.T) {
      store4<XT, VEC, CL>(p.dx, o + r * a.D, me.left, u);
      store4<GT, VEC, CL>(p.dg, o + r * a.D, me.left, dg);
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

bool vec_ok(const void* p, int dt, const int64_t* st, int64_t D) {
  const int64_t bytes = dt == NGDN2_F32 ? 16 : 8;
  return st[2] == 1 && D % 4 == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 &&
         reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

bool out_ok(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == NGDN2_F32 ? 16 : 8) == 0; }

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
constexpr int kFwdSteps = Tile<8, 8>::kSteps, kBwdSteps = Tile<8, 4>::kSteps;
constexpr int kWideSteps = Tile<32, 4>::kSteps;

struct Shape {
  int row_strips, channels;
  int64_t strips, tiles;
};

Shape shape_of(const ngdn2_scan_args* a, int steps) {
  Shape s;
  s.channels = a->T <= kWideSteps ? 128 : 32;
  s.row_strips = int((a->D + s.channels - 1) / s.channels);
  s.strips = int64_t(a->B) * s.row_strips;
  s.tiles = a->T <= kWideSteps ? 1 : (a->T + steps - 1) / steps;
  return s;
}

int validate_scan(const ngdn2_scan_args* a, bool outputs) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->g_dtype)) return NGDN2_ERR_DTYPE;
  // The strips of all tiles are counted in 31 bits.
  if (a->B < 1 || a->T < 1 || a->D < 1 || a->T >= (int64_t(1) << 31) ||
      a->D >= (int64_t(1) << 31) ||
      (a->D + 31) / 32 * ((a->T + kBwdSteps - 1) / kBwdSteps) > ((int64_t(1) << 31) - 1) / a->B)
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

size_t workspace_bytes(const ngdn2_scan_args* a) {
  const Shape f = shape_of(a, kFwdSteps), b = shape_of(a, kBwdSteps);
  const size_t x = chain_bytes(f.strips, f.tiles, f.channels),
               y = chain_bytes(b.strips, b.tiles, b.channels);
  return x > y ? x : y;
}

// The chain of one launch, its counter and state words cleared.
int start_chain(const Shape& s, void* ws, size_t ws_bytes, cudaStream_t st, Chain* c) {
  const size_t need = chain_bytes(s.strips, s.tiles, s.channels);
  if (need && (!ws || ws_bytes < need)) return NGDN2_ERR_WORKSPACE;
  *c = make_chain(ws, s.strips, s.tiles, s.channels);
  if (need && cudaMemsetAsync(c->ticket, 0, chain_flag_bytes(s.strips, s.tiles), st) != cudaSuccess)
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
  *bytes = workspace_bytes(a);
  return NGDN2_OK;
}

NGDN2_API int ngdn2_scan(const ngdn2_scan_args* a, void* stream) {
  int rc = validate_scan(a, true);
  if (rc != NGDN2_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Shape s = shape_of(a, kFwdSteps);
  Chain chain;
  rc = start_chain(s, a->workspace, a->workspace_bytes, st, &chain);
  if (rc != NGDN2_OK) return rc;
  const bool vec = vec_ok(a->x, a->x_dtype, a->x_stride, a->D) &&
                   vec_ok(a->g, a->g_dtype, a->g_stride, a->D) && out_ok(a->h, a->x_dtype) &&
                   out_ok(a->carries, NGDN2_F32);
  const unsigned grid = unsigned(s.strips * s.tiles);
  const cudaError_t err = by_types(a->x_dtype, a->g_dtype, [&](auto X, auto G) {
    constexpr int XT = decltype(X)::value, GT = decltype(G)::value;
    if (s.channels == 128) {
      if (vec) scan_kernel<XT, GT, true, 32, 4><<<grid, kThreads, 0, st>>>(*a, chain, s.row_strips);
      else scan_kernel<XT, GT, false, 32, 4><<<grid, kThreads, 0, st>>>(*a, chain, s.row_strips);
    } else {
      if (vec) scan_kernel<XT, GT, true, 8, 8><<<grid, kThreads, 0, st>>>(*a, chain, s.row_strips);
      else scan_kernel<XT, GT, false, 8, 8><<<grid, kThreads, 0, st>>>(*a, chain, s.row_strips);
    }
    return cudaGetLastError();
  });
  return err == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_scan_bwd(const ngdn2_scan_bwd_args* p, void* stream) {
  int rc = validate_scan_bwd(p);
  if (rc != NGDN2_OK) return rc;
  const ngdn2_scan_args* a = &p->fwd;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Shape s = shape_of(a, kBwdSteps);
  Chain chain;
  rc = start_chain(s, p->workspace, p->workspace_bytes, st, &chain);
  if (rc != NGDN2_OK) return rc;
  const bool vec = vec_ok(a->x, a->x_dtype, a->x_stride, a->D) &&
                   vec_ok(a->g, a->g_dtype, a->g_stride, a->D) &&
                   vec_ok(p->d_h, p->d_h_dtype, p->d_h_stride, a->D) && out_ok(p->dx, a->x_dtype) &&
                   out_ok(p->dg, a->g_dtype);
  const unsigned grid = unsigned(s.strips * s.tiles);
  const cudaError_t err = by_types(a->x_dtype, a->g_dtype, [&](auto X, auto G) {
    constexpr int XT = decltype(X)::value, GT = decltype(G)::value;
    if (s.channels == 128) {
      if (vec) scan_bwd_kernel<XT, GT, true, 32, 4><<<grid, kThreads, 0, st>>>(*p, chain, s.row_strips);
      else scan_bwd_kernel<XT, GT, false, 32, 4><<<grid, kThreads, 0, st>>>(*p, chain, s.row_strips);
    } else {
      if (vec) scan_bwd_kernel<XT, GT, true, 8, 4><<<grid, kThreads, 0, st>>>(*p, chain, s.row_strips);
      else scan_bwd_kernel<XT, GT, false, 8, 4><<<grid, kThreads, 0, st>>>(*p, chain, s.row_strips);
    }
    return cudaGetLastError();
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
