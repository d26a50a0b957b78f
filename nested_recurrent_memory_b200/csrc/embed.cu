// Scaled embedding lookup and its gradient:
//   out[n]     = scale * weight[ids[n]]
//   dweight[v] = scale * sum over {n : ids[n] = v} of d_out[n]
// Products and sums in fp32, rounded once to the output's type.

#include "common.cuh"

using namespace ngdn2;

namespace {

constexpr int kThreads = 256;

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

__device__ __forceinline__ int64_t load_id(const void* ids, int i32, int64_t n) {
  return i32 ? int64_t(reinterpret_cast<const int32_t*>(ids)[n])
             : reinterpret_cast<const int64_t*>(ids)[n];
}

// A token a CTA. A token outside [0, V) reads nothing: its row is NaN, so
// that it cannot pass as a result, and the status word says why.
__global__ void __launch_bounds__(kThreads) embed_kernel(ngdn2_embed_args a) {
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    const int64_t v = load_id(a.ids, a.ids_i32, n);
    const bool ok = v >= 0 && v < a.V;
    if (!ok && threadIdx.x == 0) atomicOr(a.status, NGDN2_STATUS_BAD_INDEX);
    for (int64_t d = threadIdx.x; d < a.D; d += kThreads) {
      const float x = ok ? a.scale * load_elem(a.weight, v * a.weight_stride + d, a.dtype)
                         : __int_as_float(0x7fc00000);
      store_elem(a.out, n * a.D + d, x, a.dtype);
    }
  }
}

// Sixteen rows of dweight by 256 columns a CTA: all tokens are looked
// through in order, and those of the CTA's rows added to their row.
constexpr int kRows = 16;

__global__ void __launch_bounds__(kThreads) embed_bwd_kernel(ngdn2_embed_bwd_args a) {
  __shared__ float acc[kRows][kThreads];
  __shared__ int list[kThreads];
  __shared__ int count[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t v0 = int64_t(blockIdx.x) * kRows, d = int64_t(blockIdx.y) * kThreads + tid;
  for (int r = 0; r < kRows; ++r) acc[r][tid] = 0.f;
  for (int64_t n0 = 0; n0 < a.N; n0 += kThreads) {
    const int64_t n = n0 + tid;
    int64_t v = n < a.N ? load_id(a.ids, a.ids_i32, n) : -1;
    if (n < a.N && (v < 0 || v >= a.V)) atomicOr(a.status, NGDN2_STATUS_BAD_INDEX);
    const bool mine = n < a.N && v >= v0 && v < v0 + kRows && v < a.V && v != a.padding_idx;
    const unsigned m = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) count[warp] = __popc(m);
    __syncthreads();
    int at = __popc(m & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += count[w];
      total += count[w];
    }
    if (mine) list[at] = tid * kRows + int(v - v0);
    __syncthreads();
    if (d < a.D)
      for (int i = 0; i < total; ++i) {
        const int e = list[i];
        acc[e % kRows][tid] += load_elem(a.d_out, (n0 + e / kRows) * a.d_stride + d, a.dtype);
      }
    __syncthreads();
  }
  if (d < a.D)
    for (int r = 0; r < kRows; ++r)
      if (v0 + r < a.V) store_elem(a.dweight, (v0 + r) * a.D + d, a.scale * acc[r][tid], a.out_dtype);
}

int validate_embed(const ngdn2_embed_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype)) return NGDN2_ERR_DTYPE;
  if (a->N < 0 || a->V < 1 || a->D < 1 || a->N >= (int64_t(1) << 31) ||
      a->V >= (int64_t(1) << 31) || a->weight_stride < 0)
    return NGDN2_ERR_SHAPE;
  if (!a->weight || !a->status || (a->N > 0 && (!a->ids || !a->out))) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

int validate_embed_bwd(const ngdn2_embed_bwd_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype)) return NGDN2_ERR_DTYPE;
  if (a->N < 0 || a->V < 1 || a->D < 1 || a->N >= (int64_t(1) << 31) ||
      a->V >= (int64_t(1) << 31) || a->d_stride < 0)
    return NGDN2_ERR_SHAPE;
  if (!a->dweight || !a->status || (a->N > 0 && (!a->ids || !a->d_out))) return NGDN2_ERR_NULL;
  return NGDN2_OK;
}

}  // namespace

extern "C" {

NGDN2_API size_t ngdn2_sizeof_embed_args(void) { return sizeof(ngdn2_embed_args); }
NGDN2_API size_t ngdn2_sizeof_embed_bwd_args(void) { return sizeof(ngdn2_embed_bwd_args); }

NGDN2_API int ngdn2_embed(const ngdn2_embed_args* a, void* stream) {
  const int rc = validate_embed(a);
  if (rc != NGDN2_OK) return rc;
  if (a->N == 0) return NGDN2_OK;
  const unsigned grid = unsigned(a->N < (1 << 20) ? a->N : (1 << 20));
  embed_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_embed_bwd_workspace_size(const ngdn2_embed_bwd_args* a, size_t* bytes) {
  const int rc = validate_embed_bwd(a);
  if (rc != NGDN2_OK) return rc;
  if (!bytes) return NGDN2_ERR_NULL;
  *bytes = 0;
  return NGDN2_OK;
}

NGDN2_API int ngdn2_embed_bwd(const ngdn2_embed_bwd_args* a, void* stream) {
  const int rc = validate_embed_bwd(a);
  if (rc != NGDN2_OK) return rc;
  const dim3 grid(unsigned((a->V + kRows - 1) / kRows), unsigned((a->D + kThreads - 1) / kThreads));
  if (grid.y > 65535) return NGDN2_ERR_SHAPE;
  embed_bwd_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
