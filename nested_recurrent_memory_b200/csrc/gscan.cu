// Gated linear recurrence, per (batch row, channel):
//   h_t = e^{g_t} h_{t-1} + x_t
// and its backward
//   u_t = dh_t + e^{g_{t+1}} u_{t+1},  dx = u,  dg_t = u_t e^{g_t} h_{t-1},  dh_0 = e^{g_1} u_1.
// The state is fp32. Written with c_t = e^{g_t} u_t the backward is itself
// such a recurrence, from the end: c_t = e^{g_t} (dh_t + c_{t+1}), c_{T+1} = d_final.

#include "common.cuh"

using namespace ngdn2;

namespace {

constexpr int kThreads = 128;

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

int64_t num_chunks(int64_t T) { return (T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK; }

// One thread a channel, token by token.
__global__ void __launch_bounds__(kThreads) scan_kernel(ngdn2_scan_args a) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= int64_t(a.B) * a.D) return;
  const int64_t b = i / a.D, d = i % a.D, NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
  float h = a.initial_state ? a.initial_state[i] : 0.f;
  for (int64_t t = 0; t < a.T; ++t) {
    if (a.carries && t % NGDN2_SCAN_CHUNK == 0)
      a.carries[(b * NC + t / NGDN2_SCAN_CHUNK) * a.D + d] = h;
    const float x = load_elem(a.x, b * a.x_stride[0] + t * a.x_stride[1] + d * a.x_stride[2], a.x_dtype);
    const float g = load_elem(a.g, b * a.g_stride[0] + t * a.g_stride[1] + d * a.g_stride[2], a.g_dtype);
    h = fmaf(expf(g), h, x);
    store_elem(a.h, (b * a.T + t) * a.D + d, h, a.x_dtype);
  }
  if (a.final_state) a.final_state[i] = h;
}

__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(ngdn2_scan_bwd_args p) {
  const ngdn2_scan_args& a = p.fwd;
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= int64_t(a.B) * a.D) return;
  const int64_t b = i / a.D, d = i % a.D, NC = (a.T + NGDN2_SCAN_CHUNK - 1) / NGDN2_SCAN_CHUNK;
  float c = p.d_final ? p.d_final[i] : 0.f;
  float prev[NGDN2_SCAN_CHUNK];
  for (int64_t n = NC - 1; n >= 0; --n) {
    const int64_t t0 = n * NGDN2_SCAN_CHUNK;
    const int len = int(a.T - t0 < NGDN2_SCAN_CHUNK ? a.T - t0 : NGDN2_SCAN_CHUNK);
    auto decay = [&](int64_t t) {
      return expf(load_elem(a.g, b * a.g_stride[0] + t * a.g_stride[1] + d * a.g_stride[2], a.g_dtype));
    };
    float h = a.carries[(b * NC + n) * a.D + d];
    for (int j = 0; j < len; ++j) {
      prev[j] = h;
      h = fmaf(decay(t0 + j), h,
               load_elem(a.x, b * a.x_stride[0] + (t0 + j) * a.x_stride[1] + d * a.x_stride[2], a.x_dtype));
    }
    for (int j = len - 1; j >= 0; --j) {
      const int64_t t = t0 + j, o = (b * a.T + t) * a.D + d;
      const float u = c + load_elem(p.d_h, b * p.d_h_stride[0] + t * p.d_h_stride[1] +
                                               d * p.d_h_stride[2], p.d_h_dtype);
      c = decay(t) * u;
      store_elem(p.dx, o, u, a.x_dtype);
      store_elem(p.dg, o, c * prev[j], a.g_dtype);
    }
  }
  if (p.d_initial) p.d_initial[i] = c;
}

__global__ void __launch_bounds__(kThreads) scan_step_kernel(ngdn2_scan_step_args a) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= int64_t(a.B) * a.D) return;
  const int64_t b = i / a.D, d = i % a.D;
  const float x = load_elem(a.x, b * a.x_stride[0] + d * a.x_stride[1], a.x_dtype);
  const float g = load_elem(a.g, b * a.g_stride[0] + d * a.g_stride[1], a.g_dtype);
  const float h = fmaf(expf(g), a.state_in[i], x);
  a.state_out[i] = h;
  store_elem(a.h, i, h, a.x_dtype);
}

int validate_scan(const ngdn2_scan_args* a, bool outputs) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->g_dtype)) return NGDN2_ERR_DTYPE;
  if (a->B < 1 || a->T < 1 || a->D < 1 || a->T >= (int64_t(1) << 31) ||
      a->D >= (int64_t(1) << 31) || int64_t(a->B) * a->D >= (int64_t(1) << 36))
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

}  // namespace

extern "C" {

NGDN2_API size_t ngdn2_sizeof_scan_args(void) { return sizeof(ngdn2_scan_args); }
NGDN2_API size_t ngdn2_sizeof_scan_bwd_args(void) { return sizeof(ngdn2_scan_bwd_args); }
NGDN2_API size_t ngdn2_sizeof_scan_step_args(void) { return sizeof(ngdn2_scan_step_args); }

NGDN2_API int ngdn2_scan_workspace_size(const ngdn2_scan_args* a, size_t* bytes) {
  const int rc = validate_scan(a, false);
  if (rc != NGDN2_OK) return rc;
  if (!bytes) return NGDN2_ERR_NULL;
  *bytes = 0;
  return NGDN2_OK;
}

NGDN2_API int ngdn2_scan(const ngdn2_scan_args* a, void* stream) {
  const int rc = validate_scan(a, true);
  if (rc != NGDN2_OK) return rc;
  const int64_t n = int64_t(a->B) * a->D;
  scan_kernel<<<unsigned((n + kThreads - 1) / kThreads), kThreads, 0,
                static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_scan_bwd(const ngdn2_scan_bwd_args* a, void* stream) {
  const int rc = validate_scan_bwd(a);
  if (rc != NGDN2_OK) return rc;
  const int64_t n = int64_t(a->fwd.B) * a->fwd.D;
  scan_bwd_kernel<<<unsigned((n + kThreads - 1) / kThreads), kThreads, 0,
                    static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

NGDN2_API int ngdn2_scan_step(const ngdn2_scan_step_args* a, void* stream) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->g_dtype)) return NGDN2_ERR_DTYPE;
  const int64_t n = int64_t(a->B) * a->D;
  if (a->B < 1 || a->D < 1 || a->D >= (int64_t(1) << 31) || n >= (int64_t(1) << 36))
    return NGDN2_ERR_SHAPE;
  if (!a->x || !a->g || !a->state_in || !a->state_out || !a->h) return NGDN2_ERR_NULL;
  scan_step_kernel<<<unsigned((n + kThreads - 1) / kThreads), kThreads, 0,
                     static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
