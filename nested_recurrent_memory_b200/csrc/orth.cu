// Newton-Schulz orthogonalisation of weight updates: X_0 = G / (|G|_F + eps),
// then X <- a X + (b A + c A A) X with A = X X^T, on the smaller side of G
// (a tall G is worked on transposed). fp32 products and sums.

#include <math.h>

#include "common.cuh"

using namespace ngdn2;

namespace {

constexpr int kThreads = 256;

bool dtype_ok(int d) { return d == NGDN2_F32 || d == NGDN2_BF16 || d == NGDN2_F16; }

struct OrthLayout {
  int64_t m, n;      // smaller and larger side
  int64_t x, y, A, Bm, inv, total;  // float offsets
};

OrthLayout layout(const ngdn2_orth_args* a) {
  OrthLayout L;
  L.m = a->rows < a->cols ? a->rows : a->cols;
  L.n = a->rows < a->cols ? a->cols : a->rows;
  L.x = 0;
  L.y = L.x + a->batch * L.m * L.n;
  L.A = L.y + a->batch * L.m * L.n;
  L.Bm = L.A + a->batch * L.m * L.m;
  L.inv = L.Bm + a->batch * L.m * L.m;
  L.total = L.inv + a->batch;
  return L;
}

// inv[b] = 1 / (|G_b|_F + eps); squares summed in 64 bits, so that neither
// large nor small gradients leave the range.
__global__ void __launch_bounds__(kThreads) norm_kernel(ngdn2_orth_args a, float* inv) {
  __shared__ double red[kThreads];
  const int64_t b = blockIdx.x;
  double s = 0.0;
  for (int64_t e = threadIdx.x; e < a.rows * a.cols; e += kThreads) {
    const double x = load_elem(a.update, b * a.update_stride[0] + (e / a.cols) * a.update_stride[1] +
                                             (e % a.cols) * a.update_stride[2], a.dtype);
    s += x * x;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) inv[b] = float(1.0 / (sqrt(red[0]) + double(a.eps)));
}

__global__ void __launch_bounds__(kThreads)
load_kernel(ngdn2_orth_args a, int64_t m, int64_t n, const float* inv, float* x) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * m * n) return;
  const int64_t b = i / (m * n), r = i / n % m, c = i % n;
  const bool tall = a.rows > a.cols;
  x[i] = inv[b] * load_elem(a.update, b * a.update_stride[0] + (tall ? c : r) * a.update_stride[1] +
                                          (tall ? r : c) * a.update_stride[2], a.dtype);
}

__global__ void __launch_bounds__(kThreads)
store_kernel(ngdn2_orth_args a, int64_t m, int64_t n, const float* x) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * m * n) return;
  const int64_t b = i / (m * n), r = i / n % m, c = i % n;
  const bool tall = a.rows > a.cols;
  store_elem(a.out, b * m * n + (tall ? c * m + r : r * n + c), x[i], a.out_dtype);
}

// C = alpha P Q + beta R for row-major matrices of a batch: P [M x Kd],
// Q [Kd x N] (QT: Q [N x Kd] transposed), R and C [M x N].
template <bool QT>
__global__ void __launch_bounds__(kGemmThreads)
product_kernel(int64_t M, int64_t N, int64_t Kd, const float* P, const float* Q, const float* R,
               float* C, float alpha, float beta) {
  __shared__ float ps[16][65], qs[16][65];
  const int tid = threadIdx.x, tm = tid / 16, tn = tid % 16;
  const int64_t b = blockIdx.z, m0 = int64_t(blockIdx.y) * 64, n0 = int64_t(blockIdx.x) * 64;
  P += b * M * Kd;
  Q += b * Kd * N;
  C += b * M * N;
  if (R) R += b * M * N;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < Kd; k0 += 16) {
    for (int e = tid; e < 64 * 16; e += kGemmThreads) {
      const int k = e % 16, r = e / 16;
      ps[k][r] = m0 + r < M && k0 + k < Kd ? P[(m0 + r) * Kd + k0 + k] : 0.f;
      if (QT) qs[k][r] = n0 + r < N && k0 + k < Kd ? Q[(n0 + r) * Kd + k0 + k] : 0.f;
    }
    if (!QT)
      for (int e = tid; e < 64 * 16; e += kGemmThreads) {
        const int c = e % 64, k = e / 64;
        qs[k][c] = n0 + c < N && k0 + k < Kd ? Q[(k0 + k) * N + n0 + c] : 0.f;
      }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(ps[k][tm + 16 * i], qs[k][tn + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + tm + 16 * i, c = n0 + tn + 16 * j;
      if (r < M && c < N)
        C[r * N + c] = alpha * acc[i][j] + (R ? beta * R[r * N + c] : 0.f);
    }
}

// The scalar iteration s <- s (a + b s^2 + c s^4) from every start in [0, 1]
// (a grid) has to stay in [0, 4].
bool coefficients_ok(const ngdn2_orth_args* a) {
  for (int i = 0; i <= 1024; ++i) {
    double s = i / 1024.0;
    for (int k = 0; k < a->steps; ++k) {
      const double q = s * s;
      s *= a->coef[0] + q * (a->coef[1] + q * a->coef[2]);
      if (!(s >= -4.0 && s <= 4.0)) return false;
    }
  }
  return true;
}

int validate_orth(const ngdn2_orth_args* a) {
  if (!a) return NGDN2_ERR_NULL;
  if (a->abi_version != NGDN2_ABI_VERSION) return NGDN2_ERR_ABI;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype)) return NGDN2_ERR_DTYPE;
  if (a->batch < 1 || a->rows < 1 || a->cols < 1 || a->batch > 65535 || a->rows > (1 << 20) ||
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
  *bytes = size_t(layout(a).total) * sizeof(float);
  return NGDN2_OK;
}

NGDN2_API int ngdn2_orth(const ngdn2_orth_args* a, void* stream) {
  const int rc = validate_orth(a);
  if (rc != NGDN2_OK) return rc;
  const OrthLayout L = layout(a);
  if (!a->workspace || a->workspace_bytes < size_t(L.total) * sizeof(float))
    return NGDN2_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* ws = static_cast<float*>(a->workspace);
  float *x = ws + L.x, *y = ws + L.y, *A = ws + L.A, *Bm = ws + L.Bm;
  const unsigned flat = unsigned((a->batch * L.m * L.n + kThreads - 1) / kThreads);
  norm_kernel<<<unsigned(a->batch), kThreads, 0, st>>>(*a, ws + L.inv);
  load_kernel<<<flat, kThreads, 0, st>>>(*a, L.m, L.n, ws + L.inv, x);
  const unsigned bm = unsigned((L.m + 63) / 64), bn = unsigned((L.n + 63) / 64);
  const dim3 small(bm, bm, unsigned(a->batch)), wide(bn, bm, unsigned(a->batch));
  for (int k = 0; k < a->steps; ++k) {
    product_kernel<true><<<small, kGemmThreads, 0, st>>>(L.m, L.m, L.n, x, x, nullptr, A, 1.f, 0.f);
    product_kernel<true><<<small, kGemmThreads, 0, st>>>(L.m, L.m, L.m, A, A, A, Bm, a->coef[2], a->coef[1]);
    product_kernel<false><<<wide, kGemmThreads, 0, st>>>(L.m, L.n, L.m, Bm, x, x, y, 1.f, a->coef[0]);
    float* t = x;
    x = y;
    y = t;
  }
  store_kernel<<<flat, kThreads, 0, st>>>(*a, L.m, L.n, x);
  return cudaGetLastError() == cudaSuccess ? NGDN2_OK : NGDN2_ERR_CUDA;
}

}  // extern "C"
