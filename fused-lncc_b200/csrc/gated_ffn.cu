// The gated feed-forward block, forward and backward:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu
//   dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// One 64 x 64 tile of a product a block, 16 of its inner axis at a time through shared memory, fp32 throughout.
#include "lncc_block.cuh"

namespace lncc {
namespace ffn {

using namespace blk;

constexpr int kTile = 64, kInner = 16;

// out[m][n] = sum_k a[m*a_m + k*a_k] * b[n*b_n + k*b_k], and where a2 is given the same sum of a2 and b2 on top
template <typename TA, typename TB, typename TO>
__global__ void __launch_bounds__(256) product_kernel(const TA* a, const TA* a2, int64_t a_m, int64_t a_k, const TB* b,
                                                      const TB* b2, int64_t b_n, int64_t b_k, TO* out, int64_t M,
                                                      int64_t N, int64_t K) {
  __shared__ float sa[kInner][kTile + 1], sb[kInner][kTile + 1];
  const int64_t m0 = int64_t(blockIdx.x) * kTile, n0 = int64_t(blockIdx.y) * kTile;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int pair = 0; pair < (a2 ? 2 : 1); pair++) {
    for (int64_t k0 = 0; k0 < K; k0 += kInner) {
      for (int i = threadIdx.x; i < kTile * kInner; i += 256) {
        const int r = i / kInner, k = i % kInner;
        sa[k][r] = m0 + r < M && k0 + k < K ? to_f((pair ? a2 : a)[(m0 + r) * a_m + (k0 + k) * a_k]) : 0.f;
        sb[k][r] = n0 + r < N && k0 + k < K ? to_f((pair ? b2 : b)[(n0 + r) * b_n + (k0 + k) * b_k]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kInner; k++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] += sa[k][ty * 4 + i] * sb[k][tx * 4 + j];
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < M && n < N && LNCC_IN(m * N + n, 1, M * N)) out[m * N + n] = from_f<TO>(acc[i][j]);
    }
}

// act(g) and act'(g)
__device__ __forceinline__ void activate(int act, float g, float& a, float& da) {
  if (act == LNCC_ACT_RELU) {
    a = g < 0.f ? 0.f : g;
    da = g > 0.f ? 1.f : 0.f;
  } else if (act == LNCC_ACT_SILU) {
    const float p = 1.f / (1.f + expf(-g));
    a = g * p;
    da = p * (1.f + g * (1.f - p));
  } else {
    const float p = 0.5f * (1.f + erff(g * 0.70710678f));
    a = g * p;
    da = p + g * expf(-0.5f * g * g) * 0.39894228f;
  }
}

__global__ void __launch_bounds__(256) hidden_kernel(int act, float* g, float* u, float* h, const float* dh, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    float a, da;
    activate(act, g[i], a, da);
    const float up = u[i];
    h[i] = a * up;
    if (dh) {
      g[i] = dh[i] * up * da;
      u[i] = dh[i] * a;
    }
  }
}

template <typename TA, typename TB, typename TO>
static void product(const TA* a, const TA* a2, int64_t a_m, int64_t a_k, const TB* b, const TB* b2, int64_t b_n,
                    int64_t b_k, TO* out, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
  product_kernel<<<dim3(unsigned(ceil_div(M, kTile)), unsigned(ceil_div(N, kTile))), 256, 0, st>>>(
      a, a2, a_m, a_k, b, b2, b_n, b_k, out, M, N, K);
}

struct Args {
  const void *x, *wg, *wu, *wd, *dy;
  int64_t x_stride, dy_stride, M, K, F, N;
  int act;
  void *y, *dx, *dwg, *dwu, *dwd;
  float *g, *u, *h, *dh;
};

template <typename T> static void forward(const Args& p, cudaStream_t st) {
  const T *x = static_cast<const T*>(p.x), *wg = static_cast<const T*>(p.wg), *wu = static_cast<const T*>(p.wu);
  const T *wd = static_cast<const T*>(p.wd), *none = nullptr;
  const float* nof = nullptr;
  product(x, none, p.x_stride, 1, wg, none, p.K, 1, p.g, p.M, p.F, p.K, st);
  product(x, none, p.x_stride, 1, wu, none, p.K, 1, p.u, p.M, p.F, p.K, st);
  hidden_kernel<<<sm_count() * 4, 256, 0, st>>>(p.act, p.g, p.u, p.h, nullptr, p.M * p.F);
  product((const float*)p.h, nof, p.F, 1, wd, none, p.F, 1, static_cast<T*>(p.y), p.M, p.N, p.F, st);
}
template <typename T> static void backward(const Args& p, cudaStream_t st) {
  const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy), *wd = static_cast<const T*>(p.wd);
  const T *wg = static_cast<const T*>(p.wg), *wu = static_cast<const T*>(p.wu), *none = nullptr;
  const float *nof = nullptr, *g = p.g, *u = p.u;
  product(x, none, p.x_stride, 1, wg, none, p.K, 1, p.g, p.M, p.F, p.K, st);
  product(x, none, p.x_stride, 1, wu, none, p.K, 1, p.u, p.M, p.F, p.K, st);
  product(dy, none, p.dy_stride, 1, wd, none, 1, p.F, p.dh, p.M, p.F, p.N, st);
  hidden_kernel<<<sm_count() * 4, 256, 0, st>>>(p.act, p.g, p.u, p.h, p.dh, p.M * p.F);
  if (p.dx) product(g, u, p.F, 1, wg, wu, 1, p.K, static_cast<T*>(p.dx), p.M, p.K, p.F, st);
  if (p.dwg) product(g, nof, 1, p.F, x, none, 1, p.x_stride, static_cast<T*>(p.dwg), p.F, p.K, p.M, st);
  if (p.dwu) product(u, nof, 1, p.F, x, none, 1, p.x_stride, static_cast<T*>(p.dwu), p.F, p.K, p.M, st);
  if (p.dwd) product(dy, none, 1, p.dy_stride, (const float*)p.h, nof, 1, p.F, static_cast<T*>(p.dwd), p.N, p.F, p.M, st);
}

static int check_sizes(int dtype, int act, int64_t M, int64_t K, int64_t F, int64_t N) {
  if (!valid_dtype(dtype)) return LNCC_ERR_DTYPE;
  if (act < LNCC_ACT_SILU || act > LNCC_ACT_RELU || M < 0 || K < 1 || F < 1 || N < 1) return LNCC_ERR_BAD_ARG;
  if (K > (1 << 20) || F > (1 << 20) || N > (1 << 20) || M > INT32_MAX / 2) return LNCC_ERR_TOO_LARGE;
  return LNCC_OK;
}
static bool good(const void* p, int dtype) { return p && aligned(p, elem_size(dtype)); }

}  // namespace ffn
}  // namespace lncc

using namespace lncc;

extern "C" {

size_t lncc_gated_ffn_scratch_bytes(int64_t M, int64_t K, int64_t F, int64_t N, int dtype, int backward) {
  if (ffn::check_sizes(dtype, 0, M, K, F, N) != LNCC_OK) return 0;
  return size_t(backward ? 4 : 3) * size_t(M) * size_t(F) * sizeof(float);
}

int lncc_gated_ffn_forward(const void* x, int64_t x_stride, const void* w_gate, const void* w_up, const void* w_down,
                           int dtype, int act, int64_t M, int64_t K, int64_t F, int64_t N, void* y, void* scratch,
                           size_t scratch_bytes, cudaStream_t stream) {
  const int st = ffn::check_sizes(dtype, act, M, K, F, N);
  if (st != LNCC_OK) return st;
  if (M == 0) return LNCC_OK;
  if (!ffn::good(x, dtype) || !ffn::good(w_gate, dtype) || !ffn::good(w_up, dtype) || !ffn::good(w_down, dtype) ||
      !ffn::good(y, dtype) || (x_stride < K && M > 1))
    return LNCC_ERR_BAD_ARG;
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < lncc_gated_ffn_scratch_bytes(M, K, F, N, dtype, 0))
    return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  ffn::Args p = {};
  p.x = x, p.x_stride = x_stride, p.wg = w_gate, p.wu = w_up, p.wd = w_down, p.act = act, p.y = y;
  p.M = M, p.K = K, p.F = F, p.N = N;
  p.g = static_cast<float*>(scratch), p.u = p.g + M * F, p.h = p.u + M * F;
  if (dtype == LNCC_F32) ffn::forward<float>(p, stream);
  else if (dtype == LNCC_BF16) ffn::forward<__nv_bfloat16>(p, stream);
  else ffn::forward<__half>(p, stream);
  return blk::check_end(stream);
}

int lncc_gated_ffn_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* w_gate,
                            const void* w_up, const void* w_down, int dtype, int act, int64_t M, int64_t K, int64_t F,
                            int64_t N, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* scratch,
                            size_t scratch_bytes, cudaStream_t stream) {
  const int st = ffn::check_sizes(dtype, act, M, K, F, N);
  if (st != LNCC_OK) return st;
  void* const grads[4] = {dx, dw_gate, dw_up, dw_down};
  for (void* g : grads)
    if (!blk::aligned(g, blk::elem_size(dtype))) return LNCC_ERR_BAD_ARG;
  if (M == 0) {  // sums over no tokens
    const size_t up = size_t(F) * K * blk::elem_size(dtype), down = size_t(N) * F * blk::elem_size(dtype);
    for (int i = 1; i < 4; i++)
      if (grads[i] && cudaMemsetAsync(grads[i], 0, i < 3 ? up : down, stream) != cudaSuccess) return LNCC_ERR_CUDA;
    return LNCC_OK;
  }
  if (!ffn::good(x, dtype) || !ffn::good(w_gate, dtype) || !ffn::good(w_up, dtype) || !ffn::good(w_down, dtype) ||
      !ffn::good(dy, dtype) || (x_stride < K && M > 1) || (dy_stride < N && M > 1))
    return LNCC_ERR_BAD_ARG;
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < lncc_gated_ffn_scratch_bytes(M, K, F, N, dtype, 1))
    return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  ffn::Args p = {};
  p.x = x, p.x_stride = x_stride, p.dy = dy, p.dy_stride = dy_stride, p.wg = w_gate, p.wu = w_up, p.wd = w_down;
  p.act = act, p.dx = dx, p.dwg = dw_gate, p.dwu = dw_up, p.dwd = dw_down, p.M = M, p.K = K, p.F = F, p.N = N;
  p.g = static_cast<float*>(scratch), p.u = p.g + M * F, p.h = p.u + M * F, p.dh = p.h + M * F;
  if (dtype == LNCC_F32) ffn::backward<float>(p, stream);
  else if (dtype == LNCC_BF16) ffn::backward<__nv_bfloat16>(p, stream);
  else ffn::backward<__half>(p, stream);
  return blk::check_end(stream);
}

}  // extern "C"
