// The gated linear recurrence over (B, T, C), forward and backward:
//
//   a_t = sigmoid(gate_t), h_t = a_t h_{t-1} + (1 - a_t) x_t, h_0 = state (or 0)
//   q_t = dh_t + a_{t+1} q_{t+1}, with dlast added to dh_T
//   dx_t = (1 - a_t) q_t, dgate_t = q_t (h_{t-1} - x_t) a_t (1 - a_t), dstate = a_1 q_1
//
// Steps compose: (A, S) after (A', S') is (A A', A S' + S), so T is cut into chunks of kChunk steps. A first kernel
// forms each chunk's (A, S) from a zero state, a second carries the state over the chunks, a third runs each chunk from
// its state. Backward the same runs from the end, and h is formed again from states that the forward pass kept every
// kKeep steps.
#include "lncc_block.cuh"

namespace lncc {
namespace scan {

using namespace blk;

constexpr int kChunk = 64, kKeep = 16, kThreads = 128;

struct Args {
  const void *x, *gate, *dh;
  int64_t x_b, x_t, gate_b, gate_t, dh_b, dh_t;  // strides in elements; time strides are negative for reverse scans
  void *h, *dx, *dgate;
  int64_t out_b, out_t;
  const float *state, *dlast;
  float *last, *dstate;
  float *kept;            // [B][ceil(T / kKeep)][C] states before steps 0, kKeep, ...
  float *agg_a, *agg_s;   // [B][chunks][C]
  int64_t B, T, C, chunks;
};

// a = sigmoid(g) and keep = 1 - a = sigmoid(-g), both to fp32 accuracy (1 - a would cancel for open gates).
__device__ __forceinline__ void gates(float g, float& a, float& keep) {
  const float e = expf(-fabsf(g)), r = 1.f / (1.f + e);
  a = g >= 0.f ? r : e * r;
  keep = g >= 0.f ? e * r : r;
  if (g != g) a = keep = g;
}

template <typename T> __global__ void __launch_bounds__(kThreads) sum_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, k = blockIdx.y, b = blockIdx.z;
  if (c >= p.C) return;
  const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b + c;
  const T* x = static_cast<const T*>(p.x) + b * p.x_b + c;
  float A = 1.f, S = 0.f;
  for (int64_t t = k * kChunk; t < min(p.T, (k + 1) * kChunk); t++) {
    float a, keep;
    gates(to_f(gate[t * p.gate_t]), a, keep);
    S = a * S + keep * to_f(x[t * p.x_t]);
    A *= a;
  }
  p.agg_a[(b * p.chunks + k) * p.C + c] = A;
  p.agg_s[(b * p.chunks + k) * p.C + c] = S;
}

// agg_s[k] becomes the state before chunk k.
__global__ void __launch_bounds__(kThreads) carry_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, b = blockIdx.y;
  if (c >= p.C) return;
  float h = p.state ? p.state[b * p.C + c] : 0.f;
  for (int64_t k = 0; k < p.chunks; k++) {
    const int64_t i = (b * p.chunks + k) * p.C + c;
    const float next = p.agg_a[i] * h + p.agg_s[i];
    p.agg_s[i] = h;
    h = next;
  }
  p.last[b * p.C + c] = h;
}

template <typename T> __global__ void __launch_bounds__(kThreads) run_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, k = blockIdx.y, b = blockIdx.z;
  if (c >= p.C) return;
  const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b + c;
  const T* x = static_cast<const T*>(p.x) + b * p.x_b + c;
  T* out = static_cast<T*>(p.h) + b * p.out_b + c;
  const int64_t keeps = (p.T + kKeep - 1) / kKeep;
  float h = p.agg_s[(b * p.chunks + k) * p.C + c];
  for (int64_t t = k * kChunk; t < min(p.T, (k + 1) * kChunk); t++) {
    if (p.kept && t % kKeep == 0) p.kept[(b * keeps + t / kKeep) * p.C + c] = h;
    float a, keep;
    gates(to_f(gate[t * p.gate_t]), a, keep);
    h = a * h + keep * to_f(x[t * p.x_t]);
    out[t * p.out_t] = from_f<T>(h);
  }
}

// backward: (A, S) of the chunk for what it hands on to the step before it, a_t q_t
template <typename T> __global__ void __launch_bounds__(kThreads) back_sum_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, k = blockIdx.y, b = blockIdx.z;
  if (c >= p.C) return;
  const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b + c;
  const T* dh = static_cast<const T*>(p.dh) + b * p.dh_b + c;
  float A = 1.f, S = 0.f;
  for (int64_t t = min(p.T, (k + 1) * kChunk) - 1; t >= k * kChunk; t--) {
    float a, keep;
    gates(to_f(gate[t * p.gate_t]), a, keep);
    S = a * (S + to_f(dh[t * p.dh_t]));
    A *= a;
  }
  p.agg_a[(b * p.chunks + k) * p.C + c] = A;
  p.agg_s[(b * p.chunks + k) * p.C + c] = S;
}

__global__ void __launch_bounds__(kThreads) back_carry_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, b = blockIdx.y;
  if (c >= p.C) return;
  float q = p.dlast ? p.dlast[b * p.C + c] : 0.f;
  for (int64_t k = p.chunks - 1; k >= 0; k--) {
    const int64_t i = (b * p.chunks + k) * p.C + c;
    const float next = p.agg_a[i] * q + p.agg_s[i];
    p.agg_s[i] = q;
    q = next;
  }
  if (p.dstate) p.dstate[b * p.C + c] = q;
}

template <typename T> __global__ void __launch_bounds__(kThreads) back_run_kernel(const Args p) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x, k = blockIdx.y, b = blockIdx.z;
  if (c >= p.C) return;
  const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b + c;
  const T* x = static_cast<const T*>(p.x) + b * p.x_b + c;
  const T* dh = static_cast<const T*>(p.dh) + b * p.dh_b + c;
  T* dx = static_cast<T*>(p.dx) + b * p.out_b + c;
  T* dgate = static_cast<T*>(p.dgate) + b * p.out_b + c;
  const int64_t keeps = (p.T + kKeep - 1) / kKeep;
  float q = p.agg_s[(b * p.chunks + k) * p.C + c];
  for (int64_t t0 = (min(p.T, (k + 1) * kChunk) - 1) / kKeep * kKeep; t0 >= k * kChunk; t0 -= kKeep) {
    float a[kKeep], keep[kKeep], v[kKeep], before[kKeep];
    float h = p.kept[(b * keeps + t0 / kKeep) * p.C + c];
#pragma unroll
    for (int i = 0; i < kKeep; i++) {
      const int64_t t = t0 + i;
      if (t < p.T) {
        gates(to_f(gate[t * p.gate_t]), a[i], keep[i]);
        v[i] = to_f(x[t * p.x_t]);
        before[i] = h;
        h = a[i] * h + keep[i] * v[i];
      }
    }
#pragma unroll
    for (int i = kKeep - 1; i >= 0; i--) {
      const int64_t t = t0 + i;
      if (t < p.T) {
        q += to_f(dh[t * p.dh_t]);
        dx[t * p.out_t] = from_f<T>(keep[i] * q);
        dgate[t * p.out_t] = from_f<T>(q * (before[i] - v[i]) * (a[i] * keep[i]));
        q *= a[i];
      }
    }
  }
}

// T = 0: the state passes through.
__global__ void __launch_bounds__(kThreads) pass_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

template <typename T> static void forward(const Args& p, cudaStream_t st) {
  const dim3 grid(unsigned(ceil_div(p.C, kThreads)), unsigned(p.chunks), unsigned(p.B));
  sum_kernel<T><<<grid, kThreads, 0, st>>>(p);
  carry_kernel<<<dim3(grid.x, grid.z), kThreads, 0, st>>>(p);
  run_kernel<T><<<grid, kThreads, 0, st>>>(p);
}
template <typename T> static void backward(const Args& p, cudaStream_t st) {
  const dim3 grid(unsigned(ceil_div(p.C, kThreads)), unsigned(p.chunks), unsigned(p.B));
  back_sum_kernel<T><<<grid, kThreads, 0, st>>>(p);
  back_carry_kernel<<<dim3(grid.x, grid.z), kThreads, 0, st>>>(p);
  back_run_kernel<T><<<grid, kThreads, 0, st>>>(p);
}

static int check_sizes(int dtype, int64_t B, int64_t T, int64_t C) {
  if (!valid_dtype(dtype)) return LNCC_ERR_DTYPE;
  if (B < 0 || T < 0 || C < 1) return LNCC_ERR_BAD_ARG;
  if (B > 65535 || T > int64_t(65535) * kChunk || C > (1 << 24)) return LNCC_ERR_TOO_LARGE;
  return LNCC_OK;
}
static bool good(const void* p, int dtype) { return p && aligned(p, elem_size(dtype)); }

}  // namespace scan
}  // namespace lncc

using namespace lncc;

extern "C" {

size_t lncc_gated_scan_kept_bytes(int64_t B, int64_t T, int64_t C) {
  if (scan::check_sizes(0, B, T, C) != LNCC_OK) return 0;
  return size_t(B) * size_t(blk::ceil_div(T, scan::kKeep)) * size_t(C) * sizeof(float);
}

size_t lncc_gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t C) {
  if (scan::check_sizes(0, B, T, C) != LNCC_OK) return 0;
  return 2 * size_t(B) * size_t(blk::ceil_div(T, scan::kChunk)) * size_t(C) * sizeof(float);
}

int lncc_gated_scan_forward(const void* x, int64_t x_b, int64_t x_t, const void* gate, int64_t gate_b, int64_t gate_t,
                            const float* state, int dtype, int64_t B, int64_t T, int64_t C, int reverse, void* h,
                            float* last, float* kept, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  const int st = scan::check_sizes(dtype, B, T, C);
  if (st != LNCC_OK) return st;
  if (B == 0) return LNCC_OK;
  if (!last || !blk::aligned(last, 4) || !blk::aligned(state, 4)) return LNCC_ERR_BAD_ARG;
  if (T == 0) {
    scan::pass_kernel<<<unsigned(blk::ceil_div(B * C, scan::kThreads)), scan::kThreads, 0, stream>>>(state, last, B * C);
    return blk::check_end(stream);
  }
  if (!scan::good(x, dtype) || !scan::good(gate, dtype) || !scan::good(h, dtype) || !blk::aligned(kept, 4))
    return LNCC_ERR_BAD_ARG;
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < lncc_gated_scan_scratch_bytes(B, T, C))
    return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  scan::Args p = {};
  const int64_t e = blk::elem_size(dtype), from = reverse ? T - 1 : 0, sign = reverse ? -1 : 1;
  p.x = static_cast<const char*>(x) + from * x_t * e, p.x_b = x_b, p.x_t = sign * x_t;
  p.gate = static_cast<const char*>(gate) + from * gate_t * e, p.gate_b = gate_b, p.gate_t = sign * gate_t;
  p.h = static_cast<char*>(h) + from * C * e, p.out_b = T * C, p.out_t = sign * C;
  p.state = state, p.last = last, p.kept = kept, p.B = B, p.T = T, p.C = C;
  p.chunks = blk::ceil_div(T, scan::kChunk);
  p.agg_a = static_cast<float*>(scratch), p.agg_s = p.agg_a + B * p.chunks * C;
  if (dtype == LNCC_F32) scan::forward<float>(p, stream);
  else if (dtype == LNCC_BF16) scan::forward<__nv_bfloat16>(p, stream);
  else scan::forward<__half>(p, stream);
  return blk::check_end(stream);
}

int lncc_gated_scan_backward(const void* dh, int64_t dh_b, int64_t dh_t, const float* dlast, const void* x, int64_t x_b,
                             int64_t x_t, const void* gate, int64_t gate_b, int64_t gate_t, const float* kept, int dtype,
                             int64_t B, int64_t T, int64_t C, int reverse, void* dx, void* dgate, float* dstate,
                             void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  const int st = scan::check_sizes(dtype, B, T, C);
  if (st != LNCC_OK) return st;
  if (B == 0) return LNCC_OK;
  if (!blk::aligned(dlast, 4) || !blk::aligned(dstate, 4)) return LNCC_ERR_BAD_ARG;
  if (T == 0) {
    if (dstate)
      scan::pass_kernel<<<unsigned(blk::ceil_div(B * C, scan::kThreads)), scan::kThreads, 0, stream>>>(dlast, dstate, B * C);
    return blk::check_end(stream);
  }
  if (!scan::good(x, dtype) || !scan::good(gate, dtype) || !scan::good(dh, dtype) || !scan::good(dx, dtype) ||
      !scan::good(dgate, dtype) || !kept || !blk::aligned(kept, 4))
    return LNCC_ERR_BAD_ARG;
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < lncc_gated_scan_scratch_bytes(B, T, C))
    return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  scan::Args p = {};
  const int64_t e = blk::elem_size(dtype), from = reverse ? T - 1 : 0, sign = reverse ? -1 : 1;
  p.x = static_cast<const char*>(x) + from * x_t * e, p.x_b = x_b, p.x_t = sign * x_t;
  p.gate = static_cast<const char*>(gate) + from * gate_t * e, p.gate_b = gate_b, p.gate_t = sign * gate_t;
  p.dh = static_cast<const char*>(dh) + from * dh_t * e, p.dh_b = dh_b, p.dh_t = sign * dh_t;
  p.dx = static_cast<char*>(dx) + from * C * e, p.dgate = static_cast<char*>(dgate) + from * C * e;
  p.out_b = T * C, p.out_t = sign * C;
  p.dlast = dlast, p.dstate = dstate, p.kept = const_cast<float*>(kept), p.B = B, p.T = T, p.C = C;
  p.chunks = blk::ceil_div(T, scan::kChunk);
  p.agg_a = static_cast<float*>(scratch), p.agg_s = p.agg_a + B * p.chunks * C;
  if (dtype == LNCC_F32) scan::backward<float>(p, stream);
  else if (dtype == LNCC_BF16) scan::backward<__nv_bfloat16>(p, stream);
  else scan::backward<__half>(p, stream);
  return blk::check_end(stream);
}

}  // extern "C"
