// The gated linear recurrence over (B, T, C), forward and backward:
//
//   a_t = sigmoid(gate_t), h_t = a_t h_{t-1} + (1 - a_t) x_t, h_0 = state (or 0)
//   q_t = dh_t + a_{t+1} q_{t+1}, with dlast added to dh_T
//   dx_t = (1 - a_t) q_t, dgate_t = q_t (h_{t-1} - x_t) a_t (1 - a_t), dstate = a_1 q_1
//
// Steps compose: (A, S) after (A', S') is (A A', A S' + S). A thread takes 4 bytes of channels of a run of steps, one
// step after the other with the state in fp32 registers, 16 steps' loads in flight: a warp reads 128 bytes of a row (or two
// rows' 64, or four rows' 32, where that leaves fewer lanes without a channel). Runs are as long as leaves the GPU full
// of threads; with enough channels one run is all of T, and one kernel does everything. Otherwise a first kernel forms
// each run's (A, S) from a zero state, and a second one starts each run from its state, which a block folds from the runs
// before it: its threads share the earlier blocks' (A, S) out, and meet in shared memory. All in a fixed order. The second
// kernel finds most of what it reads again in L2. Backward the same runs from the end, and h is formed again, 16 steps at a
// time, from the fp32 states that the forward pass kept before each 16; that reads h's 2 or 4 bytes a step less than
// saving h would, and h_{t-1} is not rounded to 16 bits.
// Measured: 2 x 32768 x 256 fp16 16 + 21 us (its bytes once: 15), 107520 x 96 bf16 11 + 16 forward and 13 + 29 backward (10, 17),
// 6 x 4093 x 389 fp32 19 + 26 and 23 + 44 (18, 29). One kernel that reads everything once, tiles waiting for earlier tiles' sums,
// took 47 us for the first: at four blocks an SM too few bytes are in flight while tiles wait. Registers are at the caps that the
// launch bounds set (64, and 128 backward), and 16 steps' loads do not quite fit beside the arithmetic: most first passes and runs
// spill up to 40 bytes a thread, back_run 32 to 104; it also forms each gate twice, once for h and once for the gradients.
#include "lncc_block.cuh"

#include <type_traits>

namespace lncc {
namespace scan {

using namespace blk;

constexpr int kKeep = 16;       // steps from one kept state to the next, and steps whose loads are in flight
constexpr int kThreads = 256;

struct Args {
  const void *x, *gate, *dh;
  int64_t x_b, x_t, gate_b, gate_t, dh_b, dh_t;  // strides in elements; time strides are negative for reverse scans
  void *h, *dx, *dgate;
  int64_t out_b, out_t;
  const float *state, *dlast;
  float *last, *dstate;
  float *kept;             // [B][ceil(T / kKeep)][C] states before steps 0, kKeep, ...
  float *run_a, *run_s;    // [B][runs][C]
  float *block_a, *block_s;  // [B][blocks of runs][C]
  int64_t B, T, C;
  int run;                 // steps of a run, a multiple of kKeep
  int runs, run_blocks;    // runs of a sequence; blocks of them
};

// V channels' products and sums; two channels as one packed instruction.
template <int V> __device__ __forceinline__ void mul(const float (&a)[V], const float (&b)[V], float (&d)[V]) {
  if constexpr (V == 2) {
    const float2 r = mul2(make_float2(a[0], a[1]), make_float2(b[0], b[1]));
    d[0] = r.x, d[1] = r.y;
  } else {
    for (int v = 0; v < V; v++) d[v] = a[v] * b[v];
  }
}
template <int V> __device__ __forceinline__ void fma(const float (&a)[V], const float (&b)[V], const float (&c)[V], float (&d)[V]) {
  if constexpr (V == 2) {
    const float2 r = fma2(make_float2(a[0], a[1]), make_float2(b[0], b[1]), make_float2(c[0], c[1]));
    d[0] = r.x, d[1] = r.y;
  } else {
    for (int v = 0; v < V; v++) d[v] = fmaf(a[v], b[v], c[v]);
  }
}

// a = sigmoid(g) and keep = 1 - a = sigmoid(-g), each to a few u32 of itself (1 - a would cancel for open gates).
// fp32: e = exp(-|g|) by the exponential of 2, with the rounding of |g| log2 e carried along, and 1 / (1 + e) with one step of
// Newton's; gates of -inf and +inf give exactly 0 and 1. 16-bit types: e = exp(-g), held below 2^126 so that its reciprocal
// stays a normal number (a then is 1e-38 where it should be less), a = 1 / (1 + e), keep = e a: e is off by |g| u32 at
// most, far below their own u. The two special functions of each gate, at 16 an SM and clock, are what bounds 16-bit scans
// next to their bytes: at 16.8M gates 7.5 us a pass over them.
template <bool EXACT, int V> __device__ __forceinline__ void gates(const float (&g)[V], float (&a)[V], float (&keep)[V]) {
  if constexpr (EXACT) {
#pragma unroll
    for (int v = 0; v < V; v++) {
      const float z = -fabsf(g[v]), t = z * 1.4426950408889634f;
      const float lost = fmaf(z, 1.4426950408889634f, -t) + z * 1.925963033e-8f;  // log2 e = 1.44269502162933 + 1.93e-8
      float e, r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
      e = z > -126.f ? fmaf(e, lost * 0.69314718f, e) : 0.f;
      const float d = 1.f + e;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
      r = fmaf(r, fmaf(-d, r, 1.f), r);
      const float er = e * r;
      a[v] = g[v] >= 0.f ? r : er;
      keep[v] = g[v] >= 0.f ? er : r;
      if (g[v] != g[v]) a[v] = keep[v] = g[v];
    }
  } else {
    float t[V], e[V], d[V], minus_log2e[V], one[V];
#pragma unroll
    for (int v = 0; v < V; v++) minus_log2e[v] = -1.44269504f, one[v] = 1.f;
    mul<V>(g, minus_log2e, t);
#pragma unroll
    for (int v = 0; v < V; v++) {
      asm("min.NaN.f32 %0, %1, 0f42FB0000;" : "=f"(t[v]) : "f"(t[v]));  // 125.5
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[v]) : "f"(t[v]));
    }
    fma<V>(e, one, one, d);
#pragma unroll
    for (int v = 0; v < V; v++) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a[v]) : "f"(d[v]));
    mul<V>(e, a, keep);
  }
}

// A register's worth of channels.
template <int BYTES> struct Word;
template <> struct Word<4> {
  typedef uint32_t type;
  static __device__ __forceinline__ void pin(uint32_t& w) { asm volatile("" : "+r"(w)); }
};
template <> struct Word<2> {
  typedef uint16_t type;
  static __device__ __forceinline__ void pin(uint16_t& w) { asm volatile("" : "+h"(w)); }
};

// Where a thread stands: sequence b, channels c .. c + V - 1, run (of the sequence), its place in the block.
template <int V, int LANES> struct Place {
  static constexpr int PER_BLOCK = kThreads / LANES;  // runs a block takes
  int64_t c, b, from, to;
  int slot, run, lane;
  bool live;  // has channels and steps
  __device__ __forceinline__ explicit Place(const Args& p) {
    lane = threadIdx.x % LANES;
    slot = threadIdx.x / LANES;
    c = (int64_t(blockIdx.x) * LANES + lane) * V;
    run = blockIdx.y * PER_BLOCK + slot;
    b = blockIdx.z;
    from = int64_t(run) * p.run;
    to = min(p.T, from + p.run);
    live = c < p.C && from < p.T;
  }
};

// (A, S) of the runs of this block before this thread's own (backward: after it), on top of the state that the earlier
// blocks leave: the threads share the blocks' sums out, then each folds the block's runs up to its own.
// h: the given state on entry, the run's on return.
template <int V, int LANES>
__device__ __forceinline__ void start_state(const Args& p, const Place<V, LANES>& at, bool reverse, float (&h)[V]) {
  constexpr int N = Place<V, LANES>::PER_BLOCK;
  __shared__ float sa[2][N][LANES][V], ss[2][N][LANES][V];  // shares of the blocks before, and the block's own runs
  const bool channel = at.c < p.C;
  const int before = reverse ? p.run_blocks - 1 - int(blockIdx.y) : int(blockIdx.y);
  float A[V], S[V];
#pragma unroll
  for (int v = 0; v < V; v++) A[v] = 1.f, S[v] = 0.f;
  if (channel) {
    const int i0 = int(int64_t(before) * at.slot / N), i1 = int(int64_t(before) * (at.slot + 1) / N);
#pragma unroll 8
    for (int i = i0; i < i1; i++) {
      const int64_t k = (at.b * p.run_blocks + (reverse ? p.run_blocks - 1 - i : i)) * p.C + at.c;
      float a2[V], s2[V];
      load_vec<float, V>(p.block_a + k, a2);
      load_vec<float, V>(p.block_s + k, s2);
#pragma unroll
      for (int v = 0; v < V; v++) S[v] = fmaf(a2[v], S[v], s2[v]), A[v] *= a2[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; v++) sa[0][at.slot][at.lane][v] = A[v], ss[0][at.slot][at.lane][v] = S[v];
  if (at.live) {
    const int64_t k = (at.b * p.runs + at.run) * p.C + at.c;
    load_vec<float, V>(p.run_a + k, A);
    load_vec<float, V>(p.run_s + k, S);
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) A[v] = 1.f, S[v] = 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; v++) sa[1][at.slot][at.lane][v] = A[v], ss[1][at.slot][at.lane][v] = S[v];
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; v++) {
    for (int i = 0; i < N; i++) h[v] = fmaf(sa[0][i][at.lane][v], h[v], ss[0][i][at.lane][v]);
    if (reverse)
      for (int i = N - 1; i > at.slot; i--) h[v] = fmaf(sa[1][i][at.lane][v], h[v], ss[1][i][at.lane][v]);
    else
      for (int i = 0; i < at.slot; i++) h[v] = fmaf(sa[1][i][at.lane][v], h[v], ss[1][i][at.lane][v]);
  }
}

// (A, S) of this thread's run, and the block's, to scratch.
template <int V, int LANES>
__device__ __forceinline__ void put_sums(const Args& p, const Place<V, LANES>& at, const float (&A)[V], const float (&S)[V],
                                         bool reverse) {
  constexpr int N = Place<V, LANES>::PER_BLOCK;
  __shared__ float sa[N][LANES][V], ss[N][LANES][V];
#pragma unroll
  for (int v = 0; v < V; v++) sa[at.slot][at.lane][v] = A[v], ss[at.slot][at.lane][v] = S[v];
  if (at.live) {
    const int64_t k = (at.b * p.runs + at.run) * p.C + at.c;
    if (LNCC_IN(k, V, p.B * p.runs * p.C)) {
      store_vec<float, V>(p.run_a + k, A);
      store_vec<float, V>(p.run_s + k, S);
    }
  }
  __syncthreads();
  if (at.slot != 0 || at.c >= p.C) return;
  float A2[V], S2[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    A2[v] = 1.f, S2[v] = 0.f;
    for (int j = 0; j < N; j++) {
      const int i = reverse ? N - 1 - j : j;
      S2[v] = fmaf(sa[i][at.lane][v], S2[v], ss[i][at.lane][v]);
      A2[v] *= sa[i][at.lane][v];
    }
  }
  const int64_t k = (at.b * p.run_blocks + blockIdx.y) * p.C + at.c;
  if (!LNCC_IN(k, V, p.B * p.run_blocks * p.C)) return;
  store_vec<float, V>(p.block_a + k, A2);
  store_vec<float, V>(p.block_s + k, S2);
}

// Up to kKeep steps of V channels, as they lie in memory; a step at or past `to` is never looked at.
template <typename T, int V> struct Steps {
  typedef typename Word<sizeof(T) * V>::type W;
  W e[kKeep];
  template <bool FULL> __device__ __forceinline__ void load(const T* p, int64_t stride, int64_t t, int64_t to) {
    p += t * stride;
#pragma unroll
    for (int i = 0; i < kKeep; i++, p += stride)
      if (FULL || t + i < to) e[i] = *reinterpret_cast<const W*>(p);
  }
  // The empty statement keeps the arithmetic on step i from moving ahead of the step before it: done for all steps at
  // once it would take hundreds of registers.
  __device__ __forceinline__ void open(int i) { Word<sizeof(T) * V>::pin(e[i]); }
  __device__ __forceinline__ void get(int i, float (&f)[V]) const {
#pragma unroll
    for (int v = 0; v < V; v++) f[v] = to_f(reinterpret_cast<const Vec<T, V>&>(e[i]).e[v]);
  }
};

// the kernel's launch may begin before the one ahead of it in the stream has ended; what that one wrote is read after this
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_begin() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename T, int V, int LANES> __global__ void __launch_bounds__(kThreads, 4) sum_kernel(const Args p) {
  const Place<V, LANES> at(p);
  let_next_kernel_begin();
  float A[V], S[V];
#pragma unroll
  for (int v = 0; v < V; v++) A[v] = 1.f, S[v] = 0.f;
  if (at.live) {
    const T* gate = static_cast<const T*>(p.gate) + at.b * p.gate_b + at.c;
    const T* x = static_cast<const T*>(p.x) + at.b * p.x_b + at.c;
    const auto block = [&](auto full, int64_t t) {
      constexpr bool FULL = decltype(full)::value;
      Steps<T, V> sg, sx;
      sg.template load<FULL>(gate, p.gate_t, t, at.to);
      sx.template load<FULL>(x, p.x_t, t, at.to);
#pragma unroll
      for (int i = 0; i < kKeep; i++) {
        if (!FULL && t + i >= at.to) break;
        sg.open(i), sx.open(i);
        float g[V], x_t[V], a[V], keep[V];
        sg.get(i, g), sx.get(i, x_t);
        gates<sizeof(T) == 4, V>(g, a, keep);
        mul<V>(keep, x_t, keep);
        fma<V>(a, S, keep, S);
        mul<V>(A, a, A);
      }
    };
    int64_t t = at.from;
    for (; t + kKeep <= at.to; t += kKeep) block(std::true_type(), t);
    if (t < at.to) block(std::false_type(), t);
  }
  put_sums<V, LANES>(p, at, A, S, false);
}

template <typename T, int V, int LANES, bool SPLIT> __global__ void __launch_bounds__(kThreads, 4) run_kernel(const Args p) {
  const Place<V, LANES> at(p);
  float h[V];
  if (SPLIT) wait_for_previous_kernel();
#pragma unroll
  for (int v = 0; v < V; v++) h[v] = p.state && at.c < p.C ? p.state[at.b * p.C + at.c + v] : 0.f;
  if (SPLIT) start_state<V, LANES>(p, at, false, h);
  if (!at.live) return;
  const T* gate = static_cast<const T*>(p.gate) + at.b * p.gate_b + at.c;
  const T* x = static_cast<const T*>(p.x) + at.b * p.x_b + at.c;
  T* out = static_cast<T*>(p.h) + at.b * p.out_b + at.c;
  const int64_t keeps = (p.T + kKeep - 1) / kKeep;
  const auto block = [&](auto full, int64_t t) {
    constexpr bool FULL = decltype(full)::value;
    Steps<T, V> sg, sx;
    sg.template load<FULL>(gate, p.gate_t, t, at.to);
    sx.template load<FULL>(x, p.x_t, t, at.to);
    if (p.kept) {
      const int64_t k = (at.b * keeps + t / kKeep) * p.C + at.c;
      if (LNCC_IN(k, V, p.B * keeps * p.C)) store_vec<float, V>(p.kept + k, h);
    }
    T* to = out + t * p.out_t;
#pragma unroll
    for (int i = 0; i < kKeep; i++, to += p.out_t) {
      if (!FULL && t + i >= at.to) break;
      sg.open(i), sx.open(i);
      float g[V], x_t[V], a[V], keep[V];
      sg.get(i, g), sx.get(i, x_t);
      gates<sizeof(T) == 4, V>(g, a, keep);
      mul<V>(keep, x_t, keep);
      fma<V>(a, h, keep, h);
      store_vec<T, V>(to, h);
    }
  };
  int64_t t = at.from;
  for (; t + kKeep <= at.to; t += kKeep) block(std::true_type(), t);
  if (t < at.to) block(std::false_type(), t);
  if (at.to == p.T && LNCC_IN(at.b * p.C + at.c, V, p.B * p.C)) store_vec<float, V>(p.last + at.b * p.C + at.c, h);
}

// backward: (A, S) of what a run hands on to the step before it, a_t q_t
template <typename T, int V, int LANES> __global__ void __launch_bounds__(kThreads, 4) back_sum_kernel(const Args p) {
  const Place<V, LANES> at(p);
  let_next_kernel_begin();
  float A[V], S[V];
#pragma unroll
  for (int v = 0; v < V; v++) A[v] = 1.f, S[v] = 0.f;
  if (at.live) {
    const T* gate = static_cast<const T*>(p.gate) + at.b * p.gate_b + at.c;
    const T* dh = static_cast<const T*>(p.dh) + at.b * p.dh_b + at.c;
    const auto block = [&](auto full, int64_t t) {
      constexpr bool FULL = decltype(full)::value;
      Steps<T, V> sg, sd;
      sg.template load<FULL>(gate, p.gate_t, t, at.to);
      sd.template load<FULL>(dh, p.dh_t, t, at.to);
#pragma unroll
      for (int i = kKeep - 1; i >= 0; i--) {
        if (!FULL && t + i >= at.to) continue;
        sg.open(i), sd.open(i);
        float g[V], d[V], a[V], keep[V];
        sg.get(i, g), sd.get(i, d);
        gates<sizeof(T) == 4, V>(g, a, keep);
#pragma unroll
        for (int v = 0; v < V; v++) d[v] += S[v];
        mul<V>(a, d, S);
        mul<V>(A, a, A);
      }
    };
    int64_t t = (at.to - 1) / kKeep * kKeep;
    if (t + kKeep > at.to) block(std::false_type(), t), t -= kKeep;
    for (; t >= at.from; t -= kKeep) block(std::true_type(), t);
  }
  put_sums<V, LANES>(p, at, A, S, true);
}

template <typename T, int V, int LANES, bool SPLIT> __global__ void __launch_bounds__(kThreads, 2) back_run_kernel(const Args p) {
  const Place<V, LANES> at(p);
  const T* gate = static_cast<const T*>(p.gate) + at.b * p.gate_b + at.c;
  const T* x = static_cast<const T*>(p.x) + at.b * p.x_b + at.c;
  const T* dh = static_cast<const T*>(p.dh) + at.b * p.dh_b + at.c;
  const int64_t keeps = (p.T + kKeep - 1) / kKeep, last = at.live ? (at.to - 1) / kKeep * kKeep : 0;
  Steps<T, V> sg, sx, sd;
  // fp32: the last steps come in while the state is formed (48 -> 43 us at 6 x 4093 x 389; two 16-bit channels a thread have no
  // registers left for it, 31 -> 35 us at 107520 x 96)
  const bool ahead = SPLIT && sizeof(T) == 4 && at.live && last + kKeep <= at.to;
  if (ahead) {
    sg.template load<true>(gate, p.gate_t, last, at.to);
    sx.template load<true>(x, p.x_t, last, at.to);
    sd.template load<true>(dh, p.dh_t, last, at.to);
  }
  float q[V];
  if (SPLIT) wait_for_previous_kernel();
#pragma unroll
  for (int v = 0; v < V; v++) q[v] = p.dlast && at.c < p.C ? p.dlast[at.b * p.C + at.c + v] : 0.f;
  if (SPLIT) start_state<V, LANES>(p, at, true, q);
  if (!at.live) return;
  T* dx = static_cast<T*>(p.dx) + at.b * p.out_b + at.c;
  T* dgate = static_cast<T*>(p.dgate) + at.b * p.out_b + at.c;
  const auto block = [&](auto full, int64_t t) {
    constexpr bool FULL = decltype(full)::value;
    float h[V], apart[kKeep][V];  // apart: h_{t-1} - x_t
    load_vec<float, V>(p.kept + (at.b * keeps + t / kKeep) * p.C + at.c, h);
    if (!ahead || t != last) {
      sg.template load<FULL>(gate, p.gate_t, t, at.to);
      sx.template load<FULL>(x, p.x_t, t, at.to);
      sd.template load<FULL>(dh, p.dh_t, t, at.to);
    }
#pragma unroll
    for (int i = 0; i < kKeep; i++) {
      if (!FULL && t + i >= at.to) break;
      sg.open(i), sx.open(i);
      float g[V], x_t[V], a[V], keep[V];
      sg.get(i, g), sx.get(i, x_t);
      gates<sizeof(T) == 4, V>(g, a, keep);
#pragma unroll
      for (int v = 0; v < V; v++) apart[i][v] = h[v] - x_t[v];
      mul<V>(keep, x_t, keep);
      fma<V>(a, h, keep, h);
    }
    T *to_x = dx + (t + kKeep - 1) * p.out_t, *to_gate = dgate + (t + kKeep - 1) * p.out_t;
#pragma unroll
    for (int i = kKeep - 1; i >= 0; i--, to_x -= p.out_t, to_gate -= p.out_t) {
      if (!FULL && t + i >= at.to) continue;
      sg.open(i), sd.open(i);
      float g[V], d[V], a[V], keep[V], ox[V], og[V], aq[V];
      sg.get(i, g), sd.get(i, d);
      gates<sizeof(T) == 4, V>(g, a, keep);
#pragma unroll
      for (int v = 0; v < V; v++) q[v] += d[v];
      mul<V>(keep, q, ox);
      mul<V>(a, q, aq);
      mul<V>(ox, apart[i], og);
      mul<V>(og, a, og);
#pragma unroll
      for (int v = 0; v < V; v++) q[v] = aq[v];
      store_vec<T, V>(to_x, ox);
      store_vec<T, V>(to_gate, og);
    }
  };
  int64_t t = last;
  if (t + kKeep > at.to) block(std::false_type(), t), t -= kKeep;
  for (; t >= at.from; t -= kKeep) block(std::true_type(), t);
  if (at.from == 0 && p.dstate && LNCC_IN(at.b * p.C + at.c, V, p.B * p.C))
    store_vec<float, V>(p.dstate + at.b * p.C + at.c, q);
}

// T = 0: the state passes through.
__global__ void __launch_bounds__(kThreads) pass_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

// Lanes of a warp for a row's channels: 32, or 16 or 8 where that leaves a tenth fewer of them idle.
static int lanes_for(int64_t threads) {
  const auto idle = [&](int64_t l) { return double(ceil_div(threads, l) * l) / double(threads); };
  int lanes = 32;
  if (idle(16) < 0.9 * idle(lanes)) lanes = 16;
  if (idle(8) < 0.9 * idle(lanes)) lanes = 8;
  return lanes;
}

// Runs of a sequence: as few as give the GPU 2048 threads an SM at one channel each (1024 at two), of at least 2 x 16 steps
// (a shorter run would not pay for its fold). The sizes alone decide.
struct Cut {
  int run, runs, run_blocks;
};
constexpr int kMinPerBlock = kThreads / 32;  // runs a block takes at 32 lanes, the fewest
static Cut cut_for(int64_t B, int64_t T, int64_t C) {
  const int64_t want = int64_t(sm_count()) * 2048, have = B * C;
  int64_t runs = ceil_div(want, have > 0 ? have : 1);
  int64_t run = ceil_div(ceil_div(T, runs), kKeep) * kKeep;
  if (run < 2 * kKeep) run = 2 * kKeep;
  if (run > T) run = ceil_div(T, kKeep) * kKeep;
  Cut c;
  c.run = int(run > 0 ? run : kKeep);
  c.runs = int(ceil_div(T > 0 ? T : 1, c.run));
  c.run_blocks = int(ceil_div(c.runs, kMinPerBlock));
  return c;
}

template <typename K> static void launch_after(K kernel, dim3 grid, const Args& p, cudaStream_t st) {
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = dim3(kThreads), cfg.stream = st, cfg.attrs = &early, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, p);
}
template <typename T, int V, int LANES> static void launch(Args& p, bool backward, cudaStream_t st) {
  p.run_blocks = int(ceil_div(p.runs, Place<V, LANES>::PER_BLOCK));
  const dim3 grid(unsigned(ceil_div(p.C, LANES * V)), unsigned(p.run_blocks), unsigned(p.B));
  if (p.runs == 1) {
    if (backward) back_run_kernel<T, V, LANES, false><<<grid, kThreads, 0, st>>>(p);
    else run_kernel<T, V, LANES, false><<<grid, kThreads, 0, st>>>(p);
  } else if (backward) {
    back_sum_kernel<T, V, LANES><<<grid, kThreads, 0, st>>>(p);
    launch_after(back_run_kernel<T, V, LANES, true>, grid, p, st);
  } else {
    sum_kernel<T, V, LANES><<<grid, kThreads, 0, st>>>(p);
    launch_after(run_kernel<T, V, LANES, true>, grid, p, st);
  }
}
template <typename T, int V> static void launch_lanes(Args& p, bool backward, cudaStream_t st) {
  const int lanes = lanes_for(ceil_div(p.C, V));
  if (lanes == 32) launch<T, V, 32>(p, backward, st);
  else if (lanes == 16) launch<T, V, 16>(p, backward, st);
  else launch<T, V, 8>(p, backward, st);
}
static bool in_pairs(const Args& p) {
  const int64_t strides[] = {p.x_b, p.x_t, p.gate_b, p.gate_t, p.dh_b, p.dh_t, p.C};
  for (int64_t s : strides)
    if (s % 2) return false;
  return aligned(p.x, 4) && aligned(p.gate, 4) && aligned(p.dh, 4) && aligned(p.h, 4) && aligned(p.dx, 4) &&
         aligned(p.dgate, 4) && aligned(p.kept, 8) && aligned(p.last, 8) && aligned(p.dstate, 8);
}
// Two channels a thread for 16-bit types where every row starts on 4 bytes.
static void dispatch(Args& p, int dtype, bool backward, cudaStream_t st) {
  if (dtype == LNCC_F32) launch_lanes<float, 1>(p, backward, st);
  else if (dtype == LNCC_BF16 && in_pairs(p)) launch_lanes<__nv_bfloat16, 2>(p, backward, st);
  else if (dtype == LNCC_BF16) launch_lanes<__nv_bfloat16, 1>(p, backward, st);
  else if (in_pairs(p)) launch_lanes<__half, 2>(p, backward, st);
  else launch_lanes<__half, 1>(p, backward, st);
}

static int check_sizes(int dtype, int64_t B, int64_t T, int64_t C) {
  if (!valid_dtype(dtype)) return LNCC_ERR_DTYPE;
  if (B < 0 || T < 0 || C < 1) return LNCC_ERR_BAD_ARG;
  if (B > 65535 || T > (int64_t(1) << 30) || C > (1 << 24)) return LNCC_ERR_TOO_LARGE;
  if (cut_for(B, T, C).run_blocks > 65535) return LNCC_ERR_TOO_LARGE;
  return LNCC_OK;
}
static void place_scratch(Args& p, void* scratch) {
  const Cut c = cut_for(p.B, p.T, p.C);
  p.run = c.run, p.runs = c.runs;
  float* at = static_cast<float*>(scratch);  // an even number of floats each, so that pairs of channels stay aligned
  const int64_t n = (p.B * c.runs * p.C + 1) / 2 * 2, m = (p.B * c.run_blocks * p.C + 1) / 2 * 2;
  p.run_a = at, p.run_s = at + n, p.block_a = at + 2 * n, p.block_s = at + 2 * n + m;
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
  const scan::Cut c = scan::cut_for(B, T, C);
  return 2 * size_t(B) * size_t(c.runs + c.run_blocks) * size_t(C) * sizeof(float) + 64;
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
  scan::place_scratch(p, scratch);
  scan::dispatch(p, dtype, false, stream);
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
  scan::place_scratch(p, scratch);
  scan::dispatch(p, dtype, true, stream);
  return blk::check_end(stream);
}

}  // extern "C"
