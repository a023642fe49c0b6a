// Layer norm over the last axis, forward and backward, with the gradients of the weight and the bias.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1/sqrt(v + eps), n = (x - mu) r, y = n w + b
//   g = dy w, dx = r (g - mean(g) - n mean(g n)), dw = sum over rows of dy n, db = sum over rows of dy
//
// A row lives in the registers of LANES threads, E = 12 or 16 elements each, from its one load to its one store: the mean and
// then the centred squares are summed in fp32 without a second read (the two-step variance does not cancel). LANES is
// a power of two and E the smaller one that holds the row, so a warp takes 8 rows of 64 or one of 384 or 512, and a block one
// of up to 8192. Arithmetic is packed, two elements an instruction: at 107520 x 384 the kernels were bound by issuing 257
// instructions a row forward and 391 backward. Both directions are bound by their bytes now: 107520 x 384 bf16 forward 28 us
// (5.9 TB/s), backward 46 us (5.4 TB/s). Thread blocks stay and walk over the rows, so that the weight is loaded once and,
// backward, each thread keeps the fp32 sums of dw and db of its own columns. The next three rows are
// under way meanwhile, copied asynchronously into shared memory that only the thread itself reads (so no barrier waits for
// them): with one row ahead in registers 24 KB an SM were in flight, and the forward pass took 60 us where its bytes
// take 25 (107520 x 384 bf16). The sums of the threads of a block meet in shared memory and those of the blocks in a
// second kernel, each in a fixed order: the gradients are the same bits run after run.
// Rows off 16 bytes move single elements, and cost it: 32749 x 97 fp32 12 + 21 us for bytes of 4 + 6, 90001 x 389 bf16 50 + 77 for 21 +
// 32, where most backward kernels also spill 24 to 138 bytes a thread.
// Rows wider than 8192 take the looping kernels at the end of this file, which read a row again for each step.
#include "lncc_block.cuh"

#include <type_traits>

namespace lncc {
namespace norm {

using namespace blk;

constexpr int kElems = 16;       // the most elements of a row that one thread holds
constexpr int kThreads = 256;    // threads of a block (LANES where that is more)
constexpr int kMaxWidth = 8192;  // widest row that 512 threads hold

struct Args {
  const void* x;
  int64_t x_stride;   // elements from row to row
  const void* dy;     // backward
  int64_t dy_stride;
  const void* w;      // null: ones
  const void* b;      // null: zeros
  int wdtype;
  int64_t rows;
  int width;
  float eps;
  void* y;            // forward: y, backward: dx (may be null)
  float* mean;        // per row, written forward (may be null), read backward
  float* rstd;
  float* partial;     // backward: [blocks][2][width] sums of dy n and of dy (null: not wanted)
};

__device__ __forceinline__ float load_param(const void* p, int dtype, int c) {
  if (dtype == LNCC_F32) return static_cast<const float*>(p)[c];
  if (dtype == LNCC_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[c]);
  return to_f(static_cast<const __half*>(p)[c]);
}

// Sum over the LANES threads of a row; every one of them gets it. `red` holds one float a warp and is not used again
// before another barrier has been passed.
template <int LANES> __device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (LANES > 32) {
    constexpr int WARPS = LANES / 32 > 0 ? LANES / 32 : 1;
    const int warp = threadIdx.x / 32;
    if (threadIdx.x % 32 == 0) red[warp] = v;
    __syncthreads();
    const float* mine = red + warp / WARPS * WARPS;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; i++) v += mine[i];
  }
  return v;
}

// One thread's shares of the rows to come: NV vectors of VEC elements each, vector v at column (v*LANES + lane)*VEC. A ring
// of rows in shared memory, filled by asynchronous copies of 4 to 16 bytes; single 16-bit elements, which have
// none, wait in registers instead, one row ahead.
template <typename T, int LANES, int VEC, int E, int THREADS> struct Rows {
  static constexpr int NV = E / VEC, BYTES = VEC * int(sizeof(T));
  static constexpr int kStages = sizeof(T) == 4 ? 3 : 4;  // at most 48 KB a ring for 256 threads
  static constexpr bool ASYNC = BYTES >= 4;
  typedef Vec<T, VEC> V;
  struct Empty {};
  typename std::conditional<ASYNC, Empty, V[NV]>::type held;
  const T* base;
  int64_t stride, rows;
  int width, lane;
  V* ring;  // this thread's vector 0 of stage 0
  int in, out;

  __host__ __device__ static constexpr int smem() { return ASYNC ? kStages * NV * THREADS * BYTES : 0; }
  __device__ __forceinline__ Rows(const void* p, int64_t stride_, int64_t rows_, int width_, int lane_, void* smem_at)
      : base(static_cast<const T*>(p)), stride(stride_), rows(rows_), width(width_), lane(lane_),
        ring(static_cast<V*>(smem_at) + threadIdx.x), in(0), out(0) {}
  // begin to fetch a row (past the end: zeros)
  __device__ __forceinline__ void fetch(int64_t row) {
    const T* from = base + (row < rows ? row * stride : 0);
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = (v * LANES + lane) * VEC;
      const bool live = row < rows && c < width && LNCC_IN(c, VEC, width);
      if constexpr (ASYNC) {
        const uint32_t dst = uint32_t(__cvta_generic_to_shared(ring + (in * NV + v) * THREADS));
        const T* src = live ? from + c : base;
        const int bytes = live ? BYTES : 0;  // what is not copied is zero
        if constexpr (BYTES == 8)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
        else if constexpr (BYTES == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) held[v].e[i] = live ? from[c + i] : from_f<T>(0.f);
      }
    }
    in = in + 1 == kStages ? 0 : in + 1;
  }
  // the oldest row fetched, as pairs of floats
  __device__ __forceinline__ void take(float2 (&pairs)[E / 2]) {
    float f[E];
#pragma unroll
    for (int v = 0; v < NV; v++) {
      V r;
      if constexpr (ASYNC) r = ring[(out * NV + v) * THREADS];
      else r = held[v];
#pragma unroll
      for (int i = 0; i < VEC; i++) f[v * VEC + i] = to_f(r.e[i]);
    }
#pragma unroll
    for (int i = 0; i < E / 2; i++) pairs[i] = make_float2(f[2 * i], f[2 * i + 1]);
    out = out + 1 == kStages ? 0 : out + 1;
  }
};
__device__ __forceinline__ void close_fetch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER> __device__ __forceinline__ void wait_fetch() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

template <int LANES> __host__ __device__ constexpr int threads_of() { return LANES > kThreads ? LANES : kThreads; }

// column of element e of a lane
template <int LANES, int VEC> __device__ __forceinline__ int column(int e, int lane) { return (e / VEC * LANES + lane) * VEC + e % VEC; }
__device__ __forceinline__ float sum2(float2 v) { return v.x + v.y; }

template <typename T, int LANES, int VEC, int E>
__global__ void __launch_bounds__(threads_of<LANES>(), LANES > kThreads ? 1 : VEC * sizeof(T) >= 4 ? 3 : 2) forward_kernel(const Args a) {
  constexpr int THREADS = LANES > kThreads ? LANES : kThreads;
  constexpr int ROWS = THREADS / LANES, NV = E / VEC;
  typedef Rows<T, LANES, VEC, E, THREADS> R;
  constexpr int AHEAD = R::ASYNC ? R::kStages - 1 : 1;
  extern __shared__ __align__(16) unsigned char stage[];
  __shared__ float red[2][THREADS / 32];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  T* y = static_cast<T*>(a.y);
  const int64_t step = int64_t(gridDim.x) * ROWS;
  int64_t row = int64_t(blockIdx.x) * ROWS + group;
  R rows(a.x, a.x_stride, a.rows, a.width, lane, stage);
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    rows.fetch(row + i * step);
    close_fetch();
  }
  float2 w[E / 2], b[E / 2];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int c = column<LANES, VEC>(e, lane);
    (e % 2 ? w[e / 2].y : w[e / 2].x) = a.w && c < a.width ? load_param(a.w, a.wdtype, c) : 1.f;
    (e % 2 ? b[e / 2].y : b[e / 2].x) = a.b && c < a.width ? load_param(a.b, a.wdtype, c) : 0.f;
  }
  const float inv = 1.f / float(a.width);
  // every group of the block takes the same number of turns: the row sums hold barriers
  for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += step, row += step) {
    float2 x[E / 2];
    if (R::ASYNC) wait_fetch<AHEAD - 1>();
    rows.take(x);
    rows.fetch(row + AHEAD * step);
    close_fetch();
    float2 s = x[0];
#pragma unroll
    for (int i = 1; i < E / 2; i++) s = add2(s, x[i]);
    const float mu = row_sum<LANES>(sum2(s), red[0]) * inv;
    float2 q = both(0.f);
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      x[i] = add2(x[i], both(-mu));
      // past the row's end nothing is summed (vectors end where rows do; single elements are looked at one by one)
      if (VEC > 1) {
        if (column<LANES, VEC>(2 * i, lane) < a.width) q = fma2(x[i], x[i], q);
      } else {
        if (column<LANES, VEC>(2 * i, lane) < a.width) q.x = fmaf(x[i].x, x[i].x, q.x);
        if (column<LANES, VEC>(2 * i + 1, lane) < a.width) q.y = fmaf(x[i].y, x[i].y, q.y);
      }
    }
    const float rs = rsqrtf(row_sum<LANES>(sum2(q), red[1]) * inv + a.eps);
    if (row >= a.rows) continue;
    if (lane == 0 && a.mean && LNCC_IN(row, 1, a.rows)) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
#pragma unroll
    for (int i = 0; i < E / 2; i++) x[i] = fma2(mul2(x[i], both(rs)), w[i], b[i]);
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = (v * LANES + lane) * VEC;
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) o[i] = (v * VEC + i) % 2 ? x[(v * VEC + i) / 2].y : x[(v * VEC + i) / 2].x;
      if (c < a.width && LNCC_IN(row * a.width + c, VEC, a.rows * a.width)) store_vec<T, VEC>(y + row * a.width + c, o);
    }
  }
  if (R::ASYNC) wait_fetch<0>();  // nothing is under way to shared memory any more
}

template <typename T, int LANES, int VEC, int E>
__global__ void __launch_bounds__(threads_of<LANES>(), LANES <= kThreads && VEC * sizeof(T) >= 4 ? 2 : 1) backward_kernel(const Args a) {
  constexpr int THREADS = LANES > kThreads ? LANES : kThreads;
  constexpr int ROWS = THREADS / LANES, NV = E / VEC;
  typedef Rows<T, LANES, VEC, E, THREADS> R;
  constexpr int AHEAD = R::ASYNC ? R::kStages - 1 : 1;
  extern __shared__ __align__(16) unsigned char stage[];
  __shared__ float red[2][THREADS / 32];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  T* dx = static_cast<T*>(a.y);
  const int64_t step = int64_t(gridDim.x) * ROWS;
  int64_t row = int64_t(blockIdx.x) * ROWS + group;
  R rows_x(a.x, a.x_stride, a.rows, a.width, lane, stage), rows_dy(a.dy, a.dy_stride, a.rows, a.width, lane, stage + R::smem());
#pragma unroll
  for (int i = 0; i < AHEAD; i++) {
    rows_x.fetch(row + i * step);
    rows_dy.fetch(row + i * step);
    close_fetch();
  }
  float2 w[E / 2], dw[E / 2], db[E / 2];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int c = column<LANES, VEC>(e, lane);
    (e % 2 ? w[e / 2].y : w[e / 2].x) = a.w && c < a.width ? load_param(a.w, a.wdtype, c) : 1.f;
    dw[e / 2] = db[e / 2] = both(0.f);
  }
  const float inv = 1.f / float(a.width);
  float mu_next = row < a.rows ? a.mean[row] : 0.f, rs_next = row < a.rows ? a.rstd[row] : 0.f;
  for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += step, row += step) {
    float2 n[E / 2], d[E / 2];
    const float mu = mu_next, rs = rs_next;
    mu_next = row + step < a.rows ? a.mean[row + step] : 0.f;
    rs_next = row + step < a.rows ? a.rstd[row + step] : 0.f;
    if (R::ASYNC) wait_fetch<AHEAD - 1>();
    rows_x.take(n);
    rows_dy.take(d);
    rows_x.fetch(row + AHEAD * step);
    rows_dy.fetch(row + AHEAD * step);
    close_fetch();
    float2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < E / 2; i++) {  // past the row's end dy is 0, and with it every term
      n[i] = mul2(add2(n[i], both(-mu)), both(rs));
      db[i] = add2(db[i], d[i]);
      dw[i] = fma2(d[i], n[i], dw[i]);
      d[i] = mul2(d[i], w[i]);
      s1 = add2(s1, d[i]);
      s2 = fma2(d[i], n[i], s2);
    }
    if (a.y == nullptr) continue;  // the same for every thread
    const float m1 = row_sum<LANES>(sum2(s1), red[0]) * inv, m2 = row_sum<LANES>(sum2(s2), red[1]) * inv;
    if (row >= a.rows) continue;
#pragma unroll
    for (int i = 0; i < E / 2; i++) d[i] = fma2(n[i], both(-m2 * rs), mul2(add2(d[i], both(-m1)), both(rs)));
#pragma unroll
    for (int v = 0; v < NV; v++) {
      const int c = (v * LANES + lane) * VEC;
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) o[i] = (v * VEC + i) % 2 ? d[(v * VEC + i) / 2].y : d[(v * VEC + i) / 2].x;
      if (c < a.width && LNCC_IN(row * a.width + c, VEC, a.rows * a.width)) store_vec<T, VEC>(dx + row * a.width + c, o);
    }
  }
  if (R::ASYNC) wait_fetch<0>();
  if (a.partial == nullptr) return;
  // the block's rows meet: thread t < LANES adds the other groups' sums to its own, group by group
  float* out = a.partial + int64_t(blockIdx.x) * 2 * a.width;
  __shared__ float meet[ROWS > 1 ? THREADS : 1];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int c = column<LANES, VEC>(e, lane);
#pragma unroll
    for (int which = 0; which < 2; which++) {
      const float2 pair = which ? db[e / 2] : dw[e / 2];
      float v = e % 2 ? pair.y : pair.x;
      if (ROWS > 1) {
        __syncthreads();
        meet[threadIdx.x] = v;
        __syncthreads();
        if (group == 0) {
          v = 0.f;
          for (int g = 0; g < ROWS; g++) v += meet[g * LANES + lane];
        }
      }
      if (group == 0 && c < a.width) out[which * a.width + c] = v;
    }
  }
}

// dw and db: column sums of the blocks' partial sums, 32 strands of blocks in order and then the strands in order.
__global__ void __launch_bounds__(1024) reduce_kernel(const float* __restrict__ partial, int blocks, int width, void* dw,
                                                      void* db, int wdtype) {
  __shared__ float sum[32][33];
  const int strand = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t c = int64_t(blockIdx.x) * 32 + lane, cols = 2 * int64_t(width);
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int p = strand; p < blocks; p += 32) s += partial[p * cols + c];
  }
  sum[strand][lane] = s;
  __syncthreads();
  if (strand != 0 || c >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; i++) s += sum[i][lane];
  void* to = c < width ? dw : db;
  const int64_t i = c < width ? c : c - width;
  if (to == nullptr || !LNCC_IN(i, 1, width)) return;
  if (wdtype == LNCC_F32) static_cast<float*>(to)[i] = s;
  else if (wdtype == LNCC_BF16) static_cast<__nv_bfloat16*>(to)[i] = from_f<__nv_bfloat16>(s);
  else static_cast<__half*>(to)[i] = from_f<__half>(s);
}

// Rows that no block's registers hold: a block of 1024 takes one row and reads it once for each step.
template <typename T> __global__ void __launch_bounds__(1024) wide_forward_kernel(const Args a) {
  __shared__ float red[2][32];
  const float inv = 1.f / float(a.width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* y = static_cast<T*>(a.y) + row * a.width;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.width; c += 1024) s += to_f(x[c]);
    const float mu = row_sum<1024>(s, red[0]) * inv;
    for (int c = threadIdx.x; c < a.width; c += 1024) q += (to_f(x[c]) - mu) * (to_f(x[c]) - mu);
    const float rs = rsqrtf(row_sum<1024>(q, red[1]) * inv + a.eps);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
    for (int c = threadIdx.x; c < a.width; c += 1024) {
      const float w = a.w ? load_param(a.w, a.wdtype, c) : 1.f, b = a.b ? load_param(a.b, a.wdtype, c) : 0.f;
      if (LNCC_IN(row * a.width + c, 1, a.rows * a.width)) y[c] = from_f<T>((to_f(x[c]) - mu) * rs * w + b);
    }
  }
}
template <typename T> __global__ void __launch_bounds__(1024) wide_dx_kernel(const Args a) {
  __shared__ float red[2][32];
  const float inv = 1.f / float(a.width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    T* dx = static_cast<T*>(a.y) + row * a.width;
    const float mu = a.mean[row], rs = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.width; c += 1024) {
      const float g = to_f(dy[c]) * (a.w ? load_param(a.w, a.wdtype, c) : 1.f);
      s1 += g;
      s2 += g * (to_f(x[c]) - mu) * rs;
    }
    const float m1 = row_sum<1024>(s1, red[0]) * inv, m2 = row_sum<1024>(s2, red[1]) * inv;
    for (int c = threadIdx.x; c < a.width; c += 1024) {
      const float g = to_f(dy[c]) * (a.w ? load_param(a.w, a.wdtype, c) : 1.f), n = (to_f(x[c]) - mu) * rs;
      if (LNCC_IN(row * a.width + c, 1, a.rows * a.width)) dx[c] = from_f<T>(rs * (g - m1 - n * m2));
    }
  }
}
// Column sums over the rows of strand blockIdx.y, one thread a column.
template <typename T> __global__ void __launch_bounds__(kThreads) wide_columns_kernel(const Args a) {
  const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = to_f(static_cast<const T*>(a.dy)[row * a.dy_stride + c]);
    dw += d * (to_f(static_cast<const T*>(a.x)[row * a.x_stride + c]) - a.mean[row]) * a.rstd[row];
    db += d;
  }
  float* out = a.partial + int64_t(blockIdx.y) * 2 * a.width;
  out[c] = dw;
  out[a.width + c] = db;
}

// Elements of a thread and threads of a row: the smallest product that holds it, of 12 or 16 by a power of two from 4.
struct Shape {
  int lanes, elems;
};
static Shape shape_for(int64_t width) {
  for (int lanes = 4;; lanes *= 2)
    for (int elems = 12; elems <= kElems; elems += 4)
      if (int64_t(lanes) * elems >= width) return {lanes, elems};
}
static int lanes_for(int64_t width) { return shape_for(width).lanes; }

// Thread blocks of a call: as many as have rows, at most what the GPU holds at once (three of 256 threads an SM forward, two
// backward, whose sums take 120 registers; one of 512).
static int blocks_for(int64_t rows, int64_t width, bool backward) {
  const int sms = sm_count();
  if (width > kMaxWidth) return int(rows < sms * 2 ? rows : sms * 2);
  const int lanes = lanes_for(width), threads = lanes > kThreads ? lanes : kThreads;
  const int64_t need = ceil_div(rows, threads / lanes), fit = int64_t(sms) * (threads > kThreads ? 1 : backward ? 2 : 3);
  return int(need < fit ? need : fit);
}
static int strands_for(int64_t rows, int64_t width) {
  if (width <= kMaxWidth) return blocks_for(rows, width, true);
  return int(rows < 64 ? rows : 64);
}

template <typename T, int VEC, int E, int LANES> static void launch_lanes(const Args& a, bool backward, int grid, cudaStream_t st) {
  constexpr int threads = threads_of<LANES>();
  const int ring = Rows<T, LANES, VEC, E, threads>::smem(), smem = backward ? 2 * ring : ring;
  const auto kernel = backward ? backward_kernel<T, LANES, VEC, E> : forward_kernel<T, LANES, VEC, E>;
  static Asked asked[2];
  int dev = 0;
  if (smem > 40 * 1024 && cudaGetDevice(&dev) == cudaSuccess && !asked[backward].has(dev)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess) asked[backward].mark(dev);
  }
  kernel<<<grid, threads, smem, st>>>(a);
}
template <typename T, int VEC, int E> static void launch(const Args& a, bool backward, cudaStream_t st) {
  const int grid = blocks_for(a.rows, a.width, backward);
  switch (lanes_for(a.width)) {
    case 4: launch_lanes<T, VEC, E, 4>(a, backward, grid, st); break;
    case 8: launch_lanes<T, VEC, E, 8>(a, backward, grid, st); break;
    case 16: launch_lanes<T, VEC, E, 16>(a, backward, grid, st); break;
    case 32: launch_lanes<T, VEC, E, 32>(a, backward, grid, st); break;
    case 64: launch_lanes<T, VEC, E, 64>(a, backward, grid, st); break;
    case 128: launch_lanes<T, VEC, E, 128>(a, backward, grid, st); break;
    case 256: launch_lanes<T, VEC, E, 256>(a, backward, grid, st); break;
    default: launch_lanes<T, VEC, E, 512>(a, backward, grid, st); break;
  }
}

// 16-byte accesses (8 for 12 elements of 16 bits) where every row of every array starts on a 16-byte boundary, else single
// elements.
template <typename T> static void run(const Args& a, bool backward, cudaStream_t st) {
  constexpr int VEC = 16 / int(sizeof(T));
  const bool vec = a.width % VEC == 0 && a.x_stride % VEC == 0 && aligned(a.x, 16) && (!a.y || aligned(a.y, 16)) &&
                   (!backward || (a.dy_stride % VEC == 0 && aligned(a.dy, 16)));
  if (a.width > kMaxWidth) {
    const int grid = blocks_for(a.rows, a.width, backward);
    if (!backward) {
      wide_forward_kernel<T><<<grid, 1024, 0, st>>>(a);
      return;
    }
    if (a.y) wide_dx_kernel<T><<<grid, 1024, 0, st>>>(a);
    if (a.partial)
      wide_columns_kernel<T><<<dim3(unsigned(ceil_div(a.width, kThreads)), strands_for(a.rows, a.width)), kThreads, 0, st>>>(a);
    return;
  }
  const bool twelve = shape_for(a.width).elems == 12;
  if (vec && twelve) launch<T, 4, 12>(a, backward, st);
  else if (vec) launch<T, VEC, 16>(a, backward, st);
  else if (twelve) launch<T, 1, 12>(a, backward, st);
  else launch<T, 1, 16>(a, backward, st);
}

static void dispatch(const Args& a, int dtype, bool backward, cudaStream_t st) {
  if (dtype == LNCC_F32) run<float>(a, backward, st);
  else if (dtype == LNCC_BF16) run<__nv_bfloat16>(a, backward, st);
  else run<__half>(a, backward, st);
}

static int check_common(int dtype, int wdtype, int64_t rows, int64_t width, const void* x, int64_t x_stride) {
  if (!valid_dtype(dtype) || !valid_dtype(wdtype)) return LNCC_ERR_DTYPE;
  if (wdtype != dtype && wdtype != LNCC_F32) return LNCC_ERR_DTYPE;
  if (rows < 0 || width < 1) return LNCC_ERR_BAD_ARG;
  if (width > INT32_MAX / 4) return LNCC_ERR_TOO_LARGE;
  if (rows > 0 && (!x || !aligned(x, elem_size(dtype)) || (x_stride < width && rows > 1))) return LNCC_ERR_BAD_ARG;
  return LNCC_OK;
}

}  // namespace norm
}  // namespace lncc

using namespace lncc;

extern "C" {

int lncc_layer_norm_forward(const void* x, int64_t x_stride, const void* weight, const void* bias, int dtype, int wdtype,
                            int64_t rows, int64_t width, float eps, void* y, float* mean, float* rstd,
                            cudaStream_t stream) {
  const int st = norm::check_common(dtype, wdtype, rows, width, x, x_stride);
  if (st != LNCC_OK) return st;
  if (rows == 0) return LNCC_OK;
  const int we = blk::elem_size(wdtype);
  if (!y || !blk::aligned(y, blk::elem_size(dtype)) || !blk::aligned(weight, we) || !blk::aligned(bias, we) ||
      (mean == nullptr) != (rstd == nullptr) || !blk::aligned(mean, 4) || !blk::aligned(rstd, 4))
    return LNCC_ERR_BAD_ARG;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  norm::Args a = {};
  a.x = x, a.x_stride = x_stride, a.w = weight, a.b = bias, a.wdtype = wdtype, a.rows = rows, a.width = int(width);
  a.eps = eps, a.y = y, a.mean = mean, a.rstd = rstd;
  norm::dispatch(a, dtype, false, stream);
  return blk::check_end(stream);
}

size_t lncc_layer_norm_scratch_bytes(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > INT32_MAX / 4) return 0;
  return size_t(norm::strands_for(rows, width)) * 2 * size_t(width) * sizeof(float);
}

int lncc_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* weight,
                             int dtype, int wdtype, int64_t rows, int64_t width, const float* mean, const float* rstd,
                             void* dx, void* dweight, void* dbias, void* scratch, size_t scratch_bytes,
                             cudaStream_t stream) {
  const int st = norm::check_common(dtype, wdtype, rows, width, x, x_stride);
  if (st != LNCC_OK) return st;
  const bool params = dweight || dbias;
  const int we = blk::elem_size(wdtype);
  if (!blk::aligned(dweight, we) || !blk::aligned(dbias, we)) return LNCC_ERR_BAD_ARG;
  if (rows == 0) {  // sums over no rows
    const size_t n = size_t(width) * blk::elem_size(wdtype);
    if (dweight && cudaMemsetAsync(dweight, 0, n, stream) != cudaSuccess) return LNCC_ERR_CUDA;
    if (dbias && cudaMemsetAsync(dbias, 0, n, stream) != cudaSuccess) return LNCC_ERR_CUDA;
    return LNCC_OK;
  }
  const int e = blk::elem_size(dtype);
  if (!dy || !blk::aligned(dy, e) || (dy_stride < width && rows > 1) || !blk::aligned(weight, we) || !mean || !rstd ||
      !blk::aligned(mean, 4) || !blk::aligned(rstd, 4) || (dx && !blk::aligned(dx, e)))
    return LNCC_ERR_BAD_ARG;
  if (params && (!scratch || !blk::aligned(scratch, 4) || scratch_bytes < lncc_layer_norm_scratch_bytes(rows, width)))
    return LNCC_ERR_WORKSPACE;
  if (!dx && !params) return LNCC_OK;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  norm::Args a = {};
  a.x = x, a.x_stride = x_stride, a.dy = dy, a.dy_stride = dy_stride, a.w = weight, a.wdtype = wdtype, a.rows = rows;
  a.width = int(width), a.y = dx, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.partial = params ? static_cast<float*>(scratch) : nullptr;
  norm::dispatch(a, dtype, true, stream);
  if (params)
    norm::reduce_kernel<<<unsigned(blk::ceil_div(2 * width, 32)), 1024, 0, stream>>>(
        a.partial, norm::strands_for(rows, width), a.width, dweight, dbias, wdtype);
  return blk::check_end(stream);
}

}  // extern "C"
