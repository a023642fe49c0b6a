// The gated feed-forward block, forward and backward:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu
//   dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Every product runs on the tensor cores, in one kernel whose epilogue does what follows it: UP forms g and u side by side
// in tensor memory and writes h alone; HIDDEN forms dh, g and u (again, from x) and writes dg, du and h (for fp32 GATES
// writes g and u, DH dh, and a kernel of its own reads the three); the others write a result or, where a long inner axis is
// split over the GPU, fp32 partial sums that a last kernel adds in order.
//
// A pair of CTAs takes a tile of 256 rows by up to 256 columns (cta_group::2): each loads its 128 rows of A and half the
// columns of B, 64 steps of the inner axis at a time, into a ring of TMA stages; one thread of the pair issues
// the products into tensor memory, and sixteen warps of each CTA read finished tiles back while the next one runs.
// Halving B between the pair matters: a tile of 256 x 256 asks L2 for 64 bytes a clock and SM at the full rate of the
// tensor cores, one of 128 x 256 for 96. The grid stays (one pair for each two SMs) and walks over the tiles, columns
// first, so that the pairs at work share rows of A and the weights stay in L2.
// Measured at 16384 x 1024 x 4096 bf16, each kernel by itself: UP 174 us (1580 TFLOP/s), DOWN 96 and DX 186 (1430 and 1480, four rounds of tiles for 3.46);
// DW_UP 185, DW_DOWN 96, HIDDEN 363 (1140, its dh on 128 columns). The products alone,
// with no loads and no epilogue, take 588 clocks a block of a tile of 256 x 256, DX's 609. At 107520 x 96 x 256, where bytes count: UP 34 us
// (2.2 TB/s), HIDDEN 61 (3.4 TB/s), the epilogue's instructions and latency bounding both.
//
// Nothing of the hidden layer is kept between forward and backward. Forming g and u again costs 4 of 22 M F K products of a
// training step, and saves writing and reading 4 M F bytes and a rounding of g and u.
//
// Roundings. For 16-bit types h, dg and du are rounded to the type's bits, since they are operands of the next product (for fp16
// times a power of 2 a row, see below: its range would not hold them); g, u and dh never leave fp32. The result then holds two
// roundings of like size, its own and h's, and is sqrt 2 as far off as one that keeps h in fp32 (more than four tokens, fp16:
// 2.9e-4 of the result against 2.1e-4, bf16 2.4e-3 against 1.7e-3); in calls of a few hundred values the factor scatters, at 5 x
// 48 x 79 between 1.25 and 1.63 in nine draws of ten. fp32 operands are taken apart into three bf16 numbers of 8 bits each,
// which hold all 24 bits, and six of the nine products are summed, smallest first (the other three are below 2^-24 of the
// result). An infinity taken apart meets zeros: it gives NaN where fp32 would give an infinity.
// The tensor cores cut, not round, what they add to an accumulator: over an inner axis of 4096 that came to 1e-5 of an fp32
// result. So for fp32 an accumulator takes 256 of the inner axis, and the epilogue adds these sums in registers, rounding each
// time. The 16-bit products with long inner axes do so every 2048: sums over 131072 tokens that do not cancel came out 8.5e-4 too
// small in one accumulator, more than fp16's own rounding, and 2.4e-5 now, at the same speed. (g, u and dh, whose inner axes are
// the block's widths, take one accumulator for 16-bit types: 8e-6 at 1024.)
#include "lncc_tc.cuh"

#include <type_traits>

namespace lncc {
namespace ffn {

using namespace blk;
using namespace tc;

constexpr uint32_t kNaN = 0x7fffffff;  // what a tile gets whose products were given up

enum Kind { UP, GATES, HIDDEN, DH, DOWN, DX, DW_UP, DW_DOWN };

constexpr int kEpilogueWarps = 16;         // of a CTA: four for each quarter of the lanes of tensor memory
constexpr int kThreads = 128 + 32 * kEpilogueWarps;  // warps 0 TMA, 1 products, 4 - 19 epilogue
constexpr int kATile = 128 * 64 * 2;       // bytes of a CTA's share of A in a stage
constexpr int kChunk = 4, kChunk16 = 32;   // blocks of 64 that an accumulator takes: fp32, and 16-bit types where sums are long

__host__ __device__ constexpr bool a_mn(int kind) { return kind == DW_UP || kind == DW_DOWN; }
__host__ __device__ constexpr bool b_mn(int kind) { return kind == DH || kind == DX || kind == DW_UP || kind == DW_DOWN; }
__host__ __device__ constexpr bool gated(int kind) { return kind == UP || kind == GATES || kind == HIDDEN; }
__host__ __device__ constexpr int b_tile(int bn) { return bn / 2 * 64 * 2; }  // a CTA's share of B
__host__ __device__ constexpr int stages(int bn) { return bn == 256 ? 6 : 8; }
__host__ __device__ constexpr int smem_bytes(int bn) { return 1024 + stages(bn) * (kATile + b_tile(bn)) + 256 + kEpilogueWarps * 32 * 9 * 4; }

// Planes of the six products of operands that are taken apart, smallest first.
__device__ __constant__ const int8_t kPlaneA[6] = {2, 1, 0, 1, 0, 0}, kPlaneB[6] = {0, 1, 2, 0, 1, 0};

struct Gemm {
  CUtensorMap a0, a1, b0, b1, b2;
  int64_t rows, cols;        // of a result
  int m_tiles, n_tiles, whichs, splits;
  int k_steps, k_steps2;     // blocks of 64 of the inner axis (HIDDEN: of g and u, and of dh)
  int blocks, per_split;     // of a tile: k_steps times the products summed into it (DX: 2); those of a split
  int bf16;
  void *out0, *out1, *out2;  // results (DW_UP: of which = 0, 1; HIDDEN: dg, du, h; GATES: g, u)
  int64_t ld, plane;         // of the results; plane for h taken apart
  int align;                 // bytes on which every row of the results starts: 32, 16 or the element's
  float* partial;            // [splits][whichs][rows][cols rounded up to 4], where splits > 1
  int8_t* levels;            // fp16: of the hidden matrices, as the gated kinds write them
  const int *row_h, *row_d, *most;  // and as level_kernel leaves them
  int level_blocks;
  unsigned* abort_word;
  int clear_abort;
};

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// act(g) and act'(g). For 16-bit types by the fast exponential of 2 and reciprocal (a few u32, and |g| u32 for the
// exponential), and erfc(z)/2, z = |g|/sqrt 2, as t P(t) exp(-z^2) with t = 1/(1 + 0.3 |g|). The exponential is the one of the
// derivative, and P is the polynomial of degree 5 that minimises the largest relative error for |g| up to 13.3, where the
// exponential ends: 7.5e-6 of the value everywhere, 1/65 of a rounding to fp16, in the lower tail too. (A form that is right
// absolutely, like Abramowitz and Stegun 7.1.26 to 1.5e-7, is off by 9e-4 of gelu(-4.5) and 1e-2 of gelu(-8).) The epilogue is
// bound by its instructions where K is small: constants are folded (log2 e into the exponent, 1/2 into the coefficients).
template <int ACT, bool FAST> __device__ __forceinline__ void activate(float g, float& a, float& da) {
  if (ACT == LNCC_ACT_RELU) {
    a = g < 0.f ? 0.f : g;
    da = g > 0.f ? 1.f : 0.f;
  } else if (ACT == LNCC_ACT_SILU) {
    const float p = FAST ? rcp_fast(1.f + exp2_fast(g * -1.44269504f)) : 1.f / (1.f + expf(-g));
    a = g * p;
    da = FAST ? fmaf(a, 1.f - p, p) : p * (1.f + g * (1.f - p));
  } else if (FAST) {
    const float e = exp2_fast(g * g * -0.72134752f), t = rcp_fast(fmaf(0.3f, fabsf(g), 1.f));
    const float q =
        e * t *
        fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.0776683912f, 0.217757061f), -0.0189181864f), 0.145261124f), 0.113472365f),
             0.120099664f);
    const float p = g < 0.f ? q : 1.f - q;
    a = g * p;
    da = fmaf(g * 0.39894228f, e, p);
  } else {
    const float p = 0.5f * erfcf(-g * 0.70710678f);
    a = g * p;
    da = fmaf(g * 0.39894228f, expf(-0.5f * g * g), p);
  }
}

// two values rounded to 16 bits, the first in the lower half
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// NW words (16 or 32 bytes) of 32 rows, a row a lane, from column col on: what lies inside rows x cols. Whole pieces of rows
// that start on 16 or 32 bytes go straight out. The rest goes through shared memory and out again with the lanes side by
// side along a row: element by element with a row a lane, a product with 333 columns took 130 us of which 95 were its stores.
constexpr int kStageWords = 32 * 9;
template <typename T, int NW>
__device__ __forceinline__ void emit(T* base, int64_t ld, int64_t row0, int64_t col, int64_t rows, int64_t cols, int align,
                                     const uint32_t (&w)[NW], uint32_t* stage) {
  constexpr int N = NW * 4 / int(sizeof(T)), PITCH = NW + 1;  // elements; words from row to row of the stage
  const int lane = threadIdx.x % 32;
  if (col >= cols) return;  // the same for all lanes, like the next
  if (col + N <= cols && align >= 16) {
    const int64_t row = row0 + lane;
    if (row >= rows || !LNCC_IN(row * ld + col, N, (rows - 1) * ld + cols)) return;
    uint32_t* p = reinterpret_cast<uint32_t*>(base + row * ld + col);
    if (NW == 8 && align >= 32) {
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                   "r"(w[4 % NW]), "r"(w[5 % NW]), "r"(w[6 % NW]), "r"(w[7 % NW])
                   : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < NW; i += 4) *reinterpret_cast<uint4*>(p + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NW; i++) stage[lane * PITCH + i] = w[i];
    __syncwarp();
    const int c = lane % N, per_turn = 32 / N;
    T* p = base + (row0 + lane / N) * ld + col + c;
    if (col + c < cols) {
#pragma unroll 4
      for (int r = lane / N; r < 32; r += per_turn, p += per_turn * ld)
        if (row0 + r < rows && LNCC_IN((row0 + r) * ld + col + c, 1, (rows - 1) * ld + cols))
          *p = reinterpret_cast<const T*>(stage + r * PITCH)[c];
    }
    __syncwarp();
  }
}
// fp32 as three bf16 numbers that add up to it. The first is cut, not rounded, so that it stays finite; all 24 bits are held.
__device__ __forceinline__ void take_apart(float v, __nv_bfloat16& hi, __nv_bfloat16& mid, __nv_bfloat16& lo) {
  hi = __float2bfloat16_rz(v);
  const float r = v - __bfloat162float(hi);
  const bool fine = fabsf(v) <= 3.4028235e38f;
  mid = __float2bfloat16_rn(fine ? r : 0.f);
  lo = __float2bfloat16_rn(fine ? r - __bfloat162float(mid) : 0.f);
}
// Eight results of a row in fp32, as the three bf16 matrices that hold them.
__device__ __forceinline__ void emit_parts(void* base, const Gemm& g, int64_t row0, int64_t col, const float (&v)[8],
                                           uint32_t* stage) {
  float part[3][8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    __nv_bfloat16 hi, mid, lo;
    take_apart(v[i], hi, mid, lo);
    part[0][i] = to_f(hi), part[1][i] = to_f(mid), part[2][i] = to_f(lo);
  }
#pragma unroll
  for (int k = 0; k < 3; k++) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = pack2<__nv_bfloat16>(part[k][2 * i], part[k][2 * i + 1]);
    emit<__nv_bfloat16, 4>(static_cast<__nv_bfloat16*>(base) + k * g.plane, g.ld, row0, col, g.rows, g.cols, g.align, w, stage);
  }
}

// ---- the range of fp16 -------------------------------------------------------------------------------------------------
// h, dg and du are operands of the next product, and as they are they need not lie in fp16's range: gates and up projections
// of some hundreds give hidden values past 65504 in a block whose result is small, and the gradients of a mean over many tokens
// lie among the subnormal numbers. So with fp16 a row of them is stored times a power of 2. Its largest value is not known
// while its tiles are written (a bound like |x|_1 max|W| is some 2^16 above the values of a dense row, and more where a few
// weights stand out), so each piece of 8 columns gets a power of its own, 2^(11 - 8k) with the smallest k that keeps the piece
// below 2^15, and level_kernel then brings the pieces of a row to the power of the row's largest k. Steps of 8, of which k = 0
// holds pieces whose largest value lies between 2^-4 and 2^4, leave few or none to rewrite. What is 2^-21 of its row's largest
// value and more keeps fp16's 11 bits at least; the rest is right to 2^-32 of it.
// The product that reads a row takes its power back out in the epilogue (DOWN, DX). The weights' gradients sum over rows of
// different powers: there the other operand, x or dy, is copied with the row's power taken out of it, relative to the largest
// of the call. dg and du share a power, since dx adds their products up. Measured beside bf16: 4096 x 768 x 2048 forward 52 us
// (43), 107520 x 96 x 256 training 275 (197), 16384 x 1024 x 4096 training 1384 (1315); level_kernel's backward part 19, 33 and
// 62 us of them, 101 where every row has pieces to rewrite. As two bf16 numbers each, 16 bits in fp32's range, h, dg and du took
// three products for one: 69, 349 and 2575 us.
constexpr int kStep = 8;
constexpr int kNoLevel = -64;      // k of zeros
constexpr int kLowest = -13;       // the least k otherwise
enum Most { MOST_DY_H, MOST_X_D, MOSTS };  // largest e + kStep k of |dy| < 2^e and h, and of |x| and dg, du

__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((max(-126, min(126, e)) + 127) << 23); }
// k of numbers whose largest absolute value is v
__device__ __forceinline__ int level_of(float v) {
  return v > 0.f ? max(kLowest, ((__float_as_int(v) >> 23) - 123) >> 3) : kNoLevel;
}
__device__ __forceinline__ float power_of_level(int k) { return power_of_2(11 - kStep * max(k, kLowest)); }
// the largest finite |v[i]|, and `least`
template <int N> __device__ __forceinline__ float largest(const float (&v)[N], float least) {
  float m = least;
#pragma unroll
  for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(v[i]));
  if (m > 3.4028235e38f) {
    m = least;
#pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(v[i]) <= 3.4028235e38f ? fabsf(v[i]) : 0.f);
  }
  return m;
}
// one of the call's largest, of the blocks' ones, for a whole warp
__device__ __forceinline__ int most_of(const int* most, int blocks, int which) {
  int e = kStep * kNoLevel;
  for (int i = threadIdx.x % 32; i < blocks; i += 32) e = max(e, most[which * blocks + i]);
  return __reduce_max_sync(0xffffffffu, e);
}

// A call's kernels but the first are launched before the one ahead has ended. Each lets the next begin at once and waits here
// before it touches memory, so that one kernel's set-up hides behind the other's end.
__device__ __forceinline__ void begin_after_previous() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One tile: 256 rows m, columns n, one of the results, blocks [from, to) of its inner axis. One division where nothing is
// split: the thread that issues the products works this out between tiles, and the tensor cores wait for it (five
// divisions, two of them of 64 bits, cost UP 24 of 198 us).
struct Tile {
  int n, m, which, split, from, to;
};
__device__ __forceinline__ Tile tile_of(const Gemm& g, int t) {
  Tile r;
  r.m = t / g.n_tiles, r.n = t - r.m * g.n_tiles, r.which = r.split = 0, r.from = 0, r.to = g.blocks;
  if (g.whichs * g.splits > 1) {
    t = r.m;
    r.split = t / (g.m_tiles * g.whichs), t -= r.split * g.m_tiles * g.whichs;
    r.which = t / g.m_tiles, r.m = t - r.which * g.m_tiles;
    r.from = r.split * g.per_split, r.to = min(g.blocks, r.from + g.per_split);
  }
  return r;
}

// T: type of the results (for float, bf16 operands taken apart). KIND, BN: see above; gated kinds hold BN/2 columns of g
// and of u, HIDDEN BN/2 of dh beside them. ACT: the activation of UP and HIDDEN.
template <int KIND, int BN, int ACT, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ Gemm g) {
  constexpr int STAGES = stages(BN), BT = b_tile(BN), HALF = BN / 2;
  constexpr bool AM = a_mn(KIND), BM = b_mn(KIND), F32 = sizeof(T) == 4;
  // Tiles of accumulators in tensor memory. HIDDEN of 256 columns has one: dh then alternates between two places, so it may
  // run while the last tile is read, and g and u wait for that.
  constexpr bool ONE = KIND == HIDDEN && BN == 256;
  constexpr int ACCS = ONE ? 1 : 2;
  constexpr int DH_BYTES = BN == 256 ? 8192 : 4096;    // a CTA's share of Wd in a stage: 64 or 32 columns
  constexpr int PARTS = F32 ? 6 : 1;                   // products of parts of the operands
  constexpr bool PROMOTED = F32 || !gated(KIND);       // accumulators take a chunk each, and are added up in registers
  constexpr int CHUNK = F32 ? kChunk : PROMOTED ? kChunk16 : 1 << 30;
  static_assert(KIND != HIDDEN || !F32, "fp32 has GATES and DH");
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((uintptr_t(raw) + 1023) / 1024 * 1024);
  const uint32_t tiles_at = smem_addr(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * (kATile + BT));
  const uint32_t full = smem_addr(bars), empty = full + 8 * STAGES, acc_full = empty + 8 * STAGES, acc_empty = acc_full + 16;
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up_flag;
  volatile int* gave_up = &gave_up_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cta_rank();

  if (threadIdx.x == 0) {
    gave_up_flag = 0;
    for (int i = 0; i < STAGES; i++) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, 2 * kEpilogueWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 64) {  // the maps are the launch's own: they may come in before the kernel ahead has ended
    prefetch_map(&g.a0);
    prefetch_map(&g.b0);
    if (KIND == HIDDEN || KIND == DX || KIND == DW_UP) prefetch_map(&g.a1);
    if (gated(KIND) || KIND == DX) prefetch_map(&g.b1);
    if (KIND == HIDDEN) prefetch_map(&g.b2);
  }
  if (warp == 1) {
    tmem_alloc<512>(smem_addr(&tmem_at));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  begin_after_previous();  // all of the above runs while the kernel before this one ends
  const uint32_t tmem = tmem_at;
  if (g.clear_abort && blockIdx.x == 0 && threadIdx.x == 0) *g.abort_word = 0u;  // waits give up seconds later
  const int pairs_at_work = gridDim.x / 2, tiles = g.n_tiles * g.m_tiles * g.whichs * g.splits;

  if (warp == 0 && lane == 0) {
    // ---- TMA: this CTA's shares of A and B, counted on the first CTA's barrier
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full_of_pair = peer_addr(full, 0);
    for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs_at_work) {
      const Tile w = tile_of(g, t);
      const int m0 = w.m * 256 + int(rank) * 128;
      const CUtensorMap* a_first = KIND == DW_UP && w.which ? &g.a1 : &g.a0;
      for (int c = w.from; c < w.to && ok; c += CHUNK) {
        const int c_end = PROMOTED ? min(c + CHUNK, w.to) : w.to;
        for (int part = 0; part < PARTS && ok; part++) {
          const int pa = F32 ? kPlaneA[part] : 0, pb = F32 ? kPlaneB[part] : 0;
          for (int b = c; b < c_end; b++) {
            if (!(ok = mbar_wait(empty + 8 * stage, phase ^ 1, gave_up))) break;
            const uint32_t at = tiles_at + stage * (kATile + BT), bt = at + kATile, bar = full_of_pair + 8 * stage;
            const bool dh = KIND == HIDDEN && b < g.k_steps2;              // HIDDEN: dh first
            const bool second = KIND == DX && b >= g.k_steps;              // DX: du Wu after dg Wg
            const int k = 64 * (KIND == HIDDEN && !dh ? b - g.k_steps2 : second ? b - g.k_steps : b);
            if (rank == 0) mbar_expect(full + 8 * stage, 2 * (kATile + (dh ? DH_BYTES : BT)));
            const CUtensorMap* am = dh || second ? &g.a1 : a_first;
            if (AM) {
              tma_load(am, at, bar, m0, k, pa);
              tma_load(am, at + kATile / 2, bar, m0 + 64, k, pa);
            } else {
              tma_load(am, at, bar, k, m0, pa);
            }
            if (dh) {  // half of the tile's columns of Wd, which memory holds along F
              tma_load(&g.b2, bt, bar, w.n * HALF + int(rank) * (HALF / 2), k, pb);
            } else if (gated(KIND)) {  // the gate's rows in one CTA, the up projection's in the other
              tma_load(rank ? &g.b1 : &g.b0, bt, bar, k, w.n * HALF, pb);
            } else if (BM) {
              const CUtensorMap* bm = second ? &g.b1 : &g.b0;
#pragma unroll
              for (int i = 0; i < HALF; i += 64) tma_load(bm, bt + i / 64 * 8192, bar, w.n * BN + int(rank) * HALF + i, k, pb);
            } else {
              tma_load(&g.b0, bt, bar, k, w.n * BN + int(rank) * HALF, pb);
            }
            if (++stage == STAGES) stage = 0, phase ^= 1;
          }
        }
      }
    }
    // every copy has landed once its stage has been read; after giving up, copies in flight get 10 ms to land
    for (int i = 0; i < STAGES && ok; i++) {
      ok = mbar_wait(empty + 8 * stage, phase ^ 1, gave_up);
      if (++stage == STAGES) stage = 0, phase ^= 1;
    }
    if (!ok)
      for (const unsigned long long start = now_ns(); now_ns() - start < 10000000ull;) __nanosleep(1000);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- products of the pair
    int stage = 0, turn = 0;  // turn counts the accumulators filled
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t wide = instr_desc(g.bf16, AM, BM, BN), narrow = instr_desc(g.bf16, false, true, HALF);
    for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs_at_work) {
      const Tile w = tile_of(g, t);
      for (int c = w.from; c < w.to && ok; c += CHUNK, turn++) {
        const int steps = (PROMOTED ? min(CHUNK, w.to - c) : w.to - c) * PARTS;
        const int acc = ACCS == 2 ? turn & 1 : 0;
        const uint32_t acc_phase = ACCS == 2 ? (turn >> 1) & 1 : turn & 1;
        const uint32_t d = tmem + (ACCS == 2 ? acc * 256 : 0), d_dh = ONE ? tmem + BN + (turn & 1) * HALF : d + BN;
        if (!ONE) {
          if (!(ok = mbar_wait(acc_empty + 8 * acc, acc_phase ^ 1, gave_up))) break;
          fence_after();
        }
        for (int s = 0; s < steps; s++) {
          const bool dh = KIND == HIDDEN && s < g.k_steps2;
          if (ONE && s == g.k_steps2) {
            if (!(ok = mbar_wait(acc_empty, acc_phase ^ 1, gave_up))) break;
            fence_after();
          }
          if (!(ok = mbar_wait(full + 8 * stage, phase, gave_up))) break;
          fence_after();
          const uint32_t at = tiles_at + stage * (kATile + BT), bt = at + kATile;
          const uint64_t da = AM ? desc_mn(at, 8192) : desc_k(at);
          const uint64_t db = dh && BN == 128 ? desc_mn_32(bt) : BM || dh ? desc_mn(bt, 8192) : desc_k(bt);
          const uint64_t a_step = AM ? 128 : 2, b_step = dh && BN == 128 ? 64 : BM || dh ? 128 : 2;
          const bool first = s == 0 || (KIND == HIDDEN && s == g.k_steps2);
#pragma unroll
          for (int k = 0; k < 4; k++)
            mma(dh ? d_dh : d, da + k * a_step, db + k * b_step, dh ? narrow : wide, k > 0 || !first);
          commit_pair(empty + 8 * stage);
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        if (ok) commit_pair(acc_full + 8 * acc);
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue: lanes are rows; four warps share a row, a quarter of the columns each
    const int sub = warp & 3, quarter = (warp - 4) / 4;
    constexpr int COLS = gated(KIND) ? HALF / 4 : BN / 4;  // columns of a result that a warp takes
    uint32_t* const stage = reinterpret_cast<uint32_t*>(smem + STAGES * (kATile + BT) + 256) + (warp - 4) * kStageWords;
    int turn = 0;
    constexpr bool LEVELS = std::is_same<T, __half>::value;
    // weights' gradients: what their operands lack together
    const float power_all =
        LEVELS && AM ? power_of_2(most_of(g.most, g.level_blocks, KIND == DW_UP ? MOST_X_D : MOST_DY_H) - 26) : 1.f;
    for (int t = blockIdx.x / 2; t < tiles; t += pairs_at_work) {
      const Tile w = tile_of(g, t);
      const int64_t row0 = int64_t(w.m) * 256 + rank * 128 + sub * 32;
      const int64_t col0 = int64_t(w.n) * (gated(KIND) ? HALF : BN) + quarter * COLS;
      const bool rows_here = row0 < g.rows;
      const auto done = [&](int acc) {  // this warp has read the accumulator
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(peer_addr(acc_empty + 8 * acc, 0));
      };
      // where an ordinary 16-bit result of this tile goes: its type, or partial sums in fp32
      const auto put = [&](int64_t col, const float (&v)[16]) {
        if (g.splits > 1) {
          const int64_t ld = (g.cols + 3) / 4 * 4;
          float* to = g.partial + (int64_t(w.split) * g.whichs + w.which) * g.rows * ld;
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = __float_as_uint(v[i + j]);
            emit<float, 8>(to, ld, row0, col + i, g.rows, ld, 16, o, stage);
          }
        } else if constexpr (sizeof(T) == 2) {
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
          emit<T, 8>(static_cast<T*>(w.which ? g.out1 : g.out0), g.ld, row0, col, g.rows, g.cols, g.align, o, stage);
        }
      };

      if constexpr (PROMOTED) {
        constexpr int SUMS = gated(KIND) ? 2 * COLS : COLS;  // gated: columns of g, then of u
        int row_level = 0;  // on its way while the products run
        if (LEVELS && !AM && row0 + lane < g.rows) row_level = (KIND == DOWN ? g.row_h : g.row_d)[row0 + lane];
        float sum[SUMS];
#pragma unroll
        for (int i = 0; i < SUMS; i++) sum[i] = 0.f;
        for (int c = w.from; c < w.to; c += CHUNK, turn++) {
          const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * (turn & 1), (turn >> 1) & 1, gave_up));
          fence_after();
          const uint32_t d = tmem + (uint32_t(sub * 32) << 16) + (turn & 1) * 256 + quarter * COLS;
#pragma unroll
          for (int i = 0; i < SUMS; i += 16) {
            uint32_t v[16];
            if (ok) {
              tmem_load(d + (gated(KIND) && i >= COLS ? HALF + i - COLS : i), v);
              wait_ld(v);
            } else {
              for (int j = 0; j < 16; j++) v[j] = kNaN;
            }
#pragma unroll
            for (int j = 0; j < 16; j++) sum[i + j] += __uint_as_float(v[j]);
          }
          done(turn & 1);
        }
        if (!rows_here) continue;
        if constexpr (KIND == UP) {
#pragma unroll
          for (int c = 0; c < COLS; c += 8) {
            if (col0 + c >= g.cols) break;
            float h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              float a, da;
              activate<ACT, false>(sum[c + i], a, da);
              h[i] = a * sum[(COLS + c + i) % SUMS];
            }
            emit_parts(g.out0, g, row0, col0 + c, h, stage);
          }
        } else if constexpr (!F32) {
          if (LEVELS) {
            const float power = AM ? power_all : power_of_2(kStep * row_level - 11);
#pragma unroll
            for (int c = 0; c < SUMS; c++) sum[c] *= power;
          }
#pragma unroll
          for (int c = 0; c < SUMS; c += 16) put(col0 + c, reinterpret_cast<const float(&)[16]>(sum[c]));
        } else {
#pragma unroll
          for (int c = 0; c < SUMS; c += 8) {
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = __float_as_uint(sum[c + j]);
            const bool second = KIND == GATES && c >= COLS;
            const int64_t col = col0 + (second ? c - COLS : c), ld = (g.cols + 3) / 4 * 4;
            if (KIND != GATES && g.splits > 1)
              emit<float, 8>(g.partial + (int64_t(w.split) * g.whichs + w.which) * g.rows * ld, ld, row0, col, g.rows, ld, 16, o, stage);
            else
              emit<float, 8>(static_cast<float*>(second || w.which ? g.out1 : g.out0), g.ld, row0, col, g.rows, g.cols, g.align, o, stage);
          }
        }
      } else {
        const int acc = ACCS == 2 ? turn & 1 : 0;
        const uint32_t acc_phase = ACCS == 2 ? (turn >> 1) & 1 : turn & 1;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * acc, acc_phase, gave_up));
        fence_after();
        const uint32_t d = tmem + (uint32_t(sub * 32) << 16) + (ACCS == 2 ? acc * 256 : 0) + quarter * COLS;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 16) {
          __syncwarp();
          const int64_t col = col0 + c;
          {
            uint32_t h[8], dg[8], du[8];
            uint32_t levels = 0;  // a byte a piece: of h, and then of dg and du
#pragma unroll
            for (int half = 0; half < 2; half++) {  // eight columns at a time: 640 threads leave 102 registers each
              uint32_t v[3][8];
              const uint32_t at = d + c + half * 8;
              if (ok) {
                tmem_load(at, v[0]);
                tmem_load(at + HALF, v[1]);
                if (KIND == HIDDEN) tmem_load(at + BN + (ONE ? (turn & 1) * HALF : 0), v[2]);
                wait_ld(v[0]);
                wait_ld(v[1]);
                if (KIND == HIDDEN) wait_ld(v[2]);
              } else {
                for (int i = 0; i < 8; i++) v[0][i] = v[1][i] = v[2][i] = kNaN;
              }
              float fh[8], fdg[8], fdu[8];
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                float a[2], da[2];
#pragma unroll
                for (int j = 0; j < 2; j++) activate<ACT, true>(__uint_as_float(v[0][i + j]), a[j], da[j]);
                const float u0 = __uint_as_float(v[1][i]), u1 = __uint_as_float(v[1][i + 1]);
                fh[i] = a[0] * u0, fh[i + 1] = a[1] * u1;
                if (KIND == HIDDEN) {
                  const float d0 = __uint_as_float(v[2][i]), d1 = __uint_as_float(v[2][i + 1]);
                  fdg[i] = d0 * u0 * da[0], fdg[i + 1] = d1 * u1 * da[1];
                  fdu[i] = d0 * a[0], fdu[i + 1] = d1 * a[1];
                }
              }
              float power_h = 1.f, power_d = 1.f;
              if (LEVELS) {
                const int k = level_of(largest(fh, 0.f));
                power_h = power_of_level(k);
                levels |= uint32_t(k & 255) << 8 * half;
                if (KIND == HIDDEN) {
                  const int kd = level_of(largest(fdg, largest(fdu, 0.f)));
                  power_d = power_of_level(kd);
                  levels |= uint32_t(kd & 255) << 16 + 8 * half;
                }
              }
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                const float ph = power_h, pd = power_d;
                h[half * 4 + i / 2] = LEVELS ? pack2<T>(fh[i] * ph, fh[i + 1] * ph) : pack2<T>(fh[i], fh[i + 1]);
                if (KIND == HIDDEN) {
                  dg[half * 4 + i / 2] = LEVELS ? pack2<T>(fdg[i] * pd, fdg[i + 1] * pd) : pack2<T>(fdg[i], fdg[i + 1]);
                  du[half * 4 + i / 2] = LEVELS ? pack2<T>(fdu[i] * pd, fdu[i + 1] * pd) : pack2<T>(fdu[i], fdu[i + 1]);
                }
              }
            }
            if (c + 16 == COLS) done(acc);
            if (!rows_here) continue;
            if (KIND == HIDDEN) {
              emit<T, 8>(static_cast<T*>(g.out0), g.ld, row0, col, g.rows, g.cols, g.align, dg, stage);
              emit<T, 8>(static_cast<T*>(g.out1), g.ld, row0, col, g.rows, g.cols, g.align, du, stage);
            }
            emit<T, 8>(static_cast<T*>(KIND == HIDDEN ? g.out2 : g.out0), g.ld, row0, col, g.rows, g.cols, g.align, h, stage);
            if (LEVELS && row0 + lane < g.rows && col < g.cols) {
              const int64_t at = (row0 + lane) * ((g.cols + 15) / 16) + col / 16;
              if (!LNCC_IN(at, 1, g.rows * ((g.cols + 15) / 16))) continue;
              if (KIND == HIDDEN) reinterpret_cast<uint32_t*>(g.levels)[at] = levels;
              else reinterpret_cast<uint16_t*>(g.levels)[at] = uint16_t(levels);
            }
          }
        }
        turn++;
      }
    }
  }
  __syncwarp();
  __syncthreads();
  cluster_sync();  // no CTA leaves while the other may still signal it or read its shares
  if (*gave_up && threadIdx.x == 0) atomicOr(g.abort_word, 1u);
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Partial sums of the splits, added in order: a thread a quad of columns, or, for many splits of few columns, STRANDS threads
// with every STRANDS-th split each, whose sums are then added in order.
constexpr int kManySplits = 16;
template <typename T, int STRANDS>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, int splits, int whichs, int64_t rows,
                                                   int64_t cols, T* out0, T* out1) {
  constexpr int LANES = 256 / STRANDS;
  __shared__ float4 meet[STRANDS][LANES];
  begin_after_previous();
  const int strand = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int64_t ld = (cols + 3) / 4 * 4, quads = whichs * rows * (ld / 4), q = int64_t(blockIdx.x) * LANES + lane;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (q < quads) {
#pragma unroll 4
    for (int i = strand; i < splits; i += STRANDS) {
      const float4 v = reinterpret_cast<const float4*>(partial)[i * quads + q];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  if (STRANDS > 1) {
    meet[strand][lane] = s;
    __syncthreads();
    if (strand != 0) return;
    for (int i = 1; i < STRANDS; i++) {
      const float4 v = meet[i][lane];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  if (q >= quads) return;
  const uint32_t per_row = uint32_t(ld / 4);
  const int64_t r = q / per_row, row = r < rows ? r : r - rows, col = (q - r * per_row) * 4;
  T* out = r < rows ? out0 : out1;
  const float v[4] = {s.x, s.y, s.z, s.w};
  T* to = out + row * cols + col;
  if (cols % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0) {
    if (LNCC_IN(row * cols + col, 4, rows * cols)) store_vec<T, 4>(to, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (col + i < cols && LNCC_IN(row * cols + col + i, 1, rows * cols)) to[i] = from_f<T>(v[i]);
}

// Matrices that TMA cannot read as they lie (fp32, or rows off the 16-byte boundary) laid out as planes of aligned rows: up to
// five in one launch, each with blocks of its own.
struct Pack {
  const void* src;
  void* dst;
  int64_t stride, rows, cols, ld, plane;
  int first_block;
};
struct Packs {
  Pack job[5];
  int jobs, blocks;
};
template <typename T, typename TO> __global__ void __launch_bounds__(256) pack_kernel(const Packs p) {
  begin_after_previous();
  int j = 0;
  while (j + 1 < p.jobs && int(blockIdx.x) >= p.job[j + 1].first_block) j++;
  const Pack& m = p.job[j];
  const T* src = static_cast<const T*>(m.src);
  TO* dst = static_cast<TO*>(m.dst);
  const uint32_t per_row = uint32_t(m.ld / 8), blocks = (j + 1 < p.jobs ? p.job[j + 1].first_block : p.blocks) - m.first_block;
  const int64_t eights = m.rows * per_row;
  for (int64_t q = int64_t(blockIdx.x - m.first_block) * 256 + threadIdx.x; q < eights; q += int64_t(blocks) * 256) {
    const int64_t row = q / per_row, col = (q - row * per_row) * 8;
    Vec<TO, 8> o[3];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const T v = col + i < m.cols && LNCC_IN(row * m.stride + col + i, 1, (m.rows - 1) * m.stride + m.cols)
                      ? src[row * m.stride + col + i] : from_f<T>(0.f);
      if constexpr (sizeof(T) == 4) take_apart(v, o[0].e[i], o[1].e[i], o[2].e[i]);
      else o[0].e[i] = v;
    }
#pragma unroll
    for (int k = 0; k < (sizeof(T) == 4 ? 3 : 1); k++)
      *reinterpret_cast<Vec<TO, 8>*>(dst + k * m.plane + row * m.ld + col) = o[k];
  }
}

// fp16: brings the pieces of each hidden row to the row's largest level, and finds what the sums over tokens start from; a
// group of `lanes` threads a row.
struct LevelArgs {
  __half *h, *dg, *du;                  // dg, du, x, dy null: forward
  const __half *x, *dy;
  int64_t x_stride, dy_stride, M, K, F, N, ld;
  int lanes;                            // a power of 2 up to 32
  const int8_t* levels;
  int *row_h, *row_d, *most;            // most: [MOSTS][blocks]
};
// e with |p[i]| < 2^e for the finite ones of a row; lanes share it
__device__ __forceinline__ int exponent_of_row(const __half* p, int64_t n, int lane, int lanes) {
  uint32_t most = 0;
  const auto one = [&](uint32_t bits) {
    bits &= 0x7fffu;
    if (bits < 0x7c00u) most = max(most, bits);
  };
  int64_t done = 0;
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    done = n / 8 * 8;
    for (int64_t i = lane; i < n / 8; i += lanes) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      one(v.x), one(v.x >> 16), one(v.y), one(v.y >> 16), one(v.z), one(v.z >> 16), one(v.w), one(v.w >> 16);
    }
  }
  for (int64_t i = done + lane; i < n; i += lanes) one(reinterpret_cast<const uint16_t*>(p)[i]);
  return most ? ilogbf(__half2float(__ushort_as_half(uint16_t(most)))) + 1 : kStep * kNoLevel;
}
template <bool BACK> __global__ void __launch_bounds__(256) level_kernel(const LevelArgs p) {
  begin_after_previous();
  __shared__ int meet[MOSTS][8];
  int most[MOSTS] = {kStep * kNoLevel, kStep * kNoLevel};
  const int lane = threadIdx.x % p.lanes, groups = 256 / p.lanes;
  const int64_t pieces = (p.F + 15) / 16;  // pairs of pieces of a row
  const auto across = [&](int k) {  // the largest of the row's lanes
    for (int o = p.lanes / 2; o > 0; o /= 2) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
    return k;
  };
  // a warp's lanes take the same number of turns
  for (int64_t r0 = int64_t(blockIdx.x) * groups; r0 < p.M; r0 += int64_t(gridDim.x) * groups) {
    const int64_t row = r0 + threadIdx.x / p.lanes;
    const bool here = row < p.M;
    const auto levels = [&](int64_t i) {  // of pair i, a byte each
      return BACK ? reinterpret_cast<const uint32_t*>(p.levels)[row * pieces + i]
                  : reinterpret_cast<const uint16_t*>(p.levels)[row * pieces + i];
    };
    const auto level = [](uint32_t w, int byte) { return int(int8_t(w >> 8 * byte)); };
    int kh = kNoLevel, kd = kNoLevel;
    for (int64_t i = lane; here && i < pieces; i += p.lanes) {
      const uint32_t w = levels(i);
      kh = max(kh, max(level(w, 0), level(w, 1)));
      if (BACK) kd = max(kd, max(level(w, 2), level(w, 3)));
    }
    kh = across(kh), kd = BACK ? across(kd) : kd;
    for (int64_t i = lane; here && i < pieces; i += p.lanes) {
      const uint32_t w = levels(i);
      constexpr int PIECES = BACK ? 6 : 2;  // two of h, of dg and of du
      typedef Vec<__half, 8> V;
      V v[PIECES];
      V* at[PIECES];
      int steps[PIECES];
#pragma unroll
      for (int j = 0; j < PIECES; j++) {  // all loads first
        const int64_t from = row * p.ld + i * 16 + j % 2 * 8;
        const int k = level(w, j < 2 ? j : 2 + j % 2);
        at[j] = reinterpret_cast<V*>((j < 2 ? p.h : j < 4 ? p.dg : p.du) + from);
        steps[j] = k == kNoLevel || !LNCC_IN(from, 8, p.M * p.ld) ? 0 : k - (j < 2 ? kh : kd);
        if (steps[j]) v[j] = *at[j];
      }
#pragma unroll
      for (int j = 0; j < PIECES; j++) {
        if (!steps[j]) continue;
        const float power = power_of_2(kStep * steps[j]);
#pragma unroll
        for (int c = 0; c < 8; c++) v[j].e[c] = __float2half_rn(__half2float(v[j].e[c]) * power);
        *at[j] = v[j];
      }
    }
    int ey = 0, ex = 0;
    if (BACK) {
      ex = across(here ? exponent_of_row(p.x + row * p.x_stride, p.K, lane, p.lanes) : 0);
      ey = across(here ? exponent_of_row(p.dy + row * p.dy_stride, p.N, lane, p.lanes) : 0);
    }
    if (!here || lane != 0 || !LNCC_IN(row, 1, p.M)) continue;
    p.row_h[row] = kh;
    if (!BACK) continue;
    p.row_d[row] = kd;
    if (kh != kNoLevel) most[MOST_DY_H] = max(most[MOST_DY_H], ey + kStep * kh);
    if (kd != kNoLevel) most[MOST_X_D] = max(most[MOST_X_D], ex + kStep * kd);
  }
  if (!BACK) return;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < MOSTS; i++) {
    const int e = __reduce_max_sync(0xffffffffu, most[i]);
    if (threadIdx.x % 32 == 0) meet[i][threadIdx.x / 32] = e;
  }
  __syncthreads();
  if (threadIdx.x >= MOSTS) return;
  int e = meet[threadIdx.x][0];
  for (int i = 1; i < 8; i++) e = max(e, meet[threadIdx.x][i]);
  if (LNCC_IN(threadIdx.x * gridDim.x + blockIdx.x, 1, MOSTS * gridDim.x)) p.most[threadIdx.x * gridDim.x + blockIdx.x] = e;
}
// x and dy for the weights' gradients, in aligned rows: a row times the power of 2 that its dg and du, or its h, lack.
struct Rescale {
  const __half *x, *dy;  // null: not wanted
  int64_t x_stride, dy_stride, M, K, N, ld_x, ld_dy;
  __half *to_x, *to_dy;
  const int *row_h, *row_d, *most;
  int level_blocks;
};
__global__ void __launch_bounds__(256) rescale_kernel(const Rescale p) {
  begin_after_previous();
#pragma unroll
  for (int which = 0; which < 2; which++) {
    const __half* src = which ? p.dy : p.x;
    if (src == nullptr) continue;
    const int most = most_of(p.most, p.level_blocks, which ? MOST_DY_H : MOST_X_D);
    const int* levels = which ? p.row_h : p.row_d;
    __half* dst = which ? p.to_dy : p.to_x;
    const int64_t stride = which ? p.dy_stride : p.x_stride, cols = which ? p.N : p.K, ld = which ? p.ld_dy : p.ld_x;
    const bool whole = reinterpret_cast<uintptr_t>(src) % 16 == 0 && stride % 8 == 0;
    const uint32_t per_row = uint32_t(ld / 8);
    for (int64_t q = int64_t(blockIdx.x) * 256 + threadIdx.x; q < p.M * per_row; q += int64_t(gridDim.x) * 256) {
      const int64_t row = q / per_row, col = (q - row * per_row) * 8;
      const int k = levels[row], e = 15 - most + kStep * k;
      const float power = k == kNoLevel || e < -126 ? 0.f : power_of_2(e);
      const __half* from = src + row * stride + col;
      Vec<__half, 8> v;
      if (whole && col + 8 <= cols) {
        v = *reinterpret_cast<const Vec<__half, 8>*>(from);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v.e[i] = col + i < cols ? from[i] : __half(0.f);
      }
#pragma unroll
      for (int i = 0; i < 8; i++) v.e[i] = __float2half_rn(__half2float(v.e[i]) * power);
      if (LNCC_IN(row * ld + col, 8, p.M * ld)) *reinterpret_cast<Vec<__half, 8>*>(dst + row * ld + col) = v;
    }
  }
}

// Euclidean norms of the rows of x and then of Wg, a warp a row: 0 for a row of zeros alone, NaN for one that holds a NaN. Where
// the squares leave the range of fp32 the row is taken relative to its largest element.
__global__ void __launch_bounds__(256) norms_kernel(const float* __restrict__ x, int64_t x_stride, const float* __restrict__ w,
                                                    float* norms, int64_t M, int64_t F, int64_t K) {
  begin_after_previous();
  const int64_t row = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
  if (row >= M + F) return;
  const float* p = row < M ? x + row * x_stride : w + (row - M) * K;
  const int lane = threadIdx.x % 32;
  const auto squares = [&](float scale) {  // the same number in every lane
    float s = 0.f;
    for (int64_t k = lane; k < K; k += 32) s = fmaf(p[k] * scale, p[k] * scale, s);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  float s = squares(1.f), norm = sqrtf(s);
  if (s < 1e-30f || s > 1e30f) {
    float most = 0.f;
    for (int64_t k = lane; k < K; k += 32) most = fmaxf(most, fabsf(p[k]));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int e = most > 0.f && most <= 3.4028235e38f ? max(-126, min(126, -ilogbf(most))) : 0;
    norm = ldexpf(sqrtf(squares(ldexpf(1.f, e))), -e);
  }
  if (lane == 0 && LNCC_IN(row, 1, M + F)) norms[row] = norm;
}
struct NearZero {  // what a gate of ReLU is formed again from
  const float *x, *w, *norms;
  int64_t x_stride, M, F, K, ld;
};
// A gate of ReLU by fp32 multiply-adds in the order of k, by a whole warp: it loads 128 of k side by side, and every lane
// adds them up.
__device__ __noinline__ float gate_in_order(const NearZero& z, int64_t row, int64_t col, float2* stage) {
  const float *x = z.x + row * z.x_stride, *w = z.w + col * z.K;
  const int lane = threadIdx.x % 32;
  float s = 0.f;
  for (int64_t k0 = 0; k0 < z.K; k0 += 128) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t k = k0 + i * 32 + lane;
      stage[i * 32 + lane] = k < z.K ? make_float2(x[k], w[k]) : make_float2(0.f, 0.f);  // adding 0 * 0 changes nothing
    }
    __syncwarp();
#pragma unroll 16
    for (int i = 0; i < 128; i++) s = fmaf(stage[i].x, stage[i].y, s);
  }
  return s;
}

// fp32: dg, du and h, taken apart, from g, u and dh (rows ld apart, like the results). Eight neighbours a thread.
// ReLU's derivative jumps at g = 0, where the last bits of g decide and one element that falls the other way is off by all of
// its gradient. The plain fp32 sum in the order of k is within K 2^-24 |x| |w| of the exact one, and the sum of the tensor
// cores within (64 + K/256) 2^-24 |x| |w|: 16 cut additions in each accumulator, the parts left out, one rounding for each
// 256 of K. Where g is closer to 0 than both together, it is formed again as the plain sum (about one gate in 2700 of dense
// normal rows at K = 389; forming all of them so took 100 us of 413 at 4093 x 389 x 1037). Rows of zeros (padded tokens) and of
// NaN are left out: every order of summation gives 0 and NaN there (half the tokens of 4096 x 1024 x 2048 zero: 21 ms with them).
template <int ACT>
__global__ void __launch_bounds__(256) parts_kernel(const float* __restrict__ g, const float* __restrict__ u,
                                                    const float* __restrict__ dh, __nv_bfloat16* dg, __nv_bfloat16* du,
                                                    __nv_bfloat16* h, int64_t n, int64_t plane, const NearZero z) {
  begin_after_previous();
  __shared__ float2 stages[ACT == LNCC_ACT_RELU ? 8 : 1][128];
  const int lane = threadIdx.x % 32;
  // a warp's lanes take the same number of turns
  for (int64_t i0 = (int64_t(blockIdx.x) * 256 + threadIdx.x - lane) * 8; i0 < n; i0 += int64_t(gridDim.x) * 256 * 8) {
    const int64_t i = i0 + lane * 8;
    const bool here = i < n;
    float vg[8], vu[8], vd[8], o[3][8];
    if (here) {
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        load_vec<float, 4>(g + i + k, reinterpret_cast<float(&)[4]>(vg[k]));
        load_vec<float, 4>(u + i + k, reinterpret_cast<float(&)[4]>(vu[k]));
        load_vec<float, 4>(dh + i + k, reinterpret_cast<float(&)[4]>(vd[k]));
      }
    }
    if (ACT == LNCC_ACT_RELU) {
      const int64_t row = i / z.ld, col = i - row * z.ld;
      const float norm = here ? z.norms[row] : 0.f, near = norm * (float(z.K + 64 + z.K / 256) * 5.9604645e-8f);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float norm_w = here && col + k < z.F ? z.norms[z.M + col + k] : 0.f, bound = near * norm_w;
        const bool again = norm != 0.f && norm_w != 0.f && bound == bound && !(fabsf(vg[k]) > bound);
        for (unsigned rest = __ballot_sync(0xffffffffu, again); rest; rest &= rest - 1) {
          const int who = __ffs(rest) - 1;
          const float v = gate_in_order(z, __shfl_sync(0xffffffffu, row, who), __shfl_sync(0xffffffffu, col, who) + k, stages[threadIdx.x / 32]);
          if (lane == who) vg[k] = v;
        }
      }
    }
    if (!here) continue;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      float a, da;
      activate<ACT, false>(vg[k], a, da);
      o[0][k] = vd[k] * vu[k] * da;
      o[1][k] = vd[k] * a;
      o[2][k] = a * vu[k];
    }
#pragma unroll
    for (int r = 0; r < 3; r++) {
      Vec<__nv_bfloat16, 8> part[3];
#pragma unroll
      for (int k = 0; k < 8; k++) take_apart(o[r][k], part[0].e[k], part[1].e[k], part[2].e[k]);
      __nv_bfloat16* to = (r == 0 ? dg : r == 1 ? du : h) + i;
#pragma unroll
      for (int k = 0; k < 3; k++)
        if (LNCC_IN(i, 8, n)) *reinterpret_cast<Vec<__nv_bfloat16, 8>*>(to + k * plane) = part[k];
    }
  }
}

// ---- a few tokens ----------------------------------------------------------------------------------------------------
// Up to four tokens need each weight once and little else: a warp reads rows of the weights, 16 bytes a lane, and multiplies
// them with the tokens, which wait in shared memory in fp32 (of each eight the first four in one half of the row and the last
// four in the other, so that lanes read 16 bytes side by side). h stays fp32 between the two kernels. Measured for one token,
// 1024 x 2816 bf16 (17 MB of weights, 2.7 us at the copy rate): the tensor kernels' pair tiles took 14 + 10 + 3 us. In calls one
// after the other, the weights then in L2: 10 us for one token, 12 for two, 18.5 for four; the pair tiles 20.5 to 22.5 for 5 to 32
// tokens. fp32: 9, 12 and 16 us, and 64 to 68 from five tokens on.
constexpr int kFewTokens = 4, kFewBytes = 96 * 1024;  // of fp32 tokens in shared memory, K or F wide
constexpr int kRowWarps = 4;                         // warps that share a row of Wd

template <typename T, int V> __device__ __forceinline__ void to_floats(const Vec<T, V>& v, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = to_f(v.e[i]);
}
// where element k of a token lies in its row of `width`
template <int V> __device__ __forceinline__ int token_place(int k, int width) {
  return V == 8 ? k / 8 * 4 + k % 4 + (k & 4 ? width / 2 : 0) : k;
}
// acc[m] += sum over this lane's V elements of w[at] x[m][at]
template <int V, int MT>
__device__ __forceinline__ void multiply(const float (&w)[V], const float* x, int width, int at, float (&acc)[MT]) {
  constexpr int PIECE = V == 8 ? 4 : V;
#pragma unroll
  for (int m = 0; m < MT; m++) {
#pragma unroll
    for (int j = 0; j < V; j += PIECE) {
      const Vec<float, PIECE> t = *reinterpret_cast<const Vec<float, PIECE>*>(x + m * width + token_place<V>(at + j, width));
#pragma unroll
      for (int i = 0; i < PIECE; i++) acc[m] = fmaf(w[j + i], t.e[i], acc[m]);
    }
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// h[m][f], one f a warp at a time. V: weights of a lane's load.
template <typename T, int V, int MT, int ACT>
__global__ void __launch_bounds__(256) few_up_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ wg,
                                                     const T* __restrict__ wu, float* __restrict__ h, int64_t M, int64_t K,
                                                     int64_t F, unsigned* abort_word) {
  extern __shared__ __align__(128) float tokens[];  // [MT][width], zeros past M and K
  asm volatile("griddepcontrol.launch_dependents;");
  if (blockIdx.x == 0 && threadIdx.x == 0) *abort_word = 0u;  // these kernels wait for nothing
  const int width = int((K + 32 * V - 1) / (32 * V) * (32 * V));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int HELD = 4, STEP = 32 * V;  // loads of each matrix under way at once; the first ones before the tokens are here
  typedef Vec<T, V> W;
  W held_g[HELD], held_u[HELD];
  const auto load = [&](int64_t f, int from) {
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      if (f < F && from + i * STEP < K) {  // K is a multiple of V
        held_g[i] = *reinterpret_cast<const W*>(wg + f * K + from + i * STEP);
        held_u[i] = *reinterpret_cast<const W*>(wu + f * K + from + i * STEP);
      }
    }
  };
  const int64_t first_f = int64_t(blockIdx.x) * 8 + warp;
  const int first = lane * V;
  load(first_f, first);
  for (int m = 0; m < MT; m++)
    for (int k = threadIdx.x; k < width; k += 256)
      tokens[m * width + token_place<V>(k, width)] = m < M && k < K ? to_f(x[m * x_stride + k]) : 0.f;
  __syncthreads();
  for (int64_t f = first_f; f < F; f += int64_t(gridDim.x) * 8) {
    float ag[MT] = {}, au[MT] = {};
    for (int from = first; from < K; from += HELD * STEP) {
      if (from != first || f != first_f) load(f, from);
#pragma unroll
      for (int i = 0; i < HELD; i++) {
        if (from + i * STEP < K) {
          float g[V], u[V];
          to_floats(held_g[i], g);
          to_floats(held_u[i], u);
          multiply<V, MT>(g, tokens, width, from + i * STEP, ag);
          multiply<V, MT>(u, tokens, width, from + i * STEP, au);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const float g = warp_sum(ag[m]), u = warp_sum(au[m]);
      float a, da;
      activate<ACT, sizeof(T) == 2>(g, a, da);
      if (lane == 0 && m < M && LNCC_IN(m * F + f, 1, M * F)) h[m * F + f] = a * u;
    }
  }
}

// y[m][n]: kRowWarps warps share a row of Wd, whose first loads are under way before h is waited for.
template <typename T, int V, int MT>
__global__ void __launch_bounds__(256) few_down_kernel(const float* __restrict__ h, const T* __restrict__ wd,
                                                       T* __restrict__ y, int64_t M, int64_t F, int64_t N) {
  extern __shared__ __align__(128) float tokens[];  // [MT][width], zeros past M and F
  __shared__ float meet[8][MT];
  constexpr int ROWS = 8 / kRowWarps, STEP = 32 * V * kRowWarps, HELD = 4;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, mine = warp % kRowWarps;
  const int width = int((F + STEP - 1) / STEP * STEP), first = (mine * 32 + lane) * V;
  typedef Vec<T, V> W;
  W held[HELD];
  const auto load = [&](int64_t n, int from) {
#pragma unroll
    for (int i = 0; i < HELD; i++)
      if (n < N && from + i * STEP < F) held[i] = *reinterpret_cast<const W*>(wd + n * F + from + i * STEP);
  };
  int64_t n = int64_t(blockIdx.x) * ROWS + warp / kRowWarps;
  load(n, first);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int m = 0; m < MT; m++)
    for (int f = threadIdx.x; f < width; f += 256)
      tokens[m * width + token_place<V>(f, width)] = m < M && f < F ? h[m * F + f] : 0.f;
  __syncthreads();
  for (int64_t n0 = int64_t(blockIdx.x) * ROWS; n0 < N; n0 += int64_t(gridDim.x) * ROWS) {
    float acc[MT] = {};
    for (int from = first; from < F; from += HELD * STEP) {
      if (from != first || n0 != int64_t(blockIdx.x) * ROWS) load(n, from);
#pragma unroll
      for (int i = 0; i < HELD; i++) {
        if (n < N && from + i * STEP < F) {
          float w[V];
          to_floats(held[i], w);
          multiply<V, MT>(w, tokens, width, from + i * STEP, acc);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const float s = warp_sum(acc[m]);
      if (lane == 0) meet[warp][m] = s;
    }
    __syncthreads();
    if (mine == 0 && lane < M && n < N && LNCC_IN(lane * N + n, 1, M * N)) {
      float s = 0.f;
      for (int i = 0; i < kRowWarps; i++) s += meet[warp + i][lane];
      y[lane * N + n] = from_f<T>(s);
    }
    __syncthreads();
    n += int64_t(gridDim.x) * ROWS;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
struct Args {
  const void *x, *wg, *wu, *wd, *dy;
  int64_t x_stride, dy_stride, M, K, F, N;
  int act, dtype;
  void *y, *dx, *dwg, *dwu, *dwd;
};

constexpr size_t kHeader = 256;  // the abort word, as in the loss's workspace
inline size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
inline int64_t lead(int64_t cols) { return (cols + 15) / 16 * 16; }  // rows of hidden and packed matrices: 32-byte starts

// How a product is cut into tiles and its inner axis into splits: the cheapest by a model of the time in clocks. A block of
// 64 of a tile of 256 columns takes 590 and one of 128 columns 515 (measured; the tensor cores then wait for A's share of
// shared memory, not for products), a tile 1500 around them; partial sums are written and read at 2200 bytes a clock, and
// their join costs a launch (9000 clocks with what the host pays for it). Of equal ones the fewest splits.
struct Cut {
  int bn, m_tiles, n_tiles, splits, per_split;
};
static Cut cut_for(int kind, int dtype, int64_t rows, int64_t cols, int whichs, int64_t blocks) {
  const int pairs = sm_count() / 2, parts = dtype == LNCC_F32 ? 6 : 1;
  Cut best = {};
  double least = 0;
  for (int bn = 256; bn >= 128; bn -= 128) {
    const int width = gated(kind) ? bn / 2 : bn;
    const int64_t m_tiles = ceil_div(rows, 256), n_tiles = ceil_div(cols, width), tiles = m_tiles * n_tiles * whichs;
    for (const int want : {1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 12, 14, 16, 18, 20, 24, 28, 32, 37, 48, 64}) {
      if (want > 1 && (gated(kind) || kind == DH || blocks < 4 * want)) break;
      const int64_t per = ceil_div(blocks, want), splits = ceil_div(blocks, per);
      double t = double(ceil_div(tiles * splits, pairs)) * (double(per) * parts * (bn == 256 ? 590 : 515) + 1500);
      // HIDDEN on 256 columns: g and u of the next tile wait for the epilogue, and only dh, half of the blocks, runs meanwhile.
      // On 128 columns everything overlaps, but a block costs more. Measured, clocks a tile: 10900 and 5000 at 2 + 2 blocks
      // (107520 x 96 x 256: 69 us against 61), 11800 and 7000 at 4 + 4 (68 against 74), 15700 and 11750 at 8 + 8.
      if (kind == HIDDEN) {
        const double half = double(per) / 2, wide = 9700 + 590 * half;
        t = double(ceil_div(tiles, pairs)) * (bn == 128 ? 2600 + 1200 * half : wide > 1690 * half ? wide : 1690 * half);
      }
      if (splits > 1) t += 9000 + 8.0 * double(splits) * whichs * double(rows) * double(cols) / 2200;
      if (best.bn == 0 || t < 0.98 * least) {
        best = {bn, int(m_tiles), int(n_tiles), int(splits), int(per)};
        least = t;
      }
    }
  }
  return best;
}

// Scratch of a call, laid out in one place for its size and its use.
struct Plan {
  int planes;
  size_t x, wg, wu, wd, dy, h, dg, du, gate, up, dh, norms, levels, row_h, row_d, most, scaled_x, scaled_dy, partial, total;
  int64_t ldf;
};
static size_t partial_bytes(int kind, int dtype, int64_t rows, int64_t cols, int whichs, int64_t blocks) {
  const Cut c = cut_for(kind, dtype, rows, cols, whichs, blocks);
  return c.splits > 1 ? size_t(c.splits) * whichs * rows * ((cols + 3) / 4 * 4) * 4 : 0;
}
static int64_t k_steps(int64_t k) { return ceil_div(k, 64); }
static int level_blocks() { return 8 * sm_count(); }
static bool few(const Args& a);
static Plan plan_for(const Args& a, bool backward) {
  Plan p = {};
  if (!backward && few(a)) {
    p.total = kHeader + round_up(size_t(a.M) * a.F * 4);
    return p;
  }
  p.planes = a.dtype == LNCC_F32 ? 3 : 1;
  p.ldf = lead(a.F);
  size_t at = kHeader;
  const auto take = [&](int64_t rows, int64_t ld) {
    const size_t here = at;
    at += round_up(size_t(p.planes) * rows * ld * 2);
    return here;
  };
  p.x = take(a.M, lead(a.K));
  p.wg = take(a.F, lead(a.K));
  p.wu = take(a.F, lead(a.K));
  p.wd = take(a.N, p.ldf);
  p.h = take(a.M, p.ldf);
  if (a.dtype == LNCC_F16) {
    p.levels = at, at += round_up(size_t(a.M) * ceil_div(a.F, 16) * (backward ? 4 : 2));
    p.row_h = at, at += round_up(size_t(a.M) * 4);
    if (backward) {
      p.row_d = at, at += round_up(size_t(a.M) * 4);
      p.most = at, at += round_up(size_t(MOSTS) * level_blocks() * 4);
      p.scaled_x = take(a.M, lead(a.K));
      p.scaled_dy = take(a.M, lead(a.N));
    }
  }
  size_t most = 0;
  const auto partial = [&](size_t n) { most = n > most ? n : most; };
  if (backward) {
    p.dy = take(a.M, lead(a.N));
    p.dg = take(a.M, p.ldf);
    p.du = take(a.M, p.ldf);
    if (a.dtype == LNCC_F32) {
      p.gate = at, at += round_up(size_t(a.M) * p.ldf * 4);
      p.up = at, at += round_up(size_t(a.M) * p.ldf * 4);
      p.dh = at, at += round_up(size_t(a.M) * p.ldf * 4);
      p.norms = at, at += round_up(size_t(a.M + a.F) * 4);
    }
    partial(partial_bytes(DX, a.dtype, a.M, a.K, 1, 2 * k_steps(a.F)));
    partial(partial_bytes(DW_UP, a.dtype, a.F, a.K, 2, k_steps(a.M)));
    partial(partial_bytes(DW_UP, a.dtype, a.F, a.K, 1, k_steps(a.M)));
    partial(partial_bytes(DW_DOWN, a.dtype, a.N, a.F, 1, k_steps(a.M)));
  } else {
    partial(partial_bytes(DOWN, a.dtype, a.M, a.N, 1, k_steps(a.F)));
  }
  p.partial = at;
  p.total = at + round_up(most);
  return p;
}

// Unnamed, so that the marks of what this library has asked the device for are its own: the checked build, loaded beside it, has
// kernels of its own under the same names.
namespace {
struct Call {
  const Args& a;
  Plan plan;
  char* scratch;
  cudaStream_t stream;
  int status;
  bool first = true;      // the next product kernel is the call's first
  bool launched = false;  // a kernel of this call is in the stream
  Packs packs = {};

  // every kernel of a call but its first may be launched while the one before it ends (begin_after_previous)
  template <typename K, typename... A> void run(K kernel, dim3 grid, int threads, int smem, const A&... args) {
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = dim3(unsigned(threads)), cfg.dynamicSmemBytes = size_t(smem), cfg.stream = stream;
    cfg.attrs = &early, cfg.numAttrs = launched ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) status = LNCC_ERR_LAUNCH;
    launched = true;
  }

  // src as TMA reads it: in place, or packed to `to` by pack()
  Matrix operand(const void* src, int64_t rows, int64_t cols, int64_t stride, size_t to) {
    Matrix m = {const_cast<void*>(src), rows, cols, stride, 0, 1, a.dtype != LNCC_F16};
    if (a.dtype != LNCC_F32 && aligned(src, 16) && (stride % 8 == 0 || rows == 1)) {
      if (rows == 1) m.ld = lead(cols);
      return m;
    }
    m.p = scratch + to;
    m.ld = lead(cols);
    m.plane = rows * m.ld;
    m.planes = plan.planes;
    const int64_t blocks = ceil_div(rows * (m.ld / 8), 256), most = int64_t(sm_count()) * 8;
    packs.job[packs.jobs++] = {src, m.p, stride, rows, cols, m.ld, m.plane, packs.blocks};
    packs.blocks += int(blocks < most ? blocks : most);
    return m;
  }
  void pack() {
    if (packs.jobs == 0) return;
    const dim3 grid = dim3(unsigned(packs.blocks));
    if (a.dtype == LNCC_F32) run(pack_kernel<float, __nv_bfloat16>, grid, 256, 0, packs);
    else if (a.dtype == LNCC_BF16) run(pack_kernel<__nv_bfloat16, __nv_bfloat16>, grid, 256, 0, packs);
    else run(pack_kernel<__half, __half>, grid, 256, 0, packs);
  }
  // fp16: after the hidden matrices, their rows' levels; the copies of x and dy that the sums over tokens take
  void level() {
    int lanes = 4;
    while (lanes < 32 && lanes * 64 < a.F) lanes *= 2;  // four pairs of pieces a lane, or more
    const LevelArgs r = {halves(plan.h), halves(plan.dg), halves(plan.du), static_cast<const __half*>(a.x), static_cast<const __half*>(a.dy),
                         a.x_stride, a.dy_stride, a.M, a.K, a.F, a.N, plan.ldf, lanes,
                         reinterpret_cast<const int8_t*>(scratch + plan.levels), ints(plan.row_h), ints(plan.row_d), ints(plan.most)};
    run(a.dy ? level_kernel<true> : level_kernel<false>, dim3(unsigned(level_blocks())), 256, 0, r);
  }
  void rescale(Matrix& x, Matrix& dy) {
    const bool want_x = a.dwg || a.dwu, want_dy = a.dwd != nullptr;
    if (!want_x && !want_dy) return;
    x = {scratch + plan.scaled_x, a.M, a.K, lead(a.K), 0, 1, false};
    dy = {scratch + plan.scaled_dy, a.M, a.N, lead(a.N), 0, 1, false};
    const Rescale r = {want_x ? static_cast<const __half*>(a.x) : nullptr, want_dy ? static_cast<const __half*>(a.dy) : nullptr,
                       a.x_stride, a.dy_stride, a.M, a.K, a.N, x.ld, dy.ld, halves(plan.scaled_x), halves(plan.scaled_dy),
                       ints(plan.row_h), ints(plan.row_d), ints(plan.most), level_blocks()};
    const int64_t blocks = ceil_div(a.M * (x.ld > dy.ld ? x.ld : dy.ld) / 8, 256), most = int64_t(sm_count()) * 8;
    run(rescale_kernel, dim3(unsigned(blocks < most ? blocks : most)), 256, 0, r);
  }
  int* ints(size_t at) const { return reinterpret_cast<int*>(scratch + at); }
  __half* halves(size_t at) const { return reinterpret_cast<__half*>(scratch + at); }

  Matrix hidden(size_t at) const {
    return {scratch + at, a.M, a.F, plan.ldf, a.M * plan.ldf, plan.planes, a.dtype != LNCC_F16};
  }

  template <int KIND, int BN, int ACT, typename T> void launch(Gemm& g) {
    const int smem = smem_bytes(BN), pairs = sm_count() / 2;
    static Asked asked;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || !asked.has(dev)) {
      if (cudaFuncSetAttribute(product_kernel<KIND, BN, ACT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
          cudaSuccess) {
        cudaGetLastError();
        status = LNCC_ERR_SMEM;
        return;
      }
      asked.mark(dev);
    }
    const int64_t tiles = int64_t(g.m_tiles) * g.n_tiles * g.whichs * g.splits;
    run(product_kernel<KIND, BN, ACT, T>, dim3(unsigned(2 * (tiles < pairs ? tiles : pairs))), kThreads, smem, g);
  }
  template <int KIND, int BN, typename T> void launch_act(Gemm& g) {
    if constexpr (KIND == UP || KIND == HIDDEN) {
      if (a.act == LNCC_ACT_SILU) launch<KIND, BN, LNCC_ACT_SILU, T>(g);
      else if (a.act == LNCC_ACT_GELU) launch<KIND, BN, LNCC_ACT_GELU, T>(g);
      else launch<KIND, BN, LNCC_ACT_RELU, T>(g);
    } else {
      launch<KIND, BN, 0, T>(g);
    }
  }
  template <int KIND, typename T> void launch_type(Gemm& g, int bn) {
    if (bn == 256) launch_act<KIND, 256, T>(g);
    else launch_act<KIND, 128, T>(g);
  }

  template <typename T> void join(const Gemm& g) {
    const int64_t quads = g.whichs * g.rows * ceil_div(g.cols, 4);
    T *out0 = static_cast<T*>(g.out0), *out1 = static_cast<T*>(g.out1);
    if (g.splits < kManySplits)
      run(join_kernel<T, 1>, dim3(unsigned(ceil_div(quads, 256))), 256, 0, static_cast<const float*>(g.partial), g.splits,
          g.whichs, g.rows, g.cols, out0, out1);
    else
      run(join_kernel<T, 8>, dim3(unsigned(ceil_div(quads, 32))), 256, 0, static_cast<const float*>(g.partial), g.splits,
          g.whichs, g.rows, g.cols, out0, out1);
  }

  // One product: A (a0, a1) and B (b0, b1, b2) as the kind takes them, results out (rows x cols, ld apart).
  template <int KIND>
  void product(const Matrix& a0, const Matrix& a1, const Matrix& b0, const Matrix& b1, const Matrix& b2, int64_t rows,
               int64_t cols, int whichs, int64_t inner, int64_t inner2, void* out0, void* out1, void* out2, int64_t ld,
               int64_t plane) {
    if (status != LNCC_OK) return;
    Gemm g = {};
    g.k_steps = int(k_steps(inner));
    g.k_steps2 = int(k_steps(inner2));
    g.blocks = KIND == DX ? 2 * g.k_steps : KIND == HIDDEN ? g.k_steps + g.k_steps2 : g.k_steps;
    const Cut c = cut_for(KIND, a.dtype, rows, cols, whichs, g.blocks);
    g.m_tiles = c.m_tiles, g.n_tiles = c.n_tiles, g.splits = c.splits, g.whichs = whichs, g.per_split = c.per_split;
    const int a_box = a_mn(KIND) ? 64 : 128, b_box = b_mn(KIND) ? 64 : c.bn / 2;
    constexpr bool second_a = KIND == HIDDEN || KIND == DX || KIND == DW_UP, second_b = gated(KIND) || KIND == DX;
    if (!make_map(&g.a0, a0, a_box) || (second_a && !make_map(&g.a1, a1, a_box)) || !make_map(&g.b0, b0, b_box) ||
        (second_b && !make_map(&g.b1, b1, b_box)) || (KIND == HIDDEN && !make_map(&g.b2, b2, 64, c.bn / 4))) {
      status = LNCC_ERR_CUDA;
      return;
    }
    g.rows = rows, g.cols = cols, g.bf16 = a0.bf16;
    g.out0 = out0, g.out1 = out1, g.out2 = out2, g.ld = ld, g.plane = plane;
    const int es = KIND == UP || KIND == HIDDEN ? 2 : elem_size(a.dtype);
    g.align = es;
    for (int al = 16; al <= 32; al *= 2)
      if (aligned(out0, al) && aligned(out1, al) && aligned(out2, al) && ld * es % al == 0) g.align = al;
    g.partial = reinterpret_cast<float*>(scratch + plan.partial);
    if (a.dtype == LNCC_F16) {
      g.levels = reinterpret_cast<int8_t*>(scratch + plan.levels);
      g.row_h = ints(plan.row_h), g.row_d = ints(plan.row_d), g.most = ints(plan.most), g.level_blocks = level_blocks();
    }
    g.abort_word = reinterpret_cast<unsigned*>(scratch);
    g.clear_abort = first;
    first = false;
    if constexpr (KIND == GATES || KIND == DH) {
      launch_type<KIND, float>(g, c.bn);
    } else if (a.dtype == LNCC_F32) {
      if constexpr (KIND != HIDDEN) launch_type<KIND, float>(g, c.bn);
    } else if (a.dtype == LNCC_BF16) {
      launch_type<KIND, __nv_bfloat16>(g, c.bn);
    } else {
      launch_type<KIND, __half>(g, c.bn);
    }
    if (g.splits > 1 && status == LNCC_OK) {
      if (a.dtype == LNCC_F32) join<float>(g);
      else if (a.dtype == LNCC_BF16) join<__nv_bfloat16>(g);
      else join<__half>(g);
    }
  }
};

}  // namespace

static int tokens_of(int64_t M) { return M <= 1 ? 1 : M <= 2 ? 2 : 4; }
static bool few(const Args& a) {
  const int64_t widest = (a.K > a.F ? a.K : a.F) + 1024;  // rounded up to a block's step
  return a.M <= kFewTokens && tokens_of(a.M) * widest * 4 <= kFewBytes;
}
template <typename T, int V, int MT> static int few_run(const Args& a, float* h, cudaStream_t st) {
  const auto up = a.act == LNCC_ACT_SILU ? few_up_kernel<T, V, MT, LNCC_ACT_SILU>
                  : a.act == LNCC_ACT_GELU ? few_up_kernel<T, V, MT, LNCC_ACT_GELU> : few_up_kernel<T, V, MT, LNCC_ACT_RELU>;
  const auto down = few_down_kernel<T, V, MT>;
  const int up_smem = int(MT * ceil_div(a.K, 32 * V) * 32 * V * 4), step = 32 * V * kRowWarps;
  const int down_smem = int(MT * ceil_div(a.F, step) * step * 4);
  constexpr int kFree = 40 * 1024;  // dynamic shared memory that any kernel may have beside its static
  if (up_smem > kFree && cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, up_smem) != cudaSuccess)
    return LNCC_ERR_SMEM;
  if (down_smem > kFree && cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, down_smem) != cudaSuccess)
    return LNCC_ERR_SMEM;
  const int64_t most = int64_t(sm_count()) * 4, up_blocks = ceil_div(a.F, 8), down_blocks = ceil_div(a.N, 8 / kRowWarps);
  up<<<unsigned(up_blocks < most ? up_blocks : most), 256, up_smem, st>>>(
      static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.wg), static_cast<const T*>(a.wu), h, a.M, a.K, a.F,
      reinterpret_cast<unsigned*>(reinterpret_cast<char*>(h) - kHeader));
  cudaLaunchAttribute early = {};  // begins while the first kernel ends
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(down_blocks < most ? down_blocks : most)), cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = down_smem, cfg.stream = st, cfg.attrs = &early, cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, down, static_cast<const float*>(h), static_cast<const T*>(a.wd),
                                           static_cast<T*>(a.y), a.M, a.F, a.N);
  return e == cudaSuccess ? LNCC_OK : LNCC_ERR_LAUNCH;
}
template <typename T, int V> static int few_tokens(const Args& a, float* h, cudaStream_t st) {
  switch (tokens_of(a.M)) {
    case 1: return few_run<T, V, 1>(a, h, st);
    case 2: return few_run<T, V, 2>(a, h, st);
    default: return few_run<T, V, 4>(a, h, st);
  }
}
template <typename T> static int few_forward(const Args& a, void* scratch, cudaStream_t st) {
  constexpr int V = 16 / int(sizeof(T));
  float* h = reinterpret_cast<float*>(static_cast<char*>(scratch) + kHeader);
  if (a.K % V == 0 && a.F % V == 0 && aligned(a.wg, 16) && aligned(a.wu, 16) && aligned(a.wd, 16))
    return few_tokens<T, V>(a, h, st);
  return few_tokens<T, 1>(a, h, st);
}

static int forward(const Args& a, const Plan& plan, void* scratch, cudaStream_t stream) {
  if (few(a)) {
    if (a.dtype == LNCC_F32) return few_forward<float>(a, scratch, stream);
    if (a.dtype == LNCC_BF16) return few_forward<__nv_bfloat16>(a, scratch, stream);
    return few_forward<__half>(a, scratch, stream);
  }
  Call c = {a, plan, static_cast<char*>(scratch), stream, LNCC_OK};
  const Matrix x = c.operand(a.x, a.M, a.K, a.x_stride, c.plan.x), wg = c.operand(a.wg, a.F, a.K, a.K, c.plan.wg),
               wu = c.operand(a.wu, a.F, a.K, a.K, c.plan.wu), wd = c.operand(a.wd, a.N, a.F, a.F, c.plan.wd),
               h = c.hidden(c.plan.h);
  c.pack();
  c.product<UP>(x, x, wg, wu, wg, a.M, a.F, 1, a.K, 0, h.p, nullptr, nullptr, h.ld, h.plane);
  if (a.dtype == LNCC_F16) c.level();
  c.product<DOWN>(h, h, wd, wd, wd, a.M, a.N, 1, a.F, 0, a.y, nullptr, nullptr, a.N, 0);
  return c.status;
}

static int backward(const Args& a, const Plan& plan, void* scratch, cudaStream_t stream) {
  Call c = {a, plan, static_cast<char*>(scratch), stream, LNCC_OK};
  const Matrix x = c.operand(a.x, a.M, a.K, a.x_stride, c.plan.x), dy = c.operand(a.dy, a.M, a.N, a.dy_stride, c.plan.dy),
               wg = c.operand(a.wg, a.F, a.K, a.K, c.plan.wg), wu = c.operand(a.wu, a.F, a.K, a.K, c.plan.wu),
               wd = c.operand(a.wd, a.N, a.F, a.F, c.plan.wd);
  const Matrix h = c.hidden(c.plan.h), dg = c.hidden(c.plan.dg), du = c.hidden(c.plan.du);
  c.pack();
  if (a.dtype == LNCC_F32) {
    float *const gate = reinterpret_cast<float*>(c.scratch + c.plan.gate), *const up = reinterpret_cast<float*>(c.scratch + c.plan.up),
                *const dh = reinterpret_cast<float*>(c.scratch + c.plan.dh);
    const NearZero z = {static_cast<const float*>(a.x), static_cast<const float*>(a.wg),
                        reinterpret_cast<const float*>(c.scratch + c.plan.norms), a.x_stride, a.M, a.F, a.K, h.ld};
    if (a.act == LNCC_ACT_RELU)
      c.run(norms_kernel, dim3(unsigned(ceil_div(a.M + a.F, 8))), 256, 0, z.x, a.x_stride, z.w, const_cast<float*>(z.norms), a.M, a.F, a.K);
    c.product<GATES>(x, x, wg, wu, wg, a.M, a.F, 1, a.K, 0, gate, up, nullptr, h.ld, 0);
    c.product<DH>(dy, dy, wd, wd, wd, a.M, a.F, 1, a.N, 0, dh, nullptr, nullptr, h.ld, 0);
    const auto parts = a.act == LNCC_ACT_SILU ? parts_kernel<LNCC_ACT_SILU>
                       : a.act == LNCC_ACT_GELU ? parts_kernel<LNCC_ACT_GELU> : parts_kernel<LNCC_ACT_RELU>;
    const int64_t n = a.M * h.ld, blocks = ceil_div(n, 2048), most = int64_t(sm_count()) * 8;
    c.run(parts, dim3(unsigned(blocks < most ? blocks : most)), 256, 0, static_cast<const float*>(gate), static_cast<const float*>(up),
          static_cast<const float*>(dh), static_cast<__nv_bfloat16*>(dg.p), static_cast<__nv_bfloat16*>(du.p),
          static_cast<__nv_bfloat16*>(h.p), n, h.plane, z);
  } else {
    c.product<HIDDEN>(x, dy, wg, wu, wd, a.M, a.F, 1, a.K, a.N, dg.p, du.p, h.p, h.ld, h.plane);
  }
  Matrix sum_x = x, sum_dy = dy;  // as the sums over tokens take them
  if (a.dtype == LNCC_F16) {
    c.level();
    c.rescale(sum_x, sum_dy);
  }
  if (a.dx) c.product<DX>(dg, du, wg, wu, wg, a.M, a.K, 1, a.F, 0, a.dx, nullptr, nullptr, a.K, 0);
  if (a.dwg || a.dwu) {
    // one product for both where both are wanted
    const Matrix& first = a.dwg ? dg : du;
    c.product<DW_UP>(first, du, sum_x, sum_x, sum_x, a.F, a.K, a.dwg && a.dwu ? 2 : 1, a.M, 0, a.dwg ? a.dwg : a.dwu, a.dwu, nullptr, a.K, 0);
  }
  if (a.dwd) c.product<DW_DOWN>(sum_dy, sum_dy, h, h, h, a.N, a.F, 1, a.M, 0, a.dwd, nullptr, nullptr, a.F, 0);
  return c.status;
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
  if (ffn::check_sizes(dtype, 0, M, K, F, N) != LNCC_OK || M == 0) return 0;
  ffn::Args a = {};
  a.M = M, a.K = K, a.F = F, a.N = N, a.dtype = dtype, a.act = LNCC_ACT_RELU;  // the activation that needs most
  return ffn::plan_for(a, backward != 0).total;
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
  ffn::Args p = {};
  p.x = x, p.x_stride = x_stride, p.wg = w_gate, p.wu = w_up, p.wd = w_down, p.act = act, p.dtype = dtype, p.y = y;
  p.M = M, p.K = K, p.F = F, p.N = N;
  const ffn::Plan plan = ffn::plan_for(p, false);
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < plan.total) return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  const int run = ffn::forward(p, plan, scratch, stream);
  const int ended = blk::check_end(stream);
  return run != LNCC_OK ? run : ended;
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
  ffn::Args p = {};
  p.x = x, p.x_stride = x_stride, p.dy = dy, p.dy_stride = dy_stride, p.wg = w_gate, p.wu = w_up, p.wd = w_down;
  p.act = act, p.dtype = dtype, p.dx = dx, p.dwg = dw_gate, p.dwu = dw_up, p.dwd = dw_down;
  p.M = M, p.K = K, p.F = F, p.N = N;
  const ffn::Plan plan = ffn::plan_for(p, true);
  if (!scratch || !blk::aligned(scratch, 16) || scratch_bytes < plan.total) return LNCC_ERR_WORKSPACE;
  const int cb = blk::check_begin();
  if (cb != LNCC_OK) return cb;
  const int run = ffn::backward(p, plan, scratch, stream);
  const int ended = blk::check_end(stream);
  return run != LNCC_OK ? run : ended;
}

}  // extern "C"
