// Arguments of linear_act.hip's products and how they are cut into tiles; the tile kernels themselves are compiled one element type
// a translation unit.
#pragma once
#include "half_types.hpp"

namespace acktr {

struct LinArgs {
    const void *a, *b;                  // A: M x K, B: N x K
    long lda, ldb;
    int M, N, K;
    void* y;
    long ldy;
    const void *bias, *res;             // nullable
    void* pre;                          // slopes for the backward pass; nullable
    long ldr, ldp;
    int act;
    float* slabs;                       // split reduction: fp32 partial products [slices][M][N] instead of y
    int kslice;                         // k per slice (a multiple of the K step), K without a split
    int tiles_m, tiles_n;
    // the weight gradient's launch also forms the bias gradient db[M] from `blocks` rows of column sums [blocks][M]; nullable
    const float* sums;
    void* db;
    int blocks;
};

constexpr int KSTEP_BYTES = 128, MAX_SLICES = 32, SUM_BLOCKS = 256, SUM_COLS = 32, SUM_GROUPS = 8;
constexpr long SUM_WIDE = 1 << 18;        // results from which the sum of slices takes 8 columns a thread

static inline long up(long v, long a) { return (v + a - 1) / a * a; }
static inline bool rows16(const void* p, long ld, long e) { return ((uintptr_t)p & 15) == 0 && ld * e % 16 == 0; }

// Tile and reduction split of an M x N x K product, by an estimate of its time.  A K step (128 bytes of k) of a 64 x 64 piece is the
// unit.  `rate`: units per microsecond that a CU full of such workgroups gets through; `step`: microseconds a step takes a workgroup
// that has a CU to itself.  Measured (bf16; 16384 x 2048 x 2048 for the rates, the weight gradients of 2048 x 2048 x 16384 and
// 512 x 1568 x 4096 for the steps): 256 x 256 1352 TFLOP/s, 1.13 us; 128 x 128 1137, 0.61; 128 x 64 886, 0.37; 64 x 64 718, 0.31.
// fp32 is bound by its matrix instructions from 64 x 64 tiles on (143 TFLOP/s; 0.47 us a unit): larger ones only lose parallelism.
// Big tiles read the least, small ones fill the chip; a long reduction with few tiles is cut into slices, whose fp32 partial products
// cost a second pass (3 bytes per picosecond and a launch).
struct Tile { int bm, bn; float rate, step; };
struct Plan { int tile, slices; long kslice; float us; };
constexpr Tile TILES[] = {{64, 64, 5.0f, 0.31f}, {128, 64, 6.6f, 0.37f}, {128, 128, 8.7f, 0.61f}, {256, 256, 10.2f, 1.13f}};
constexpr Tile TILES32[] = {{64, 64, 2.1f, 0.75f}, {128, 64, 2.15f, 1.25f}};
static inline const Tile& tile_of(int t, int e) { return e == 4 ? TILES32[t] : TILES[t]; }
static inline long steps_of(long K, int e) { return (K * e + KSTEP_BYTES - 1) / KSTEP_BYTES; }
static inline float slices_us(int slices, long M, long N) { return slices > 1 ? 3.f + (slices + 1) * 4.f * M * N / 3e6f : 0.f; }
// f(slices, K steps in each) over the splits worth trying: at least 4 steps a slice
template <class F>
static inline void each_split(long steps, F&& f) {
    for (int want = 1; want <= MAX_SLICES && (want == 1 || steps / want >= 4); want += want < 4 ? 1 : want / 2) {
        const long per = (steps + want - 1) / want;
        f(steps ? (int)((steps + per - 1) / per) : 1, per);
    }
}
static Plan plan_of(long M, long N, long K, int e) {
    const long kt = KSTEP_BYTES / e, steps = steps_of(K, e);
    Plan best{0, 1, up(K, kt), 0.f};
    for (int t = 0; t < (e == 4 ? 2 : 4); ++t) {
        const Tile& ti = tile_of(t, e);
        const long tiles = (long)cdiv(M, ti.bm) * cdiv(N, ti.bn), units = (long)ti.bm * ti.bn / 4096;
        each_split(steps, [&](int slices, long per) {
            const float busy = (float)cdiv(tiles * slices, 256) * units / ti.rate;
            const float us = 3.f + per * (busy > ti.step ? busy : ti.step) + slices_us(slices, M, N);
            if (best.us == 0.f || us < best.us) best = Plan{t, slices, slices > 1 ? per * kt : up(K, kt), us};
        });
    }
    return best;
}
// Both gradients of a layer in one launch (tile < 0: better apart): the units of both share the chip, the longer chain of steps bounds
// them from below.  The weight gradient, with the long reduction, takes 64 x 64 tiles; `tile` is the input gradient's, 64 x 64 or
// 128 x 64 (measured, bf16, 4096 rows, 512 x 1568 weights: 29.0 and 26.7 us, apart 36; 512 rows, 512 x 512: 5.6, 6.6, apart 10.6).
struct PairPlan { int tile, slices; long kslice; };
static PairPlan pair_plan_of(const LinArgs& dw, const LinArgs& dx, int e) {
    const long kt = KSTEP_BYTES / e, steps = steps_of(dw.K, e), dx_steps = steps_of(dx.K, e);
    PairPlan best{-1, 1, 0};
    float least = plan_of(dw.M, dw.N, dw.K, e).us + plan_of(dx.M, dx.N, dx.K, e).us;
    if (steps == 0 || dx_steps == 0) return best;
    const Tile& tw = tile_of(0, e);
    const long dw_tiles = (long)cdiv(dw.M, tw.bm) * cdiv(dw.N, tw.bn);
    for (int t = 0; t < 2; ++t) {
        const Tile& tx = tile_of(t, e);
        const long dx_units = (long)cdiv(dx.M, tx.bm) * cdiv(dx.N, tx.bn) * dx_steps * (tx.bm * tx.bn / 4096);
        each_split(steps, [&](int slices, long per) {
            const float busy = ((float)dw_tiles * slices * per / tw.rate + dx_units / tx.rate) / 256.f;
            const float chain = max(per * tw.step, dx_steps * tx.step);
            const float us = 4.f + max(busy, chain) + slices_us(slices, dw.M, dw.N);
            if (us < least) least = us, best = PairPlan{t, slices, slices > 1 ? per * kt : up(dw.K, kt)};
        });
    }
    return best;
}
static long slab_bytes(long M, long N, int slices) { return slices > 1 ? up(4 * M * N * slices, 256) : 0; }

// One product with its epilogue; `slabs` holds the slices of a split reduction.  FORWARD: both operands k-contiguous, bias / activation /
// residual; DX: A k-contiguous, B row-contiguous; DW: both row-contiguous.
enum LinKind { LIN_FORWARD, LIN_DX, LIN_DW };
template <class T> int linear_product(LinKind kind, const LinArgs& p, float* slabs, hipStream_t s);
// DW and DX of one layer, in one launch where that is faster
template <class T> int linear_gradients(LinArgs dw, LinArgs dx, float* slabs, hipStream_t s);
// the bias's gradient alone: M, sums, blocks and db of its arguments
template <class T> int linear_bias(const LinArgs& dw, hipStream_t s);

}  // namespace acktr
