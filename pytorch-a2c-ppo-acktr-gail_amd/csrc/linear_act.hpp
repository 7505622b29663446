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
    int act, vec;                       // vec: 16-byte stores of 8 columns are possible everywhere
    float* slabs;                       // split reduction: fp32 partial products [slices][M][N] instead of y
    int kslice;                         // k per slice (a multiple of the K step), K without a split
    int tiles_m, tiles_n;
};

constexpr int KSTEP_BYTES = 128, MAX_SLICES = 32, SUM_BLOCKS = 256;

static inline long up(long v, long a) { return (v + a - 1) / a * a; }
static inline bool rows16(const void* p, long ld, long e) { return ((uintptr_t)p & 15) == 0 && ld * e % 16 == 0; }

// Tile and reduction split of an M x N x K product, by an estimate of its time.  A K step (128 bytes of k) of a 64 x 64 piece is the
// unit.  `rate`: units per microsecond that a CU full of such workgroups gets through; `step`: microseconds a step takes a workgroup
// that has a CU to itself (measured on 16384 x 2048 x 2048 and on 2048 x 2048 x 16384: 256 x 256 tiles 1.65 us a step full, 1.17 us
// alone; 128 x 128 1.0 us for two, 0.61 alone; 128 x 64 0.30 for one of many, 0.5 alone; 64 x 64 0.19, 0.45 alone; fp32 is bound by its
// matrix instructions, 0.47 us a unit, from 64 x 64 tiles on, so larger ones only lose parallelism).  Big tiles read the least, small
// ones fill the chip; a long reduction with few tiles is cut into slices, whose fp32 partial products cost a second pass
// (3 bytes per picosecond and a launch).  The estimates are within 15 % of the times measured at 4096 x 512 x 1568.
struct Tile { int bm, bn; float rate, step; };
struct Plan { int tile, slices; long kslice; };
constexpr Tile TILES[] = {{64, 64, 5.3f, 0.45f}, {128, 64, 6.6f, 0.5f}, {128, 128, 8.0f, 0.62f}, {256, 256, 9.7f, 1.17f}};
constexpr Tile TILES32[] = {{64, 64, 2.1f, 0.75f}, {128, 64, 2.15f, 1.2f}};
static Plan plan_of(long M, long N, long K, int e) {
    const long kt = KSTEP_BYTES / e, steps = (K + kt - 1) / kt;
    Plan best{0, 1, up(K, kt)};
    float least = 0.f;
    for (int t = 0; t < (e == 4 ? 2 : 4); ++t) {
        const Tile& ti = e == 4 ? TILES32[t] : TILES[t];
        const long tiles = (long)cdiv(M, ti.bm) * cdiv(N, ti.bn), units = (long)ti.bm * ti.bn / 4096;
        for (int want = 1; want <= MAX_SLICES && (want == 1 || steps / want >= 4); want += want < 4 ? 1 : want / 2) {
            const long per = (steps + want - 1) / want, slices = steps ? (steps + per - 1) / per : 1;
            const float busy = (float)cdiv(tiles * slices, 256) * units / ti.rate;
            float us = 3.f + per * (busy > ti.step ? busy : ti.step);
            if (slices > 1) us += 3.f + (slices + 1) * 4.f * M * N / 3e6f;
            if (least == 0.f || us < least) {
                least = us;
                best = Plan{t, (int)slices, slices > 1 ? per * kt : up(K, kt)};
            }
        }
    }
    return best;
}

static long slab_bytes(long M, long N, long K, int e) {
    const Plan pl = plan_of(M, N, K, e);
    return pl.slices > 1 ? up(4 * M * N * pl.slices, 256) : 0;
}

// One product with its epilogue; `slabs` holds the slices of a split reduction.  FORWARD: both operands k-contiguous, bias / activation /
// residual; DX: A k-contiguous, B row-contiguous; DW: both row-contiguous.
enum LinKind { LIN_FORWARD, LIN_DX, LIN_DW };
template <class T> int linear_product(LinKind kind, const LinArgs& p, float* slabs, hipStream_t s);

}  // namespace acktr
