// Matrix-core tile product for bf16 / fp16 / fp32 operands that are read as they lie in memory.
//
//   D(m, n) = sum_k A(m, k) B(n, k)         A: M x K, B: N x K, each with either k or its own row index contiguous
//
// * Tiles go from memory straight into LDS (16 bytes a lane, no registers in between).  A lane's LDS place is fixed by the
//   instruction (base + 16 * lane), so bank conflicts are kept away by choosing which 16 bytes of memory a lane FETCHES:
//     k contiguous   : the tile is [rows][128 bytes]; chunk c of row r lies at c ^ ((r >> 1) & 7).  A fragment read (16 rows, one
//                      chunk each) then covers all 64 banks once.
//     rows contiguous: the tile is [k][rows]; 32-byte unit u of line k lies at u ^ ((k & 3) | (k >> 1 & 4)) (as many of these
//                      bits as the line has units).  16-bit fragments are
//                      read with the transposing ds_read_b64_tr_b16 (a group of 16 lanes reads 4 lines x 16 rows and gets 4
//                      consecutive k of its row each); fp32 fragments with one ds_read_b32 per k.
// * A K step is 128 bytes of k (64 16-bit or 32 fp32 values), cut into two halves that alternate in registers: while the
//   matrix cores work on one half, the other half is read from LDS.  STAGES K steps have a place in LDS: memory loads are in
//   flight for STAGES - 1 K steps (a large tile computes long enough on one step to cover the latency with 2 stages, the small
//   ones take 3; 5 to 8 were no faster).  One barrier per K step, which waits for the oldest loads only.
// * The products are formed transposed (B's rows on the matrix instruction's row side), so that a lane ends up with four
//   consecutive n of one m.  fp32 uses v_mfma_f32_16x16x4 on the same fragments: a lane group's four consecutive k are four
//   instructions, each pairing the same k of A and B.
// * What bounds it (16384 x 2048 x 2048, bf16, one part of the loop at a time): 64 x 64 tiles 183 us, of which the copies into LDS
//   alone take 162 (4.3 GB at 26 TB/s, whether or not the L2 caches hit), products 67, LDS reads 80; 128 x 128 tiles 125: 105, 66, 52;
//   256 x 256 tiles 107: 79, 79, 46.  So small tiles are bound by the copies, and the largest one by how far copies, products and
//   reads overlap.  Two wave groups half a step apart were slower there (127 us): their extra barriers cost more than the overlap.
// * Memory loads are written as inline assembly because the compiler, which cannot tell the LDS stages apart, would wait for
//   all of them in front of every LDS read.  They write no register; tile_sync() waits for them.
#pragma once
#include "half_types.hpp"

namespace acktr {

#define ACKTR_LDS __attribute__((address_space(3)))

typedef short s16v4 __attribute__((ext_vector_type(4)));
typedef short s16v8 __attribute__((ext_vector_type(8)));

// 16 zero bytes of the reduction's tail
__device__ const uint4 g_tile_zero = {0, 0, 0, 0};

// memory -> LDS, 16 bytes a lane: from `base` (uniform) + off (per lane); to lds (uniform) + 16 * lane
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma16_ptr(const void* p, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
// all but the newest LEFT loads and every LDS access of this wave are done, then the workgroup's
template <int LEFT>
__device__ __forceinline__ void tile_sync() {
    static_assert(LEFT >= 0 && LEFT < 64, "the counter has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

__device__ __forceinline__ f32v4 mfma_half(const s16v8& a, const s16v8& b, const f32v4& c, __bf16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32v4 mfma_half(const s16v8& a, const s16v8& b, const f32v4& c, _Float16) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32v4 mfma_half(const s16v8& a, const s16v8& b, f32v4 c, float) {
    const f32v4 x = __builtin_bit_cast(f32v4, a), y = __builtin_bit_cast(f32v4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
}

// One operand's tile: R rows x 128 bytes of k per K step.  KC: k contiguous.
template <class T, bool KC, int R, int NT>
struct TileOperand {
    static constexpr int E = sizeof(T), V = 16 / E;              // values in 16 bytes
    static constexpr int KT = 128 / E;                           // k per K step
    static constexpr int BYTES = R * 128;                        // either layout
    static constexpr int CHUNKS = BYTES / 16, ITERS = CHUNKS / NT;
    static constexpr int LINE = KC ? 128 : R * E;                // bytes of an LDS line
    static_assert(CHUNKS % NT == 0, "whole loads");
    // the unit permutation of line k (rows contiguous)
    __device__ static __forceinline__ int twist(int k) { return ((k & 3) | ((k >> 1) & 4)) & (LINE / 32 - 1); }

    unsigned off[ITERS];      // per lane, from the tile's base
    int kk[ITERS];            // first k of the lane's chunk within the K step
    const char* base;         // uniform: tile's first row, current K step
    long step;                // bytes from one K step to the next

    // rows [row0, row0 + R) of `rows`, first K step at k0; ld in elements
    __device__ __forceinline__ void init(const void* p, long ld, int row0, int rows, int k0, int tid) {
        if constexpr (KC) {
            base = (const char*)p + ((long)row0 * ld + k0) * E;
            step = 128;
        } else {
            base = (const char*)p + ((long)k0 * ld + row0) * E;
            step = (long)KT * ld * E;
        }
#pragma unroll
        for (int i = 0; i < ITERS; ++i) {
            const int id = i * NT + tid;
            if constexpr (KC) {
                const int r = id >> 3, c = (id & 7) ^ ((r >> 1) & 7);
                int rr = row0 + r < rows ? r : rows - 1 - row0;   // rows behind the last one: the last one's values, never stored
                off[i] = (unsigned)((long)rr * ld * E) + c * 16;
                kk[i] = c * V;
            } else {
                constexpr int CPL = LINE / 16;                   // chunks in a line
                const int k = id / CPL, c = id % CPL, f = twist(k);
                int g = (((c >> 1) ^ f) << 1 | (c & 1)) * V;     // first row of the fetched chunk
                if (row0 + g >= rows) g = (rows - 1 - row0) / V * V;
                off[i] = (unsigned)((long)k * ld * E) + g * E;
                kk[i] = k;
            }
        }
    }
    // kleft: k that are left at this K step; lds: uniform address of the stage
    __device__ __forceinline__ void load(int kleft, unsigned lds, int wave) {
        if (kleft >= KT) {                           // (uniform)
#pragma unroll
            for (int i = 0; i < ITERS; ++i) dma16(base, off[i], lds + (i * NT + wave * 64) * 16);
        } else {
#pragma unroll
            for (int i = 0; i < ITERS; ++i)
                dma16_ptr(kk[i] < kleft ? (const void*)(base + off[i]) : (const void*)&g_tile_zero, lds + (i * NT + wave * 64) * 16);
        }
        base += step;
    }
    // fragment of rows [r0, r0 + 16), half h of the K step at LDS stage s
    __device__ static __forceinline__ s16v8 frag(const ACKTR_LDS char* s, int r0, int h, int lane) {
        if constexpr (KC) {
            const int r = r0 + (lane & 15), c = (h * 4 + (lane >> 4)) ^ ((r >> 1) & 7);
            return *reinterpret_cast<const ACKTR_LDS s16v8*>(s + r * 128 + c * 16);
        } else if constexpr (E == 2) {
            const int k = h * 32 + 8 * (lane >> 4) + ((lane & 15) >> 2);
            // k + 4 has the same (k & 3) and (k >> 3 & 1): both reads sit in the same unit
            const int u = (r0 >> 4) ^ twist(k);
            ACKTR_LDS char* p = const_cast<ACKTR_LDS char*>(s) + k * LINE + u * 32 + (lane & 3) * 8;
            const s16v4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ACKTR_LDS s16v4*>(p));
            const s16v4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<ACKTR_LDS s16v4*>(p + 4 * LINE));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            f32v4 v;
            const int r = r0 + (lane & 15);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = h * 16 + 4 * (lane >> 4) + j;
                const int u = (r >> 3) ^ twist(k);
                v[j] = *reinterpret_cast<const ACKTR_LDS float*>(s + k * LINE + u * 32 + (r & 7) * 4);
            }
            return __builtin_bit_cast(s16v8, v);
        }
    }
};

// A workgroup's BM x BN tile by WM x WN waves.  After run(): lane holds acc[mi][ni][i] = D(m, n) with
// m = wave's first row + 16 mi + lane % 16, n = wave's first column + 16 ni + 4 (lane / 16) + i.
template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int STAGES>
struct TileGemm {
    static constexpr int NT = WM * WN * 64, MI = BM / WM / 16, NI = BN / WN / 16;
    typedef TileOperand<T, AKC, BM, NT> OpA;
    typedef TileOperand<T, BKC, BN, NT> OpB;
    static constexpr int KT = OpA::KT, STAGE = OpA::BYTES + OpB::BYTES, LDS = STAGES * STAGE;
    static constexpr int LOADS = OpA::ITERS + OpB::ITERS;         // a wave's load instructions for a K step

    f32v4 acc[MI][NI];

    __device__ __forceinline__ void frags(const ACKTR_LDS char* s, int h, int wm, int wn, int lane, s16v8 (&fa)[MI], s16v8 (&fb)[NI]) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[i] = OpA::frag(s, wm + 16 * i, h, lane);
#pragma unroll
        for (int i = 0; i < NI; ++i) fb[i] = OpB::frag(s + OpA::BYTES, wn + 16 * i, h, lane);
    }
    __device__ __forceinline__ void products(const s16v8 (&fa)[MI], const s16v8 (&fb)[NI]) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i][j] = mfma_half(fb[j], fa[i], acc[i][j], T{});
    }
    // Order of a half step: its LDS reads are spread over its products instead of being gathered where registers are scarcest
    // (the compiler's own order leaves their latency in front of the next half).
    __device__ __forceinline__ void interleave() {
        constexpr int PER = sizeof(T) == 4 ? 4 : 1;
        constexpr int READS = MI * (AKC ? 1 : sizeof(T) == 4 ? 4 : 2) + NI * (BKC ? 1 : sizeof(T) == 4 ? 4 : 2), PRODUCTS = MI * NI * PER;
        constexpr int EACH = PRODUCTS >= 2 * READS ? PRODUCTS * 3 / 4 / READS : 1;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
    }
    __device__ __forceinline__ void run(const void* a, long lda, int m0, int M, const void* b, long ldb, int n0, int N, int k0, int k1,
                                        ACKTR_LDS char* sm) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
        const unsigned lds = (unsigned)(uintptr_t)sm;
        OpA oa;
        OpB ob;
        oa.init(a, lda, m0, M, k0, tid);
        ob.init(b, ldb, n0, N, k0, tid);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = f32v4{0.f, 0.f, 0.f, 0.f};
        int left = k1 - k0;                              // k not yet requested
        const int steps = (k1 - k0 + KT - 1) / KT;
        if (steps <= 0) return;
        // the request for the K step that follows the last one requested; behind the end it fetches zeros, so that the number of
        // loads in flight stays what the waits count on
        auto request = [&](unsigned stage) __attribute__((always_inline)) {
            oa.load(left, lds + stage, wave);
            ob.load(left, lds + stage + OpA::BYTES, wave);
            left -= KT;
        };
        s16v8 fa0[MI], fb0[NI], fa1[MI], fb1[NI];
#pragma unroll
        for (int i = 0; i < STAGES; ++i) request(i * STAGE);
        tile_sync<(STAGES - 1) * LOADS>();
        frags(sm, 0, wm, wn, lane, fa0, fb0);
        unsigned cur = 0;
        for (int t = 0; t + 1 < steps; ++t) {
            frags(sm + cur, 1, wm, wn, lane, fa1, fb1);
            products(fa0, fb0);
            interleave();
            tile_sync<(STAGES - 2) * LOADS>();           // this stage is read, the next one has arrived
            request(cur);
            cur = cur + STAGE == LDS ? 0 : cur + STAGE;
            frags(sm + cur, 0, wm, wn, lane, fa0, fb0);
            products(fa1, fb1);
            interleave();
        }
        frags(sm + cur, 1, wm, wn, lane, fa1, fb1);
        products(fa0, fb0);
        products(fa1, fb1);
        tile_sync<0>();                                  // LDS is the caller's again
    }
};

}  // namespace acktr
