// Tile kernels of linear_act.hip and their launches.
#pragma once
#include <atomic>
#include <type_traits>

#include "act_terms.hpp"
#include "linear_act.hpp"
#include "tile_gemm.hpp"

namespace acktr {

// act(v + bias) + res for 8 columns n.. of row m, and their stores (rows may start anywhere).  v: the product; bias and residual are
// already in registers (b, r; zero where there is none).
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish8(const LinArgs& p, int m, int n, float (&v)[8], const float (&b)[8], const vec_t<T, 8>& r, bool res) {
    typedef typename SlopeOf<T>::type ST;
    vec_t<T, 8> y;
    vec_t<ST, 8> z;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float slope;
        float o = act_of<ACT, SLOPE, sizeof(T) == 4>(v[i] + b[i], slope);
        if (res) o += to_f32(r[i]);
        y[i] = from_f32<T>(o);
        if (SLOPE) {
            ST c;
            put_slope(c, slope);
            z[i] = c;
        }
    }
    *reinterpret_cast<uvec_t<T, 8>*>((T*)p.y + (long)m * p.ldy + n) = y;
    if (SLOPE) *reinterpret_cast<uvec_t<ST, 8>*>((ST*)p.pre + (long)m * p.ldp + n) = z;
}
// one value, for the columns behind the last 8; b, r: bias and residual as above
template <class T, int ACT, bool SLOPE>
__device__ __forceinline__ void finish1(const LinArgs& p, int m, int n, float v, float b, T r, bool res) {
    typedef typename SlopeOf<T>::type ST;
    float slope;
    float o = act_of<ACT, SLOPE, sizeof(T) == 4>(v + b, slope);
    if (res) o += to_f32(r);
    ((T*)p.y)[(long)m * p.ldy + n] = from_f32<T>(o);
    if (SLOPE) put_slope(((ST*)p.pre)[(long)m * p.ldp + n], slope);
}
// f(activation code, whether slopes are wanted) as compile-time constants
template <class F>
__device__ __forceinline__ void with_act(const LinArgs& p, F&& f) {
    using std::integral_constant;
    auto both = [&](auto act) __attribute__((always_inline)) {
        if (p.pre) f(act, std::true_type{});
        else f(act, std::false_type{});
    };
    switch (p.act) {
        case ACKTR_ACT_RELU: both(integral_constant<int, ACKTR_ACT_RELU>{}); break;
        case ACKTR_ACT_TANH: both(integral_constant<int, ACKTR_ACT_TANH>{}); break;
        case ACKTR_ACT_SILU: both(integral_constant<int, ACKTR_ACT_SILU>{}); break;
        case ACKTR_ACT_GELU: both(integral_constant<int, ACKTR_ACT_GELU>{}); break;
        default: both(integral_constant<int, ACKTR_ACT_NONE>{});
    }
}
template <class T>
__device__ __forceinline__ void load_bias8(const LinArgs& p, int n, float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.f;
    if (p.bias && n + 8 <= p.N) {
        const vec_t<T, 8> x = *reinterpret_cast<const uvec_t<T, 8>*>((const T*)p.bias + n);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = to_f32(x[i]);
    }
}

// Row blocks [base, base + P) of the accumulators into LDS.  The registers of each turn are picked by comparison (they have no
// address), so one copy of the epilogue serves all turns.
template <class G, int P, int PITCH, int TURN>
__device__ __forceinline__ void spill_turn(const f32v4 (&acc)[G::MI][G::NI], int base, ACKTR_LDS float* at) {
    if (base == TURN) {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int j = 0; j < G::NI; ++j) *reinterpret_cast<ACKTR_LDS f32v4*>(at + i * 16 * PITCH + j * 16) = acc[TURN + i][j];
        asm volatile("; turn %0" ::"n"(TURN));               // keeps the turns' stores apart: merged, they would index the registers
    }
    if constexpr (TURN + P < G::MI) spill_turn<G, P, PITCH, TURN + P>(acc, base, at);
}

// One tile of a product: workgroup `id` of the p.tiles_m * p.tiles_n ones of slice `slice`.
// FULL: bias / activation / residual; otherwise the product is stored as it is.
template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int STAGES, bool FULL>
__device__ __forceinline__ void linear_tile(const LinArgs& p, int id, int slice, ACKTR_LDS char* sm) {
    typedef TileGemm<T, AKC, BKC, BM, BN, WM, WN, STAGES> G;
    // Neighbouring tiles share operand rows, so each of the 8 L2 caches (workgroups go to them in turn) gets a contiguous piece
    // of the tile order, and the order walks blocks of 8 row tiles.
    const int total = p.tiles_m * p.tiles_n;
    const int per = (total + 7) / 8, full = total - 8 * (per - 1);            // XCDs 0 .. full-1 have `per` tiles, the others per-1
    const int x = id & 7, q = id >> 3;
    const int t = x < full ? x * per + q : full * per + (x - full) * (per - 1) + q;
    const int band = t / (8 * p.tiles_n), inband = t % (8 * p.tiles_n);
    const int rows_in = min(8, p.tiles_m - band * 8);
    const int tm = band * 8 + inband % rows_in, tn = inband / rows_in;
    const int m0 = tm * BM, n0 = tn * BN;
    const int k0 = slice * p.kslice, k1 = k0 + min(p.K - k0, p.kslice);       // (k0 + kslice may pass 2^31 behind the last row)

    G g;
    g.run(p.a, p.lda, m0, p.M, p.b, p.ldb, n0, p.N, k0, k1, sm);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = m0 + (wave / WN) * (BM / WM), wn = n0 + (wave % WN) * (BN / WN);
    // The accumulators pass through a wave's own piece of LDS (P row blocks at a time) and come back as 8 consecutive columns of a
    // row, so stores cover whole lines and the epilogue is one loop.  Row pitch + 4 floats: 16 rows meet 16 different bank groups.
    constexpr int WTN = BN / WN, PITCH = WTN + 4, BLK = 16 * PITCH * 4;
    constexpr int FIT = G::LDS / (WM * WN) / BLK;
    constexpr int P = FIT >= G::MI ? G::MI : FIT >= 4 && G::MI % 4 == 0 ? 4 : FIT >= 2 && G::MI % 2 == 0 ? 2 : 1;
    static_assert(FIT >= 1, "epilogue block");
    constexpr int LPR = WTN / 8, RPI = 64 / LPR, IT = P * 16 / RPI;           // lanes a row, rows an iteration, iterations a turn
    __syncthreads();
    ACKTR_LDS float* mine = reinterpret_cast<ACKTR_LDS float*>(sm) + wave * (P * BLK / 4);
    const int lr = lane / LPR, n = wn + (lane % LPR) * 8;
    const ACKTR_LDS float* src = mine + lr * PITCH + (lane % LPR) * 8;
    auto spill = [&](int base) __attribute__((always_inline)) {
        spill_turn<G, P, PITCH, 0>(g.acc, base, mine + (lane & 15) * PITCH + 4 * (lane >> 4));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                    // the wave's own piece: no barrier
    };
    auto fetch8 = [&](int k, float(&v)[8]) __attribute__((always_inline)) {
        const f32v4 lo = *reinterpret_cast<const ACKTR_LDS f32v4*>(src + k * RPI * PITCH);
        const f32v4 hi = *reinterpret_cast<const ACKTR_LDS f32v4*>(src + k * RPI * PITCH + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
    };
    // the columns behind the last whole 8 (from `whole` on): a column a lane, so that a row's stores still lie side by side, eight rows
    // in flight
    const int whole = p.N & ~7;
    constexpr int LA = WTN < 64 ? WTN : 64, RP1 = 64 / LA, CG = WTN / LA, U = 8;
    static_assert(P * 16 / RP1 % U == 0, "whole groups of rows");
    auto finish_rest = [&](auto act, auto slope, auto slab) __attribute__((always_inline)) {
        if (whole == p.N || wn + WTN <= whole || wn >= p.N) return;           // (uniform)
        constexpr int ACT = decltype(act)::value;
        constexpr bool SLOPE = decltype(slope)::value, SLAB = decltype(slab)::value;
        const bool res = !SLAB && p.res;
#pragma unroll 1
        for (int base = 0; base < G::MI; base += P) {
            spill(base);
#pragma unroll 1
            for (int k = 0; k < CG * (P * 16 / RP1 / U); ++k) {
                const int c = (k % CG) * LA + lane % LA, r0 = (k / CG) * U * RP1 + lane / LA, nn = wn + c;
                const bool in = nn >= whole && nn < p.N;
                const float b = !SLAB && FULL && p.bias && in ? to_f32(((const T*)p.bias)[nn]) : 0.f;
                float v[U];
                T rr[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = r0 + u * RP1, m = wm + base * 16 + r;
                    v[u] = mine[r * PITCH + c];
                    rr[u] = res && in && m < p.M ? ((const T*)p.res)[(long)m * p.ldr + nn] : (T)0.f;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int m = wm + base * 16 + r0 + u * RP1;
                    if (!in || m >= p.M) continue;
                    if (SLAB) p.slabs[((long)slice * p.M + m) * p.N + nn] = v[u];
                    else finish1<T, ACT, SLOPE>(p, m, nn, v[u], b, rr[u], res);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };
    using std::integral_constant;
    if (p.slabs) {
#pragma unroll 1
        for (int base = 0; base < G::MI; base += P) {
            spill(base);
#pragma unroll 1
            for (int k = 0; k < IT; ++k) {
                const int m = wm + base * 16 + k * RPI + lr;
                float v[8];
                fetch8(k, v);
                if (m >= p.M || n + 8 > p.N) continue;
                float* s = p.slabs + ((long)slice * p.M + m) * p.N + n;
                *reinterpret_cast<uvec_t<float, 4>*>(s) = f32v4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<uvec_t<float, 4>*>(s + 4) = f32v4{v[4], v[5], v[6], v[7]};
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        return finish_rest(integral_constant<int, ACKTR_ACT_NONE>{}, std::false_type{}, std::true_type{});
    }
    auto finish = [&](auto act, auto slope) __attribute__((always_inline)) {
        constexpr int ACT = decltype(act)::value;
        constexpr bool SLOPE = decltype(slope)::value;
        float b[8];
        if constexpr (FULL) load_bias8<T>(p, n, b);
        else
            for (int i = 0; i < 8; ++i) b[i] = 0.f;
        const bool res = p.res;
        vec_t<T, 8> r[IT];
        // a turn's residual rows are requested a turn ahead: their latency passes under the turn before
        auto residual = [&](int base) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int m = wm + base * 16 + k * RPI + lr;
                if (res && m < p.M && n + 8 <= p.N) r[k] = *reinterpret_cast<const uvec_t<T, 8>*>((const T*)p.res + (long)m * p.ldr + n);
            }
        };
        residual(0);
#pragma unroll 1
        for (int base = 0; base < G::MI; base += P) {
            spill(base);
            vec_t<T, 8> now[IT];
#pragma unroll
            for (int k = 0; k < IT; ++k) now[k] = r[k];
            if (base + P < G::MI) residual(base + P);
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int m = wm + base * 16 + k * RPI + lr;
                float v[8];
                fetch8(k, v);
                if (m < p.M && n + 8 <= p.N) finish8<T, ACT, SLOPE>(p, m, n, v, b, now[k], res);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        finish_rest(act, slope, std::false_type{});
    };
    if constexpr (FULL) with_act(p, finish);
    else finish(std::integral_constant<int, ACKTR_ACT_NONE>{}, std::false_type{});
}

// db = sum of the row blocks' column sums for SUM_COLS columns, in fixed order: SUM_GROUPS groups of threads add every eighth block each,
// then their sums are added in order.  It rides in the weight gradient's launch, beside the tiles: by itself it is 2.8 us of latency
// (4096 rows, 512 columns).
template <class T>
__device__ __forceinline__ void bias_sums(const LinArgs& p, int id, ACKTR_LDS char* sm) {
    const int c = threadIdx.x % SUM_COLS, j = threadIdx.x / SUM_COLS, col = id * SUM_COLS + c;
    ACKTR_LDS float* part = reinterpret_cast<ACKTR_LDS float*>(sm);
    float t = 0.f;
    if (j < SUM_GROUPS && col < p.M) {
#pragma unroll 16
        for (int b = j; b < p.blocks; b += SUM_GROUPS) t += p.sums[(long)b * p.M + col];
        part[threadIdx.x] = t;
    }
    __syncthreads();
    if (j > 0 || col >= p.M) return;
    t = 0.f;
#pragma unroll
    for (int g = 0; g < SUM_GROUPS; ++g) t += part[g * SUM_COLS + c];
    ((T*)p.db)[col] = from_f32<T>(t);
}
static inline int bias_groups(const LinArgs& p) { return p.db ? cdiv(p.M, SUM_COLS) : 0; }

// A product in tiles (bf16, 16384 x 2048 x 2048, each in a loop of its own; the clock moves them by 10 %): forward 103 us (1335 TFLOP/s),
// with bias, silu, residual and slopes 154 us; input gradient 102 (1352); weight gradient in 4 slices 121 (1133).  Small ones are bound by launch, first loads and epilogue: 512 x 512 x 512
// takes 5.4 us.
// waves a SIMD: the largest tile has it to itself with two, the others share it
constexpr int waves_of(int bm, int bn, int waves) { return bm * bn > 128 * 128 ? waves / 4 : 2; }

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int STAGES, bool FULL>
__global__ __launch_bounds__(WM * WN * 64, waves_of(BM, BN, WM * WN)) void linear_tile_kernel(const LinArgs p) {
    extern __shared__ char smem[];
    if constexpr (!AKC && !BKC) {
        const int tiles = p.tiles_m * p.tiles_n;
        if ((int)blockIdx.x >= tiles) {
            if (blockIdx.y == 0) bias_sums<T>(p, blockIdx.x - tiles, (ACKTR_LDS char*)smem);
            return;
        }
    }
    linear_tile<T, AKC, BKC, BM, BN, WM, WN, STAGES, FULL>(p, blockIdx.x, blockIdx.y, (ACKTR_LDS char*)smem);
}
// All gradients of a layer in one launch: the weight gradient's tiles (long reductions) first, the input gradient's fill up behind
// them, then the bias's.  Apart, each leaves part of the chip idle at its end, and of a small layer most of it.
template <class T, int XM, int STAGES, int XSTAGES>
__global__ __launch_bounds__(256, 2) void linear_pair_kernel(const LinArgs dw, const LinArgs dx, int dw_groups, int tile_groups) {
    extern __shared__ char smem[];
    const int id = blockIdx.x, per = dw.tiles_m * dw.tiles_n;
    if (id < dw_groups) linear_tile<T, false, false, 64, 64, 2, 2, STAGES, false>(dw, id % per, id / per, (ACKTR_LDS char*)smem);
    else if (id >= tile_groups) bias_sums<T>(dw, id - tile_groups, (ACKTR_LDS char*)smem);
    else linear_tile<T, true, false, XM, 64, 2, 2, XSTAGES, false>(dx, id - dw_groups, 0, (ACKTR_LDS char*)smem);
}

template <class T>
__global__ __launch_bounds__(SUM_COLS * SUM_GROUPS) void bias_kernel(const LinArgs p) {
    __shared__ float part[SUM_COLS * SUM_GROUPS];
    bias_sums<T>(p, blockIdx.x, (ACKTR_LDS char*)part);
}

// Sum of the slices of a split reduction in slice order, then the epilogue: bound by reading them (4 slices of
// 2048 x 2048 13 us, 6.5 TB/s out of the caches that the tiles left them in).  V: columns a thread; 8
// halve the accesses of a large matrix, one a thread gives a small one more loads in flight (with 8 and 1: 2048 x 2048 13.9 and 16.5 us,
// 512 x 512 4.0 and 4.0, 256 x 256 5.3 and 4.4, 17 x 847 of 32 slices 22 and 4.6).
template <class T, int V>
__global__ __launch_bounds__(256) void linear_slabs_kernel(const LinArgs p, int slices) {
    const int groups = p.N / V;
    const long total = (long)p.M * groups, plane = (long)p.M * p.N;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const int m = (int)(i / groups), n = (int)(i % groups) * V;
        const float* s = p.slabs + (long)m * p.N + n;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.f;
#pragma unroll 4
        for (int z = 0; z < slices; ++z) {
            if constexpr (V == 8) {
                const f32v4 lo = *reinterpret_cast<const f32v4*>(s + z * plane), hi = *reinterpret_cast<const f32v4*>(s + z * plane + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += lo[j], v[4 + j] += hi[j];
            } else {
                v[0] += s[z * plane];
            }
        }
        if constexpr (V == 8) {
            float b[8];
            load_bias8<T>(p, n, b);
            vec_t<T, 8> r;
            if (p.res) r = *reinterpret_cast<const uvec_t<T, 8>*>((const T*)p.res + (long)m * p.ldr + n);
            with_act(p, [&](auto act, auto slope) { finish8<T, decltype(act)::value, decltype(slope)::value>(p, m, n, v, b, r, p.res); });
        } else {
            const float b = p.bias ? to_f32(((const T*)p.bias)[n]) : 0.f;
            const T r = p.res ? ((const T*)p.res)[(long)m * p.ldr + n] : (T)0.f;
            with_act(p, [&](auto act, auto slope) { finish1<T, decltype(act)::value, decltype(slope)::value>(p, m, n, v[0], b, r, p.res); });
        }
    }
}

// more than 64 KiB of LDS are granted once per kernel and device
static int allow_lds(const void* kern, int lds, std::atomic<unsigned>& allowed) {
    if (lds <= 65536) return 0;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && !(allowed.load(std::memory_order_relaxed) >> (dev & 31) & 1u)) {
        e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e == hipSuccess) allowed.fetch_or(1u << (dev & 31), std::memory_order_relaxed);
    }
    if (e == hipSuccess) return 0;
    set_error("linear_act: %d bytes of LDS refused: %s", lds, hipGetErrorString(e));
    return (int)e;
}

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int STAGES, bool FULL>
static int launch_tile(LinArgs& p, const Plan& pl, hipStream_t s) {
    auto kern = linear_tile_kernel<T, AKC, BKC, BM, BN, WM, WN, STAGES, FULL>;
    constexpr int lds = TileGemm<T, AKC, BKC, BM, BN, WM, WN, STAGES>::LDS;
    static std::atomic<unsigned> allowed{0};
    if (int rc = allow_lds((const void*)kern, lds, allowed)) return rc;
    p.tiles_m = cdiv(p.M, BM);
    p.tiles_n = cdiv(p.N, BN);
    const int more = AKC || BKC ? 0 : bias_groups(p);
    kern<<<dim3((unsigned)(p.tiles_m * p.tiles_n + more), pl.slices), dim3(WM * WN * 64), lds, s>>>(p);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

template <class T>
static int sum_slices(const LinArgs& p, int slices, hipStream_t s) {
    const long count = (long)p.M * p.N;
    if (p.N % 8 == 0 && count >= SUM_WIDE) linear_slabs_kernel<T, 8><<<min(cdiv(count / 8, 256), 2048), 256, 0, s>>>(p, slices);
    else linear_slabs_kernel<T, 1><<<min(cdiv(count, 256), 4096), 256, 0, s>>>(p, slices);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

template <class T, bool AKC, bool BKC, bool FULL>
static int product(LinArgs p, float* slabs, hipStream_t s) {
    const Plan pl = plan_of(p.M, p.N, p.K, sizeof(T));
    p.kslice = (int)pl.kslice;
    p.slabs = pl.slices > 1 ? slabs : nullptr;
    int rc;
    if constexpr (sizeof(T) == 4) {
        if (pl.tile == 0) rc = launch_tile<T, AKC, BKC, 64, 64, 2, 2, 2, FULL>(p, pl, s);
        else rc = launch_tile<T, AKC, BKC, 128, 64, 2, 2, 3, FULL>(p, pl, s);
    } else {
        switch (pl.tile) {
            case 0: rc = launch_tile<T, AKC, BKC, 64, 64, 2, 2, 3, FULL>(p, pl, s); break;
            case 1: rc = launch_tile<T, AKC, BKC, 128, 64, 2, 2, 3, FULL>(p, pl, s); break;
            case 2: rc = launch_tile<T, AKC, BKC, 128, 128, 2, 2, 2, FULL>(p, pl, s); break;
            default: rc = launch_tile<T, AKC, BKC, 256, 256, 2, 4, 2, FULL>(p, pl, s);
        }
    }
    if (rc || pl.slices == 1) return rc;
    return sum_slices<T>(p, pl.slices, s);
}

template <class T, int XM, int STAGES, int XSTAGES>
static int launch_pair(LinArgs& dw, LinArgs& dx, int slices, hipStream_t s) {
    auto kern = linear_pair_kernel<T, XM, STAGES, XSTAGES>;
    constexpr int lw = TileGemm<T, false, false, 64, 64, 2, 2, STAGES>::LDS, lx = TileGemm<T, true, false, XM, 64, 2, 2, XSTAGES>::LDS;
    constexpr int lds = lw > lx ? lw : lx;
    static std::atomic<unsigned> allowed{0};
    if (int rc = allow_lds((const void*)kern, lds, allowed)) return rc;
    dw.tiles_m = cdiv(dw.M, 64), dw.tiles_n = cdiv(dw.N, 64);
    dx.tiles_m = cdiv(dx.M, XM), dx.tiles_n = cdiv(dx.N, 64);
    const int first = dw.tiles_m * dw.tiles_n * slices, tiles = first + dx.tiles_m * dx.tiles_n;
    kern<<<tiles + bias_groups(dw), 256, lds, s>>>(dw, dx, first, tiles);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

template <class T>
int linear_gradients(LinArgs dw, LinArgs dx, float* slabs, hipStream_t s) {
    const PairPlan pl = pair_plan_of(dw, dx, sizeof(T));
    if (pl.tile < 0) {
        if (int rc = product<T, true, false, false>(dx, slabs, s)) return rc;
        return product<T, false, false, false>(dw, slabs, s);
    }
    dw.kslice = (int)pl.kslice, dw.slabs = pl.slices > 1 ? slabs : nullptr;
    dx.kslice = dx.K, dx.slabs = nullptr;
    constexpr int ST = sizeof(T) == 4 ? 2 : 3;
    const int rc = pl.tile == 0 ? launch_pair<T, 64, ST, ST>(dw, dx, pl.slices, s) : launch_pair<T, 128, ST, 3>(dw, dx, pl.slices, s);
    if (rc || pl.slices == 1) return rc;
    return sum_slices<T>(dw, pl.slices, s);
}

template <class T>
int linear_bias(const LinArgs& dw, hipStream_t s) {
    bias_kernel<T><<<bias_groups(dw), SUM_COLS * SUM_GROUPS, 0, s>>>(dw);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

template <class T>
int linear_product(LinKind kind, const LinArgs& p, float* slabs, hipStream_t s) {
    switch (kind) {
        case LIN_FORWARD: return product<T, true, true, true>(p, slabs, s);
        case LIN_DX: return product<T, true, false, false>(p, slabs, s);
        default: return product<T, false, false, false>(p, slabs, s);
    }
}

}  // namespace acktr
