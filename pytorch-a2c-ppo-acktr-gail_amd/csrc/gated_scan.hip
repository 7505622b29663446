// Gated linear recurrence over [T, N, H] and its backward pass:
//   f = s(g),  h_t = f_t (m_t h_{t-1}) + (1 - f_t) v_t                       (m_t = 0 restarts the channel: nothing before it counts)
//   E_t = m_t f_t D_t,  D_t = dout_t + E_{t+1},  E_T = dlast
//   dv = D (1 - f),  dg = D (m h_{t-1} - v) f (1 - f),  dh0 = E_0
// A step is linear in the state, h -> a h + b, and steps compose: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2).  So time is cut
// into pieces that are composed in parallel, the pieces' states follow from a short scan over them, and a second walk over the
// piece -- its inputs still in registers -- gives every state.  One read of each input, one write of each output.
//
// A wave owns 64 * V neighbouring channels (n, h flattened; V a lane) and 16 consecutive steps; the waves of a workgroup follow one
// another in time, and the workgroup walks on in superchunks of 16 steps a wave.  A whole wave per step keeps loads and stores in full
// lines, addresses in scalar registers (one 32-bit offset a lane serves all steps) and the composition free of cross-lane traffic:
// waves meet in LDS once a superchunk.  The next superchunk's inputs are requested before the present one is worked on.
// States, products and sums are fp32 whatever the storage type.
#include <type_traits>

#include "act_terms.hpp"
#include "half_types.hpp"

namespace acktr {

constexpr int SCAN_L = 16;
constexpr int SCAN_SAVE = 64;                       // steps between saved states; divides the superchunk of more than 64 steps

// A value as the compiler sees it for the first time: what was derived from it before is derived again rather than kept in a register.
template <class X>
__device__ __forceinline__ void forget(X& x) {
    typedef typename std::conditional<sizeof(X) == 8, unsigned long, typename std::conditional<sizeof(X) == 4, unsigned, unsigned short>::type>::type U;
    U u = __builtin_bit_cast(U, x);
    asm volatile("" : "+v"(u));
    x = __builtin_bit_cast(X, u);
}

// product that is 0 where a factor is, even if the other one is not finite: what a mask of 0 drops leaves no trace
extern "C" __device__ float acktr_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");      // v_mul_legacy_f32
__device__ __forceinline__ float cut_mul(float a, float x) { return acktr_mul_legacy(a, x); }
// Such a product must not become 0 by itself, however many steps it spans: a state that is not finite stays so until a mask drops it.  A
// composed factor without a zero in it is held at 2^-126 (what it adds to a finite state is what a shut gate's f adds).
__device__ __forceinline__ float held(float A) { return fabsf(A) < 1.17549435e-38f ? 1.17549435e-38f : A; }
// Products of factors, and the least of them, which tells a mask from an underflow.
template <int V>
struct Factor {
    float prod[V], least[V];
    __device__ __forceinline__ Factor() {
#pragma unroll
        for (int i = 0; i < V; ++i) prod[i] = least[i] = 1.f;
    }
    __device__ __forceinline__ void take(int i, float a) {
        prod[i] *= a;
        least[i] = fminf(least[i], fabsf(a));
    }
    __device__ __forceinline__ float value(int i) const { return least[i] == 0.f ? 0.f : held(prod[i]); }
};

// f = 1 / (1 + e^-x) and 1 - f = e^-x f, both relative to their own size.  x is held above -87, where f is fp32's smallest normal number
// and e^-x still finite (maximum() keeps a NaN).  ACC (fp32 storage): the product x log2(e) is carried with its rounding error,
// without which e^-x is off by |x| 6e-8 -- nothing beside the rounding of a 16-bit x.  That error is infinity - infinity where the
// product overflows, so there x is held below 200 too, where e^-x is 0 already.
template <bool ACC>
__device__ __forceinline__ void gate_of(float x, float& f, float& nf) {
    x = __builtin_elementwise_maximum(x, -87.f);
    if (ACC) x = __builtin_elementwise_minimum(x, 200.f);
    const float e = exp_of<ACC>(-x);
    f = fast_rcp(1.f + e);
    nf = e * f;
}

struct ScanArgs {
    const void *gate, *value, *dout;
    long gt, gn, vt, vn, ot, on, dt, dn;            // strides over t and n, in elements; h is contiguous
    const float *h0, *masks;                        // [N, H] and [T, N]; nullable
    void* out;
    float *last, *saved;                            // saved: state before every SCAN_SAVE-th step, [count, N * H]; nullable
    const float* dlast;                             // nullable
    void *dgate, *dvalue;
    long dgt, dgn, dvt, dvn;
    float* dh0;                                     // nullable
    float *agg;                                     // time split over workgroups: composed blocks [blocks][2][C]
    int T, N, H, blocks, block_steps;               // block_steps: a multiple of the superchunk
};

// How a tile's channels lie: WHOLE: all in one sequence (H is a multiple of the tile, or N is 1), so masks are scalars; MIXED: of
// several; FAR: MIXED with offsets that need 64 bits.
enum ScanMode { SCAN_WHOLE, SCAN_MIXED, SCAN_FAR };

template <class T, int V, int NW, int MODE>
struct Scan {
    static constexpr bool FAR = MODE == SCAN_FAR;
    static constexpr int CT = 64 * V, SC = NW * SCAN_L;
    typedef vec_t<T, V> vv;
    typedef vec_t<float, 2 * V> pairs;

    int lane, wave, tile, c, dn, j, n0;                    // n0: the tile's first sequence, dn: this lane's, counted from there
    bool live;

    __device__ __forceinline__ void place(const ScanArgs& p) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        // Workgroups go to the 8 L2 caches in turn: each cache gets a contiguous piece of the tiles, whose neighbours share lines where
        // rows do not start at a line's boundary (594 x 116 x 973, forward + backward: bf16 390 -> 314 us, fp32 633 -> 488).
        const int tiles = gridDim.x, per = (tiles + 7) / 8, whole = tiles - 8 * (per - 1), x = blockIdx.x & 7, q = blockIdx.x >> 3;
        tile = x < whole ? x * per + q : whole * per + (x - whole) * (per - 1) + q;
        const long first = (long)tile * CT, C = (long)p.N * p.H;
        live = first + lane * V < C;
        c = (int)(live ? first + lane * V : first);
        n0 = (int)(first / p.H);
        if constexpr (MODE == SCAN_WHOLE) {
            dn = 0;
            j = c - n0 * p.H;
        } else {
            const int n = c / p.H;
            dn = n - n0;
            j = c - n * p.H;
        }
    }
    // A [T, N, H] operand as this lane sees it, from step t on: a buffer whose base and step offsets are uniform (scalar registers), so
    // that one 32-bit offset a lane is all the addressing there is; FAR: plain 64-bit addresses.
    struct Rows {
        const char* base;                            // uniform: sequence n0
        long step;                                   // bytes a step
        typename std::conditional<FAR, long, int>::type off;
    };
    struct Window {
        __amdgpu_buffer_rsrc_t rsrc;
        const char* base;
        long step;
        typename std::conditional<FAR, long, int>::type off;
        __device__ __forceinline__ vv load(int l) const {
            if constexpr (FAR) return *reinterpret_cast<const vv*>(base + l * step + off);
            else if constexpr (sizeof(vv) == 2) return __builtin_bit_cast(vv, __builtin_amdgcn_raw_buffer_load_b16(rsrc, off, l * (int)step, 0));
            else if constexpr (sizeof(vv) == 4) return __builtin_bit_cast(vv, __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, l * (int)step, 0));
            else return __builtin_bit_cast(vv, __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, l * (int)step, 0));
        }
        __device__ __forceinline__ void store(int l, const vv& v) const {
            typedef unsigned u2 __attribute__((ext_vector_type(2)));
            if constexpr (FAR) *reinterpret_cast<vv*>(const_cast<char*>(base) + l * step + off) = v;
            else if constexpr (sizeof(vv) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rsrc, off, l * (int)step, 0);
            else if constexpr (sizeof(vv) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rsrc, off, l * (int)step, 0);
            else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, v), rsrc, off, l * (int)step, 0);
        }
    };
    __device__ __forceinline__ Rows rows(const void* p, long st, long sn) const {
        Rows r;
        r.base = (const char*)p + n0 * sn * (long)sizeof(T);
        r.step = st * (long)sizeof(T);
        r.off = (typename std::conditional<FAR, long, int>::type)((dn * sn + j) * (long)sizeof(T));
        return r;
    }
    __device__ __forceinline__ static Window at(const Rows& r, int t) {
        Window w;
        w.base = r.base + t * r.step;
        w.step = r.step;
        w.off = r.off;
        if constexpr (!FAR) w.rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(w.base), 0, 0xffffffff, 0x00020000);
        return w;
    }
    // steps [t, t + SCAN_L) of the inputs.  What lies behind the end (te), or in lanes without channels, becomes a step that changes
    // nothing: a gate of 200 (f = 1, 1 - f = 0), a value, a derivative of 0, a mask of 1.
    template <bool VALUES, bool DOUTS>
    __device__ __forceinline__ void fetch(const ScanArgs& p, const Rows& rg, const Rows& rv, const Rows& rd, int t, int te, bool all,
                                          vv (&g)[SCAN_L], vv (&v)[SCAN_L], vv (&d)[SCAN_L]) const {
        const Window wg = at(rg, t), wv = at(rv, t), wd = at(rd, t);
        const int left = te - t;
        if (all && left >= SCAN_L) {
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) {
                g[l] = wg.load(l);
                if (VALUES) v[l] = wv.load(l);
                if (DOUTS) d[l] = wd.load(l);
            }
        } else {
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) {
                g[l] = vv((T)200.f), v[l] = vv((T)0.f), d[l] = vv((T)0.f);
                if (l < left && live) {
                    g[l] = wg.load(l);
                    if (VALUES) v[l] = wv.load(l);
                    if (DOUTS) d[l] = wd.load(l);
                }
            }
        }
    }
    // (not requested ahead: they would hold registers for a whole superchunk; they are on their way while the inputs are waited for)
    __device__ __forceinline__ void masks(const ScanArgs& p, int t, int te, float (&m)[SCAN_L]) const {
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) m[l] = 1.f;
        if (p.masks) {
            const float* q = p.masks + (long)t * p.N + n0;
            if (te - t >= SCAN_L) {
#pragma unroll
                for (int l = 0; l < SCAN_L; ++l) m[l] = q[(long)l * p.N + dn];
            } else {
#pragma unroll
                for (int l = 0; l < SCAN_L; ++l)
                    if (l < te - t) m[l] = q[(long)l * p.N + dn];
            }
        }
    }
    __device__ __forceinline__ void put(const Rows& r, int t, int te, bool all, const vv (&o)[SCAN_L]) const {
        const Window w = at(r, t);
        const int left = te - t;
        if (all && left >= SCAN_L) {
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) w.store(l, o[l]);
        } else if (live) {
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l)
                if (l < left) w.store(l, o[l]);
        }
    }

    // (A, B): this wave's composed steps (REV: in descending order).  Returns the state at their start in `in` and moves `carry`
    // behind the last wave; PROD: `all` collects the product of all A.  sm: NW * CT * 2 floats; the caller alternates two of them.
    template <bool REV, bool PROD>
    __device__ __forceinline__ void exchange(const float (&A)[V], const float (&B)[V], float (&carry)[V], float (&in)[V], Factor<V>& all,
                                             pairs* sm) const {
        pairs mine;
#pragma unroll
        for (int i = 0; i < V; ++i) mine[2 * i] = A[i], mine[2 * i + 1] = B[i];
        sm[wave * 64 + lane] = mine;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const int w = REV ? NW - 1 - k : k;
            if (w == wave) {
#pragma unroll
                for (int i = 0; i < V; ++i) in[i] = carry[i];
            }
            const pairs q = sm[w * 64 + lane];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                carry[i] = cut_mul(q[2 * i], carry[i]) + q[2 * i + 1];
                if (PROD) all.take(i, q[2 * i]);
            }
        }
    }
    // the blocks before this one (REV: behind it, last to first), composed: `carry` moves over them.  A contiguous range per wave.
    template <bool REV>
    __device__ __forceinline__ void skip_blocks(const ScanArgs& p, int blk, float (&carry)[V], pairs* sm) const {
        const long C = (long)p.N * p.H;
        const int cnt = REV ? p.blocks - 1 - blk : blk, per = (cnt + NW - 1) / NW;
        const int r = REV ? NW - 1 - wave : wave, b0 = min(cnt, r * per), b1 = min(cnt, b0 + per);
        float A[V], B[V], in[V];
        Factor<V> all;
#pragma unroll
        for (int i = 0; i < V; ++i) B[i] = 0.f;
        for (int b = b0; b < b1; ++b) {
            const float* q = p.agg + 2L * (REV ? p.blocks - 1 - b : b) * C + c;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                B[i] = cut_mul(q[i], B[i]) + q[C + i];
                all.take(i, q[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = all.value(i);
        exchange<REV, false>(A, B, carry, in, all, sm);
    }
};

// --------------------------------------------------------------------------------------------------------- forward
// AGG: only the block's composition is formed (first pass of a time split).  Bound by memory: bf16, 2048 x 32 x 1024 in 89 us (4.5 TB/s
// over two reads and a write); 65536 x 1 x 512, split, 30 us for the compositions and 39 for the states.  With two channels a lane the
// registers are kept to 128, which lets two workgroups of 8 waves share a CU (that case, forward + backward, 171 us against 181 with 133).
template <class T, int V, int NW, int MODE, bool AGG>
__global__ __launch_bounds__(NW * 64, V == 2 && (NW == 8 || MODE == SCAN_WHOLE) ? 4 : 1) void scan_fwd_kernel(const ScanArgs p) {
    typedef Scan<T, V, NW, MODE> S;
    typedef typename S::vv vv;
    __shared__ typename S::pairs sm[2][NW * 64];
    S s;
    s.place(p);
    const long C = (long)p.N * p.H;
    const int blk = blockIdx.y, tb = blk * p.block_steps, te = min(p.T, tb + p.block_steps);
    const typename S::Rows rg = s.rows(p.gate, p.gt, p.gn), rv = s.rows(p.value, p.vt, p.vn), ro = s.rows(p.out, p.ot, p.on);
    const bool all = (long)(s.tile + 1) * S::CT <= C;    // every lane of the tile has channels
    float carry[V];
    Factor<V> prod;
    int par = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = !AGG && p.h0 ? p.h0[s.c + i] : 0.f;
    if (!AGG && p.blocks > 1) {
        s.template skip_blocks<false>(p, blk, carry, sm[par]);
        par ^= 1;
    }
    vv g[SCAN_L], v[SCAN_L], none[SCAN_L];
    auto fetch = [&](int t) __attribute__((always_inline)) { s.template fetch<true, false>(p, rg, rv, rg, t, te, all, g, v, none); };
    fetch(tb + s.wave * SCAN_L);
    for (int t0 = tb; t0 < te; t0 += S::SC) {
        const int tw = t0 + s.wave * SCAN_L;
        float m[SCAN_L], a[SCAN_L][V], b[SCAN_L][V], A[V], B[V], in[V], kept = 1.f;
        s.masks(p, tw, te, m);
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f;
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float f, nf;
                gate_of<sizeof(T) == 4>(to_f32(g[l][i]), f, nf);
                a[l][i] = m[l] * f;
                b[l][i] = nf * to_f32(v[l][i]);
                B[i] = cut_mul(a[l][i], B[i]) + b[l][i];
                A[i] = cut_mul(a[l][i], A[i]);
            }
            kept = cut_mul(kept, m[l]);                      // 0 where a mask of these steps is
        }
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = kept == 0.f ? 0.f : held(A[i]);
        if (t0 + S::SC < te) fetch(tw + S::SC);
        s.template exchange<false, AGG>(A, B, carry, in, prod, sm[par]);
        par ^= 1;
        if (!AGG) {
            if (p.saved && tw % SCAN_SAVE == 0 && tw < te && s.live) {
#pragma unroll
                for (int i = 0; i < V; ++i) p.saved[(long)(tw / SCAN_SAVE) * C + s.c + i] = in[i];
            }
            vv o[SCAN_L];
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    in[i] = cut_mul(a[l][i], in[i]) + b[l][i];
                    o[l][i] = from_f32<T>(in[i]);
                }
            s.put(ro, tw, te, all, o);
        }
    }
    if (s.wave == 0 && s.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (AGG) {
                p.agg[(2L * blk) * C + s.c + i] = prod.value(i);
                p.agg[(2L * blk + 1) * C + s.c + i] = carry[i];
            } else if (te == p.T && p.last) {
                p.last[s.c + i] = carry[i];
            }
        }
    }
}

// --------------------------------------------------------------------------------------------------------- backward
// The states are formed again from the saved ones, in fp32, rather than read from the rounded output.  Bound by memory: bf16,
// 2048 x 32 x 1024 in 152 us (4.4 TB/s over three reads and two writes); 65536 x 1 x 512, split, 31 + 77 us.  With two
// channels a lane the registers are kept to 256, two waves a SIMD, for a few spilled ones (forward + backward, 600 x 36 x 974 fp16 116 -> 112 us).
template <class T, int V, int NW, int MODE, bool AGG>
__global__ __launch_bounds__(NW * 64, V == 2 ? 2 : 1) void scan_bwd_kernel(const ScanArgs p) {
    typedef Scan<T, V, NW, MODE> S;
    typedef typename S::vv vv;
    __shared__ typename S::pairs sm[2][2][NW * 64];
    S s;
    s.place(p);
    const long C = (long)p.N * p.H;
    const int blk = blockIdx.y, tb = blk * p.block_steps, te = min(p.T, tb + p.block_steps);
    const typename S::Rows rg = s.rows(p.gate, p.gt, p.gn), rv = s.rows(p.value, p.vt, p.vn), rd = s.rows(p.dout, p.dt, p.dn);
    const typename S::Rows qg = s.rows(p.dgate, p.dgt, p.dgn), qv = s.rows(p.dvalue, p.dvt, p.dvn);
    const bool all = (long)(s.tile + 1) * S::CT <= C;
    float carry[V];                                          // E behind the steps that are done
    Factor<V> prod;
    int par = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = !AGG && p.dlast ? p.dlast[s.c + i] : 0.f;
    if (!AGG && p.blocks > 1) {
        s.template skip_blocks<true>(p, blk, carry, sm[0][par]);
        par ^= 1;
    }
    vv g[SCAN_L], v[SCAN_L], d[SCAN_L];
    auto fetch = [&](int t) __attribute__((always_inline)) { s.template fetch<!AGG, true>(p, rg, rv, rd, t, te, all, g, v, d); };
    const int chunks = (te - tb + S::SC - 1) / S::SC;
    fetch(tb + (chunks - 1) * S::SC + s.wave * SCAN_L);
    for (int q = chunks - 1; q >= 0; --q) {
        const int t0 = tb + q * S::SC, tw = t0 + s.wave * SCAN_L;
        float f[SCAN_L][V], nf[SCAN_L][V], A[V], B[V], P[V], Q[V], in[V], ein[V], kept = 1.f;
        vv vc[SCAN_L], dc[SCAN_L];
        float mc[SCAN_L];
        s.masks(p, tw, te, mc);
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f, P[i] = 1.f, Q[i] = 0.f;
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
            dc[l] = d[l];
            if (!AGG) vc[l] = v[l];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                gate_of<sizeof(T) == 4>(to_f32(g[l][i]), f[l][i], nf[l][i]);
                if (!AGG) {
                    const float a = mc[l] * f[l][i];
                    B[i] = cut_mul(a, B[i]) + nf[l][i] * to_f32(vc[l][i]);
                    A[i] = cut_mul(a, A[i]);
                }
            }
        }
#pragma unroll
        for (int l = SCAN_L - 1; l >= 0; --l) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float a = mc[l] * f[l][i];
                Q[i] = cut_mul(a, to_f32(dc[l][i]) + Q[i]);
                P[i] = cut_mul(a, P[i]);
            }
            kept = cut_mul(kept, mc[l]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = kept == 0.f ? 0.f : held(A[i]), P[i] = kept == 0.f ? 0.f : held(P[i]);
        if (q > 0) fetch(tw - S::SC);
        if (!AGG) {
            // fp32 copies of values and derivatives and the products m f would take 96 registers more
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) {
                forget(vc[l]), forget(dc[l]);
#pragma unroll
                for (int i = 0; i < V; ++i) forget(f[l][i]);
            }
            float start[V];
#pragma unroll
            for (int i = 0; i < V; ++i) start[i] = p.saved ? p.saved[(long)(t0 / SCAN_SAVE) * C + s.c + i] : p.h0 ? p.h0[s.c + i] : 0.f;
            s.template exchange<false, false>(A, B, start, in, prod, sm[1][par]);
        }
        s.template exchange<true, AGG>(P, Q, carry, ein, prod, sm[0][par]);
        par ^= 1;
        if (!AGG) {
            float hp[SCAN_L][V];                             // m_t h_{t-1}
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    hp[l][i] = cut_mul(mc[l], in[i]);
                    in[i] = cut_mul(f[l][i], hp[l][i]) + nf[l][i] * to_f32(vc[l][i]);
                }
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) forget(vc[l]);
            vv og[SCAN_L], ov[SCAN_L];
#pragma unroll
            for (int l = SCAN_L - 1; l >= 0; --l)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float D = to_f32(dc[l][i]) + ein[i], y = D * nf[l][i];
                    og[l][i] = from_f32<T>((hp[l][i] - to_f32(vc[l][i])) * f[l][i] * y);
                    ov[l][i] = from_f32<T>(y);
                    ein[i] = cut_mul(mc[l] * f[l][i], D);
                }
            s.put(qg, tw, te, all, og);
            s.put(qv, tw, te, all, ov);
        }
    }
    if (s.wave == 0 && s.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (AGG) {
                p.agg[(2L * blk) * C + s.c + i] = prod.value(i);
                p.agg[(2L * blk + 1) * C + s.c + i] = carry[i];
            } else if (tb == 0 && p.dh0) {
                p.dh0[s.c + i] = carry[i];
            }
        }
    }
}

// --------------------------------------------------------------------------------------------------------- one token
// A channel a value, 8 bytes of gate and value a lane where rows allow it.  32 x 512 is one launch of latency.
template <class T, int V>
__global__ __launch_bounds__(256) void scan_step_kernel(const void* gate, long gn, const void* value, long vn, const float* from, float* to,
                                                        const float* masks, void* out, long on, int N, int H) {
    typedef vec_t<T, V> vv;
    typedef vec_t<float, V> fv;
    const long c = ((long)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= (long)N * H) return;
    const int n = (int)(c / H), j = (int)(c - (long)n * H);
    const vv g = *reinterpret_cast<const vv*>((const T*)gate + n * gn + j), v = *reinterpret_cast<const vv*>((const T*)value + n * vn + j);
    fv h = *reinterpret_cast<const fv*>(from + c);
    const float m = masks ? masks[n] : 1.f;
    vv o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float f, nf;
        gate_of<sizeof(T) == 4>(to_f32(g[i]), f, nf);
        h[i] = f * cut_mul(m, h[i]) + nf * to_f32(v[i]);
        o[i] = from_f32<T>(h[i]);
    }
    *reinterpret_cast<fv*>(to + c) = h;
    *reinterpret_cast<vv*>((T*)out + n * on + j) = o;
}
// dst = src or 0: the states of a sequence of no steps
__global__ __launch_bounds__(256) void scan_copy_kernel(const float* src, float* dst, long n) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : 0.f;
}

// --------------------------------------------------------------------------------------------------------- host side
struct ScanPlan { int v, nw, sc, ct, blocks, block_steps; };

// Time is split over workgroups (about 512 of them) where tiles of 64 channels alone would leave most of the chip without work: it costs
// a second read of gates and values, by all CUs at once.  V = 2 (16-bit storage, rows that allow it: 4 bytes a lane, half the loads)
// pays where there are tiles of 128 channels for every CU, or a split with enough steps to share.  Waves: as many as the steps fill, up
// to 8, or 4 where two workgroups and more share a CU anyway.
// Measured, forward + backward, us (bf16 unless said; H = 512):
//   split: T x N 2048 x 8 54 against 120 whole, 2048 x 16 94 / 121, 512 x 16 30 / 37, 2048 x 20 121 / 125, 1024 x 24 85 / 67,
//     2048 x 32 169 / 155; 256 x 4 21 / 20; fp32 2048 x 12 112 / 126, 512 x 16 46 / 41
//   4 waves instead of 8 (H = 1024): 300 x 64 67 against 76, 594 x 116 267 / 275, 128 x 256 120 / 131; 2048 x 32, a tile a CU, 279 / 236
//   V = 2: whole 1024 x 64 118 against 154, 2048 x 32 188 / 155; split 512 x 16 30 / 34, 1024 x 8 31 / 34, 512 x 8 26 / 23
static ScanPlan scan_plan(long T, long N, long H, int e, bool pair) {
    ScanPlan p;
    const long C = N * H;
    const bool split = T > 2 * 8 * SCAN_L && C <= 64 * (e == 2 ? 128 : 96);
    p.v = e == 2 && pair && (split ? T * C >= 1 << 22 : C >= 128 * 256) ? 2 : 1;
    p.ct = 64 * p.v;
    const long tiles = cdiv(C, p.ct);
    p.nw = T <= 16 ? 1 : T <= 64 || tiles >= 512 ? 4 : 8;
    p.sc = p.nw * SCAN_L;
    const long chunks = cdiv(T, p.sc), per = split ? cdiv(chunks, min(chunks, (long)cdiv(512, tiles))) : max(chunks, 1L);
    p.block_steps = (int)(per * p.sc);
    p.blocks = (int)max(cdiv(chunks, per), 1);
    return p;
}
// two neighbouring channels can be taken at once
static bool in_pairs(const void* p, long st, long sn, int e) { return ((uintptr_t)p & (2 * e - 1)) == 0 && st % 2 == 0 && sn % 2 == 0; }
// offsets within a tile of 128 channels or 16 steps need more than 31 bits
static bool is_far(long st, long sn, long N, long H, int e) { return (min(N, 128 / H + 2) * sn + H) * e >= (1L << 31) || SCAN_L * st * e >= (1L << 31); }

static int scan_check(long T, long N, long H, int dtype) {
    ACKTR_ARG(dtype_ok(dtype), "gated_scan: unknown dtype code %d", dtype);
    ACKTR_ARG(T >= 0 && N >= 0 && H >= 1, "gated_scan: sizes must be T >= 0, N >= 0, H >= 1 (got T %ld, N %ld, H %ld)", T, N, H);
    ACKTR_ARG(T < (1L << 30) && N * H < (1L << 30), "gated_scan: T and N * H must be below 2^30 (got T %ld, N %ld, H %ld)", T, N, H);
    return 0;
}

template <class T, bool BWD, bool AGG, int V, int MODE>
static void scan_launch_nw(const ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    const dim3 grid(cdiv((long)a.N * a.H, p.ct), p.blocks);
    auto go = [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        if constexpr (BWD) scan_bwd_kernel<T, V, NW, MODE, AGG><<<grid, NW * 64, 0, s>>>(a);
        else scan_fwd_kernel<T, V, NW, MODE, AGG><<<grid, NW * 64, 0, s>>>(a);
    };
    if constexpr (AGG) {                                     // a time split has more than 256 steps and few tiles: always 8 waves
        go(std::integral_constant<int, 8>{});
    } else {
        if (p.nw == 1) go(std::integral_constant<int, 1>{});
        else if (p.nw == 4) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 8>{});
    }
}
template <class T, bool BWD, bool AGG>
static void scan_launch(const ScanArgs& a, const ScanPlan& p, bool far, hipStream_t s) {
    const bool whole = a.N == 1 || a.H % p.ct == 0;
    if (far) return scan_launch_nw<T, BWD, AGG, 1, SCAN_FAR>(a, p, s);
    if constexpr (sizeof(T) == 2) {
        if (p.v == 2 && whole) return scan_launch_nw<T, BWD, AGG, 2, SCAN_WHOLE>(a, p, s);
        if (p.v == 2) return scan_launch_nw<T, BWD, AGG, 2, SCAN_MIXED>(a, p, s);
    }
    if (whole) scan_launch_nw<T, BWD, AGG, 1, SCAN_WHOLE>(a, p, s);
    else scan_launch_nw<T, BWD, AGG, 1, SCAN_MIXED>(a, p, s);
}
template <class T, bool BWD>
static int scan_run(ScanArgs a, const ScanPlan& p, bool far, hipStream_t s) {
    a.blocks = p.blocks;
    a.block_steps = p.block_steps;
    if (p.blocks > 1) {
        scan_launch<T, BWD, true>(a, p, far, s);
        ACKTR_LAUNCH_CHECK();
    }
    scan_launch<T, BWD, false>(a, p, far, s);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

}  // namespace acktr

using namespace acktr;

extern "C" int acktr_gated_scan_save_interval(void) { return SCAN_SAVE; }

extern "C" long acktr_gated_scan_workspace_bytes(long T, long N, long H, int dtype) {
    if (scan_check(T, N, H, dtype)) return -1;
    long most = 0;
    for (int pair = 0; pair < 2; ++pair) {
        const ScanPlan p = scan_plan(T, N, H, (int)elem_bytes(dtype), pair != 0);
        if (p.blocks > 1) most = max(most, 8L * p.blocks * N * H);
    }
    return most;
}

extern "C" int acktr_gated_scan_fwd(const void* gate, long gt, long gn, const void* value, long vt, long vn, const float* h0,
                                    const float* masks, void* out, long ot, long on, float* last, float* saved, long T, long N, long H,
                                    int dtype, void* workspace, long workspace_bytes, void* stream) {
    if (int rc = scan_check(T, N, H, dtype)) return rc;
    if (N * H == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    if (T == 0) {
        if (last) {
            scan_copy_kernel<<<cdiv(N * H, 256), 256, 0, s>>>(h0, last, N * H);
            ACKTR_LAUNCH_CHECK();
        }
        return 0;
    }
    const int e = (int)elem_bytes(dtype);
    ACKTR_ARG(gate && value && out, "gated_scan_fwd: gate, value and out are required");
    ACKTR_ARG(gt >= 0 && gn >= 0 && vt >= 0 && vn >= 0 && ot >= 0 && on >= 0, "gated_scan_fwd: negative stride");
    const bool far = is_far(gt, gn, N, H, e) || is_far(vt, vn, N, H, e) || is_far(ot, on, N, H, e);
    const bool pair = !far && H % 2 == 0 && in_pairs(gate, gt, gn, e) && in_pairs(value, vt, vn, e) && in_pairs(out, ot, on, e);
    ACKTR_ARG(workspace_bytes >= acktr_gated_scan_workspace_bytes(T, N, H, dtype), "gated_scan_fwd: workspace of %ld bytes is too small",
              workspace_bytes);
    const ScanPlan p = scan_plan(T, N, H, e, pair);
    ScanArgs a{};
    a.gate = gate, a.gt = gt, a.gn = gn, a.value = value, a.vt = vt, a.vn = vn, a.h0 = h0, a.masks = masks;
    a.out = out, a.ot = ot, a.on = on, a.last = last, a.saved = saved, a.agg = (float*)workspace;
    a.T = (int)T, a.N = (int)N, a.H = (int)H;
    return with_dtype(dtype, [&](auto t) -> int { return scan_run<decltype(t), false>(a, p, far, s); });
}

extern "C" int acktr_gated_scan_bwd(const void* dout, long dt, long dn, const void* gate, long gt, long gn, const void* value, long vt, long vn,
                                    const float* h0, const float* masks, const float* saved, const float* dlast, void* dgate, long dgt,
                                    long dgn, void* dvalue, long dvt, long dvn, float* dh0, long T, long N, long H, int dtype,
                                    void* workspace, long workspace_bytes, void* stream) {
    if (int rc = scan_check(T, N, H, dtype)) return rc;
    if (N * H == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    if (T == 0) {
        if (dh0) {
            scan_copy_kernel<<<cdiv(N * H, 256), 256, 0, s>>>(dlast, dh0, N * H);
            ACKTR_LAUNCH_CHECK();
        }
        return 0;
    }
    const int e = (int)elem_bytes(dtype);
    ACKTR_ARG(dout && gate && value && dgate && dvalue, "gated_scan_bwd: dout, gate, value, dgate and dvalue are required");
    ACKTR_ARG(dt >= 0 && dn >= 0 && gt >= 0 && gn >= 0 && vt >= 0 && vn >= 0 && dgt >= 0 && dgn >= 0 && dvt >= 0 && dvn >= 0,
              "gated_scan_bwd: negative stride");
    const bool far = is_far(gt, gn, N, H, e) || is_far(vt, vn, N, H, e) || is_far(dt, dn, N, H, e) || is_far(dgt, dgn, N, H, e) || is_far(dvt, dvn, N, H, e);
    const bool pair = !far && H % 2 == 0 && in_pairs(dout, dt, dn, e) && in_pairs(gate, gt, gn, e) && in_pairs(value, vt, vn, e) &&
                      in_pairs(dgate, dgt, dgn, e) && in_pairs(dvalue, dvt, dvn, e);
    ACKTR_ARG(workspace_bytes >= acktr_gated_scan_workspace_bytes(T, N, H, dtype), "gated_scan_bwd: workspace of %ld bytes is too small",
              workspace_bytes);
    const ScanPlan p = scan_plan(T, N, H, e, pair);
    ACKTR_ARG(saved || T <= SCAN_SAVE, "gated_scan_bwd: %ld steps need the states that the forward pass saves every %d steps", T, SCAN_SAVE);
    ScanArgs a{};
    a.dout = dout, a.dt = dt, a.dn = dn, a.gate = gate, a.gt = gt, a.gn = gn, a.value = value, a.vt = vt, a.vn = vn;
    a.h0 = h0, a.masks = masks, a.saved = const_cast<float*>(saved), a.dlast = dlast;
    a.dgate = dgate, a.dgt = dgt, a.dgn = dgn, a.dvalue = dvalue, a.dvt = dvt, a.dvn = dvn, a.dh0 = dh0, a.agg = (float*)workspace;
    a.T = (int)T, a.N = (int)N, a.H = (int)H;
    return with_dtype(dtype, [&](auto t) -> int { return scan_run<decltype(t), true>(a, p, far, s); });
}

// one step from state `from` to state `to` (the same one, or apart)
static int scan_step(const void* gate, long gn, const void* value, long vn, const float* from, float* to, const float* masks, void* out, long on,
                     long N, long H, int dtype, hipStream_t s) {
    return with_dtype(dtype, [&](auto t) -> int {
        typedef decltype(t) T;
        constexpr int W = 8 / sizeof(T);
        auto rows8 = [](const void* q, long sn) { return ((uintptr_t)q & 7) == 0 && sn * (long)sizeof(T) % 8 == 0; };
        const bool wide = H % W == 0 && rows8(gate, gn) && rows8(value, vn) && rows8(out, on) && (((uintptr_t)from | (uintptr_t)to) & 15) == 0;
        if (wide) scan_step_kernel<T, W><<<cdiv(N * H, 256 * W), 256, 0, s>>>(gate, gn, value, vn, from, to, masks, out, on, (int)N, (int)H);
        else scan_step_kernel<T, 1><<<cdiv(N * H, 256), 256, 0, s>>>(gate, gn, value, vn, from, to, masks, out, on, (int)N, (int)H);
        ACKTR_LAUNCH_CHECK();
        return 0;
    });
}

extern "C" int acktr_gated_scan_step(const void* gate, long gn, const void* value, long vn, float* state, const float* masks, void* out, long on,
                                     long N, long H, int dtype, void* stream) {
    if (int rc = scan_check(1, N, H, dtype)) return rc;
    if (N * H == 0) return 0;
    ACKTR_ARG(gate && value && state && out, "gated_scan_step: gate, value, state and out are required");
    ACKTR_ARG(gn >= 0 && vn >= 0 && on >= 0, "gated_scan_step: negative stride");
    return scan_step(gate, gn, value, vn, state, state, masks, out, on, N, H, dtype, (hipStream_t)stream);
}

// One step of the whole core.  Its three launches are those of the single entries; a caller that acts, and waits for every step, saves
// the host's work for two calls.
struct CoreSpace { long h, scratch, bytes; };
static int core_space(const void* x, long ldx, const void* w_in, const void* w_out, long N, long I, long H, int dtype, CoreSpace& sp) {
    if (int rc = scan_check(1, N, H, dtype)) return rc;
    const long e = elem_bytes(dtype);
    const long a = acktr_linear_act_fwd_workspace_bytes(x, ldx, w_in, I, N, 2 * H, I, dtype);
    const long b = acktr_linear_act_fwd_workspace_bytes(nullptr, H, w_out, H, N, H, H, dtype);        // (the states start at 256 bytes)
    if (a < 0 || b < 0) return -1;
    auto up256 = [](long v) { return (v + 255) / 256 * 256; };
    sp.h = up256(2 * N * H * e);
    sp.scratch = sp.h + up256(N * H * e);
    sp.bytes = sp.scratch + max(a, b);
    return 0;
}
extern "C" long acktr_gated_core_step_workspace_bytes(const void* x, long ldx, const void* w_in, const void* w_out, long N, long I, long H, int dtype) {
    CoreSpace sp;
    return core_space(x, ldx, w_in, w_out, N, I, H, dtype, sp) ? -1 : sp.bytes;
}
extern "C" int acktr_gated_core_step(const void* x, long ldx, const void* w_in, const void* b_in, const void* w_out, const void* b_out,
                                     const float* state, float* state_out, const float* masks, void* y, long ldy, long N, long I, long H,
                                     int dtype, void* workspace, long workspace_bytes, void* stream) {
    CoreSpace sp;
    if (int rc = core_space(x, ldx, w_in, w_out, N, I, H, dtype, sp)) return rc;
    if (N == 0) return 0;
    ACKTR_ARG(x && w_in && w_out && state && state_out && y, "gated_core_step: x, the weights, both states and y are required");
    ACKTR_ARG(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= sp.bytes,
              "gated_core_step: workspace of %ld bytes, %ld with 256-byte alignment are needed", workspace_bytes, sp.bytes);
    ACKTR_ARG(ldx >= I && ldx < (1 << 21) && ldy >= H && ldy < (1 << 21),
              "gated_core_step: row strides must be at least the rows' lengths and below 2^21 (got %ld, %ld)", ldx, ldy);
    char *proj = (char*)workspace, *h = proj + sp.h, *scratch = proj + sp.scratch;
    const long left = workspace_bytes - sp.scratch, e = elem_bytes(dtype);
    if (int rc = acktr_linear_act_fwd(x, ldx, w_in, I, b_in, nullptr, 0, proj, 2 * H, nullptr, 0, N, 2 * H, I, dtype, ACKTR_ACT_NONE, scratch, left, stream))
        return rc;
    if (int rc = scan_step(proj, 2 * H, proj + H * e, 2 * H, state, state_out, masks, h, H, N, H, dtype, (hipStream_t)stream)) return rc;
    return acktr_linear_act_fwd(h, H, w_out, H, b_out, h, H, y, ldy, nullptr, 0, N, H, H, dtype, ACKTR_ACT_SILU, scratch, left, stream);
}
