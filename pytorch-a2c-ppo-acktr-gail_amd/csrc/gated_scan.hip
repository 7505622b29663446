// Gated linear recurrence over [T, N, H] and its backward pass:
//   f = s(g),  h_t = f_t (m_t h_{t-1}) + (1 - f_t) v_t                       (m_t = 0 restarts the channel: nothing before it counts)
//   E_t = m_t f_t D_t,  D_t = dout_t + E_{t+1},  E_T = dlast
//   dv = D (1 - f),  dg = D (m h_{t-1} - v) f (1 - f),  dh0 = E_0
// A step is linear in the state, h -> a h + b, and steps compose: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2).  So time is cut
// into pieces that are composed in parallel, the pieces' states follow from a short scan over them, and a second walk over the
// piece -- its inputs still in registers -- gives every state.  One read of each input, one write of each output.
//
// A workgroup owns CT = LC * V neighbouring channels (n, h flattened) and walks time in superchunks of NW * (64 / LC) * L steps: each
// thread holds L consecutive steps of V channels.  States, products and sums are fp32 whatever the storage type.
#include "act_terms.hpp"
#include "half_types.hpp"

namespace acktr {

constexpr int SCAN_L = 8;

// restart-safe product: a zero factor drops the other one even if it is not finite
__device__ __forceinline__ float cut_mul(float a, float x) { return a == 0.f ? 0.f : a * x; }

// f = 1 / (1 + e^-x) and 1 - f without cancellation; e = exp(-|x|) <= 1 never overflows.  The product |x| log2(e) is carried
// with its rounding error: without it e is off by |x| * 6e-8.
__device__ __forceinline__ void gate_of(float x, float& f, float& nf) {
    const float a = -fabsf(x), p = a * LOG2E, lo = fmaf(a, LOG2E, -p) + a * 1.92596299e-8f;
    const float e0 = __builtin_amdgcn_exp2f(p), e = fmaf(e0, lo * 0.693147182f, e0), r = fast_rcp(1.f + e);
    const float small = e * r;
    f = x < 0.f ? small : r;
    nf = x < 0.f ? r : small;
}

// both halves of a gate in one register: the smaller one, with the sign bit set where it is f
__device__ __forceinline__ float gate_pack(float x, float f, float nf) { return x < 0.f ? -f : nf; }
__device__ __forceinline__ void gate_unpack(float s, float& f, float& nf) {
    const bool neg = __float_as_uint(s) >> 31;
    const float a = fabsf(s), b = 1.f - a;
    f = neg ? a : b;
    nf = neg ? b : a;
}

constexpr int SCAN_SAVE = 64;                       // steps between saved states; divides every superchunk of more than 32 steps

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

template <class T, int V, int LC, int NW>
struct Scan {
    static constexpr int NT = NW * 64, GW = 64 / LC, CT = LC * V, SC = NW * GW * SCAN_L;
    typedef vec_t<T, V> vv;

    int lane, wave, group, c, n, j, chl;            // chl: channel within the tile
    bool live;

    __device__ __forceinline__ void place(const ScanArgs& p) {
        lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        group = wave * GW + lane / LC;
        chl = (lane % LC) * V;
        const long cc = (long)blockIdx.x * CT + chl;
        live = cc < (long)p.N * p.H;
        c = live ? (int)cc : 0;
        n = c / p.H;
        j = c - n * p.H;
    }
    __device__ __forceinline__ static vv load(const void* base, long off) { return *reinterpret_cast<const vv*>((const T*)base + off); }

    // (A, B): this thread's composed piece, in group order (REV: in descending order).  Returns the state at the piece's start in `in`
    // and moves `carry` behind the last piece.  sm: [NW][CT][2] floats; the caller alternates two of them.
    template <bool REV>
    __device__ __forceinline__ void exchange(float (&A)[V], float (&B)[V], float (&carry)[V], float (&in)[V], float* sm) {
#pragma unroll
        for (int d = LC; d < 64; d *= 2) {
            const bool has = REV ? lane + d < 64 : lane >= d;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float pa = REV ? __shfl_down(A[i], d, 64) : __shfl_up(A[i], d, 64);
                const float pb = REV ? __shfl_down(B[i], d, 64) : __shfl_up(B[i], d, 64);
                if (has) {
                    B[i] += cut_mul(A[i], pb);
                    A[i] *= pa;
                }
            }
        }
        const bool edge = REV ? lane < LC : lane >= 64 - LC;             // holds the wave's whole composition
        if (edge) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sm[(wave * CT + chl + i) * 2] = A[i];
                sm[(wave * CT + chl + i) * 2 + 1] = B[i];
            }
        }
        float ea[V], eb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            ea[i] = 1.f, eb[i] = 0.f;
            if (LC < 64) {
                const float pa = REV ? __shfl_down(A[i], LC, 64) : __shfl_up(A[i], LC, 64);
                const float pb = REV ? __shfl_down(B[i], LC, 64) : __shfl_up(B[i], LC, 64);
                const bool first = REV ? lane >= 64 - LC : lane < LC;
                if (!first) ea[i] = pa, eb[i] = pb;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float h = carry[i], mine = h;
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const int w = REV ? NW - 1 - k : k;
                if (w == wave) mine = h;
                const float a = sm[(w * CT + chl + i) * 2], b = sm[(w * CT + chl + i) * 2 + 1];
                h = cut_mul(a, h) + b;
            }
            carry[i] = h;
            in[i] = cut_mul(ea[i], mine) + eb[i];
        }
    }
};

// --------------------------------------------------------------------------------------------------------- forward
// AGG: only the block's composition is formed (first pass of a time split).
template <class T, int V, int LC, int NW, bool AGG>
__global__ __launch_bounds__(NW * 64) void scan_fwd_kernel(const ScanArgs p) {
    typedef Scan<T, V, LC, NW> S;
    typedef typename S::vv vv;
    __shared__ float sm[2][NW * S::CT * 2];
    S s;
    s.place(p);
    const long C = (long)p.N * p.H;
    const int blk = blockIdx.y, tb = blk * p.block_steps, te = min(p.T, tb + p.block_steps);
    float carry[V];
    int par = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = !AGG && p.h0 && s.live ? p.h0[s.c + i] : 0.f;
    if (!AGG && p.blocks > 1) {                              // the blocks before this one, composed: a contiguous range per group
        const int G = NW * S::GW, per = (blk + G - 1) / G, b0 = min(blk, s.group * per), b1 = min(blk, b0 + per);
        float A[V], B[V], in[V];
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f;
        if (s.live)
            for (int b = b0; b < b1; ++b)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = p.agg[(2L * b) * C + s.c + i];
                    B[i] = cut_mul(a, B[i]) + p.agg[(2L * b + 1) * C + s.c + i];
                    A[i] *= a;
                }
        s.template exchange<false>(A, B, carry, in, sm[par]);
        par ^= 1;
    }
    float wa[V];                                             // AGG: the block's composition so far is (wa, carry)
#pragma unroll
    for (int i = 0; i < V; ++i) wa[i] = 1.f;

    vv g[SCAN_L], v[SCAN_L];
    float m[SCAN_L];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
            const int t = t0 + l;
            if (s.live && t < te) {
                g[l] = S::load(p.gate, t * p.gt + s.n * p.gn + s.j);
                v[l] = S::load(p.value, t * p.vt + s.n * p.vn + s.j);
                m[l] = p.masks ? p.masks[(long)t * p.N + s.n] : 1.f;
            }
        }
    };
    fetch(tb + s.group * SCAN_L);
    for (int t0 = tb; t0 < te; t0 += S::SC) {
        const int tg = t0 + s.group * SCAN_L;
        float a[SCAN_L][V], b[SCAN_L][V], A[V], B[V], in[V];
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f;
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
            const bool on = s.live && tg + l < te;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float f, nf;
                gate_of(on ? to_f32(g[l][i]) : 0.f, f, nf);
                a[l][i] = on ? m[l] * f : 1.f;
                b[l][i] = on ? nf * to_f32(v[l][i]) : 0.f;
                B[i] = cut_mul(a[l][i], B[i]) + b[l][i];
                A[i] *= a[l][i];
            }
        }
        if (t0 + S::SC < te) fetch(tg + S::SC);
        if (AGG) {
            // the product of all a of the superchunk: composed with a state of 1 and no addend
#pragma unroll
            for (int i = 0; i < V; ++i) in[i] = 0.f;
            float A2[V], Z[V];
#pragma unroll
            for (int i = 0; i < V; ++i) A2[i] = A[i], Z[i] = 0.f;
            float dummy[V];
            s.template exchange<false>(A2, Z, wa, dummy, sm[par]);
            par ^= 1;
        }
        s.template exchange<false>(A, B, carry, in, sm[par]);
        par ^= 1;
        if (!AGG) {
            if (p.saved && s.live && tg % SCAN_SAVE == 0 && tg < te) {
#pragma unroll
                for (int i = 0; i < V; ++i) p.saved[(long)(tg / SCAN_SAVE) * C + s.c + i] = in[i];
            }
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) {
                vv o;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    in[i] = cut_mul(a[l][i], in[i]) + b[l][i];
                    o[i] = from_f32<T>(in[i]);
                }
                const int t = tg + l;
                if (s.live && t < te) *reinterpret_cast<vv*>((T*)p.out + t * p.ot + s.n * p.on + s.j) = o;
            }
        }
    }
    if (s.group == 0 && s.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (AGG) {
                p.agg[(2L * blk) * C + s.c + i] = wa[i];
                p.agg[(2L * blk + 1) * C + s.c + i] = carry[i];
            } else if (te == p.T && p.last) {
                p.last[s.c + i] = carry[i];
            }
        }
    }
}

// --------------------------------------------------------------------------------------------------------- backward
template <class T, int V, int LC, int NW, bool AGG>
__global__ __launch_bounds__(NW * 64) void scan_bwd_kernel(const ScanArgs p) {
    typedef Scan<T, V, LC, NW> S;
    typedef typename S::vv vv;
    __shared__ float sm[2][2][NW * S::CT * 2];
    S s;
    s.place(p);
    const long C = (long)p.N * p.H;
    const int blk = blockIdx.y, tb = blk * p.block_steps, te = min(p.T, tb + p.block_steps);
    float carry[V];                                          // E behind the steps that are done
    int par = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = !AGG && p.dlast && s.live ? p.dlast[s.c + i] : 0.f;
    if (!AGG && p.blocks > 1) {                              // the blocks behind this one, last to first
        const int G = NW * S::GW, cnt = p.blocks - 1 - blk, per = (cnt + G - 1) / G;
        const int r = G - 1 - s.group, b0 = min(cnt, r * per), b1 = min(cnt, b0 + per);      // group G-1 has the last blocks
        float A[V], B[V], in[V];
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f;
        if (s.live)
            for (int b = b0; b < b1; ++b)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const long q = 2L * (p.blocks - 1 - b);
                    const float a = p.agg[q * C + s.c + i];
                    B[i] = cut_mul(a, B[i]) + p.agg[(q + 1) * C + s.c + i];
                    A[i] *= a;
                }
        s.template exchange<true>(A, B, carry, in, sm[0][par]);
        par ^= 1;
    }
    float wa[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wa[i] = 1.f;

    vv g[SCAN_L], v[SCAN_L], d[SCAN_L];
    float m[SCAN_L];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
            const int t = t0 + l;
            if (s.live && t < te) {
                g[l] = S::load(p.gate, t * p.gt + s.n * p.gn + s.j);
                if (!AGG) v[l] = S::load(p.value, t * p.vt + s.n * p.vn + s.j);
                d[l] = S::load(p.dout, t * p.dt + s.n * p.dn + s.j);
                m[l] = p.masks ? p.masks[(long)t * p.N + s.n] : 1.f;
            }
        }
    };
    const int chunks = (te - tb + S::SC - 1) / S::SC;
    fetch(tb + (chunks - 1) * S::SC + s.group * SCAN_L);
    for (int q = chunks - 1; q >= 0; --q) {
        const int t0 = tb + q * S::SC, tg = t0 + s.group * SCAN_L;
        float f[SCAN_L][V], A[V], B[V], P[V], Q[V], in[V], ein[V], start[V];
        vv vc[SCAN_L], dc[SCAN_L];
        float mc[SCAN_L];
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, B[i] = 0.f, P[i] = 1.f, Q[i] = 0.f;
#pragma unroll
        for (int l = 0; l < SCAN_L; ++l) {
            const bool on = s.live && tg + l < te;
            mc[l] = on ? m[l] : 1.f;
            if (!AGG) vc[l] = v[l];
            dc[l] = d[l];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float ff, nf;
                const float x = on ? to_f32(g[l][i]) : 0.f;
                gate_of(x, ff, nf);
                f[l][i] = gate_pack(x, ff, nf);
                if (!AGG) {
                    const float a = on ? mc[l] * ff : 1.f;
                    B[i] = cut_mul(a, B[i]) + (on ? nf * to_f32(vc[l][i]) : 0.f);
                    A[i] *= a;
                }
            }
        }
#pragma unroll
        for (int l = SCAN_L - 1; l >= 0; --l) {
            const bool on = s.live && tg + l < te;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (on) {
                    float ff, nf;
                    gate_unpack(f[l][i], ff, nf);
                    const float a = mc[l] * ff;
                    Q[i] = cut_mul(a, to_f32(dc[l][i]) + Q[i]);
                    P[i] *= a;
                }
            }
        }
        if (q > 0) fetch(tg - S::SC);
        if (!AGG) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                start[i] = !s.live ? 0.f : p.saved ? p.saved[(long)(t0 / SCAN_SAVE) * C + s.c + i] : p.h0 ? p.h0[s.c + i] : 0.f;
            s.template exchange<false>(A, B, start, in, sm[1][par]);
        } else {
            float P2[V], Z[V], dummy[V];
#pragma unroll
            for (int i = 0; i < V; ++i) P2[i] = P[i], Z[i] = 0.f;
            s.template exchange<true>(P2, Z, wa, dummy, sm[1][par]);
        }
        s.template exchange<true>(P, Q, carry, ein, sm[0][par]);
        par ^= 1;
        if (!AGG) {
            float hp[SCAN_L][V];                             // m_t h_{t-1}
#pragma unroll
            for (int l = 0; l < SCAN_L; ++l) {
                const bool on = s.live && tg + l < te;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float ff, nf;
                    gate_unpack(f[l][i], ff, nf);
                    hp[l][i] = cut_mul(mc[l], in[i]);
                    if (on) in[i] = cut_mul(ff, hp[l][i]) + nf * to_f32(vc[l][i]);
                }
            }
#pragma unroll
            for (int l = SCAN_L - 1; l >= 0; --l) {
                const int t = tg + l;
                const bool on = s.live && t < te;
                vv og, ov;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float ff, nf;
                    gate_unpack(f[l][i], ff, nf);
                    const float D = to_f32(dc[l][i]) + ein[i];
                    og[i] = from_f32<T>(D * (hp[l][i] - to_f32(vc[l][i])) * ff * nf);
                    ov[i] = from_f32<T>(D * nf);
                    if (on) ein[i] = cut_mul(mc[l] * ff, D);
                }
                if (on) {
                    *reinterpret_cast<vv*>((T*)p.dgate + t * p.dgt + s.n * p.dgn + s.j) = og;
                    *reinterpret_cast<vv*>((T*)p.dvalue + t * p.dvt + s.n * p.dvn + s.j) = ov;
                }
            }
        }
    }
    if (s.group == 0 && s.live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (AGG) {
                p.agg[(2L * blk) * C + s.c + i] = wa[i];
                p.agg[(2L * blk + 1) * C + s.c + i] = carry[i];
            } else if (tb == 0 && p.dh0) {
                p.dh0[s.c + i] = carry[i];
            }
        }
    }
}

// --------------------------------------------------------------------------------------------------------- one token
template <class T, int V>
__global__ __launch_bounds__(256) void scan_step_kernel(const void* gate, long gn, const void* value, long vn, float* state, const float* masks,
                                                        void* out, long on, int N, int H) {
    typedef vec_t<T, V> vv;
    typedef vec_t<float, V> fv;
    const long c = ((long)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= (long)N * H) return;
    const int n = (int)(c / H), j = (int)(c - (long)n * H);
    const vv g = *reinterpret_cast<const vv*>((const T*)gate + n * gn + j), v = *reinterpret_cast<const vv*>((const T*)value + n * vn + j);
    fv h = *reinterpret_cast<fv*>(state + c);
    const float m = masks ? masks[n] : 1.f;
    vv o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float f, nf;
        gate_of(to_f32(g[i]), f, nf);
        h[i] = f * cut_mul(m, h[i]) + nf * to_f32(v[i]);
        o[i] = from_f32<T>(h[i]);
    }
    *reinterpret_cast<fv*>(state + c) = h;
    *reinterpret_cast<vv*>((T*)out + n * on + j) = o;
}
// dst = src or 0: the states of a sequence of no steps
__global__ __launch_bounds__(256) void scan_copy_kernel(const float* src, float* dst, long n) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : 0.f;
}

// --------------------------------------------------------------------------------------------------------- host side
struct ScanPlan { int v, lc, nw, sc, ct, blocks, block_steps; };

static ScanPlan scan_plan(long T, long N, long H, int e, bool wide) {
    ScanPlan p;
    p.v = wide ? 8 / e : 1;
    p.lc = wide ? 16 : 64;
    const int gw = 64 / p.lc;
    p.nw = wide ? (T <= 32 ? 1 : T <= 128 ? 4 : 8) : (T <= 32 ? 4 : 8);
    p.sc = p.nw * gw * SCAN_L;
    p.ct = p.lc * p.v;
    p.blocks = 1;
    const long tiles = cdiv(N * H, p.ct), chunks = cdiv(T, p.sc);
    long per = chunks;
    if (tiles < 96 && chunks > 1) per = cdiv(chunks, min(chunks, (long)cdiv(512, tiles)));
    if (per < 1) per = 1;
    p.block_steps = (int)(per * p.sc);
    p.blocks = chunks ? cdiv(chunks, per) : 1;
    return p;
}
static bool vec8(const void* p, long st, long sn, int e) { return ((uintptr_t)p & 7) == 0 && st * e % 8 == 0 && sn * e % 8 == 0; }

static int scan_check(long T, long N, long H, int dtype) {
    ACKTR_ARG(dtype_ok(dtype), "gated_scan: unknown dtype code %d", dtype);
    ACKTR_ARG(T >= 0 && N >= 0 && H >= 1, "gated_scan: sizes must be T >= 0, N >= 0, H >= 1 (got T %ld, N %ld, H %ld)", T, N, H);
    ACKTR_ARG(T < (1L << 30) && N * H < (1L << 30), "gated_scan: T and N * H must be below 2^30 (got T %ld, N %ld, H %ld)", T, N, H);
    return 0;
}

template <class T, bool BWD, bool AGG, int V, int LC>
static void scan_launch_nw(const ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    const dim3 grid(cdiv((long)a.N * a.H, p.ct), p.blocks);
    auto go = [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        if constexpr (BWD) scan_bwd_kernel<T, V, LC, NW, AGG><<<grid, NW * 64, 0, s>>>(a);
        else scan_fwd_kernel<T, V, LC, NW, AGG><<<grid, NW * 64, 0, s>>>(a);
    };
    if (p.nw == 1) go(std::integral_constant<int, 1>{});
    else if (p.nw == 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
}
template <class T, bool BWD>
static int scan_run(ScanArgs a, const ScanPlan& p, hipStream_t s) {
    a.blocks = p.blocks;
    a.block_steps = p.block_steps;
    constexpr int W = 8 / sizeof(T);
    if (p.blocks > 1) {
        if (p.v > 1) scan_launch_nw<T, BWD, true, W, 16>(a, p, s);
        else scan_launch_nw<T, BWD, true, 1, 64>(a, p, s);
        ACKTR_LAUNCH_CHECK();
    }
    if (p.v > 1) scan_launch_nw<T, BWD, false, W, 16>(a, p, s);
    else scan_launch_nw<T, BWD, false, 1, 64>(a, p, s);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

}  // namespace acktr

using namespace acktr;

extern "C" int acktr_gated_scan_save_interval(void) { return SCAN_SAVE; }

extern "C" long acktr_gated_scan_workspace_bytes(long T, long N, long H, int dtype) {
    if (scan_check(T, N, H, dtype)) return -1;
    long most = 0;
    for (int wide = 0; wide < 2; ++wide) {
        const ScanPlan p = scan_plan(T, N, H, (int)elem_bytes(dtype), wide != 0);
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
    const bool wide = H % (8 / e) == 0 && vec8(gate, gt, gn, e) && vec8(value, vt, vn, e) && vec8(out, ot, on, e);
    ACKTR_ARG(workspace_bytes >= acktr_gated_scan_workspace_bytes(T, N, H, dtype), "gated_scan_fwd: workspace of %ld bytes is too small",
              workspace_bytes);
    const ScanPlan p = scan_plan(T, N, H, e, wide);
    ScanArgs a{};
    a.gate = gate, a.gt = gt, a.gn = gn, a.value = value, a.vt = vt, a.vn = vn, a.h0 = h0, a.masks = masks;
    a.out = out, a.ot = ot, a.on = on, a.last = last, a.saved = saved, a.agg = (float*)workspace;
    a.T = (int)T, a.N = (int)N, a.H = (int)H;
    return with_dtype(dtype, [&](auto t) -> int { return scan_run<decltype(t), false>(a, p, s); });
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
    const bool wide = H % (8 / e) == 0 && vec8(dout, dt, dn, e) && vec8(gate, gt, gn, e) && vec8(value, vt, vn, e) &&
                      vec8(dgate, dgt, dgn, e) && vec8(dvalue, dvt, dvn, e);
    ACKTR_ARG(workspace_bytes >= acktr_gated_scan_workspace_bytes(T, N, H, dtype), "gated_scan_bwd: workspace of %ld bytes is too small",
              workspace_bytes);
    const ScanPlan p = scan_plan(T, N, H, e, wide);
    ACKTR_ARG(saved || T <= SCAN_SAVE, "gated_scan_bwd: %ld steps need the states that the forward pass saves every %d steps", T, SCAN_SAVE);
    ScanArgs a{};
    a.dout = dout, a.dt = dt, a.dn = dn, a.gate = gate, a.gt = gt, a.gn = gn, a.value = value, a.vt = vt, a.vn = vn;
    a.h0 = h0, a.masks = masks, a.saved = const_cast<float*>(saved), a.dlast = dlast;
    a.dgate = dgate, a.dgt = dgt, a.dgn = dgn, a.dvalue = dvalue, a.dvt = dvt, a.dvn = dvn, a.dh0 = dh0, a.agg = (float*)workspace;
    a.T = (int)T, a.N = (int)N, a.H = (int)H;
    return with_dtype(dtype, [&](auto t) -> int { return scan_run<decltype(t), true>(a, p, s); });
}

extern "C" int acktr_gated_scan_step(const void* gate, long gn, const void* value, long vn, float* state, const float* masks, void* out, long on,
                                     long N, long H, int dtype, void* stream) {
    if (int rc = scan_check(1, N, H, dtype)) return rc;
    if (N * H == 0) return 0;
    ACKTR_ARG(gate && value && state && out, "gated_scan_step: gate, value, state and out are required");
    hipStream_t s = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto t) -> int {
        typedef decltype(t) T;
        constexpr int W = 8 / sizeof(T);
        const bool wide = H % W == 0 && vec8(gate, 0, gn, sizeof(T)) && vec8(value, 0, vn, sizeof(T)) && vec8(out, 0, on, sizeof(T)) &&
                          ((uintptr_t)state & 15) == 0;
        if (wide) scan_step_kernel<T, W><<<cdiv(N * H, 256 * W), 256, 0, s>>>(gate, gn, value, vn, state, masks, out, on, (int)N, (int)H);
        else scan_step_kernel<T, 1><<<cdiv(N * H, 256), 256, 0, s>>>(gate, gn, value, vn, state, masks, out, on, (int)N, (int)H);
        ACKTR_LAUNCH_CHECK();
        return 0;
    });
}
