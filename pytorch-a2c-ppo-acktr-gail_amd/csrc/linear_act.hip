// y = act(x w^T + b) + r with bf16, fp16 or fp32 operands and fp32 sums, and its backward pass:
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = sum over rows of dz
// Three products over the same tile kernel (tile_gemm.hpp), which reads each operand as it lies: forward k | k contiguous, input
// gradient k | rows, weight gradient rows | rows.
#include <initializer_list>
#include <type_traits>

#include "act_terms.hpp"
#include "linear_act.hpp"

namespace acktr {

// V values of a row, `left` of which it still has; 0 behind them
template <class T, int V>
__device__ __forceinline__ vec_t<T, V> row_piece(const T* p, int left) {
    if (left >= V) return *reinterpret_cast<const uvec_t<T, V>*>(p);
    vec_t<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < left ? p[j] : (T)0.f;
    return v;
}

// dst[r][c] = src[r][c] for c < cols, 0 up to ldd: a copy whose rows start at 16-byte boundaries, for operands that do not
// (an odd width, a slice of a wider row).  It costs one pass over the operand; reading such rows element by element in the
// product would cost a fetch per element of every tile that uses it.  Up to three operands a launch (4.2 us for 1011 x 777 and 390 x 777
// fp16 values together).
struct PackJob { const void* src; long lds; int rows, cols; void* dst; int ldd; };
struct PackJobs { PackJob job[3]; };
constexpr int PACK_U = 4;                    // 16-byte pieces a thread has in flight
template <class T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const PackJobs jobs) {
    const PackJob p = jobs.job[blockIdx.y];
    constexpr int V = 16 / sizeof(T);
    typedef vec_t<T, V> vv;
    const int groups = p.ldd / V;
    const long total = (long)p.rows * groups;
    for (long i0 = (long)blockIdx.x * (256 * PACK_U) + threadIdx.x; i0 < total; i0 += (long)gridDim.x * (256 * PACK_U)) {
        vv o[PACK_U];
#pragma unroll
        for (int u = 0; u < PACK_U; ++u) {
            const long i = min(i0 + u * 256, total - 1);
            const long r = total < (1L << 31) ? (long)((unsigned)i / (unsigned)groups) : i / groups;
            const int c = (int)(i - r * groups) * V;
            o[u] = row_piece<T, V>((const T*)p.src + r * p.lds + c, p.cols - c);
        }
#pragma unroll
        for (int u = 0; u < PACK_U; ++u) {
            const long i = i0 + u * 256;               // (rows of ldd values lie one behind the other)
            if (i < total) *reinterpret_cast<vv*>((T*)p.dst + i * V) = o[u];
        }
    }
}

// dz = dy slope (ACT; dz null: not wanted; without ACT dz is dy itself) and, per block of rows, the column sums of dz.
// A thread holds one group of V columns and walks the block's rows in steps of 8; sums[block][N] (nullable).  Bound by memory: bf16,
// 16384 x 2048 in 40 us (5.0 TB/s).  dz is written once, in rows that both products read, rather than formed in each of them.
// Zeros are written up to the end of dz's aligned row, which the products read.  V: 16 bytes, or 1 where a small matrix has rows that
// do not fill or start at 16 bytes (fp16, with 8 and 1: 1011 x 390 4.7 and 3.8 us, 4011 x 390 8.2 and 6.2, 8011 x 390 8.2 and 10.6,
// 8011 x 1390 15.4 and 24.9).
template <class T, bool ACT, int V>
__global__ __launch_bounds__(256) void act_bwd_kernel(const T* __restrict__ dy, long lddy, const void* __restrict__ pre, long ldp,
                                                      T* __restrict__ dz, long lddz, int M, int N, int rows_per, float* __restrict__ sums) {
    typedef typename SlopeOf<T>::type ST;
    const int cg = threadIdx.x & 31, rg = threadIdx.x >> 5;
    const int n = (blockIdx.x * 32 + cg) * V, left = N - n;
    const int r0 = blockIdx.y * rows_per, r1 = r0 + min(M - r0, rows_per);          // (r0 + rows_per may pass 2^31)
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.f;
    if (n < (ACT && dz ? (int)lddz : N)) {
#pragma unroll 4
        for (int r = r0 + rg; r < r1; r += 8) {
            const vec_t<T, V> g = row_piece<T, V>(dy + r * lddy + n, left);
            vec_t<ST, V> z;
            vec_t<T, V> o;
            if (ACT) z = row_piece<ST, V>((const ST*)pre + r * ldp + n, left);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float d = to_f32(g[i]);
                if (ACT) d *= get_slope(z[i]);
                s[i] += d;
                o[i] = from_f32<T>(d);
            }
            if (ACT && dz) *reinterpret_cast<vec_t<T, V>*>(dz + r * lddz + n) = o;
        }
    }
    if (!sums) return;
    __shared__ float part[8][32 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) part[rg][cg * V + i] = s[i];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += 256) {
        const int col = blockIdx.x * 32 * V + c;
        if (col >= N) continue;
        float t = 0.f;
        for (int j = 0; j < 8; ++j) t += part[j][c];
        sums[(long)blockIdx.y * N + col] = t;
    }
}
// packs the jobs that have rows
template <class T>
static int pack(std::initializer_list<PackJob> list, hipStream_t s) {
    PackJobs jobs{};
    int n = 0;
    long most = 0;
    for (const PackJob& j : list)
        if (j.rows > 0) {
            jobs.job[n++] = j;
            most = max(most, (long)j.rows * (j.ldd * (long)sizeof(T) / 16));
        }
    if (n == 0) return 0;
    pack_rows_kernel<T><<<dim3(min(cdiv(most, 256 * PACK_U), 4096), n), 256, 0, s>>>(jobs);
    ACKTR_LAUNCH_CHECK();
    return 0;
}

static int check_dims(long M, long K, long N, int dtype, int act) {
    ACKTR_ARG(dtype_ok(dtype), "linear_act: unknown dtype code %d", dtype);
    ACKTR_ARG(act >= 0 && act <= ACKTR_ACT_GELU, "linear_act: unknown activation code %d", act);
    ACKTR_ARG(M >= 0 && N >= 1 && K >= 1, "linear_act: sizes must be M >= 0, N >= 1, K >= 1 (got M %ld, N %ld, K %ld)", M, N, K);
    ACKTR_ARG(M < (1L << 31) - 256 && N <= (1 << 20) && K <= (1 << 20), "linear_act: M below 2^31 - 256, N and K at most 2^20 (got M %ld, N %ld, K %ld)", M, N, K);
    ACKTR_ARG((long)cdiv(M, 64) * cdiv(N, 64) < (1L << 31) - 8, "linear_act: too many tiles (M %ld, N %ld)", M, N);
    return 0;
}
static int check_ld(const char* what, long ld, long cols) {
    ACKTR_ARG(ld >= cols && ld < (1 << 21), "linear_act: row stride of %s must be at least its %ld columns and below 2^21 (got %ld)", what, cols, ld);
    return 0;
}

static constexpr long ROWS_WIDE = 1 << 21;    // values from which unaligned rows are taken 16 bytes at a time
static constexpr int per16(int e) { return 16 / e; }

}  // namespace acktr

using namespace acktr;

// Where the parts of a workspace lie (byte offsets; a part that is not needed has no bytes).
struct FwdSpace { bool px, pw; long x, w, slabs, bytes; };
static FwdSpace fwd_space(const void* x, long ldx, const void* w, long ldw, long M, long N, long K, int e) {
    FwdSpace f;
    const bool whole = K % per16(e) == 0;
    const long kp = up(K, per16(e));
    f.px = !whole || !rows16(x, ldx, e);
    f.pw = !whole || !rows16(w, ldw, e);
    f.x = 0;
    f.w = f.px ? up(M * kp * e, 256) : 0;
    f.slabs = f.w + (f.pw ? up(N * kp * e, 256) : 0);
    f.bytes = f.slabs + slab_bytes(M, N, plan_of(M, N, kp, e).slices);
    return f;
}
struct BwdSpace { bool pdy, px, pw; long dz, x, w, sums, slabs, bytes; };
static BwdSpace bwd_space(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* pre, long ldp, bool dx, bool dw,
                          bool db, long M, long N, long K, int e, int act) {
    BwdSpace f;
    const int V = per16(e);
    const long np = up(N, V), kp = up(K, V);
    f.pdy = act == ACKTR_ACT_NONE && (dx || dw) && (N % V != 0 || !rows16(dy, lddy, e));
    f.px = dw && (K % V != 0 || !rows16(x, ldx, e));
    f.pw = dx && (K % V != 0 || !rows16(w, ldw, e));
    f.dz = 0;
    f.x = act != ACKTR_ACT_NONE || f.pdy ? up(M * np * e, 256) : 0;
    f.w = f.x + (f.px ? up(M * kp * e, 256) : 0);
    f.sums = f.w + (f.pw ? up(N * kp * e, 256) : 0);
    f.slabs = f.sums + (db ? up(4L * SUM_BLOCKS * N, 256) : 0);
    long most = dx ? slab_bytes(M, K, plan_of(M, K, N, e).slices) : 0;
    if (dw) most = max(most, slab_bytes(N, K, plan_of(N, K, M, e).slices));
    if (dx && dw) {
        LinArgs pw{}, px{};
        pw.M = (int)N, pw.N = (int)K, pw.K = (int)M, px.M = (int)M, px.N = (int)K, px.K = (int)N;
        most = max(most, slab_bytes(N, K, pair_plan_of(pw, px, e).slices));
    }
    f.bytes = f.slabs + most;
    return f;
}

extern "C" long acktr_linear_act_fwd_workspace_bytes(const void* x, long ldx, const void* w, long ldw, long M, long N, long K, int dtype) {
    if (check_dims(M, K, N, dtype, 0)) return -1;
    return fwd_space(x, ldx, w, ldw, M, N, K, (int)elem_bytes(dtype)).bytes;
}

extern "C" int acktr_linear_act_fwd(const void* x, long ldx, const void* w, long ldw, const void* bias, const void* residual, long ldr,
                                    void* y, long ldy, void* pre, long ldp, long M, long N, long K, int dtype, int act,
                                    void* workspace, long workspace_bytes, void* stream) {
    if (int rc = check_dims(M, K, N, dtype, act)) return rc;
    if (check_ld("x", ldx, K) || check_ld("w", ldw, K) || check_ld("y", ldy, N)) return -1;
    if ((residual && check_ld("residual", ldr, N)) || (pre && check_ld("pre", ldp, N))) return -1;
    ACKTR_ARG(M == 0 || (x && w && y), "linear_act_fwd: x, w and y are required");
    if (M == 0) return 0;
    const FwdSpace sp = fwd_space(x, ldx, w, ldw, M, N, K, (int)elem_bytes(dtype));
    ACKTR_ARG(workspace_bytes >= sp.bytes && ((uintptr_t)workspace & 15) == 0 && (workspace || !sp.bytes),
              "linear_act_fwd: workspace of %ld bytes, %ld with 16-byte alignment are needed", workspace_bytes, sp.bytes);
    hipStream_t s = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto t) -> int {
        typedef decltype(t) T;
        constexpr int e = sizeof(T);
        LinArgs p{};
        p.a = x, p.lda = ldx, p.b = w, p.ldb = ldw;
        p.M = (int)M, p.N = (int)N, p.K = (int)K;
        p.y = y, p.ldy = ldy, p.bias = bias, p.res = residual, p.ldr = ldr, p.pre = pre, p.ldp = ldp, p.act = act;
        char* ws = (char*)workspace;
        const int kp = (int)up(K, per16(e));
        if (int rc = pack<T>({{x, ldx, sp.px ? (int)M : 0, (int)K, ws + sp.x, kp}, {w, ldw, sp.pw ? (int)N : 0, (int)K, ws + sp.w, kp}}, s)) return rc;
        if (sp.px) p.a = ws + sp.x, p.lda = kp;
        if (sp.pw) p.b = ws + sp.w, p.ldb = kp;
        p.K = kp;
        return linear_product<T>(LIN_FORWARD, p, (float*)(ws + sp.slabs), s);
    });
}

extern "C" long acktr_linear_act_bwd_workspace_bytes(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw,
                                                     const void* pre, long ldp, int dx, int dw, int db, long M, long N, long K, int dtype,
                                                     int act) {
    if (check_dims(M, K, N, dtype, act)) return -1;
    return bwd_space(dy, lddy, x, ldx, w, ldw, pre, ldp, dx != 0, dw != 0, db != 0, M, N, K, (int)elem_bytes(dtype), act).bytes;
}

extern "C" int acktr_linear_act_bwd(const void* dy, long lddy, const void* x, long ldx, const void* w, long ldw, const void* pre, long ldp,
                                    const void* dx_add, long ldxa, void* dx, long lddx, void* dw, void* db, long M, long N, long K, int dtype, int act, void* workspace,
                                    long workspace_bytes, void* stream) {
    if (int rc = check_dims(M, K, N, dtype, act)) return rc;
    if (check_ld("dy", lddy, N)) return -1;
    ACKTR_ARG(!dx || w, "linear_act_bwd: dx needs w");
    ACKTR_ARG(!dw || x || M == 0, "linear_act_bwd: dw needs x");
    if ((dx && (check_ld("w", ldw, K) || check_ld("dx", lddx, K) || (dx_add && check_ld("dx_add", ldxa, K)))) || (dw && check_ld("x", ldx, K))) return -1;
    ACKTR_ARG(act == ACKTR_ACT_NONE || pre || M == 0, "linear_act_bwd: an activation's gradient needs what the forward pass left in `pre`");
    if (act != ACKTR_ACT_NONE && check_ld("pre", ldp, N)) return -1;
    ACKTR_ARG(M == 0 || dy, "linear_act_bwd: dy is required");
    const BwdSpace sp = bwd_space(dy, lddy, x, ldx, w, ldw, pre, ldp, dx, dw, db, M, N, K, (int)elem_bytes(dtype), act);
    ACKTR_ARG(workspace_bytes >= sp.bytes && ((uintptr_t)workspace & 15) == 0 && (workspace || !sp.bytes),
              "linear_act_bwd: workspace of %ld bytes, %ld with 16-byte alignment are needed", workspace_bytes, sp.bytes);
    hipStream_t s = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto t) -> int {
        typedef decltype(t) T;
        constexpr int e = sizeof(T), V = per16(e);
        const int np = (int)up(N, V), kp = (int)up(K, V);
        char* ws = (char*)workspace;
        T *dz_ws = (T*)(ws + sp.dz), *x_ws = (T*)(ws + sp.x), *w_ws = (T*)(ws + sp.w);
        float *sums = (float*)(ws + sp.sums), *slabs = (float*)(ws + sp.slabs);

        LinArgs px{}, pw{};
        int blocks = 0;
        // dz, in aligned rows, which the two products read, and the column sums
        const void* dz = dy;
        long lddz = lddy;
        const bool write = act != ACKTR_ACT_NONE && M > 0;
        if (write) dz = dz_ws, lddz = np;
        if (M > 0 && (write || db)) {
            const bool wide = (long)M * N >= ROWS_WIDE || (N % V == 0 && rows16(dy, lddy, e) && (!write || rows16(pre, ldp, e)));
            const int gx = cdiv(write ? np : N, wide ? 32 * V : 32);
            const int want = max(1, min(SUM_BLOCKS, 2048 / gx));
            const int rows_per = (int)up(max(16, cdiv(M, want)), 8), gy = cdiv(M, rows_per);
            const auto kern = write ? (wide ? act_bwd_kernel<T, true, V> : act_bwd_kernel<T, true, 1>)
                                    : (wide ? act_bwd_kernel<T, false, V> : act_bwd_kernel<T, false, 1>);
            kern<<<dim3(gx, gy), 256, 0, s>>>((const T*)dy, lddy, pre, ldp, dz_ws, np, (int)M, (int)N, rows_per, db ? sums : nullptr);
            ACKTR_LAUNCH_CHECK();
            blocks = gy;
        }
        pw.M = (int)N, pw.N = (int)K, pw.K = (int)M;
        pw.sums = sums, pw.blocks = blocks, pw.db = db;
        if (db && !dw)                                       // no weight gradient's launch for it to ride in
            if (int rc = linear_bias<T>(pw, s)) return rc;
        if (sp.pdy) dz = dz_ws, lddz = np;                   // no activation: dy itself, in aligned rows
        if (int rc = pack<T>({{dy, lddy, sp.pdy ? (int)M : 0, (int)N, dz_ws, np}, {x, ldx, sp.px ? (int)M : 0, (int)K, x_ws, kp}, {w, ldw, sp.pw && M > 0 ? (int)N : 0, (int)K, w_ws, kp}}, s)) return rc;
        px.a = dz, px.lda = lddz, px.b = sp.pw ? w_ws : w, px.ldb = sp.pw ? kp : ldw;      // dx[M, K] = dz[M, N] w[N, K]: sum over N
        px.M = (int)M, px.N = (int)K, px.K = (int)N;
        px.y = dx, px.ldy = lddx, px.res = dx_add, px.ldr = ldxa;
        pw.a = dz, pw.lda = lddz, pw.b = sp.px ? x_ws : x, pw.ldb = sp.px ? kp : ldx;      // dw[N, K] = dz^T x: sum over M
        pw.y = dw, pw.ldy = K;
        if (dx && dw && M > 0) return linear_gradients<T>(pw, px, slabs, s);
        if (dx && M > 0) return linear_product<T>(LIN_DX, px, slabs, s);
        if (dw) return linear_product<T>(LIN_DW, pw, slabs, s);
        return 0;
    });
}
