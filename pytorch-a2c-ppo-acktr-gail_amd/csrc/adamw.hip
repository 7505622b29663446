// AdamW over many tensors:
//   g <- g min(1, c / (|g| + 1e-6))            (|g|: 2-norm over all tensors; only with a clip)
//   m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// One launch walks all tensors: their elements are cut into chunks of 2048, a table gives each workgroup its chunk.  The step counter
// and the hyperparameters live in device memory, so a captured launch sequence replays with the right bias corrections.
//
// Moments are fp32 or 8-bit.  In 8 bits, 256 elements share a power of two as scale (just above the largest magnitude, so dividing by
// it is exact) and a value is sign + 4 exponent + 3 mantissa bits (m) or 5 exponent + 3 mantissa bits (v; a running mean of squares
// spans twice the octaves).  Rounding is stochastic: with b2 = 0.999 a step changes v by at most 0.1 % of its distance to g^2, far
// below half a code's spacing of 6 %, so rounding to nearest would freeze v; rounding up with the probability of the cut-off bits
// keeps its expectation.  The random bits are a function of (seed, step, element), so runs repeat.  A positive v never becomes 0 (but in a
// block that lies below 2^-126): m may survive where v would not, and m / eps is no step.
#include "half_types.hpp"

#pragma clang fp contract(off)

namespace acktr {

constexpr int AW_THREADS = 256, AW_CHUNK = 2048, AW_BLOCK = 256, AW_PARTIALS = 1024;
// up to this many chunks, the update's workgroups sum the norm's partial sums themselves
constexpr int AW_SMALL = 1024;

// what a step's update needs besides the elements
struct AwScalars { float coef, keep, step_size, inv_bc2, b1, nb1, b2, nb2, eps; unsigned key; };

// device copy of the optimiser's state that is not per element (acktr_adamw_state_bytes)
struct AwState {
    double lr, b1, b2, eps, wd, max_norm;      // written by the host when they change
    long long step, seed;
    AwScalars now;                             // of the present step
    unsigned done;                             // finished workgroups of the norm launch; back at 0 when it ends
    double partial[AW_PARTIALS];
};

// 32-bit mixing function: multiply and xor-shift with the low-bias constants that C. Wellons published (2018)
__device__ __forceinline__ unsigned mix32(unsigned x) {
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

// min(1, c / (|g| + 1e-6)); a norm that is not a number stays one.  max_norm 0: no clip, whatever the norm (a captured step goes through
// here with and without one)
__device__ __forceinline__ float aw_coef(double sumsq, double max_norm) {
    if (max_norm == 0.0) return 1.f;
    const double c = max_norm / (sqrt(sumsq) + 1e-6);
    return (float)(c > 1.0 ? 1.0 : c);
}
// bc1 = 1 - b1^t, bc2 = 1 - b2^t
__device__ __forceinline__ AwScalars aw_scalars(const AwState* st, long long t, float coef, double bc1, double bc2) {
    AwScalars a;
    a.coef = coef;
    a.keep = (float)(1.0 - st->lr * st->wd);
    a.step_size = (float)(st->lr / bc1);
    a.inv_bc2 = (float)(1.0 / sqrt(bc2));
    a.b1 = (float)st->b1;
    a.nb1 = (float)(1.0 - st->b1);
    a.b2 = (float)st->b2;
    a.nb2 = (float)(1.0 - st->b2);
    a.eps = (float)st->eps;
    a.key = mix32((unsigned)st->seed + (unsigned)t * 0x9e3779b9u);
    return a;
}
// counts the step and writes its scalars; one lane
__device__ __forceinline__ void aw_begin(AwState* st, float coef) {
    const long long t = st->step + 1;
    st->step = t;
    st->now = aw_scalars(st, t, coef, 1.0 - pow(st->b1, (double)t), 1.0 - pow(st->b2, (double)t));
}

// Pointers that come out of the table are to device memory; said so, they are not accessed through the slower generic path.
#define ACKTR_GLB __attribute__((address_space(1)))

// 4 consecutive values from element i of a tensor of n; nothing behind the end is touched
template <class T>
__device__ __forceinline__ f32v4 ld4_as(const void* p, long i, long n, bool vec) {
    f32v4 r = {0.f, 0.f, 0.f, 0.f};
    if (vec && i + 4 <= n) {
        const vec_t<T, 4> v = *reinterpret_cast<const ACKTR_GLB vec_t<T, 4>*>((const ACKTR_GLB T*)p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = to_f32(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) r[k] = to_f32(((const ACKTR_GLB T*)p)[i + k]);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void st4_as(void* p, long i, long n, bool vec, const f32v4& v) {
    if (vec && i + 4 <= n) {
        vec_t<T, 4> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = from_f32<T>(v[k]);
        *reinterpret_cast<ACKTR_GLB vec_t<T, 4>*>((ACKTR_GLB T*)p + i) = o;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) ((ACKTR_GLB T*)p)[i + k] = from_f32<T>(v[k]);
    }
}
__device__ __forceinline__ f32v4 ld4(const void* p, int dt, long i, long n, bool vec) {
    return dt == ACKTR_F32 ? ld4_as<float>(p, i, n, vec) : dt == ACKTR_BF16 ? ld4_as<__bf16>(p, i, n, vec) : ld4_as<_Float16>(p, i, n, vec);
}
__device__ __forceinline__ void st4(void* p, int dt, long i, long n, bool vec, const f32v4& v) {
    if (dt == ACKTR_F32) st4_as<float>(p, i, n, vec, v);
    else if (dt == ACKTR_BF16) st4_as<__bf16>(p, i, n, vec, v);
    else st4_as<_Float16>(p, i, n, vec, v);
}

// Sum of squares of all gradients, in fp64.  SMALL: partial sums only (and the step is counted): the update's workgroups add them up.
// Otherwise the last workgroup to finish adds them, in the same fixed order, and writes the step's scalars: thousands of workgroups
// would read too much, while for a few hundred the chain of atomics costs more than the rest of the launch (13 us against 5 for the
// 867 thousand parameters of the NatureCNN policy).  Bound by reading: 201 million fp32 gradients in 232 us (3.5 TB/s).  Without a
// clip norm at the time of the launch nothing is read.
template <bool SMALL>
__global__ __launch_bounds__(AW_THREADS) void adamw_norm_kernel(AwState* st, const acktr_adamw_tensor* tensors, const int2* chunks, int nchunks) {
    __shared__ double sm[16];
    __shared__ bool last;
    double s = 0.0;
    constexpr int IT = AW_CHUNK / AW_THREADS / 4;
    if (SMALL && blockIdx.x == 0 && threadIdx.x == 0) st->step = st->step + 1;
    // two chunks at a time, and the table entries of the next two travel with their values
    const int step = gridDim.x;
    int q = st->max_norm == 0.0 ? nchunks : blockIdx.x;
    const int none = nchunks - 1;
    int2 c0 = chunks[min(q, none)], c1 = chunks[min(q + step, none)];
    acktr_adamw_tensor t0 = tensors[c0.x], t1 = tensors[c1.x];
    while (q < nchunks) {
        f32v4 g[2 * IT];
        const bool two = q + step < nchunks;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            g[k] = ld4(t0.g, t0.g_dtype, (long)c0.y * AW_CHUNK + (k * AW_THREADS + threadIdx.x) * 4, t0.n, t0.vec & 2);
            g[IT + k] = two ? ld4(t1.g, t1.g_dtype, (long)c1.y * AW_CHUNK + (k * AW_THREADS + threadIdx.x) * 4, t1.n, t1.vec & 2) : f32v4{0.f, 0.f, 0.f, 0.f};
        }
        q += 2 * step;
        c0 = chunks[min(q, none)], c1 = chunks[min(q + step, none)];
        t0 = tensors[c0.x], t1 = tensors[c1.x];
#pragma unroll
        for (int k = 0; k < 2 * IT; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) s += (double)g[k][j] * (double)g[k][j];
    }
    s = block_sum(s, sm);
    if (SMALL) {
        if (threadIdx.x == 0) st->partial[blockIdx.x] = s;
        return;
    }
    if (threadIdx.x == 0) {
        __hip_atomic_store(&st->partial[blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(&st->done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    double v = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += AW_THREADS) v += __hip_atomic_load(&st->partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    v = block_sum(v, sm);
    if (threadIdx.x == 0) {
        aw_begin(st, aw_coef(v, st->max_norm));
        st->done = 0;
    }
}
__global__ void adamw_begin_kernel(AwState* st) { aw_begin(st, 1.f); }

// magnitude of a code of `TOP` as largest exponent field, for a scale of 1
template <int TOP>
__device__ __forceinline__ float code_value(unsigned c) {
    const float x = __uint_as_float((c << 20) + ((127u - TOP) << 23));
    return c < 8 ? 2.f * x - __uint_as_float((128u - TOP) << 23) : x;
}
// code of 0 <= y <= 1, rounded up with probability (cut-off bits) / 2^20; below the smallest exponent the codes are evenly spaced
template <int TOP>
__device__ __forceinline__ unsigned code_of(float y, unsigned rnd) {
    const float low = __uint_as_float((128u - TOP) << 23);
    const bool small = y < low;
    const unsigned b = (__float_as_uint(small ? y + low : y) + rnd) >> 20;
    return b - ((127u - TOP) << 3) - (small ? 8u : 0u);
}
// power-of-two scale above a block's largest magnitude and its inverse; 0 for a block of zeros (or below 2^-126), a NaN scale marks
// a block with values that are not finite (or 2^126 and more)
__device__ __forceinline__ void block_scale(float most, bool bad, float& scale, float& inv) {
    const unsigned e = __float_as_uint(most) >> 23;
    const bool ok = e > 0 && e < 253;
    scale = bad || e >= 253 ? __uint_as_float(0x7fc00000u) : ok ? __uint_as_float((e + 1) << 23) : 0.f;
    inv = ok && !bad ? __uint_as_float((253 - e) << 23) : 0.f;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// SMALL: the step's scalars are formed here from `parts` partial sums, beside the loads of the elements.  Bound by memory, 201 million
// parameters: 32 bits with bf16 parameters' gradients and copies 1066 us (5.3 TB/s), 8 bits 590 us (5.5 TB/s).  A thread takes 8 elements
// of a chunk of 2048, all loads before the first use.
template <int BITS, bool SMALL>
__global__ __launch_bounds__(AW_THREADS) void adamw_update_kernel(const AwState* __restrict__ st, const acktr_adamw_tensor* __restrict__ tensors,
                                                                  const int2* __restrict__ chunks, void* mom1, void* mom2, float* scales,
                                                                  int parts) {
    const int2 ck = chunks[blockIdx.x];
    const acktr_adamw_tensor t = tensors[ck.x];
    const long base = (long)ck.y * AW_CHUNK;
    constexpr int IT = AW_CHUNK / AW_THREADS / 4;
    f32v4 pv[IT], gv[IT];
    f32v4 mv[IT], vv[IT];
    unsigned mc[IT], vc[IT];
    float ms[IT], vs[IT];
    // all loads of the thread first
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const long i = base + (k * AW_THREADS + threadIdx.x) * 4, si = t.state + i;      // a wave covers one block of 256 elements
        if (base + (k * AW_THREADS + (threadIdx.x & ~63)) * 4 >= t.n) break;
        pv[k] = ld4(t.p, t.p_dtype, i, t.n, t.vec & 1);
        gv[k] = ld4(t.g, t.g_dtype, i, t.n, t.vec & 2);
        if (BITS == 32) {
            mv[k] = *reinterpret_cast<const f32v4*>((const float*)mom1 + si);
            vv[k] = *reinterpret_cast<const f32v4*>((const float*)mom2 + si);
        } else {
            mc[k] = *reinterpret_cast<const unsigned*>((const uint8_t*)mom1 + si);
            vc[k] = *reinterpret_cast<const unsigned*>((const uint8_t*)mom2 + si);
            ms[k] = scales[si / AW_BLOCK * 2];
            vs[k] = scales[si / AW_BLOCK * 2 + 1];
        }
    }
    AwScalars a;
    if (SMALL) {
        __shared__ double sh[3];
        if (threadIdx.x < 64) {
            double v[AW_SMALL / 64], total = 0.0;
#pragma unroll
            for (int j = 0; j < AW_SMALL / 64; ++j) v[j] = st->partial[threadIdx.x + 64 * j < parts ? threadIdx.x + 64 * j : 0];
#pragma unroll
            for (int j = 0; j < AW_SMALL / 64; ++j) total += (int)threadIdx.x + 64 * j < parts ? v[j] : 0.0;
            total = wave_sum(total);
            if (threadIdx.x == 0) sh[0] = total;
        } else if (threadIdx.x == 64) {                      // (a wave each: a double pow takes as long as the sum)
            sh[1] = 1.0 - pow(st->b1, (double)st->step);
        } else if (threadIdx.x == 128) {
            sh[2] = 1.0 - pow(st->b2, (double)st->step);
        }
        __syncthreads();
        a = aw_scalars(st, st->step, aw_coef(sh[0], st->max_norm), sh[1], sh[2]);
    } else {
        a = st->now;
    }
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const long i = base + (k * AW_THREADS + threadIdx.x) * 4, si = t.state + i;
        if (base + (k * AW_THREADS + (threadIdx.x & ~63)) * 4 >= t.n) break;             // the whole wave leaves
        if (BITS == 8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned a = (mc[k] >> (8 * j)) & 255u, b = (vc[k] >> (8 * j)) & 255u;
                const float x = code_value<15>(a & 127u) * ms[k];
                mv[k][j] = a & 128u ? -x : x;
                vv[k][j] = code_value<31>(b) * vs[k];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float g = gv[k][j] * a.coef;
            const float m = mv[k][j] * a.b1 + g * a.nb1;
            const float v = vv[k][j] * a.b2 + (g * g) * a.nb2;
            const float denom = sqrtf(v) * a.inv_bc2 + a.eps;
            pv[k][j] = pv[k][j] * a.keep - (m / denom) * a.step_size;
            mv[k][j] = m;
            vv[k][j] = v;
        }
        st4(t.p, t.p_dtype, i, t.n, t.vec & 1, pv[k]);
        if (t.copy) st4(t.copy, t.copy_dtype, i, t.n, t.vec & 4, pv[k]);
        if (BITS == 32) {
            *reinterpret_cast<f32v4*>((float*)mom1 + si) = mv[k];
            *reinterpret_cast<f32v4*>((float*)mom2 + si) = vv[k];
        } else {
            float mm = 0.f, vm = 0.f;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i + j >= t.n) mv[k][j] = 0.f, vv[k][j] = 0.f;    // what lies behind a tensor's end has no state
                mm = fmaxf(mm, fabsf(mv[k][j]));
                vm = fmaxf(vm, vv[k][j]);
                bad = bad || !(fabsf(mv[k][j]) < INFINITY) || !(vv[k][j] < INFINITY);
            }
            mm = wave_max(mm);
            vm = wave_max(vm);
            bad = __any(bad);
            float sm, im, sv, iv;
            block_scale(mm, bad, sm, im);
            block_scale(vm, bad, sv, iv);
            unsigned ma = 0, va = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned r = mix32((unsigned)(si + j) ^ a.key);
                const float y = mv[k][j] * im, z = vv[k][j] * iv;
                unsigned cm = code_of<15>(fabsf(y), r & 0xfffffu), cv = code_of<31>(z, r >> 12);
                if (y < 0.f) cm += 128u;
                if (cv == 0 && z > 0.f) cv = 1;
                ma |= (bad ? 0u : cm) << (8 * j);
                va |= (bad ? 0u : cv) << (8 * j);
            }
            *reinterpret_cast<unsigned*>((uint8_t*)mom1 + si) = ma;
            *reinterpret_cast<unsigned*>((uint8_t*)mom2 + si) = va;
            if ((threadIdx.x & 63) == 0) {
                scales[si / AW_BLOCK * 2] = sm;
                scales[si / AW_BLOCK * 2 + 1] = sv;
            }
        }
    }
}

// the values that 8-bit moments stand for: 2 bytes read, 8 written an element, 201 million in 415 us (4.9 TB/s)
__global__ __launch_bounds__(256) void adamw_read_kernel(const uint8_t* __restrict__ mom1, const uint8_t* __restrict__ mom2,
                                                         const float* __restrict__ scales, float* __restrict__ m, float* __restrict__ v, long n) {
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long)gridDim.x * 1024) {
        const unsigned a4 = *reinterpret_cast<const unsigned*>(mom1 + i), b4 = *reinterpret_cast<const unsigned*>(mom2 + i);
        const float ms = scales[i / AW_BLOCK * 2], vs = scales[i / AW_BLOCK * 2 + 1];
        f32v4 om, ov;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned a = (a4 >> (8 * j)) & 255u, b = (b4 >> (8 * j)) & 255u;
            const float x = code_value<15>(a & 127u) * ms;
            om[j] = a & 128u ? -x : x;
            ov[j] = code_value<31>(b) * vs;
        }
        *reinterpret_cast<f32v4*>(m + i) = om;
        *reinterpret_cast<f32v4*>(v + i) = ov;
    }
}

}  // namespace acktr

using namespace acktr;

extern "C" int acktr_adamw_chunk(void) { return AW_CHUNK; }
extern "C" int acktr_adamw_block(void) { return AW_BLOCK; }
extern "C" long acktr_adamw_state_bytes(void) { return (long)sizeof(AwState); }

extern "C" int acktr_adamw_step(void* state, const acktr_adamw_tensor* tensors, const int* chunks, long nchunks, void* mom1, void* mom2,
                                float* scales, int bits, int clip, void* stream) {
    ACKTR_ARG(bits == 32 || bits == 8, "adamw: moments are held in 32 or 8 bits (got %d)", bits);
    ACKTR_ARG(nchunks >= 0 && nchunks < (1L << 31), "adamw: too many chunks (%ld)", nchunks);
    ACKTR_ARG(state && (nchunks == 0 || (tensors && chunks && mom1 && mom2)) && (bits == 32 || nchunks == 0 || scales), "adamw: null buffer");
    ACKTR_ARG((((uintptr_t)state | (uintptr_t)mom1 | (uintptr_t)mom2) & 15) == 0 && (((uintptr_t)tensors | (uintptr_t)chunks) & 7) == 0,
              "adamw: buffers must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    AwState* st = (AwState*)state;
    const int2* table = (const int2*)chunks;
    const int n = (int)nchunks;
    const bool small = clip && n && n <= AW_SMALL;
    if (small) adamw_norm_kernel<true><<<n, AW_THREADS, 0, s>>>(st, tensors, table, n);
    else if (clip && n) adamw_norm_kernel<false><<<min(n, AW_PARTIALS), AW_THREADS, 0, s>>>(st, tensors, table, n);
    else adamw_begin_kernel<<<1, 1, 0, s>>>(st);
    ACKTR_LAUNCH_CHECK();
    if (!n) return 0;
    if (bits == 32) {
        if (small) adamw_update_kernel<32, true><<<n, AW_THREADS, 0, s>>>(st, tensors, table, mom1, mom2, scales, n);
        else adamw_update_kernel<32, false><<<n, AW_THREADS, 0, s>>>(st, tensors, table, mom1, mom2, scales, 0);
    } else {
        if (small) adamw_update_kernel<8, true><<<n, AW_THREADS, 0, s>>>(st, tensors, table, mom1, mom2, scales, n);
        else adamw_update_kernel<8, false><<<n, AW_THREADS, 0, s>>>(st, tensors, table, mom1, mom2, scales, 0);
    }
    ACKTR_LAUNCH_CHECK();
    return 0;
}

extern "C" int acktr_adamw_read_moments(const void* mom1, const void* mom2, const float* scales, float* m, float* v, long n, void* stream) {
    ACKTR_ARG(n >= 0 && n % AW_BLOCK == 0, "adamw: the moments' length must be a multiple of %d (got %ld)", AW_BLOCK, n);
    if (n == 0) return 0;
    ACKTR_ARG(mom1 && mom2 && scales && m && v, "adamw: null buffer");
    adamw_read_kernel<<<(int)min((n + 1023) / 1024, 8192L), 256, 0, (hipStream_t)stream>>>((const uint8_t*)mom1, (const uint8_t*)mom2, scales, m, v, n);
    ACKTR_LAUNCH_CHECK();
    return 0;
}
