// Group norm with channels last, the modulation of the sample's channels and an activation, and its vector-Jacobian products:
//   n = (x - mean_g) rstd_g,  z = (n w + b)(1 + s) + h,  y = act(z)
// and with a = dy act'(z), P[b,c] = sum a n and Q[b,c] = sum a over the sample's positions
//   dh = Q,  ds = w P + b Q,  dw = sum_b (1 + s) P,  db = sum_b (1 + s) Q
//   dx = rstd (gamma a - mean_g(gamma a) - n mean_g(gamma a n)),  gamma = w (1 + s),
// where the two means over a group follow from P and Q: sum_c gamma_c Q_c and sum_c gamma_c P_c.
//
// A sample is read as rows of 16-byte vectors.  Where a row of channels is no whole number of vectors, `period` rows are taken as
// one, so that a thread that goes down the rows meets the same channels every time and keeps their sums and constants in registers.
#include <math.h>

#include <type_traits>

#include "tode_field.h"

namespace tode {

constexpr int NORM_RESIDENT_THREADS = 512;                   // (256 registers each)
constexpr int NORM_ROW_VECTORS = 256;                        // of a workgroup's part of a row at most: as many groups as values, two sums of each in LDS
// vectors a thread keeps of a tensor: 128 registers, backward twice 32.  (Backward with 16 only one workgroup fits, and with 4 fewer samples: 64 samples of
// 32 x 32 x 320, bfloat16, 54 us with 8, 69 with 16, 54 with 4; 2048 of 32 x 32 x 64, float32, 355, 528 and 507.)
constexpr int NORM_MOST = 32, NORM_MOST_BACKWARD = 8;

struct NormShape {
    long long B, S, rows;  // rows: of `period` positions each
    int C, G, width;       // width: channels of a group
    int period, chunk, V;  // chunk: channels a workgroup handles; V: vectors in its part of a row
    int chunks, splits, apply_splits;  // pieces of a sample whose sums are taken apart, and to which they are applied
    long long split_rows, apply_rows;
};

// ------------------------------------------------------------------------------------------
// parameters and activations
// ------------------------------------------------------------------------------------------

template <typename A> __device__ __forceinline__ void set_param(void *p, int dtype, long long i, A v) {
    switch (dtype) {
        case TODE_F32: ((float *)p)[i] = (float)v; break;
        case TODE_F64: ((double *)p)[i] = (double)v; break;
        case TODE_BF16: ((bf16 *)p)[i] = (bf16)(float)v; break;
        default: ((f16 *)p)[i] = (f16)(float)v; break;
    }
}

// What an activation is computed to: SHORT for results that are rounded to 16 bits.
template <typename T> constexpr bool is_short() { return sizeof(T) == 2; }

// 1 / (1 + exp(-z)).  The hardware's power of two and reciprocal are off by one unit each; the product z log2(e) has an error that grows
// with |z|, which float32 results carry along as `lo` (2^(hi + lo)).  Where the power ends at 0 or infinity, z may be anything: it is cut off beyond
// that, so that neither hi nor lo overflows.
template <bool SHORT> __device__ __forceinline__ float sigmoid(float z) {
    constexpr float L = 1.44269502162933349609375f;
    if (SHORT) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -L));
    const float t = __builtin_amdgcn_fmed3f(-z, -128.0f, 128.0f), hi = t * L, lo = fmaf(t, L, -hi) + t * 1.9259629911266174e-8f;
    return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(hi), fmaf(lo, 0.693147180559945286f, 1.0f), 1.0f));
}
template <bool SHORT> __device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

// 16 bits: 1 - 2 / (1 + exp(2 z)), off by 2^-24; z itself where that is too much (off by z^2 / 3 of it)
template <bool SHORT> __device__ __forceinline__ float tangent(float z) {
    if (!SHORT) return tanhf(z);
    const float y = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * 2.88539004325866699219f)), 1.0f);
    return fabsf(z) < 0.00390625f ? z : y;
}
template <bool SHORT> __device__ __forceinline__ double tangent(double z) { return tanh(z); }

// The normal distribution's function and density times sqrt(2 pi).  The tail is density times a polynomial in t = 1 / (1 + c |z|): its ratio to
// the density falls slowly and is smooth in t.  Coefficients by weighted least squares to the smallest relative error for |z| < 14, where the
// density ends: 1.5e-7 for 16 bits (whose parameters may have float32 gradients), 2e-8 for float32, whose |z| < 1 take an odd polynomial about 1/2
// instead (4e-8 of it; differences from 1 would double the error).  One power and one reciprocal; erfcf takes several times as long (512 float32 samples of 64 x 64 x 16: 76 us; 66 with five
// coefficients for everything, which were off by 7e-8 of 1 and by a tenth of a per cent at -4; 37 float16 ones of 45 x 53 x 120: 31).
template <bool SHORT> __device__ __forceinline__ void normal(float z, float &below, float &density) {
    const float x = fabsf(z), s = z * z;
    density = __builtin_amdgcn_exp2f(s * -0.72134752044448170368f);
    const float t = __builtin_amdgcn_rcpf(fmaf(x, SHORT ? 0.3f : 0.2625f, 1.0f));
    float p;
    if (SHORT) {
        p = fmaf(0.0355736409f, t, -0.156781816f), p = fmaf(p, t, 0.205628049f), p = fmaf(p, t, -0.0530165609f), p = fmaf(p, t, 0.128209209f);
        p = fmaf(p, t, 0.100020071f), p = fmaf(p, t, 0.120736926f), p = fmaf(p, t, 0.119630405f);
    } else {
        p = fmaf(0.0306574329f, t, -0.148385007f), p = fmaf(p, t, 0.233887704f), p = fmaf(p, t, -0.132396963f), p = fmaf(p, t, 0.148453724f);
        p = fmaf(p, t, 0.0561404901f), p = fmaf(p, t, 0.102743951f), p = fmaf(p, t, 0.104149397f), p = fmaf(p, t, 0.104749262f);
    }
    p *= t * density;
    below = z < 0 ? p : 1.0f - p;
    if (!SHORT) {
        float q = fmaf(9.42358652e-5f, s, -1.16935511e-3f);
        q = fmaf(q, s, 9.96719793e-3f), q = fmaf(q, s, -6.6489583e-2f), q = fmaf(q, s, 0.398942264f);
        below = x < 1.0f ? fmaf(q, z, 0.5f) : below;
    }
}
template <bool SHORT> __device__ __forceinline__ void normal(double z, double &below, double &density) {
    below = 0.5 * erfc(-0.70710678118654752440 * z), density = exp(-0.5 * z * z);
}

template <int N, bool SHORT, typename A> __device__ __forceinline__ void activate(int act, A *z) {
    if (act == TODE_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] *= sigmoid<SHORT>(z[i]);
    } else if (act == TODE_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            A below, density;
            normal<SHORT>(z[i], below, density);
            z[i] *= below;
        }
    } else if (act == TODE_ACT_TANH) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = tangent<SHORT>(z[i]);
    } else if (act == TODE_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = z[i] > 0 ? z[i] : (z[i] != z[i] ? z[i] : (A)0);
    }
}

// h[i] *= act'(z[i])
template <int N, bool SHORT, typename A> __device__ __forceinline__ void activate_backward(int act, const A *z, A *h) {
    if (act == TODE_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const A e = sigmoid<SHORT>(z[i]);
            h[i] *= fma(z[i] * e, 1 - e, e);
        }
    } else if (act == TODE_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            A below, density;
            normal<SHORT>(z[i], below, density);
            h[i] *= fma(z[i] * (A)0.398942280401432678, density, below);
        }
    } else if (act == TODE_ACT_TANH) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const A e = tangent<SHORT>(z[i]);
            h[i] *= (1 - e) * (1 + e);
        }
    } else if (act == TODE_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = z[i] > 0 ? h[i] : (z[i] != z[i] ? z[i] : (A)0);
    }
}

// f(act) with act known to the compiler.  A loop that is unrolled for values in registers has the code of one activation in a row that way, and not
// that of all of them between any two of its steps, which is more than the instruction cache holds (512 float32 samples of 64 x 64 x 16 with
// SiLU: 60 us, 76 the other way; 128 bfloat16 ones of 64 x 64 x 256: 142 against 150).
template <typename F> __device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
        case TODE_ACT_SILU: f(std::integral_constant<int, TODE_ACT_SILU>()); break;
        case TODE_ACT_GELU: f(std::integral_constant<int, TODE_ACT_GELU>()); break;
        case TODE_ACT_TANH: f(std::integral_constant<int, TODE_ACT_TANH>()); break;
        case TODE_ACT_RELU: f(std::integral_constant<int, TODE_ACT_RELU>()); break;
        default: f(std::integral_constant<int, TODE_ACT_NONE>());
    }
}

// N parameters from `i` on, `other` where there are none.  (One branch for all of them: their loads are under way together.)
template <int N, typename S, typename A> __device__ __forceinline__ void params_as(const void *p, long long i, A *v) {
    S w[N];
    __builtin_memcpy(w, (const S *)p + i, sizeof(w));
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (A)(typename Wide<S>::type)w[e];
}
template <int N, typename A> __device__ __forceinline__ void params(const void *p, int dtype, long long i, A other, A *v) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = other;
    } else if (dtype == TODE_F32)
        params_as<N, float>(p, i, v);
    else if (dtype == TODE_F64)
        params_as<N, double>(p, i, v);
    else if (dtype == TODE_BF16)
        params_as<N, bf16>(p, i, v);
    else
        params_as<N, f16>(p, i, v);
}

// gain = w (1 + s) and offset of N channels from c0 on, which may wrap round behind the last
template <int N, typename A> __device__ __forceinline__ void channel_parameters(const tode_group_norm_args &a, const NormShape &n, long long b, int c0, A *gain, A *offset) {
    A w[N], o[N], s[N], h[N];
    const long long sample = b * n.C, own = a.affine_per_sample ? sample : 0;
    if (c0 + N <= n.C) {
        params<N>(a.weight, a.affine_dtype, own + c0, (A)1, w), params<N>(a.bias, a.affine_dtype, own + c0, (A)0, o);
        params<N>(a.scale, a.modulation_dtype, sample + c0, (A)0, s), params<N>(a.shift, a.modulation_dtype, sample + c0, (A)0, h);
    } else {
        int c = c0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            params<1>(a.weight, a.affine_dtype, own + c, (A)1, w + i), params<1>(a.bias, a.affine_dtype, own + c, (A)0, o + i);
            params<1>(a.scale, a.modulation_dtype, sample + c, (A)0, s + i), params<1>(a.shift, a.modulation_dtype, sample + c, (A)0, h + i);
            if (++c == n.C) c = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += 1, gain[i] = w[i] * s[i], offset[i] = fma(o[i], s[i], h[i]);
}

// The groups of N channels from c0 on.
template <int N> __device__ __forceinline__ void groups_of(const NormShape &n, int c0, int *group) {
    int g = c0 / n.width, r = c0 - g * n.width;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        group[i] = g;
        if (++r == n.width) r = 0, g = g + 1 == n.G ? 0 : g + 1;
    }
}

// What becomes of P and Q of one channel of a sample; returns gamma.
template <typename A> __device__ __forceinline__ A channel_gradients(const tode_group_norm_args &a, const NormShape &n, long long b, int c, A p, A q, A *products) {
    const long long at = b * n.C + c, at1 = a.affine_per_sample ? at : c;
    A w, o, s;
    params<1>(a.weight, a.affine_dtype, at1, (A)1, &w), params<1>(a.bias, a.affine_dtype, at1, (A)0, &o), params<1>(a.scale, a.modulation_dtype, at, (A)0, &s);
    s += 1;
    products[2 * at] = s * p, products[2 * at + 1] = s * q;
    if (a.dscale) set_param(a.dscale, a.modulation_dtype, at, fma(w, p, o * q));
    if (a.dshift) set_param(a.dshift, a.modulation_dtype, at, q);
    if (a.affine_per_sample && a.dweight) set_param(a.dweight, a.affine_dtype, at, s * p);
    if (a.affine_per_sample && a.dbias) set_param(a.dbias, a.affine_dtype, at, s * q);
    return w * s;
}

template <typename A> __device__ __forceinline__ A wave_total(A v) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// Workgroups of one sample lie on one XCD (they go round the eight), so that cache lines two of them share are fetched once.
__device__ __forceinline__ bool place_sample(unsigned block, unsigned chunks, long long samples, long long &b, int &chunk) {
    if (samples >= 8) {
        const unsigned round = block / 8 / chunks;
        b = round * 8ll + block % 8, chunk = (int)(block / 8 - round * chunks);
        return b < samples;
    }
    const unsigned sample = block / chunks;
    b = sample, chunk = (int)(block - sample * chunks);
    return b < samples;
}

// What a thread has to know of its N channels: n = (x - mean) rstd, z = n gain + offset.  The mean is taken off first: x rstd - mean rstd would
// leave a unit of mean rstd, which in a group without spread has sqrt(eps) for its divisor (float16, 30 000 everywhere: 0.5 in place of 0; 37 float16 samples of
// 45 x 53 x 120 with GELU: 29.9 us, that way 28.4; 128 bfloat16 ones of 64 x 64 x 256 with SiLU 152 either way).
template <int N, typename A> struct Channels {
    A mean[N], rstd[N], gain[N], offset[N];
    __device__ __forceinline__ A normal(A x, int i) const { return (x - mean[i]) * rstd[i]; }
    __device__ __forceinline__ void load(const tode_group_norm_args &a, const NormShape &n, long long b, int c0) {
        channel_parameters<N>(a, n, b, c0, gain, offset);
        int group[N];
        groups_of<N>(n, c0, group);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const long long g = b * n.G + group[i];
            rstd[i] = ((const A *)a.rstd)[g], mean[i] = ((const A *)a.mean)[g];
        }
    }
};

// Reads N values of a row of the sample that ends at `end` values; zeros behind it.
template <typename T, int N> struct Vec {
    typedef typename Wide<T>::type A;
    static __device__ __forceinline__ void load(const T *p, long long left, A *v) {
        if (N == Raw<T>::N && left >= N) {
            Raw<T> r;
            r.load(p);
            unpack(r, v);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < left ? (A)p[i] : (A)0;
        }
    }
    static __device__ __forceinline__ void store(T *p, long long left, const A *v) {
        if (N == Raw<T>::N && left >= N) {
            Raw<T> r;
            pack(r, v);
            r.store(p);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) p[i] = (T)v[i];
        }
    }
};

// (n, mean, sum of squared distances) of two sets of values joined
template <typename A> __device__ __forceinline__ void join(A &n, A &mean, A &m2, A nb, A meanb, A m2b) {
    const A total = n + nb;
    if (nb == 0) return;
    const A d = meanb - mean, f = nb / total;
    mean += d * f;
    m2 += m2b + d * d * n * f;
    n = total;
}

// ------------------------------------------------------------------------------------------
// the resident form: a workgroup keeps its part of a sample -- all positions of some whole groups -- in registers
// ------------------------------------------------------------------------------------------

// Thread t has vector t % V of rows t / V, t / V + lanes, ...: at most R of them.  What is summed goes through LDS, [lanes][columns].
// WRAPPED: rows of several positions (period > 1), whose last one may end within a vector.
template <typename T, int R, bool WRAPPED> struct Resident {
    typedef typename Wide<T>::type A;
    static constexpr int N = Raw<T>::N;
    long long b, first, step;  // of the sample's part, and between a thread's rows: the same for all threads
    int lanes, j, lane_row, c0, chunk0, groups, rows, thread_offset;
    bool there, active;
    __device__ __forceinline__ Resident(const NormShape &n) {
        int chunk;
        there = place_sample(block_number(), n.chunks, n.B, b, chunk);
        lanes = blockDim.x / n.V, j = threadIdx.x % n.V, lane_row = threadIdx.x / n.V;
        active = lane_row < lanes, rows = active ? (int)n.rows : 0;
        chunk0 = chunk * n.chunk, c0 = WRAPPED ? N * j % n.C : chunk0 + N * j, groups = n.chunk / n.width;
        const int stride = n.period * n.C;
        first = b * n.S * n.C + chunk0, step = (long long)lanes * stride, thread_offset = lane_row * stride + N * j;
    }
    // values there are of vector i: none, N, or fewer where the sample ends
    __device__ __forceinline__ int left(const NormShape &n, int i) const {
        if (lane_row + i * lanes >= rows) return 0;
        if (!WRAPPED) return N;
        const long long k = n.S * n.C - i * step - thread_offset;
        return k < N ? (int)k : N;
    }
    __device__ __forceinline__ void load(const NormShape &n, const void *of, Raw<T> *r) const {
        const T *p = (const T *)of + first;
#pragma unroll
        for (int i = 0; i < R; ++i, p += step) {
            const int k = left(n, i);
            r[i].zero();
            if (k == N)
                r[i].load(p + thread_offset);
            else if (WRAPPED && k > 0) {
                T v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = e < k ? p[thread_offset + e] : (T)0.0f;
                __builtin_memcpy(r[i].w, v, 16);
            }
        }
    }
    __device__ __forceinline__ void store(void *of, int i, int left, const A *v) const { Vec<T, N>::store((T *)of + first + i * step + thread_offset, left, v); }
    // Means over the workgroup by group, into total[0 .. groups-1].  One value a thread where its vector lies in one group, else N.
    // `buffer`: room for blockDim.x * N values, then one a group or wavefront, of which there are more.
    // S: what they are taken in there.  Returns them divided by `count`.
    template <typename S> __device__ __forceinline__ void mean_of_groups(const NormShape &n, const A *v, A *buffer, S count, A *total) const {
        const int threads = blockDim.x;
        const bool one = !WRAPPED && n.width % N == 0;
        const int cols = one ? n.V : n.V * N, width = one ? n.width / N : n.width;
        if (active) {
            if (one) {
                A t = v[0];
#pragma unroll
                for (int i = 1; i < N; ++i) t += v[i];
                buffer[lane_row * cols + j] = t;
            } else
#pragma unroll
                for (int i = 0; i < N; ++i) buffer[lane_row * cols + j * N + i] = v[i];
        }
        __syncthreads();
        const int waves = threads / 64, wave = threadIdx.x / 64, lane = threadIdx.x % 64, share = groups < waves ? waves / groups : 1;
        S *const parts = (S *)(buffer + threads * N);
        for (int k = wave; k < groups * share; k += waves) {
            const int g = k / share, row = WRAPPED ? n.period * width : width, stride = 64 * share, rows_step = stride / row, rest = stride % row;
            int e = lane + 64 * (k % share), r = e / row;
            e %= row;
            S t = 0;
            while (r < lanes) {
                const int p = WRAPPED ? e / width : 0;
                t += buffer[r * cols + p * n.C + g * width + (e - p * width)];
                e += rest, r += rows_step;
                if (e >= row) e -= row, ++r;
            }
            t = wave_total(t);
            if (lane == 0) parts[g * share + k % share] = t;
        }
        __syncthreads();
        for (int g = threadIdx.x; g < groups; g += threads) {
            S t = parts[g * share];
            for (int k = 1; k < share; ++k) t += parts[g * share + k];
            total[g] = (A)(t / count);
        }
        __syncthreads();
    }
};

// Vectors are worked on one after the other: interleaved by the compiler, their unpacked values take the registers that hold the others.
__device__ __forceinline__ void one_at_a_time() { __builtin_amdgcn_sched_barrier(0); }
// Nor are they kept unpacked from one pass over them to the next, which would take twice the registers.
template <int R, typename T> __device__ __forceinline__ void keep_packed(Raw<T> *r) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(r[i].w[k]));
}

template <typename T, int R, bool WRAPPED> __global__ void __launch_bounds__(NORM_RESIDENT_THREADS) norm_resident_kernel(tode_group_norm_args a, NormShape n) {
    typedef Resident<T, R, WRAPPED> W;
    typedef typename W::A A;
    constexpr int N = W::N;
    extern __shared__ __align__(16) char lds[];
    const W w(n);
    if (!w.there) return;
    // Sums of 16-bit values that are all the same are exact in a thread (32 values of 11 bits), and between threads in float64: their mean
    // has to be theirs to the last bit, as what is left of them is divided by sqrt(eps).
    typedef typename std::conditional<is_short<T>(), double, A>::type S;
    A *const buffer = (A *)lds, *const means = (A *)((S *)(buffer + blockDim.x * N) + max(w.groups, (int)blockDim.x / 64)), *const variances = means + w.groups;
    Raw<T> x[R];
    w.load(n, a.x, x);
    A sum[N], mean[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        A v[N];
        unpack(x[i], v);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += v[e];  // (zeros behind the end)
        one_at_a_time();
    }
    w.mean_of_groups(n, sum, buffer, (S)n.S * (S)n.width, means);
    keep_packed<R>(x);
    const A count = (A)n.S * (A)n.width;
    int group[N];
    groups_of<N>(n, w.c0, group);
    const int group0 = w.chunk0 / n.width;
#pragma unroll
    for (int e = 0; e < N; ++e) mean[e] = means[group[e] - group0], sum[e] = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int left = w.left(n, i);
        if (left > 0) {
            A v[N];
            unpack(x[i], v);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const A d = v[e] - mean[e];
                sum[e] = !WRAPPED || e < left ? fma(d, d, sum[e]) : sum[e];
            }
        }
        one_at_a_time();
    }
    w.mean_of_groups(n, sum, buffer, count, variances);
    keep_packed<R>(x);
    for (int g = threadIdx.x; g < w.groups; g += blockDim.x) {
        const long long k = w.b * n.G + w.chunk0 / n.width + g;
        if (a.mean) ((A *)a.mean)[k] = means[g];
        if (a.rstd) ((A *)a.rstd)[k] = 1 / sqrt(variances[g] + (A)a.eps);
    }
    if (!w.active) return;
    A gain[N], shift[N];
    channel_parameters<N>(a, n, w.b, w.c0, gain, shift);
#pragma unroll
    for (int e = 0; e < N; ++e) gain[e] *= 1 / sqrt(variances[group[e] - group0] + (A)a.eps);
    with_activation(a.activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int left = w.left(n, i);
            if (left > 0) {
                A v[N];
                unpack(x[i], v);
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = fma(v[e] - mean[e], gain[e], shift[e]);
                activate<N, is_short<T>()>(act(), v);
                w.store(a.y, i, left, v);
            }
            if (i % 2) one_at_a_time();
        }
    });
}

// P, Q, the gradients of scale and shift, and x's, from x and dy in registers; products[b,c] = (1 + s) (P, Q) for the shared weights'.
template <typename T, int R, bool WRAPPED>
__global__ void __launch_bounds__(NORM_RESIDENT_THREADS) norm_resident_backward_kernel(tode_group_norm_args a, NormShape n, typename Wide<T>::type *products) {
    typedef Resident<T, R, WRAPPED> W;
    typedef typename W::A A;
    constexpr int N = W::N;
    extern __shared__ __align__(16) char lds[];
    const W w(n);
    if (!w.there) return;
    const int threads = blockDim.x;
    Raw<T> x[R], dy[R];
    w.load(n, a.x, x);
    w.load(n, a.dy, dy);
    Channels<N, A> ch;
    ch.load(a, n, w.b, w.c0);
    A P[N], Q[N];
#pragma unroll
    for (int e = 0; e < N; ++e) P[e] = Q[e] = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (w.left(n, i) > 0) {
            A v[N], h[N], z[N];
            unpack(x[i], v);
            unpack(dy[i], h);  // (zeros behind the end: nothing is added there)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = ch.normal(v[e], e), z[e] = fma(v[e], ch.gain[e], ch.offset[e]);
            activate_backward<N, is_short<T>()>(a.activation, z, h);
#pragma unroll
            for (int e = 0; e < N; ++e) P[e] = fma(h[e], v[e], P[e]), Q[e] += h[e];
        }
        one_at_a_time();
    }
    keep_packed<R>(x), keep_packed<R>(dy);
    // columns over the lanes: `pieces` threads a column, then one a channel
    const int cols = n.V * N, pieces = threads / cols > 1 ? threads / cols : 1;
    A *const s_p = (A *)lds, *const s_q = s_p + threads * N, *const piece_p = s_q + threads * N, *const piece_q = piece_p + pieces * cols;
    A *const channel_p = s_p, *const channel_q = s_q, *const m1 = piece_q + pieces * cols, *const m2 = m1 + w.groups;  // (s_p and s_q are read by then)
    if (w.active)
#pragma unroll
        for (int e = 0; e < N; ++e) s_p[w.lane_row * cols + w.j * N + e] = P[e], s_q[w.lane_row * cols + w.j * N + e] = Q[e];
    __syncthreads();
    for (int k = threadIdx.x; k < pieces * cols; k += threads) {
        const int piece = k / cols, col = k % cols;
        A p = 0, q = 0;
        for (int r = piece; r < w.lanes; r += pieces) p += s_p[r * cols + col], q += s_q[r * cols + col];
        piece_p[k] = p, piece_q[k] = q;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < n.chunk; c += threads) {
        A p = 0, q = 0;
        for (int k = 0; k < pieces; ++k)
            for (int r = 0; r < n.period; ++r) p += piece_p[k * cols + r * n.C + c], q += piece_q[k * cols + r * n.C + c];
        const A gamma = channel_gradients(a, n, w.b, w.chunk0 + c, p, q, products);
        channel_p[c] = gamma * p, channel_q[c] = gamma * q;
    }
    if (!a.dx) return;
    __syncthreads();
    const A count = (A)n.S * (A)n.width;
    const int waves = threads / 64, lane = threadIdx.x % 64;
    for (int g = threadIdx.x / 64; g < w.groups; g += waves) {
        A p = 0, q = 0;
        for (int c = lane; c < n.width; c += 64) p += channel_p[g * n.width + c], q += channel_q[g * n.width + c];
        p = wave_total(p), q = wave_total(q);
        if (lane == 0) m1[g] = q / count, m2[g] = p / count;
    }
    __syncthreads();
    if (!w.active) return;
    A k1[N], k2[N];
    int group[N];
    groups_of<N>(n, w.c0, group);
    const int group0 = w.chunk0 / n.width;
#pragma unroll
    for (int e = 0; e < N; ++e) k1[e] = m1[group[e] - group0], k2[e] = m2[group[e] - group0];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int left = w.left(n, i);
        if (left > 0) {
            A v[N], h[N], z[N];
            unpack(x[i], v);
            unpack(dy[i], h);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = ch.normal(v[e], e), z[e] = fma(v[e], ch.gain[e], ch.offset[e]);
            activate_backward<N, is_short<T>()>(a.activation, z, h);
#pragma unroll
            for (int e = 0; e < N; ++e) h[e] = ch.rstd[e] * (fma(ch.gain[e], h[e], -k1[e]) - v[e] * k2[e]);
            w.store(a.dx, i, left, h);
        }
        one_at_a_time();
    }
}

// ------------------------------------------------------------------------------------------
// the general form: partial sums per channel of a piece of a sample's rows, joined by a second kernel, applied by a third
// ------------------------------------------------------------------------------------------

constexpr int NORM_THREADS = 256;
constexpr int NORM_BATCH = 8;  // rows whose loads a thread has in flight

struct NormPlace {  // of a thread in its workgroup
    int lane_row, lanes, j, c0, chunk0;
    bool active;
    __device__ __forceinline__ NormPlace(const NormShape &n, int N, int chunk) {
        lanes = NORM_THREADS / n.V;
        j = threadIdx.x % n.V, lane_row = threadIdx.x / n.V;
        active = lane_row < lanes;
        chunk0 = chunk * n.chunk;
        if (chunk0 + N * j >= n.C && n.period == 1) active = false;  // (the last chunk may be narrower)
        c0 = (chunk0 + N * j) % n.C;
    }
};

// Mean and sum of squares of a piece of a sample's rows, by channel.
template <typename T, int N>
__global__ void __launch_bounds__(NORM_THREADS) norm_statistics_kernel(tode_group_norm_args a, NormShape n, typename Wide<T>::type *partial) {
    typedef typename Wide<T>::type A;
    const int chunk = blockIdx.x % n.chunks, split = blockIdx.x / n.chunks;
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    const NormPlace at(n, N, chunk);
    const long long first = split * n.split_rows, last = min(first + n.split_rows, n.rows), end = n.S * n.C;
    const T *x = (const T *)a.x + b * end + at.chunk0 + N * at.j;
    const long long stride = (long long)n.period * n.C, limit = end - at.chunk0 - N * at.j;
    A count[N], mean[N], m2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) count[i] = mean[i] = m2[i] = 0;
    if (at.active) {
        // rows in full, a batch at a time: its own mean and squares, joined to those before
        const long long full = limit < N ? 0 : min(last, (limit - N) / stride + 1);
        long long r = first + at.lane_row;
        A k = 0;
        for (; r + (NORM_BATCH - 1) * at.lanes < full; r += NORM_BATCH * at.lanes) {
            Raw<T> raw[NORM_BATCH];
            A sum[N], squares[N];
            if (N > 1) {
#pragma unroll
                for (int u = 0; u < NORM_BATCH; ++u) raw[u].load(x + (r + u * at.lanes) * stride);
            }
            auto value = [&](int u, A *v) {
                if (N > 1)
                    unpack(raw[u], v);
                else
                    v[0] = (A)x[(r + u * at.lanes) * stride];
            };
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = squares[i] = 0;
#pragma unroll
            for (int u = 0; u < NORM_BATCH; ++u) {
                A v[Raw<T>::N];
                value(u, v);
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[i];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] *= (A)(1.0 / NORM_BATCH);
#pragma unroll
            for (int u = 0; u < NORM_BATCH; ++u) {
                A v[Raw<T>::N];
                value(u, v);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const A d = v[i] - sum[i];
                    squares[i] = fma(d, d, squares[i]);
                }
            }
            const A f = NORM_BATCH / (k + NORM_BATCH), kf = k * f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const A d = sum[i] - mean[i];
                mean[i] = fma(d, f, mean[i]);
                m2[i] += fma(d * d, kf, squares[i]);
            }
            k += NORM_BATCH;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) count[i] = k;
        for (; r < last; r += at.lanes) {  // the others one by one; the last one may end within a vector
            const long long left = limit - r * stride;
            if (left <= 0) break;
            A v[N];
            Vec<T, N>::load(x + r * stride, left, v);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) {
                    const A d = v[i] - mean[i];
                    count[i] += 1;
                    mean[i] += d / count[i];
                    m2[i] = fma(d, v[i] - mean[i], m2[i]);
                }
        }
    }
    // threads of one column, then columns of one channel
    __shared__ A s_count[NORM_THREADS * N], s_mean[NORM_THREADS * N], s_m2[NORM_THREADS * N];
    const int cols = n.V * N;
    if (at.lane_row < at.lanes)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = at.lane_row * cols + at.j * N + i;
            s_count[k] = count[i], s_mean[k] = mean[i], s_m2[k] = m2[i];
        }
    for (int half = at.lanes; half > 1;) {
        const int upper = half / 2, kept = half - upper;  // rows kept .. half-1 are joined into rows 0 .. upper-1
        __syncthreads();
        for (int k = threadIdx.x; k < upper * cols; k += NORM_THREADS) {
            const int o = k + kept * cols;
            join(s_count[k], s_mean[k], s_m2[k], s_count[o], s_mean[o], s_m2[o]);
        }
        half = kept;
    }
    __syncthreads();
    const int width = min(n.chunk, n.C - at.chunk0);
    A *out = partial + ((b * n.splits + split) * n.C + at.chunk0) * 2;
    for (int c = threadIdx.x; c < width; c += NORM_THREADS) {
        A k = 0, m = 0, q = 0;
        for (int p = 0; p < n.period; ++p) {
            const int o = p * n.C + c;
            join(k, m, q, s_count[o], s_mean[o], s_m2[o]);
        }
        out[2 * c] = m, out[2 * c + 1] = q;
    }
}

// A wavefront joins the statistics of all channels and pieces of group g: the mean, and 1 / sqrt(variance + eps).
template <typename A> __device__ __forceinline__ void join_group(const NormShape &n, const A *partial, long long b, int g, A eps, A &mean, A &rstd) {
    const int lane = threadIdx.x % 64;
    A count = 0, m2 = 0;
    mean = 0;
    int split = lane / n.width, c = lane - split * n.width;
    const int splits_step = 64 / n.width, rest = 64 - splits_step * n.width;
    const A *const from = partial + (b * n.splits * n.C + g * n.width) * 2;
    while (split < n.splits) {
        A p[4], q[4], k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // (four loads under way)
            const bool there = split < n.splits;
            const A *const o = from + (there ? 2ll * split * n.C + 2 * c : 0);
            const long long first = split * n.split_rows * n.period, last = min((split + 1) * n.split_rows * n.period, n.S);
            k[u] = there ? (A)(last - first) : (A)0, p[u] = o[0], q[u] = o[1];
            c += rest, split += splits_step;
            if (c >= n.width) c -= n.width, ++split;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) join(count, mean, m2, k[u], p[u], q[u]);
    }
    for (int off = 32; off > 0; off >>= 1) {
        const A c1 = __shfl_xor(count, off), m1 = __shfl_xor(mean, off), q1 = __shfl_xor(m2, off);
        // (both lanes of a pair take the same order, so that all lanes end with the same bits)
        const bool upper = lane & off;
        A c0 = upper ? c1 : count, m0 = upper ? m1 : mean, q0 = upper ? q1 : m2;
        join(c0, m0, q0, upper ? count : c1, upper ? mean : m1, upper ? m2 : q1);
        count = c0, mean = m0, m2 = q0;
    }
    rstd = 1 / sqrt(m2 / count + eps);
}

// Where there are many pieces: one wavefront for each group of each sample.
template <typename A>
__global__ void __launch_bounds__(64) norm_join_statistics_kernel(NormShape n, const A *partial, A eps, A *mean_out, A *rstd_out) {
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    const int g = blockIdx.x;
    A mean, rstd;
    join_group(n, partial, b, g, eps, mean, rstd);
    if (threadIdx.x == 0) mean_out[b * n.G + g] = mean, rstd_out[b * n.G + g] = rstd;
}

// partial: the pieces' statistics, where there are so few that every workgroup joins them by itself; else mean and rstd are there.
template <typename T, int N> __global__ void __launch_bounds__(NORM_THREADS) norm_apply_kernel(tode_group_norm_args a, NormShape n, const typename Wide<T>::type *partial) {
    typedef typename Wide<T>::type A;
    const int chunk = blockIdx.x % n.chunks, split = blockIdx.x / n.chunks;
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    const NormPlace at(n, N, chunk);
    const long long first = split * n.apply_rows, last = min(first + n.apply_rows, n.rows), end = n.S * n.C;
    const long long stride = (long long)n.period * n.C, offset = b * end + at.chunk0 + N * at.j, limit = end - at.chunk0 - N * at.j;
    const T *x = (const T *)a.x + offset;
    T *y = (T *)a.y + offset;
    A gain[N], shift[N], mean[N], rstd[N];
    int group[N];
    channel_parameters<N>(a, n, b, at.c0, gain, shift);
    groups_of<N>(n, at.c0, group);
    if (partial) {
        extern __shared__ __align__(16) char lds[];
        A *const s_mean = (A *)lds;
        const int g0 = at.chunk0 / n.width, g1 = (min(at.chunk0 + n.chunk, n.C) - 1) / n.width, groups = g1 - g0 + 1;
        A *const s_rstd = s_mean + groups;
        for (int g = g0 + threadIdx.x / 64; g <= g1; g += NORM_THREADS / 64) {
            A m, r;
            join_group(n, partial, b, g, (A)a.eps, m, r);
            if (threadIdx.x % 64 == 0) {
                s_mean[g - g0] = m, s_rstd[g - g0] = r;
                if (split == 0 && g * n.width >= at.chunk0 && a.mean) ((A *)a.mean)[b * n.G + g] = m, ((A *)a.rstd)[b * n.G + g] = r;
            }
        }
        __syncthreads();
        if (!at.active) return;
#pragma unroll
        for (int i = 0; i < N; ++i) mean[i] = s_mean[group[i] - g0], rstd[i] = s_rstd[group[i] - g0];
    } else {
        if (!at.active) return;
#pragma unroll
        for (int i = 0; i < N; ++i) mean[i] = ((const A *)a.mean)[b * n.G + group[i]], rstd[i] = ((const A *)a.rstd)[b * n.G + group[i]];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) gain[i] *= rstd[i];
    auto apply = [&](A *v) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fma(v[i] - mean[i], gain[i], shift[i]);
        activate<N, is_short<T>()>(a.activation, v);
    };
    const long long full = limit < N ? 0 : min(last, (limit - N) / stride + 1);
    long long r = first + at.lane_row;
    if (N > 1)
        for (; r + 3 * at.lanes < full; r += 4 * at.lanes) {
            Raw<T> raw[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) raw[u].load(x + (r + u * at.lanes) * stride);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                A v[Raw<T>::N];
                unpack(raw[u], v);
                apply(v);
                pack(raw[u], v);
                raw[u].store(y + (r + u * at.lanes) * stride);
            }
        }
    for (; r < last; r += at.lanes) {
        const long long left = limit - r * stride;
        if (left <= 0) break;
        A v[N];
        Vec<T, N>::load(x + r * stride, left, v);
        apply(v);
        Vec<T, N>::store(y + r * stride, left, v);
    }
}

// P and Q of a piece of a sample's rows, by channel.
template <typename T, int N>
__global__ void __launch_bounds__(NORM_THREADS) norm_products_kernel(tode_group_norm_args a, NormShape n, typename Wide<T>::type *partial) {
    typedef typename Wide<T>::type A;
    const int chunk = blockIdx.x % n.chunks, split = blockIdx.x / n.chunks;
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    const NormPlace at(n, N, chunk);
    const long long first = split * n.split_rows, last = min(first + n.split_rows, n.rows), end = n.S * n.C;
    const long long stride = (long long)n.period * n.C, offset = b * end + at.chunk0 + N * at.j, limit = end - at.chunk0 - N * at.j;
    A P[N], Q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) P[i] = Q[i] = 0;
    if (at.active) {
        const T *x = (const T *)a.x + offset, *dy = (const T *)a.dy + offset;
        Channels<N, A> ch;
        ch.load(a, n, b, at.c0);
        auto add = [&](A *v, A *h) {
            A z[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = ch.normal(v[i], i), z[i] = fma(v[i], ch.gain[i], ch.offset[i]);
            activate_backward<N, is_short<T>()>(a.activation, z, h);
#pragma unroll
            for (int i = 0; i < N; ++i) P[i] = fma(h[i], v[i], P[i]), Q[i] += h[i];
        };
        const long long full = limit < N ? 0 : min(last, (limit - N) / stride + 1);
        long long r = first + at.lane_row;
        if (N > 1)
            for (; r + 3 * at.lanes < full; r += 4 * at.lanes) {
                Raw<T> raw[4], grad[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) raw[u].load(x + (r + u * at.lanes) * stride), grad[u].load(dy + (r + u * at.lanes) * stride);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    A v[Raw<T>::N], h[Raw<T>::N];
                    unpack(raw[u], v);
                    unpack(grad[u], h);
                    add(v, h);
                }
            }
        for (; r < last; r += at.lanes) {
            const long long left = limit - r * stride;
            if (left <= 0) break;
            A v[N], h[N];
            Vec<T, N>::load(x + r * stride, left, v);
            Vec<T, N>::load(dy + r * stride, left, h);  // (zero behind the sample's end: nothing is added there)
            add(v, h);
        }
    }
    __shared__ A s_p[NORM_THREADS * N], s_q[NORM_THREADS * N];
    const int cols = n.V * N;
    if (at.lane_row < at.lanes)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = at.lane_row * cols + at.j * N + i;
            s_p[k] = P[i], s_q[k] = Q[i];
        }
    for (int half = at.lanes; half > 1;) {
        const int upper = half / 2, kept = half - upper;
        __syncthreads();
        for (int k = threadIdx.x; k < upper * cols; k += NORM_THREADS) s_p[k] += s_p[k + kept * cols], s_q[k] += s_q[k + kept * cols];
        half = kept;
    }
    __syncthreads();
    const int width = min(n.chunk, n.C - at.chunk0);
    A *out = partial + ((b * n.splits + split) * n.C + at.chunk0) * 2;
    for (int c = threadIdx.x; c < width; c += NORM_THREADS) {
        A p = 0, q = 0;
        for (int k = 0; k < n.period; ++k) p += s_p[k * n.C + c], q += s_q[k * n.C + c];
        out[2 * c] = p, out[2 * c + 1] = q;
    }
}

// A wavefront adds up P and Q of all pieces of group g's channels, writes what becomes of those in [from, to), and returns the group's two means.
template <typename A>
__device__ __forceinline__ void join_products(const tode_group_norm_args &a, const NormShape &n, const A *partial, long long b, int g, int from, int to, A *products, A &m1, A &m2) {
    const int lane = threadIdx.x % 64, wide = n.width < 64 ? n.width : 64, parts = 64 / wide, part = lane / wide;
    A sp = 0, sq = 0;
    for (int k0 = 0; k0 < n.width; k0 += wide) {
        const int k = k0 + lane % wide, c = g * n.width + k;
        const bool there = part < parts && k < n.width;
        A p = 0, q = 0;
        if (there) {
            const A *const o = partial + (b * n.splits * n.C + c) * 2;
#pragma unroll 8
            for (int piece = part; piece < n.splits; piece += parts) p += o[2ll * piece * n.C], q += o[2ll * piece * n.C + 1];
        }
        A tp = p, tq = q;
        for (int i = 1; i < parts; ++i) tp += __shfl(p, lane % wide + i * wide), tq += __shfl(q, lane % wide + i * wide);
        if (there && part == 0) {
            A gamma, unused;
            if (c >= from && c < to)
                gamma = channel_gradients(a, n, b, c, tp, tq, products);
            else
                channel_parameters<1>(a, n, b, c, &gamma, &unused);
            sp = fma(gamma, tp, sp), sq = fma(gamma, tq, sq);
        }
    }
    const A size = (A)n.S * (A)n.width;
    m1 = wave_total(sq) / size, m2 = wave_total(sp) / size;
}

// Where there are many pieces: one wavefront for each group of each sample; `products` [B,C] of pairs, `means` [B,G] of pairs.
template <typename A>
__global__ void __launch_bounds__(64) norm_join_products_kernel(tode_group_norm_args a, NormShape n, const A *partial, A *products, A *means) {
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    A m1, m2;
    join_products(a, n, partial, b, (int)blockIdx.x, 0, n.C, products, m1, m2);
    if (threadIdx.x == 0) means[(b * n.G + blockIdx.x) * 2] = m1, means[(b * n.G + blockIdx.x) * 2 + 1] = m2;
}

// partial: the pieces' P and Q, where there are so few that every workgroup joins them by itself; else the two means are there.
template <typename T, int N>
__global__ void __launch_bounds__(NORM_THREADS) norm_apply_backward_kernel(tode_group_norm_args a, NormShape n, const typename Wide<T>::type *partial, typename Wide<T>::type *products,
                                                                           const typename Wide<T>::type *means) {
    typedef typename Wide<T>::type A;
    const int chunk = blockIdx.x % n.chunks, split = blockIdx.x / n.chunks;
    const long long b = blockIdx.y + (long long)blockIdx.z * 32768;
    if (b >= n.B) return;
    const NormPlace at(n, N, chunk);
    const long long first = split * n.apply_rows, last = min(first + n.apply_rows, n.rows), end = n.S * n.C;
    const long long stride = (long long)n.period * n.C, offset = b * end + at.chunk0 + N * at.j, limit = end - at.chunk0 - N * at.j;
    const T *x = (const T *)a.x + offset, *dy = (const T *)a.dy + offset;
    T *dx = (T *)a.dx + offset;
    Channels<N, A> ch;
    ch.load(a, n, b, at.c0);
    A m1[N], m2[N];
    int group[N];
    groups_of<N>(n, at.c0, group);
    if (partial) {
        extern __shared__ __align__(16) char lds[];
        A *const s_means = (A *)lds;
        const int c1 = min(at.chunk0 + n.chunk, n.C), g0 = at.chunk0 / n.width, g1 = (c1 - 1) / n.width;
        for (int g = g0 + threadIdx.x / 64; g <= g1; g += NORM_THREADS / 64) {
            A p, q;
            join_products(a, n, partial, b, g, split == 0 ? at.chunk0 : c1, c1, products, p, q);
            if (threadIdx.x % 64 == 0) s_means[2 * (g - g0)] = p, s_means[2 * (g - g0) + 1] = q;
        }
        __syncthreads();
        if (!at.active || !a.dx) return;
#pragma unroll
        for (int i = 0; i < N; ++i) m1[i] = s_means[2 * (group[i] - g0)], m2[i] = s_means[2 * (group[i] - g0) + 1];
    } else {
        if (!at.active) return;
#pragma unroll
        for (int i = 0; i < N; ++i) m1[i] = means[2 * (b * n.G + group[i])], m2[i] = means[2 * (b * n.G + group[i]) + 1];
    }
    auto apply = [&](A *v, A *h) {
        A z[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ch.normal(v[i], i), z[i] = fma(v[i], ch.gain[i], ch.offset[i]);
        activate_backward<N, is_short<T>()>(a.activation, z, h);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = ch.rstd[i] * (fma(ch.gain[i], h[i], -m1[i]) - v[i] * m2[i]);
    };
    const long long full = limit < N ? 0 : min(last, (limit - N) / stride + 1);
    long long r = first + at.lane_row;
    if (N > 1)
        for (; r + 3 * at.lanes < full; r += 4 * at.lanes) {
            Raw<T> raw[4], grad[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) raw[u].load(x + (r + u * at.lanes) * stride), grad[u].load(dy + (r + u * at.lanes) * stride);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                A v[Raw<T>::N], h[Raw<T>::N];
                unpack(raw[u], v);
                unpack(grad[u], h);
                apply(v, h);
                pack(grad[u], h);
                grad[u].store(dx + (r + u * at.lanes) * stride);
            }
        }
    for (; r < last; r += at.lanes) {
        const long long left = limit - r * stride;
        if (left <= 0) break;
        A v[N], h[N];
        Vec<T, N>::load(x + r * stride, left, v);
        Vec<T, N>::load(dy + r * stride, left, h);
        apply(v, h);
        Vec<T, N>::store(dx + r * stride, left, h);
    }
}

// dweight and dbias of weights that all samples share: 16 channels by 64 samples a workgroup, the samples in a fixed order.
template <typename A> __global__ void __launch_bounds__(1024) norm_affine_gradients_kernel(tode_group_norm_args a, long long B, int C, const A *products) {
    const int lane = threadIdx.x % 16, row = threadIdx.x / 16, c = blockIdx.x * 16 + lane;
    A p = 0, q = 0;
    if (c < C)
#pragma unroll 8
        for (long long b = row; b < B; b += 64) p += products[2 * (b * C + c)], q += products[2 * (b * C + c) + 1];
    __shared__ A s_p[1024], s_q[1024];
    for (int half = 32; half > 0; half /= 2) {
        if (row >= half && row < 2 * half) s_p[threadIdx.x - 16 * half] = p, s_q[threadIdx.x - 16 * half] = q;
        __syncthreads();
        if (row < half) p += s_p[threadIdx.x], q += s_q[threadIdx.x];
        __syncthreads();
    }
    if (row || c >= C) return;
    if (a.dweight) set_param(a.dweight, a.affine_dtype, c, p);
    if (a.dbias) set_param(a.dbias, a.affine_dtype, c, q);
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------

static int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// N: values of a vector, or 1 where a period of rows would be wider than a workgroup
static NormShape shape_of(const tode_group_norm_args &a, int &N) {
    NormShape n = {};
    n.B = a.batch, n.S = a.positions, n.C = a.channels, n.G = a.n_groups, n.width = a.channels / a.n_groups;
    const int full = 16 / bytes_of(a.dtype), g = gcd(n.C, full);
    N = full;
    if (g == full || n.C / g > NORM_THREADS) {  // whole vectors in a row, or none at all
        if (g != full) N = 1;
        n.period = 1;
        const int vectors = n.C / N;
        n.V = vectors < 64 ? vectors : 64;
        n.chunks = (vectors + n.V - 1) / n.V;
    } else {
        n.period = full / g, n.V = n.C / g, n.chunks = 1;
    }
    n.chunk = n.period == 1 ? n.V * N : n.C;
    n.rows = (n.S + n.period - 1) / n.period;
    // about 2048 workgroups (eight a compute unit), of a batch of rows a thread or more
    const int lanes = NORM_THREADS / n.V;
    auto pieces = [&](long long least, long long wanted, long long &rows) {  // of whole batches of `least` rows a thread
        const long long batch = lanes * least, there = (n.rows + batch - 1) / batch;
        const long long each = wanted < there ? (there + wanted - 1) / wanted : 1;
        rows = each * batch;
        return (int)((there + each - 1) / each);
    };
    const long long wanted = 2048 / (n.B * n.chunks > 0 ? n.B * n.chunks : 1) + 1;
    n.apply_splits = pieces(4, wanted, n.apply_rows);
    n.splits = pieces(NORM_BATCH, wanted, n.split_rows);
    return n;
}
// A workgroup joins the sums of its groups' pieces by itself where its wavefronts have two groups each at most, of no more than 256 values:
// 2 us, where a launch of its own takes 4 to 8 us (40 groups a workgroup: 25 us against 5).
static bool joins_itself(const NormShape &n) { return n.chunk / n.width + 2 <= 2 * NORM_THREADS / 64 && (long long)n.splits * n.width <= 256; }

// The resident form, where a workgroup's part fits: at most `most` vectors a thread.  Its part is as many whole groups as fit and make whole
// vectors.
struct ResidentPlan {
    NormShape n;
    int threads, R;  // R = 0: it does not fit
    long long blocks;
};
static ResidentPlan resident_of(const tode_group_norm_args &a, int most) {
    ResidentPlan p = {};
    NormShape &n = p.n;
    n.B = a.batch, n.S = a.positions, n.C = a.channels, n.G = a.n_groups, n.width = a.channels / a.n_groups;
    const int N = 16 / bytes_of(a.dtype), g = gcd(n.C, N);
    n.splits = 1;
    if (g < N) {
        n.period = N / g, n.V = n.C / g, n.chunk = n.C, n.chunks = 1;
        n.rows = (n.S + n.period - 1) / n.period;
        if (n.V > NORM_ROW_VECTORS) return p;
    } else {
        n.period = 1, n.rows = n.S;
        const int base = n.width / gcd(n.width, N) * N, units = n.C / base;  // the least part, and how many of them there are
        // the widest part that fits and leaves 1024 workgroups or more, but 64 bytes in any case where they fit
        int best = 0;
        for (int m = 1; m <= units; ++m) {
            if (units % m) continue;
            const long long vectors = n.S * (m * (base / N));
            if (m * (base / N) > NORM_ROW_VECTORS || vectors > (long long)NORM_RESIDENT_THREADS * most) break;
            if (best && m * base * bytes_of(a.dtype) > 64 && n.B * (units / m) < 1024) break;
            best = m;
        }
        // (64 float32 samples of 32 channels in 8 groups: 16 384 positions, 16 bytes of each 92 us, in the general form 69; 8192 positions, 32 bytes
        // of each 32 us, in the general form 39)
        if (!best || best * base * bytes_of(a.dtype) < 32) return p;
        n.chunk = best * base, n.V = n.chunk / N, n.chunks = units / best;
    }
    p.blocks = (n.B >= 8 ? (n.B + 7) / 8 * 8 : n.B) * n.chunks;
    if (p.blocks > (1ll << 31) - 1) return p;
    if (n.period > 1) most /= 2;  // (which value is the last takes registers too)
    if (n.rows * n.period * n.C * bytes_of(a.dtype) > (1ll << 31)) return p;  // (a thread's place in the sample is a 32-bit number)
    // Too few workgroups for the chip, of more than 64 KiB each (us here and in the general form; float32, 64 channels in 8 groups: parts of 256 KiB, 64
    // workgroups 18.7 and 17.9, 128 workgroups 22.6 and 24.5; of 94 to 128 KiB, up to 64 workgroups 10 to 11 and 12 to 15, but rows of several positions, 5000 of 6
    // channels, 16.2 and 13.5, and float64 12.6 and 11.8; float16, 45 x 53 positions of 120 channels in 12, 186 KiB, 96 workgroups 26.5 and 25.0, 192
    // workgroups 28.7 and 32.9)
    if (p.blocks < 128 && n.rows * n.V > 4096) return p;
    // up to eight vectors a thread as long as there are two wavefronts a SIMD, else as many threads as there may be
    auto with = [&](int R) {
        const long long lanes = (n.rows + R - 1) / R, threads = (lanes * n.V + 63) / 64 * 64;
        if (threads > NORM_RESIDENT_THREADS) return false;
        p.threads = (int)threads, p.R = R;
        return true;
    };
    for (int R = most < 8 ? most : 8; R >= 1; R /= 2)
        if (with(R) && p.blocks * (p.threads / 64) >= 2048) return p;
    for (int R = 1; R <= most; R *= 2)
        if (with(R)) return p;
    p.R = 0;
    return p;
}

static int check(const tode_group_norm_args *a) {
    if (!a) return fail(TODE_E_INVALID, "null argument struct");
    if (!known_field_dtype(a->dtype)) return fail(TODE_E_INVALID, "unknown dtype %d", a->dtype);
    for (const int32_t type : {a->affine_dtype, a->modulation_dtype})
        if (type != a->dtype && (type != TODE_F32 || a->dtype == TODE_F64))
            return fail(TODE_E_INVALID, "parameters of dtype %d with data of dtype %d: they are of the data's type or float32", type, a->dtype);
    if (a->activation < TODE_ACT_NONE || a->activation > TODE_ACT_RELU) return fail(TODE_E_INVALID, "unknown activation %d", a->activation);
    if (a->batch < 0 || a->positions < 0 || a->channels < 1 || a->n_groups < 1 || a->channels % a->n_groups)
        return fail(TODE_E_INVALID, "bad sizes: batch=%lld positions=%lld channels=%d groups=%d", (long long)a->batch, (long long)a->positions, a->channels, a->n_groups);
    if (!(a->eps >= 0)) return fail(TODE_E_INVALID, "eps must not be negative");
    if (a->channels > (1 << 20) || a->n_groups > (1 << 20)) return fail(TODE_E_UNSUPPORTED, "more than 2^20 channels");
    if (a->batch > (1ll << 30) || a->positions > (1ll << 40) / a->channels || (a->batch > 0 && a->positions * a->channels > (1ll << 42) / a->batch))
        return fail(TODE_E_UNSUPPORTED, "more than 2^42 values");
    return TODE_OK;
}

struct NormScratch {  // in values of the statistics' type
    long long partial, statistics, products, means, total;
};
static NormScratch scratch_of(const tode_group_norm_args &a, const NormShape &n, bool backward) {
    NormScratch s = {};
    s.partial = 0;
    s.statistics = n.B * n.splits * n.C * 2;
    s.products = s.statistics + (backward ? 0 : n.B * n.G * 2);
    s.means = s.products + (backward ? n.B * n.C * 2 : 0);
    s.total = s.means + (backward ? n.B * n.G * 2 : 0);
    return s;
}

// LDS for two values of each group that a chunk touches
static size_t group_bytes(const NormShape &n, size_t size) { return 2 * size * (n.chunk / n.width + 2); }
static dim3 grid_of(const NormShape &n, int x) { return dim3(x, (unsigned)(n.B < 32768 ? n.B : 32768), (unsigned)((n.B + 32767) / 32768)); }

template <typename T, int R, bool WRAPPED> static int launch_resident(const tode_group_norm_args &a, const ResidentPlan &p, hipStream_t s) {
    typedef typename Wide<T>::type A;
    const NormShape &n = p.n;
    const int groups = n.chunk / n.width, waves = p.threads / 64;
    const size_t bytes = ((size_t)p.threads * Raw<T>::N + 2 * groups) * sizeof(A) + (groups > waves ? groups : waves) * sizeof(double);
    static_assert(((NORM_RESIDENT_THREADS + 2 * NORM_ROW_VECTORS) * sizeof(A) + NORM_ROW_VECTORS * sizeof(double)) * Raw<T>::N <= 64 * 1024, "what a launch may have without asking");
    hipLaunchKernelGGL((norm_resident_kernel<T, R, WRAPPED>), grid_line(p.blocks), dim3(p.threads), bytes, s, a, n);
    return check_hip(hipGetLastError(), "tode_group_norm launch");
}
template <typename T, int R, bool WRAPPED> static int launch_resident_backward(const tode_group_norm_args &a, const ResidentPlan &p, hipStream_t s) {
    typedef typename Wide<T>::type A;
    const NormShape &n = p.n;
    const int cols = n.V * Raw<T>::N, pieces = p.threads / cols > 1 ? p.threads / cols : 1;
    const size_t bytes = ((size_t)2 * p.threads * Raw<T>::N + 2 * pieces * cols + 2 * (n.chunk / n.width)) * sizeof(A);
    static_assert((2 * NORM_RESIDENT_THREADS + 4 * NORM_ROW_VECTORS) * Raw<T>::N * sizeof(A) <= 64 * 1024, "what a launch may have without asking");
    A *const products = (A *)a.workspace;
    hipLaunchKernelGGL((norm_resident_backward_kernel<T, R, WRAPPED>), grid_line(p.blocks), dim3(p.threads), bytes, s, a, n, products);
    if (!a.affine_per_sample && (a.dweight || a.dbias))
        hipLaunchKernelGGL((norm_affine_gradients_kernel<A>), dim3((n.C + 15) / 16), dim3(1024), 0, s, a, n.B, n.C, (const A *)products);
    return check_hip(hipGetLastError(), "tode_group_norm_backward launch");
}
#define TODE_NORM_R(CALL, R) return p.n.period > 1 ? CALL<T, R, true>(a, p, s) : CALL<T, R, false>(a, p, s)
template <typename T> static int forward_resident(const tode_group_norm_args &a, const ResidentPlan &p, hipStream_t s) {
    switch (p.R) {
        case 1: TODE_NORM_R(launch_resident, 1);
        case 2: TODE_NORM_R(launch_resident, 2);
        case 4: TODE_NORM_R(launch_resident, 4);
        case 8: TODE_NORM_R(launch_resident, 8);
        case 16: TODE_NORM_R(launch_resident, 16);
        default: return launch_resident<T, 32, false>(a, p, s);  // (rows of several positions take half as many)
    }
}
template <typename T> static int backward_resident(const tode_group_norm_args &a, const ResidentPlan &p, hipStream_t s) {
    switch (p.R) {
        case 1: TODE_NORM_R(launch_resident_backward, 1);
        case 2: TODE_NORM_R(launch_resident_backward, 2);
        case 4: TODE_NORM_R(launch_resident_backward, 4);
        default: return launch_resident_backward<T, 8, false>(a, p, s);
    }
}
#undef TODE_NORM_R

template <typename T, int N> static int forward_as(tode_group_norm_args a, const NormShape &n, hipStream_t s) {
    typedef typename Wide<T>::type A;
    const NormScratch at = scratch_of(a, n, false);
    A *const w = (A *)a.workspace;
    hipLaunchKernelGGL((norm_statistics_kernel<T, N>), grid_of(n, n.chunks * n.splits), dim3(NORM_THREADS), 0, s, a, n, w);
    const bool itself = joins_itself(n);
    if (!itself) {
        if (!a.mean) a.mean = w + at.statistics, a.rstd = w + at.statistics + n.B * n.G;
        hipLaunchKernelGGL((norm_join_statistics_kernel<A>), grid_of(n, n.G), dim3(64), 0, s, n, w, (A)a.eps, (A *)a.mean, (A *)a.rstd);
    }
    hipLaunchKernelGGL((norm_apply_kernel<T, N>), grid_of(n, n.chunks * n.apply_splits), dim3(NORM_THREADS), itself ? group_bytes(n, sizeof(A)) : 0, s, a, n, itself ? w : nullptr);
    return check_hip(hipGetLastError(), "tode_group_norm launch");
}

template <typename T, int N> static int backward_as(const tode_group_norm_args &a, NormShape n, hipStream_t s) {
    typedef typename Wide<T>::type A;
    const NormScratch at = scratch_of(a, n, true);
    A *const w = (A *)a.workspace;
    hipLaunchKernelGGL((norm_products_kernel<T, N>), grid_of(n, n.chunks * n.splits), dim3(NORM_THREADS), 0, s, a, n, w);
    const bool itself = joins_itself(n);
    if (!itself) hipLaunchKernelGGL((norm_join_products_kernel<A>), grid_of(n, n.G), dim3(64), 0, s, a, n, w, w + at.products, w + at.means);
    if (a.dx || itself) {
        if (!a.dx) n.apply_splits = 1;
        hipLaunchKernelGGL((norm_apply_backward_kernel<T, N>), grid_of(n, n.chunks * n.apply_splits), dim3(NORM_THREADS), itself ? group_bytes(n, sizeof(A)) : 0, s, a, n, itself ? w : nullptr,
                           w + at.products, w + at.means);
    }
    if (!a.affine_per_sample && (a.dweight || a.dbias))
        hipLaunchKernelGGL((norm_affine_gradients_kernel<A>), dim3((n.C + 15) / 16), dim3(1024), 0, s, a, n.B, n.C, w + at.products);
    return check_hip(hipGetLastError(), "tode_group_norm_backward launch");
}

// gradients of parameters that no value reaches
__global__ void __launch_bounds__(256) norm_zero_kernel(void *p, int dtype, long long n) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += 256ll * gridDim.x) set_param<double>(p, dtype, i, 0);
}

}  // namespace tode

extern "C" {

using namespace tode;

int64_t tode_group_norm_workspace_bytes(const tode_group_norm_args *a, int32_t backward) {
    if (int rc = check(a)) return rc;
    if (a->batch == 0 || a->positions == 0) return 0;
    const int size = a->dtype == TODE_F64 ? 8 : 4;
    if (resident_of(*a, backward ? NORM_MOST_BACKWARD : NORM_MOST).R) return backward ? 2 * a->batch * a->channels * size : 0;
    int N;
    const NormShape n = shape_of(*a, N);
    return scratch_of(*a, n, backward != 0).total * size;
}

#define TODE_NORM_RESIDENT(CALL, a, p, s)             \
    switch ((a)->dtype) {                             \
        case TODE_F32: return CALL<float>(*a, p, s);  \
        case TODE_F64: return CALL<double>(*a, p, s); \
        case TODE_BF16: return CALL<bf16>(*a, p, s);  \
        default: return CALL<f16>(*a, p, s);          \
    }
#define TODE_NORM(CALL, a, n, s)                                                            \
    switch ((a)->dtype) {                                                                   \
        case TODE_F32: return N == 1 ? CALL<float, 1>(*a, n, s) : CALL<float, 4>(*a, n, s);   \
        case TODE_F64: return N == 1 ? CALL<double, 1>(*a, n, s) : CALL<double, 2>(*a, n, s); \
        case TODE_BF16: return N == 1 ? CALL<bf16, 1>(*a, n, s) : CALL<bf16, 8>(*a, n, s);    \
        default: return N == 1 ? CALL<f16, 1>(*a, n, s) : CALL<f16, 8>(*a, n, s);             \
    }

int tode_group_norm(const tode_group_norm_args *a, void *stream) {
    if (int rc = check(a)) return rc;
    if (a->batch == 0 || a->positions == 0) return TODE_OK;
    if (!a->x || !a->y) return fail(TODE_E_INVALID, "null pointer");
    if (!a->mean != !a->rstd) return fail(TODE_E_INVALID, "mean and rstd are written together");
    const int64_t need = tode_group_norm_workspace_bytes(a, 0);
    if (a->workspace_bytes < need || (need > 0 && !a->workspace)) return fail(TODE_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)need);
    const hipStream_t s = (hipStream_t)stream;
    const ResidentPlan p = resident_of(*a, NORM_MOST);
    if (p.R) TODE_NORM_RESIDENT(forward_resident, a, p, s)
    int N;
    const NormShape n = shape_of(*a, N);
    TODE_NORM(forward_as, a, n, s)
}

int tode_group_norm_backward(const tode_group_norm_args *a, void *stream) {
    if (int rc = check(a)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    if (a->batch == 0 || a->positions == 0) {
        const long long per_sample = (long long)a->batch * a->channels, affine = a->affine_per_sample ? per_sample : a->channels;
        void *const out[4] = {a->dweight, a->dbias, a->dscale, a->dshift};
        for (int i = 0; i < 4; ++i)
            if (out[i] && (i < 2 ? affine : per_sample) > 0)
                hipLaunchKernelGGL(norm_zero_kernel, dim3(64), dim3(256), 0, s, out[i], i < 2 ? a->affine_dtype : a->modulation_dtype, i < 2 ? affine : per_sample);
        return check_hip(hipGetLastError(), "tode_group_norm_backward launch");
    }
    if (!a->x || !a->dy || !a->mean || !a->rstd) return fail(TODE_E_INVALID, "null pointer");
    const int64_t need = tode_group_norm_workspace_bytes(a, 1);
    if (a->workspace_bytes < need || (need > 0 && !a->workspace)) return fail(TODE_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)need);
    const ResidentPlan p = resident_of(*a, NORM_MOST_BACKWARD);
    if (p.R) TODE_NORM_RESIDENT(backward_resident, a, p, s)
    int N;
    const NormShape n = shape_of(*a, N);
    TODE_NORM(backward_as, a, n, s)
}

}  // extern "C"
