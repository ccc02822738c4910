// Cross attention on the matrix cores: tiles, operands and the rows of a head group, shared by the forward kernels
// (tode_attention.hip) and the backward ones (tode_attention_backward.hip).
//
// Everything is computed in tiles of 32 x 32 with the operand that a wavefront keeps (its 32 "columns") on the right and the one that
// streams by (32 "rows" at a time, in LDS) on the left, so that the result of one product is the right operand of the next as it
// lies in the registers: of a tile M[row][column], lane l holds column l % 32 and the rows 8 (r / 4) + 4 (l / 32) + r % 4, r = 0 .. 15, and a
// product summed over the rows may take them in any order as long as both operands take the same.
//   forward, gradient of q:  columns are queries, rows keys;  gradients of k and v: columns are keys, rows queries.
// The G = H / Hkv heads that share a head of keys are rows (columns) of one problem: row r is query r / G of head r % G of the group.
#pragma once
#include <type_traits>

#include "tode_field.h"

namespace tode {

typedef float acc16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int ATT_TILE = 32;
constexpr float LOG2E = 1.44269504088896340736f;

// One 32 x 32 product over the 16 (float32: 8) values that the two operands' 16 bytes a lane hold: value e of lane half h is number
// N h + e on both sides.
__device__ __forceinline__ acc16 mma(const Raw<bf16> &a, const Raw<bf16> &b, acc16 c) {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a.w), __builtin_bit_cast(x8, b.w), c, 0, 0, 0);
}
__device__ __forceinline__ acc16 mma(const Raw<f16> &a, const Raw<f16> &b, acc16 c) {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a.w), __builtin_bit_cast(x8, b.w), c, 0, 0, 0);
}
__device__ __forceinline__ acc16 mma(const Raw<float> &a, const Raw<float> &b, acc16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w[i]), __uint_as_float(b.w[i]), c, 0, 0, 0);
    return c;
}

// Weights are taken 2^12 times as large for float16, whose steps stop shrinking at 2^-14: those of a softmax over thousands of keys are
// smaller.
template <typename T> inline constexpr float WEIGHT_BITS = 0;
template <> inline constexpr float WEIGHT_BITS<f16> = 12;
template <typename T> inline constexpr float WEIGHT_UNIT = 1;
template <> inline constexpr float WEIGHT_UNIT<f16> = 1.0f / 4096;

__device__ __forceinline__ acc16 zero16() {
    acc16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0;
    return z;
}

// An LDS tile: 32 rows of DP values, 32 bytes between them (8 of 64 banks: the 16-byte reads of eight rows and the transposed
// reads of four touch every bank once).
template <typename T, int DP> struct Tile {
    static constexpr int STRIDE = DP + 32 / (int)sizeof(T), N = Raw<T>::N, NC = DP / (2 * N), NT = DP / 32;
    static constexpr int VALUES = ATT_TILE * STRIDE;
};

// A row's values [first, first + N), zeros from D on.
template <typename T> __device__ __forceinline__ Raw<T> row_part(const T *row, int first, int D) {
    Raw<T> r;
    r.zero();
    if (!row) return r;
    if (first + Raw<T>::N <= D)
        r.load(row + first);
    else if (first < D) {
        T v[Raw<T>::N];
#pragma unroll
        for (int i = 0; i < Raw<T>::N; ++i) v[i] = first + i < D ? row[first + i] : (T)0.0f;
        __builtin_memcpy(r.w, v, 16);
    }
    return r;
}

// What a lane holds of its column (or row) of DP values: chunk c has the values 2 N c + N h + e.
template <typename T, int DP> struct Operand {
    Raw<T> c[Tile<T, DP>::NC];
    __device__ __forceinline__ void load(const T *row, int D, int h) {
        if (D == DP && row) {
#pragma unroll
            for (int i = 0; i < Tile<T, DP>::NC; ++i) c[i].load(row + (2 * i + h) * Raw<T>::N);
            return;
        }
#pragma unroll
        for (int i = 0; i < Tile<T, DP>::NC; ++i) c[i] = row_part(row, (2 * i + h) * Raw<T>::N, D);
    }
    // The same of a row that is there, in memory, for all lanes: zeros where it does not count.  (The lanes stay together on the way: a branch of some
    // lanes would have the compiler spill what it loads within it, where the registers are as short as for 256 values.)
    __device__ __forceinline__ void load_if(const T *row, int D, int h, bool counts) {
        if (D == DP) {
#pragma unroll
            for (int i = 0; i < Tile<T, DP>::NC; ++i) c[i].load(row + (2 * i + h) * Raw<T>::N);
        } else {
#pragma unroll
            for (int i = 0; i < Tile<T, DP>::NC; ++i) c[i] = row_part(row, (2 * i + h) * Raw<T>::N, D);
        }
#pragma unroll
        for (int i = 0; i < Tile<T, DP>::NC; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) c[i].w[k] = counts ? c[i].w[k] : 0;
    }
    // ... of the other sign where the scale is negative, so that larger scores have larger weights
    __device__ __forceinline__ void load_signed(const T *row, int D, int h, bool minus) {
        load(row, D, h);
        if (minus)
#pragma unroll
            for (int i = 0; i < Tile<T, DP>::NC; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) c[i].w[k] ^= sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
    }
};

template <typename T> __device__ __forceinline__ Raw<T> lds_part(const T *p) {
    Raw<T> r;
    const uint4 v = *(const uint4 *)p;
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    return r;
}

// tile [row][d] times columns: M[row][column], summed over d
template <typename T, int DP> __device__ __forceinline__ acc16 rows_times(const T *tile, const Operand<T, DP> &columns, int lane) {
    typedef Tile<T, DP> L;
    acc16 s = zero16();
    const T *p = tile + (lane % 32) * L::STRIDE + (lane / 32) * L::N;
#pragma unroll
    for (int i = 0; i < L::NC; ++i) s = mma(lds_part(p + 2 * i * L::N), columns.c[i], s);
    return s;
}

// out[d][column] += sum over the tile's rows of tile[row][d] m[row][column], m as a product left it in the registers; for
// the 16-bit types rounded to them (out: DP / 32 tiles of 32 values of d)
template <int DP> __device__ __forceinline__ void transposed_times(const float *tile, const float *m, acc16 *out, int lane) {
    typedef Tile<float, DP> L;
    const float *p = tile + 4 * (lane / 32) * L::STRIDE + lane % 32;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(p[(8 * (r / 4) + r % 4) * L::STRIDE + 32 * t], m[r], out[t], 0, 0, 0);
}
// Sixteen lanes read four rows of 16 values and get one value of d of the four rows each; twice.
template <typename T> __device__ __forceinline__ Raw<T> transposed_part(const T *lo, const T *hi) {
    typedef __attribute__((address_space(3))) s16x4 *lds;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)lo), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)hi);
    Raw<T> r;
    __builtin_memcpy(r.w, &x, 8);
    __builtin_memcpy(r.w + 2, &y, 8);
    return r;
}
template <int DP, typename T> __device__ __forceinline__ void transposed_times(const T *tile, const float *m, acc16 *out, int lane) {
    typedef Tile<T, DP> L;
    const int h = lane / 32, block = (lane / 16) % 2, i = lane % 16;
    const T *p = tile + (4 * h + i / 4) * L::STRIDE + 16 * block + 4 * (i % 4);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        Raw<T> b;
        pack(b, m + 8 * k);
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[t] = mma(transposed_part(p + 16 * k * L::STRIDE + 32 * t, p + (16 * k + 8) * L::STRIDE + 32 * t), b, out[t]);
    }
}

// Copies 32 rows into an LDS tile by `threads` threads; row(i): its address, or null for a row of zeros.
template <typename T, int DP, typename Row> __device__ __forceinline__ void stage(T *tile, int thread, int threads, int D, Row row) {
    typedef Tile<T, DP> L;
    constexpr int PARTS = DP / L::N;
    for (int k = thread; k < ATT_TILE * PARTS; k += threads) {
        const int i = k / PARTS, part = k % PARTS;
        const Raw<T> r = row_part(row(i), part * L::N, D);
        *(uint4 *)(tile + i * L::STRIDE + part * L::N) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    }
}

// The problem of one sample's head group.
template <typename T> struct Group {
    long long b;
    int head, G, shift, D, rows, keys, length;  // rows = queries * G; shift: log2 G, or -1
    const tode_cross_attention_args &a;
    __device__ __forceinline__ Group(const tode_cross_attention_args &args, long long group) : a(args) {
        b = group / a.kv_heads, head = (int)(group % a.kv_heads), G = a.heads / a.kv_heads, D = a.head_dim;
        shift = (G & (G - 1)) ? -1 : __ffs(G) - 1;
        rows = (int)(a.queries * G), keys = (int)a.keys, length = keys;
        if (a.lengths) {
            const long long n = a.lengths_are_64 ? ((const int64_t *)a.lengths)[b] : ((const int32_t *)a.lengths)[b];
            length = (int)(n < 0 ? 0 : n > keys ? keys : n);
        }
    }
    __device__ __forceinline__ bool allowed(int key) const { return key < length && (!a.mask || a.mask[b * a.mask_stride + key]); }
    // The weight of a single key is 1 whatever its score: the gradient of scores is zero, and not what rounding leaves of a difference of equals.
    // With a mask the keys of the sample are counted until there are two: most often the first step ends it (64 samples of 64 queries over 200 keys,
    // float32, forward and backward: 68.8 us, 66.8 without the count).  Called by whole wavefronts.
    __device__ __forceinline__ bool scores_matter(int lane) const {
        if (!a.mask || length < 2) return length > 1;
        const uint8_t *const mask = a.mask + b * a.mask_stride;
        int seen = 0;
        for (int first = 0; first < length && seen < 2; first += 512) {
            int k[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) k[u] = mask[min(first + 64 * u + lane, length - 1)];  // (eight loads under way)
#pragma unroll
            for (int u = 0; u < 8; ++u) seen += __popcll(__ballot(k[u] && first + 64 * u + lane < length));
        }
        return seen > 1;
    }
    // 32 keys from `first` on, one bit each
    __device__ __forceinline__ unsigned allowed_bits(int first, int lane) const {
        return (unsigned)__ballot(lane < 32 && allowed(first + lane));
    }
    __device__ __forceinline__ int query_of(int r) const { return shift >= 0 ? r >> shift : r / G; }
    // element offsets of row r in an array [B, queries, H, ...] with these strides, and in one that is contiguous
    __device__ __forceinline__ long long at(int r, long long sb, long long sr, long long sh) const {
        const int i = query_of(r);
        return b * sb + i * sr + (head * G + r - i * G) * sh;
    }
    __device__ __forceinline__ long long flat(int r) const {
        const int i = query_of(r);
        return (b * a.queries + i) * a.heads + (head * G + r - i * G);
    }
    __device__ __forceinline__ const T *query(int r) const { return r < rows ? (const T *)a.q + at(r, a.q_strides[0], a.q_strides[1], a.q_strides[2]) : nullptr; }
    __device__ __forceinline__ const T *key(int k) const { return (const T *)a.k + b * a.k_strides[0] + k * a.k_strides[1] + head * a.k_strides[2]; }
    __device__ __forceinline__ const T *value(int k) const { return (const T *)a.v + b * a.v_strides[0] + k * a.v_strides[1] + head * a.v_strides[2]; }
    __device__ __forceinline__ const T *cotangent(int r) const { return r < rows ? (const T *)a.grad_out + at(r, a.grad_strides[0], a.grad_strides[1], a.grad_strides[2]) : nullptr; }
    __device__ __forceinline__ const T *output(int r, const void *of) const { return r < rows && of ? (const T *)of + flat(r) * D : nullptr; }
};

// The row of register r in lane half h.
__device__ __forceinline__ int row_of(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

// Other lane half's value.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// A column's 4 neighbouring values of d out of a lane's registers, rounded and written: out[t] holds d = 32 t + row_of(r, h).
template <typename T, int NT> __device__ __forceinline__ void store_column(T *row, const acc16 *out, int D, int h) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * t + 8 * q + 4 * h;
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)out[t][4 * q + e];
            if (d + 4 <= D)
                __builtin_memcpy(row + d, v, sizeof(v));
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < D) row[d + e] = v[e];
        }
}

// A product that is rounded to T twice -- to be written, and for what that takes off -- and has to be the same number both times: the compiler
// may take a multiplication and the rounding to float16 behind it as one operation with a single rounding, the first time and not the second, and
// near the middle between two steps the two then differ by a whole one.
template <typename T> __device__ __forceinline__ float settled(float v) {
    if (std::is_same<T, f16>::value) asm("" : "+v"(v));
    return v;
}

// What rounding to T takes off.
template <typename T, int NT> __device__ __forceinline__ void keep_low(acc16 *out) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[t][r] -= (float)(T)out[t][r];
}

// A row's sums of weights l, times 2^m: what it divides by and its log-sum.  Zeros and infinity where no key was met; a NaN stays one, in
// the gradients as well.
__device__ __forceinline__ float reciprocal(float l) { return l == 0 ? 0 : 1 / l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0 ? INFINITY : m + log2f(l); }

// The power of two that a column's score gradients are taken times ahead of their rounding to T.  They have the size of the
// cotangent, and float16 has neither its small values (steps stop shrinking at 2^-14) nor its large ones: the largest so far of a column is brought
// to 2^8, and its sums to another power once one reaches 2^15, as a softmax does with its maximum.  bfloat16 has float32's range.
template <typename T, int NT> struct ColumnUnit {
    __device__ __forceinline__ void fit(float *, acc16 *) {}
    __device__ __forceinline__ float undo() const { return 1; }
};
template <int NT> struct ColumnUnit<f16, NT> {
    unsigned exponent = 0;  // of the power, as float32 has it (127: 1); 0: none yet, all values were zeros
    static __device__ __forceinline__ float power(unsigned e) { return __uint_as_float(e << 23); }
    __device__ __forceinline__ void fit(float *m, acc16 *sum) {
        float top = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(m[r]));
        top = fmaxf(top, other_half(top));
        const bool grown = exponent ? top * power(exponent) >= 32768.0f : top > 0;
        if (__any(grown)) {
            const int next = min(max(262 - (int)(__float_as_uint(top) >> 23), 4), 250);  // (infinities stay what they are)
            const float shrink = grown && exponent ? power(next) * power(254 - exponent) : 1;
            exponent = grown ? next : exponent;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[t][r] *= shrink;
        }
        const float f = power(exponent);
#pragma unroll
        for (int r = 0; r < 16; ++r) m[r] *= f;
    }
    __device__ __forceinline__ float undo() const { return exponent ? power(254 - exponent) : 1; }
};

// Orders one wavefront's LDS traffic where its lanes hand values to each other.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// Which of `tiles` of which head group workgroup number n has.  Workgroups go round the eight XCDs, each with an L2 of its own, so those
// that read the same keys get numbers that are eight apart.  Samples whose keys are small for an L2 stay on one XCD with all their heads, the
// heads of a tile side by side: what lies next to each other in memory is read and written at the same time (512 samples of
// 256 x 4 x 32 over 60 keys, bfloat16: 21.8 us, with the heads on eight XCDs 25.3; gradients of 32 samples of 4096 x 8 x 64 over 96 keys: 355 against
// 384; beyond the bound, of 131 072 keys' values to a million, within 2 % either way).  False: behind the last group.
__device__ __forceinline__ bool place(const tode_cross_attention_args &a, unsigned n, unsigned tiles, long long &group, int &tile) {
    const unsigned heads = a.kv_heads, xcd = n % 8, i = n / 8;
    if (a.batch >= 8 && a.keys * a.kv_heads * a.head_dim <= 262144) {
        const unsigned round = i / (tiles * heads), rest = i - round * (tiles * heads), t = rest / heads;
        tile = (int)t, group = (round * 8ll + xcd) * heads + (rest - t * heads);
        return round * 8ll + xcd < a.batch;
    }
    const long long groups = a.batch * a.kv_heads;
    if (groups >= 8) {
        const unsigned round = i / tiles;
        group = round * 8ll + xcd, tile = (int)(i - round * tiles);
        return group < groups;
    }
    const unsigned g = n / tiles;
    group = g, tile = (int)(n - g * tiles);
    return group < groups;
}
// How many workgroups that takes.
inline long long placed(const tode_cross_attention_args &a, int tiles) {
    const long long groups = a.batch * a.kv_heads;
    if (a.batch >= 8 && a.keys * a.kv_heads * a.head_dim <= 262144) return (a.batch + 7) / 8 * 8 * a.kv_heads * tiles;
    return (groups >= 8 ? (groups + 7) / 8 * 8 : groups) * tiles;
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------

// More than 64 KiB of LDS is to be asked for, kernel by kernel.
inline int allow_lds(const void *kernel, int bytes) {
    return bytes > 64 * 1024 ? check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "hipFuncSetAttribute") : TODE_OK;
}

// The sources are compiled once for each element type.
#define TODE_ATT_JOIN_(name, suffix) name##_##suffix
#define TODE_ATT_JOIN(name, suffix) TODE_ATT_JOIN_(name, suffix)
#define TODE_ATT_NAME(name) TODE_ATT_JOIN(name, TODE_ATT_TYPE)
#define TODE_ATT_DECLARE(type)                                                             \
    int attention_forward_##type(const tode_cross_attention_args &a, hipStream_t s);       \
    int64_t attention_forward_bytes_##type(const tode_cross_attention_args &a);            \
    int attention_backward_##type(const tode_cross_attention_args &a, hipStream_t s);      \
    int64_t attention_backward_bytes_##type(const tode_cross_attention_args &a);
TODE_ATT_DECLARE(float)
TODE_ATT_DECLARE(bf16)
TODE_ATT_DECLARE(f16)
#undef TODE_ATT_DECLARE

}  // namespace tode
