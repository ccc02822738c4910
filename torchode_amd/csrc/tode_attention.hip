// Cross attention, forward: for the 32 queries that a wavefront keeps, one pass over the keys with the running maximum and sum of the
// softmax.  A score is c q.k; p = 2^(s - m) with s in units of log 2; out = (sum p v) / (sum p), in float32.
// The matrix instructions take both operands in one type, so for the 16-bit ones p is rounded to it ahead of the product with v (their sum is not): an
// output is off by 0.0023 of its size in bfloat16 (4 samples of 4096 queries over 4096 keys), where its own rounding alone is 0.0017.  Weights in two parts
// would spare that for half as many products again.  Up to eight rows a head of keys take the vector units, where p stays float32.
#include "tode_attention.h"

#ifdef TODE_ATT_TYPE

namespace tode {

constexpr int ATTENTION_SPLITS = 1024;  // pieces of a row's keys at most

// A wavefront's 32 columns written through its own LDS tile, 16 bytes a lane and side by side: out[t] of 32 t + row_of(r, h) of column lane % 32.
template <typename T, int DP> __device__ __forceinline__ void write_columns(const Group<T> &p, void *of, T *own, const acc16 *out, int row0, int lane) {
    typedef Tile<T, DP> L;
    constexpr int PARTS = DP / L::N;
    wave_sync();
    store_column<T, L::NT>(own + (lane % 32) * L::STRIDE, out, DP, lane / 32);
    wave_sync();
#pragma unroll 1
    for (int k = lane; k < 32 * PARTS; k += 64) {
        const int r = k / PARTS, part = k % PARTS * L::N, to = row0 + r;
        if (to >= p.rows || part >= p.D) continue;
        const Raw<T> v = lds_part(own + r * L::STRIDE + part);
        T *const at = (T *)of + p.flat(to) * p.D + part;
        if (part + L::N <= p.D)
            v.store(at);
        else {
            T x[L::N];
            __builtin_memcpy(x, v.w, 16);
#pragma unroll
            for (int e = 0; e < L::N; ++e)
                if (part + e < p.D) at[e] = x[e];
        }
    }
}

// ------------------------------------------------------------------------------------------
// 16-bit types, many keys: four wavefronts of 32 CT queries each share tiles of 64 (D = 256: 32) keys
// ------------------------------------------------------------------------------------------

// A tile is loaded into registers while the one before is worked on, and lies in one of two places in LDS, so that one barrier a tile is
// enough.  CT: a value of a tile goes from LDS to a wavefront once for all of its 32 CT queries.
template <typename T, int DP, int CT>
__global__ void __launch_bounds__(256, CT * DP <= 128 ? 2 : 1) attention_tiles_kernel(tode_cross_attention_args a, int tiles, int splits, float *partial) {
    typedef Tile<T, DP> L;
    constexpr int SUBS = DP > 128 ? 1 : 2, KEYS = 32 * SUBS, PARTS = DP / L::N, LOADS = KEYS * PARTS / 256, SIZE = KEYS * L::STRIDE;
    static_assert(KEYS * PARTS % 256 == 0, "whole loads");
    extern __shared__ __align__(16) char lds[];
    T *const buffer = (T *)lds;  // [2][k, v][KEYS][STRIDE]
    long long group;
    int tile;
    if (!place(a, block_number(), tiles * splits, group, tile)) return;
    const int split = tile % splits;
    tile /= splits;
    const Group<T> p(a, group);
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32, row0 = (tile * 4 + wave) * 32 * CT;
    const float c = fmaxf(fabsf((float)a.scale) * LOG2E, 1e-37f);  // (not 0: infinity times it stays what it is)
    Operand<T, DP> q[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) q[ct].load_signed(p.query(row0 + 32 * ct + lane % 32), p.D, h, a.scale < 0);
    acc16 out[CT][L::NT];
    float m[CT], l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        m[ct] = -INFINITY, l[ct] = 0;
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[ct][t] = zero16();
    }
    const int key_tiles = (p.length + KEYS - 1) / KEYS, per_split = (key_tiles + splits - 1) / splits;
    const int first = split * per_split, last = min(first + per_split, key_tiles);
    const T *const keys = p.key(0), *const values = p.value(0);
    Raw<T> k_next[LOADS], v_next[LOADS];
    // places in a tile, and which of them are values at all; tiles of which all keys may be looked at need no more
    int k_offset[LOADS], v_offset[LOADS], inside = 0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int k = thread + 256 * i, row = k / PARTS, part = k % PARTS * L::N;
        k_offset[i] = row * (int)a.k_strides[1] + part, v_offset[i] = row * (int)a.v_strides[1] + part;
        inside |= (part < p.D) << i;
        k_next[i].zero(), v_next[i].zero();
    }
    const bool simple = !a.mask && p.D % L::N == 0 && a.k_strides[1] < (1 << 24) && a.v_strides[1] < (1 << 24);
    auto fetch = [&](int t) {
        if (simple && KEYS * (t + 1) <= p.length) {
            const T *const k_from = keys + (long long)KEYS * t * a.k_strides[1], *const v_from = values + (long long)KEYS * t * a.v_strides[1];
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (inside >> i & 1) k_next[i].load(k_from + k_offset[i]);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (inside >> i & 1) v_next[i].load(v_from + v_offset[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int k = thread + 256 * i, row = KEYS * t + k / PARTS, part = k % PARTS * L::N;
            const bool there = p.allowed(row);
            k_next[i] = row_part(there ? keys + row * a.k_strides[1] : (const T *)nullptr, part, p.D);
            v_next[i] = row_part(there ? values + row * a.v_strides[1] : (const T *)nullptr, part, p.D);
        }
    };
    if (first < last) fetch(first);
    for (int t = first; t < last; ++t) {
        T *const k_tile = buffer + (t & 1) * 2 * SIZE, *const v_tile = k_tile + SIZE;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int k = thread + 256 * i, at = k / PARTS * L::STRIDE + k % PARTS * L::N;
            *(uint4 *)(k_tile + at) = make_uint4(k_next[i].w[0], k_next[i].w[1], k_next[i].w[2], k_next[i].w[3]);
            *(uint4 *)(v_tile + at) = make_uint4(v_next[i].w[0], v_next[i].w[1], v_next[i].w[2], v_next[i].w[3]);
        }
        __syncthreads();
        if (t + 1 < last) fetch(t + 1);
        if (row0 >= p.rows) continue;  // (a wavefront behind the last row only helps to load)
        acc16 s[SUBS][CT];
        const T *const k_at = k_tile + (lane % 32) * L::STRIDE + h * L::N;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) s[sub][ct] = zero16();
#pragma unroll
            for (int i = 0; i < L::NC; ++i) {
                const Raw<T> k = lds_part(k_at + 32 * sub * L::STRIDE + 2 * i * L::N);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[sub][ct] = mma(k, q[ct].c[i], s[sub][ct]);
            }
        }
        if (a.mask || KEYS * (t + 1) > p.length) {
            const unsigned long long bits = __ballot(p.allowed(KEYS * t + lane)) >> (4 * h);
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                const unsigned mine = (unsigned)(bits >> (32 * sub));
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) s[sub][ct][r] = mine >> row_of(r, 0) & 1 ? s[sub][ct][r] : -INFINITY;
            }
        }
        Raw<T> w[CT][2 * SUBS];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float top = s[0][ct][0];
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(fmaxf(top, s[0][ct][r]), s[SUBS - 1][ct][r]);
            top = fmaf(fmaxf(top, other_half(top)), c, -WEIGHT_BITS<T>);
            // weights may grow to 2^8 (float16: 2^3, on top of its 2^12) before the sums are brought to a new base
            const bool grown = top > m[ct] + (WEIGHT_BITS<T> > 0 ? 3.0f : 8.0f) || m[ct] == -INFINITY;
            if (__ballot(grown)) {
                const float next = fmaxf(m[ct], top), shrink = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - next);
                m[ct] = next, l[ct] *= shrink;
#pragma unroll
                for (int t2 = 0; t2 < L::NT; ++t2)
#pragma unroll
                    for (int r = 0; r < 16; ++r) out[ct][t2][r] *= shrink;
            }
            const float base = m[ct] == -INFINITY ? 0 : m[ct];
            float sum[SUBS] = {};
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(s[sub][ct][r], c, -base)), sum[sub] += x[r];
                pack(w[ct][2 * sub], x);
                pack(w[ct][2 * sub + 1], x + 8);
            }
            l[ct] += SUBS > 1 ? sum[0] + sum[SUBS - 1] : sum[0];
        }
        const int i = lane % 16;
        const T *const v_at = v_tile + (4 * h + i / 4) * L::STRIDE + 16 * (lane / 16 % 2) + 4 * (i % 4);
#pragma unroll
        for (int k = 0; k < 2 * SUBS; ++k)
#pragma unroll
            for (int t2 = 0; t2 < L::NT; ++t2) {
                const Raw<T> v = transposed_part(v_at + 16 * k * L::STRIDE + 32 * t2, v_at + (16 * k + 8) * L::STRIDE + 32 * t2);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) out[ct][t2] = mma(v, w[ct][k], out[ct][t2]);
            }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) l[ct] += other_half(l[ct]);

    if (splits > 1) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int row = row0 + 32 * ct + lane % 32;
            if (row >= p.rows) continue;
            float *const to = partial + ((group * splits + split) * p.rows + row) * (p.D + 2);
            if (h == 0) to[0] = m[ct], to[1] = l[ct];
            store_column<float, L::NT>(to + 2, out[ct], p.D, h);
        }
        return;
    }
    // by way of LDS, so that a row is written 16 bytes a lane and side by side
    __syncthreads();
    T *const own = buffer + wave * 32 * L::STRIDE;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int row = row0 + 32 * ct + lane % 32;
        const float f = reciprocal(l[ct]);
        if (a.lse && h == 0 && row < p.rows) a.lse[p.flat(row)] = log_sum(m[ct], l[ct]);
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[ct][t][r] = settled<T>(out[ct][t][r] * f);
        write_columns<T, DP>(p, a.out, own, out[ct], row0 + 32 * ct, lane);
        if (a.out_low) keep_low<T, L::NT>(out[ct]), write_columns<T, DP>(p, a.out_low, own, out[ct], row0 + 32 * ct, lane);
    }
}

// ------------------------------------------------------------------------------------------
// many rows, few keys (up to 32 SUBS): all keys stay in LDS, and every wavefront goes over rows of its own
// ------------------------------------------------------------------------------------------

// What is left is to read q and to write the output.  A score of every key is in registers at once, so the softmax needs no running
// maximum, and the next 32 queries are under way from the moment that the last product with these is done.
template <typename T, int DP, int SUBS, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 2) attention_short_kernel(tode_cross_attention_args a, int row_tiles, int chunks) {
    typedef Tile<T, DP> L;
    extern __shared__ __align__(16) char lds[];
    long long group;
    int chunk;
    if (!place(a, block_number(), chunks, group, chunk)) return;
    const Group<T> p(a, group);
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32;
    T *const k_tile = (T *)lds, *const v_tile = k_tile + SUBS * L::VALUES, *const own = v_tile + SUBS * L::VALUES + wave * L::VALUES;
    const float c = fmaxf(fabsf((float)a.scale) * LOG2E, 1e-37f);
    const int subs = (p.length + 31) / 32, stride = chunks * WAVES;
    int tile = chunk * WAVES + wave;
    Operand<T, DP> q;
    if (tile < row_tiles) q.load_signed(p.query(tile * 32 + lane % 32), p.D, h, a.scale < 0);
    unsigned bits[SUBS];
    int partly = 0;  // which 32 keys are not all looked at
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
        bits[sub] = p.allowed_bits(32 * sub, lane);
        partly |= (bits[sub] != 0xffffffffu) << sub;
        if (sub < subs) {
            const unsigned there = bits[sub];
            auto k_row = [&](int i) { return there >> i & 1 ? p.key(32 * sub + i) : (const T *)nullptr; };
            auto v_row = [&](int i) { return there >> i & 1 ? p.value(32 * sub + i) : (const T *)nullptr; };
            stage<T, DP>(k_tile + sub * L::VALUES, thread, 64 * WAVES, p.D, k_row);
            stage<T, DP>(v_tile + sub * L::VALUES, thread, 64 * WAVES, p.D, v_row);
        }
        bits[sub] >>= 4 * h;
    }
    __syncthreads();
    for (; tile < row_tiles; tile += stride) {
        const int row0 = tile * 32, row = row0 + lane % 32;
        float w[SUBS][16], top = -INFINITY;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            if (sub >= subs) continue;
            const acc16 s = rows_times<T, DP>(k_tile + sub * L::VALUES, q, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) w[sub][r] = s[r];
            if (partly >> sub & 1)
#pragma unroll
                for (int r = 0; r < 16; ++r) w[sub][r] = bits[sub] >> row_of(r, 0) & 1 ? w[sub][r] : -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, w[sub][r]);
        }
        if (tile + stride < row_tiles) q.load_signed(p.query(row0 + 32 * stride + lane % 32), p.D, h, a.scale < 0);
        const float m = fmaf(fmaxf(top, other_half(top)), c, -WEIGHT_BITS<T>), base = m == -INFINITY ? 0 : m;
        acc16 out[L::NT];
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[t] = zero16();
        float l = 0;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            if (sub >= subs) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) w[sub][r] = __builtin_amdgcn_exp2f(fmaf(w[sub][r], c, -base)), l += w[sub][r];
            transposed_times<DP>(v_tile + sub * L::VALUES, w[sub], out, lane);
        }
        l += other_half(l);
        const float f = reciprocal(l);
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[t][r] = settled<T>(out[t][r] * f);
        if (a.lse && h == 0 && row < p.rows) a.lse[p.flat(row)] = log_sum(m, l);
        write_columns<T, DP>(p, a.out, own, out, row0, lane);
        if (a.out_low) keep_low<T, L::NT>(out), write_columns<T, DP>(p, a.out_low, own, out, row0, lane);
    }
}

// ------------------------------------------------------------------------------------------
// float32, many keys
// ------------------------------------------------------------------------------------------

// WC: wavefronts with columns (queries) of their own, sharing the tiles of keys; WS: wavefronts with tiles of their own for the same
// columns, joined at the end.  Few rows (single tokens) take WS = 4, others WC = 4.
template <typename T, int DP, int WC, int WS>
__global__ void __launch_bounds__(64 * WC * WS) attention_kernel(tode_cross_attention_args a, int tiles, int splits, float *partial) {
    typedef Tile<T, DP> L;
    extern __shared__ __align__(16) char lds[];
    long long group;
    int tile;
    if (!place(a, block_number(), tiles * splits, group, tile)) return;
    const int split = tile % splits;
    tile /= splits;
    const Group<T> p(a, group);
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32, wc = wave % WC, ws = wave / WC;
    T *const k_tile = (T *)lds + (WS > 1 ? ws * 2 * L::VALUES : 0), *const v_tile = k_tile + L::VALUES;
    const int row = (tile * WC + wc) * 32 + lane % 32;
    Operand<T, DP> q;
    q.load(p.query(row), p.D, h);
    const float sign = a.scale < 0 ? -1.0f : 1.0f, c = fmaxf(fabsf((float)a.scale) * LOG2E, 1e-37f);  // (not 0: infinity times it stays what it is)

    acc16 out[L::NT];
#pragma unroll
    for (int t = 0; t < L::NT; ++t) out[t] = zero16();
    float m = -INFINITY, l = 0;
    const int key_tiles = (p.length + 31) / 32, per_split = (key_tiles + splits - 1) / splits;
    const int first = split * per_split, last = min(first + per_split, key_tiles);
    for (int t = first; t < last; t += WS) {
        const int at = 32 * (t + (WS > 1 ? ws : 0));
        const unsigned bits = t + (WS > 1 ? ws : 0) < last ? p.allowed_bits(at, lane) : 0;
        if (WS > 1)
            wave_sync();
        else
            __syncthreads();
        auto k_row = [&](int i) { return bits >> i & 1 ? p.key(at + i) : (const T *)nullptr; };
        auto v_row = [&](int i) { return bits >> i & 1 ? p.value(at + i) : (const T *)nullptr; };
        stage<T, DP>(k_tile, WS > 1 ? lane : thread, WS > 1 ? 64 : 64 * WC, p.D, k_row);
        stage<T, DP>(v_tile, WS > 1 ? lane : thread, WS > 1 ? 64 : 64 * WC, p.D, v_row);
        if (WS > 1)
            wave_sync();
        else
            __syncthreads();
        const acc16 s = rows_times<T, DP>(k_tile, q, lane);
        float w[16], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            w[r] = bits >> row_of(r, h) & 1 ? sign * s[r] : -INFINITY;
            top = fmaxf(top, w[r]);
        }
        top = fmaxf(top, other_half(top)) * c - WEIGHT_BITS<T>;
        const float next = fmaxf(m, top), base = next == -INFINITY ? 0 : next, shrink = __builtin_amdgcn_exp2f(m - base);
        float sum = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(fmaf(w[r], c, -base)), sum += w[r];
        l = fmaf(l, shrink, sum), m = next;
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[t][r] *= shrink;
        transposed_times<DP>(v_tile, w, out, lane);
    }
    l += other_half(l);

    if (WS > 1) {
        // [wave][value][lane]: the maxima and sums, then the sums of v
        float *const s_out = (float *)lds, *const s_m = s_out + WS * L::NT * 16 * 64, *const s_l = s_m + WS * 64;
        __syncthreads();
        s_m[ws * 64 + lane] = m, s_l[ws * 64 + lane] = l;
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) s_out[((ws * L::NT + t) * 16 + r) * 64 + lane] = out[t][r];
        __syncthreads();
        if (ws) return;
        float top = -INFINITY;
        for (int w = 0; w < WS; ++w) top = fmaxf(top, s_m[w * 64 + lane]);
        const float base = top == -INFINITY ? 0 : top;
        m = top, l = 0;
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[t] = zero16();
        for (int w = 0; w < WS; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w * 64 + lane] - base);
            l = fmaf(s_l[w * 64 + lane], f, l);
#pragma unroll
            for (int t = 0; t < L::NT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[t][r] = fmaf(s_out[((w * L::NT + t) * 16 + r) * 64 + lane], f, out[t][r]);
        }
    }
    if (row >= p.rows) return;
    if (splits > 1) {
        float *const to = partial + ((group * splits + split) * p.rows + row) * (p.D + 2);
        if (h == 0) to[0] = m, to[1] = l;
        store_column<float, L::NT>(to + 2, out, p.D, h);
        return;
    }
    const float f = reciprocal(l);
#pragma unroll
    for (int t = 0; t < L::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[t][r] *= f;
    store_column<T, L::NT>((T *)a.out + p.flat(row) * p.D, out, p.D, h);
    if (a.out_low) keep_low<T, L::NT>(out), store_column<T, L::NT>((T *)a.out_low + p.flat(row) * p.D, out, p.D, h);
    if (a.lse && h == 0) a.lse[p.flat(row)] = log_sum(m, l);
}

// ------------------------------------------------------------------------------------------
// few rows a head of keys (single tokens): keys and values from memory straight to the lanes that use them
// ------------------------------------------------------------------------------------------

template <int CONTROL> __device__ __forceinline__ float lanes_added(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}
// The sum over `lanes` neighbouring lanes (a power of two), in all of them.
__device__ __forceinline__ float neighbours_sum(float v, int lanes) {
    if (lanes > 1) v = lanes_added<0xB1>(v);   // lane ^ 1
    if (lanes > 2) v = lanes_added<0x4E>(v);   // lane ^ 2
    if (lanes > 4) v = lanes_added<0x141>(v);  // the other half of eight lanes, backwards: its four sums are the same
    if (lanes > 8) v = lanes_added<0x140>(v);  // the other half of sixteen
    if (lanes > 16) v += __shfl_xor(v, 16);
    return v;
}

// A wavefront's lanes: `width` of 16 bytes a key and head, `heads` heads side by side, and the rest different keys; every lane keeps its
// part of R rows of q, and sums of its own over the keys it meets.  WK: wavefronts that share a head's keys (else each has its own).
// Bound by reading the keys once: 2 samples of 8 heads of 128 over 60 001 keys, 4 rows each, bfloat16: 112 us (4.4 TB/s; the general form's
// tiles: 180); 4096 samples of 4 heads of 16 over up to 50 keys, float32: 16.9 us (4.8 TB/s; 169).
template <typename T, int R, int WK>
__global__ void __launch_bounds__(256) attention_token_kernel(tode_cross_attention_args a, int width, int heads, int splits, float *partial) {
    constexpr int N = Raw<T>::N, U = R > 4 ? 2 : 4;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, blocks = a.kv_heads / heads;
    const unsigned block = block_number(), unit = WK > 1 ? block / splits : block * 4 + wave;
    const int split = WK > 1 ? (int)(block - unit * splits) : 0;
    if (unit >= a.batch * blocks) return;  // (WK = 1 only: no barrier follows)
    const long long b = unit / blocks;
    const int part = lane % width * N, head = (int)(unit - b * blocks) * heads + lane / width % heads, slots = 64 / (width * heads), slot = lane / (width * heads);
    const long long group = b * a.kv_heads + head;
    const Group<T> p(a, group);
    const bool whole = part + N <= p.D, none = part >= p.D;
    const float c = fmaxf(fabsf((float)a.scale) * LOG2E, 1e-37f);
    float q[R][N], out[R][N], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unpack(row_part(p.query(r), part, p.D), q[r]);
        m[r] = -INFINITY, l[r] = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) q[r][e] = a.scale < 0 ? -q[r][e] : q[r][e], out[r][e] = 0;
    }
    const T *const keys = p.key(0) + part, *const values = p.value(0) + part;
    const int step = slots * U, pieces = splits * WK, piece = split * WK + (WK > 1 ? wave : 0);
    const int per_piece = ((p.length + pieces - 1) / pieces + step - 1) / step * step, first = min((long long)piece * per_piece, (long long)p.length), last = min(first + per_piece, p.length);
    Raw<T> k[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u].zero(), v[u].zero();
    for (int at = first; at < last; at += step) {
        bool ok[U], all = true;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = at + u * slots + slot, row = min(j, last - 1);
            ok[u] = j < last && (!a.mask || a.mask[b * a.mask_stride + row]);
            all = all && ok[u];
            if (whole)
                k[u].load(keys + row * a.k_strides[1]), v[u].load(values + row * a.v_strides[1]);
            else if (!none)
                k[u] = row_part(keys - part + row * a.k_strides[1], part, p.D), v[u] = row_part(values - part + row * a.v_strides[1], part, p.D);
        }
        float s[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[N];
            unpack(k[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float t = q[r][0] * x[0];
#pragma unroll
                for (int e = 1; e < N; ++e) t = fmaf(q[r][e], x[e], t);
                s[u][r] = neighbours_sum(t, width);
            }
        }
        if (!__all(all))
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int r = 0; r < R; ++r) s[u][r] = ok[u] ? s[u][r] : -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u].w[i] = ok[u] ? v[u].w[i] : 0;
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = s[0][r];
#pragma unroll
            for (int u = 1; u < U; ++u) top = fmaxf(top, s[u][r]);
            top *= c;
            if (__any(top > m[r] + 8.0f || m[r] == -INFINITY)) {
                const float next = fmaxf(m[r], top), shrink = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - next);
                m[r] = next, l[r] *= shrink;
#pragma unroll
                for (int e = 0; e < N; ++e) out[r][e] *= shrink;
            }
            const float base = m[r] == -INFINITY ? 0 : m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, -base)), l[r] += s[u][r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[N];
            unpack(v[u], x);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < N; ++e) out[r][e] = fmaf(s[u][r], x[e], out[r][e]);
        }
    }
    // lanes that met other keys of the head, then other wavefronts
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float top = m[r];
        for (int off = width * heads; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
        const float f = top == -INFINITY ? 0 : __builtin_amdgcn_exp2f(m[r] - top);
        m[r] = top, l[r] *= f;
#pragma unroll
        for (int e = 0; e < N; ++e) out[r][e] *= f;
        for (int off = width * heads; off < 64; off *= 2) {
            l[r] += __shfl_xor(l[r], off);
#pragma unroll
            for (int e = 0; e < N; ++e) out[r][e] += __shfl_xor(out[r][e], off);
        }
    }
    if (WK > 1) {
        __shared__ float s_out[WK][R][N + 2][64];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s_out[wave][r][N][lane] = m[r], s_out[wave][r][N + 1][lane] = l[r];
#pragma unroll
            for (int e = 0; e < N; ++e) s_out[wave][r][e][lane] = out[r][e];
        }
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
            for (int w = 1; w < WK; ++w) top = fmaxf(top, s_out[w][r][N][lane]);
            const float mine = top == -INFINITY ? 0 : __builtin_amdgcn_exp2f(m[r] - top);
            l[r] *= mine;
#pragma unroll
            for (int e = 0; e < N; ++e) out[r][e] *= mine;
            for (int w = 1; w < WK; ++w) {
                const float f = top == -INFINITY ? 0 : __builtin_amdgcn_exp2f(s_out[w][r][N][lane] - top);
                l[r] = fmaf(s_out[w][r][N + 1][lane], f, l[r]);
#pragma unroll
                for (int e = 0; e < N; ++e) out[r][e] = fmaf(s_out[w][r][e][lane], f, out[r][e]);
            }
            m[r] = top;
        }
    }
    if (slot || none) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= p.rows) break;
        if (splits > 1) {
            float *const to = partial + ((group * splits + split) * p.rows + r) * (p.D + 2);
            if (part == 0) to[0] = m[r], to[1] = l[r];
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (part + e < p.D) to[2 + part + e] = out[r][e];
            continue;
        }
        const float f = reciprocal(l[r]);
        if (a.lse && part == 0) a.lse[p.flat(r)] = log_sum(m[r], l[r]);
#pragma unroll
        for (int e = 0; e < N; ++e) out[r][e] = settled<T>(out[r][e] * f);
        auto write = [&](void *of) {
            T *const to = (T *)of + p.flat(r) * p.D + part;
            if (whole) {
                Raw<T> x;
                pack(x, out[r]);
                x.store(to);
            } else
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (part + e < p.D) to[e] = (T)out[r][e];
        };
        write(a.out);
        if (a.out_low) {
#pragma unroll
            for (int e = 0; e < N; ++e) out[r][e] -= (float)(T)out[r][e];
            write(a.out_low);
        }
    }
}

// The pieces of a row's keys joined: a workgroup a row, D values (a power of two or the next) by 256 / D pieces at a time.
template <typename T> __global__ void __launch_bounds__(256) attention_join_kernel(tode_cross_attention_args a, int splits, const float *partial) {
    const int thread = threadIdx.x, D = a.head_dim, G = a.heads / a.kv_heads, rows = (int)(a.queries * G);
    const long long n = blockIdx.x, group = n / rows, b = group / a.kv_heads;
    const int row = (int)(n - group * rows);
    const float *const from = partial + (group * splits * rows + row) * (D + 2);
    const long long step = (long long)rows * (D + 2);
    __shared__ float s_weight[ATTENTION_SPLITS], s_sum[256], s_top[4], s_total[4];
    float top = -INFINITY;
    for (int s = thread; s < splits; s += 256) top = fmaxf(top, from[s * step]);
    for (int off = 32; off > 0; off /= 2) top = fmaxf(top, __shfl_xor(top, off));
    if (thread % 64 == 0) s_top[thread / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    const float base = top == -INFINITY ? 0 : top;
    float l = 0;
    for (int s = thread; s < splits; s += 256) {
        const float f = __builtin_amdgcn_exp2f(from[s * step] - base);
        s_weight[s] = f, l = fmaf(from[s * step + 1], f, l);
    }
    for (int off = 32; off > 0; off /= 2) l += __shfl_xor(l, off);
    if (thread % 64 == 0) s_total[thread / 64] = l;
    __syncthreads();
    l = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    const int wide = D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256, d = thread % wide, parts = 256 / wide;
    float v = 0;
    if (d < D)
#pragma unroll 8
        for (int s = thread / wide; s < splits; s += parts) v = fmaf(from[s * step + 2 + d], s_weight[s], v);
    s_sum[thread] = v;
    __syncthreads();
    if (thread >= D) return;
    for (int i = 1; i < parts; ++i) v += s_sum[thread + i * wide];
    const int query = row / G;
    const long long at = (b * a.queries + query) * a.heads + (group - b * a.kv_heads) * G + row - query * G;
    v = settled<T>(v * reciprocal(l));
    ((T *)a.out)[at * D + d] = (T)v;
    if (a.out_low) ((T *)a.out_low)[at * D + d] = (T)(v - (float)(T)v);
    if (a.lse && thread == 0) a.lse[at] = log_sum(top, l);
}

struct ForwardPlan {
    bool few, token;           // float32: four wavefronts on 32 rows; up to 8 rows a head of keys
    int tiles, splits;
    int width, heads, shared;  // token: lanes a key, heads side by side, wavefronts that share keys
    long long groups, bytes;
};
static ForwardPlan plan_forward(const tode_cross_attention_args &a) {
    ForwardPlan p;
    const long long rows = a.queries * (a.heads / a.kv_heads);
    p.groups = a.batch * a.kv_heads;
    // float32: also where there are few tiles of 128 rows, each of which would go over the keys one tile after the other, as long as the
    // workgroups of 32 rows are all on the chip at once, which takes the more of it the longer the heads are (us in this form and the other one, 128 rows over
    // 200 keys: heads of 32 values, 192 groups 16.3 and 17.5, 256 groups 19.8 and 17.6; of 64, 128 groups 21.8 and 28.0, 160 groups 36.6 and 28.5; of
    // 128, 64 groups 28.4 and 48.6, 96 groups 59.9 and 51.2)
    const long long tiles = p.groups * ((rows + 127) / 128);
    p.few = a.dtype == TODE_F32 && (rows <= 32 || (a.keys > 64 && tiles <= (a.head_dim <= 32 ? 192 : a.head_dim <= 64 ? 128 : 64)));
    p.token = rows <= 8;  // (10 rows of 80 values, float32: 738 us in two blocks of 8, in the general form 566)
    if (p.token) {
        const int N = a.dtype == TODE_F32 ? 4 : 8;
        for (p.width = 1; p.width * N < a.head_dim;) p.width *= 2;
        // 256 bytes side by side where heads make that up
        for (p.heads = 1; a.kv_heads % (2 * p.heads) == 0 && 2 * p.heads * p.width <= 64 && p.heads * a.head_dim * 16 / N < 256;) p.heads *= 2;
        const int step = 64 / (p.width * p.heads) * (rows > 4 ? 2 : 4);  // keys a wavefront works on at a time
        const long long units = p.groups / p.heads;
        p.shared = a.keys >= 8 * step && units < 8192 ? 4 : 1;
        // about four workgroups a compute unit, of four steps a wavefront or more
        const long long most = a.keys / (p.shared * step * 4), wanted = units > 0 ? 1024 / units : 1;
        p.tiles = 1, p.splits = p.shared == 1 || wanted < 2 || most < 2 ? 1 : (int)(wanted < most ? wanted : most);
        if (p.splits > ATTENTION_SPLITS) p.splits = ATTENTION_SPLITS;
        p.bytes = p.splits > 1 ? p.groups * p.splits * rows * (a.head_dim + 2) * 4 : 0;
        return p;
    }
    const int tall = p.few ? 32 : a.dtype != TODE_F32 && a.head_dim <= 64 ? 256 : 128;
    p.tiles = (int)((rows + tall - 1) / tall);
    // about four workgroups a compute unit, of four tiles a wavefront or more
    const long long there = p.groups * p.tiles, most = (a.keys + 511) / 512, wanted = there > 0 ? 1024 / there : 1;
    p.splits = a.keys <= 128 ? 1 : (int)(wanted < 1 || most < 1 ? 1 : wanted < most ? wanted : most);
    if (p.splits > ATTENTION_SPLITS) p.splits = ATTENTION_SPLITS;
    p.bytes = p.splits > 1 ? p.groups * p.splits * rows * (a.head_dim + 2) * 4 : 0;
    return p;
}

template <typename T, int DP, int WC, int WS> static int launch(const tode_cross_attention_args &a, const ForwardPlan &p, hipStream_t s) {
    typedef Tile<T, DP> L;
    constexpr int tile_bytes = WS * 2 * L::VALUES * (int)sizeof(T), join_bytes = WS > 1 ? WS * (L::NT * 16 + 2) * 64 * 4 : 0;
    constexpr int bytes = tile_bytes > join_bytes ? tile_bytes : join_bytes;
    static_assert(bytes <= 160 * 1024, "LDS");
    if (int rc = allow_lds((const void *)attention_kernel<T, DP, WC, WS>, bytes)) return rc;
    hipLaunchKernelGGL((attention_kernel<T, DP, WC, WS>), grid_line(placed(a, p.tiles * p.splits)), dim3(64 * WC * WS), bytes, s, a, p.tiles, p.splits, (float *)a.workspace);
    if (p.splits > 1) {
        const long long rows = p.groups * a.queries * (a.heads / a.kv_heads);
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, s, a, p.splits, (const float *)a.workspace);
    }
    return check_hip(hipGetLastError(), "tode_cross_attention launch");
}

template <typename T, int DP, int CT> static int launch_tiles(const tode_cross_attention_args &a, const ForwardPlan &p, hipStream_t s) {
    typedef Tile<T, DP> L;
    constexpr int bytes = 4 * (DP > 128 ? 32 : 64) * L::STRIDE * (int)sizeof(T);
    static_assert(bytes <= 160 * 1024, "LDS");
    if (int rc = allow_lds((const void *)attention_tiles_kernel<T, DP, CT>, bytes)) return rc;
    hipLaunchKernelGGL((attention_tiles_kernel<T, DP, CT>), grid_line(placed(a, p.tiles * p.splits)), dim3(256), bytes, s, a, p.tiles, p.splits, (float *)a.workspace);
    if (p.splits > 1) {
        const long long rows = p.groups * a.queries * (a.heads / a.kv_heads);
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, s, a, p.splits, (const float *)a.workspace);
    }
    return check_hip(hipGetLastError(), "tode_cross_attention launch");
}

template <typename T, int DP, int SUBS> static int launch_short(const tode_cross_attention_args &a, const ForwardPlan &p, hipStream_t s) {
    typedef Tile<T, DP> L;
    // eight wavefronts share the keys where four of them leave no room for a second workgroup, and there is room for eight
    constexpr int tile = L::VALUES * (int)sizeof(T), WAVES = (2 * SUBS + 4) * tile <= 80 * 1024 || (2 * SUBS + 8) * tile > 160 * 1024 ? 4 : 8, bytes = (2 * SUBS + WAVES) * tile;
    if constexpr (bytes > 160 * 1024)
        return fail(TODE_E_UNSUPPORTED, "head_dim %d", a.head_dim);
    else {
        if (int rc = allow_lds((const void *)attention_short_kernel<T, DP, SUBS, WAVES>, bytes)) return rc;
        const long long rows = a.queries * (a.heads / a.kv_heads), row_tiles = (rows + 31) / 32;
        // a wavefront takes two tiles of rows or more where there are a thousand workgroups without it
        const long long most = (row_tiles + WAVES - 1) / WAVES, wanted = (1024 + p.groups - 1) / p.groups;
        const int chunks = (int)(wanted < most ? wanted : most);
        hipLaunchKernelGGL((attention_short_kernel<T, DP, SUBS, WAVES>), grid_line(placed(a, chunks)), dim3(64 * WAVES), bytes, s, a, (int)row_tiles, chunks);
        return check_hip(hipGetLastError(), "tode_cross_attention launch");
    }
}
template <typename T, int DP> static int launch_short(const tode_cross_attention_args &a, const ForwardPlan &p, hipStream_t s) {
    if (a.keys <= 32) return launch_short<T, DP, 1>(a, p, s);
    if (a.keys <= 64) return launch_short<T, DP, 2>(a, p, s);
    if (a.keys <= 96) return launch_short<T, DP, 3>(a, p, s);
    return launch_short<T, DP, 4>(a, p, s);
}
// The keys that a workgroup holds in LDS at once.
template <typename T> static int short_keys(int head_dim) { return sizeof(T) == 2 ? (head_dim <= 128 ? 128 : 0) : (head_dim <= 64 ? 128 : 64); }

template <typename T, int R> static int launch_token(const tode_cross_attention_args &a, const ForwardPlan &p, hipStream_t s) {
    const long long units = p.groups / p.heads;
    if (p.shared > 1)
        hipLaunchKernelGGL((attention_token_kernel<T, R, 4>), grid_line(units * p.splits), dim3(256), 0, s, a, p.width, p.heads, p.splits, (float *)a.workspace);
    else
        hipLaunchKernelGGL((attention_token_kernel<T, R, 1>), grid_line((units + 3) / 4), dim3(256), 0, s, a, p.width, p.heads, 1, (float *)nullptr);
    if (p.splits > 1)
        hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)(p.groups * a.queries * (a.heads / a.kv_heads))), dim3(256), 0, s, a, p.splits, (const float *)a.workspace);
    return check_hip(hipGetLastError(), "tode_cross_attention launch");
}

template <typename T> static int forward(const tode_cross_attention_args &a, hipStream_t s) {
    const ForwardPlan p = plan_forward(a);
    if (p.token) {
        const long long rows = a.queries * (a.heads / a.kv_heads);
        return rows <= 1 ? launch_token<T, 1>(a, p, s) : rows <= 2 ? launch_token<T, 2>(a, p, s) : rows <= 4 ? launch_token<T, 4>(a, p, s) : launch_token<T, 8>(a, p, s);
    }
    if (!p.few && a.keys <= short_keys<T>(a.head_dim)) {
        if (a.head_dim <= 32) return launch_short<T, 32>(a, p, s);
        if (a.head_dim <= 64) return launch_short<T, 64>(a, p, s);
        return launch_short<T, 128>(a, p, s);
    }
    if constexpr (sizeof(T) == 2) {
        if (a.head_dim <= 32) return launch_tiles<T, 32, 2>(a, p, s);
        if (a.head_dim <= 64) return launch_tiles<T, 64, 2>(a, p, s);
        if (a.head_dim <= 96) return launch_tiles<T, 96, 1>(a, p, s);
        if (a.head_dim <= 128) return launch_tiles<T, 128, 1>(a, p, s);
        return launch_tiles<T, 256, 1>(a, p, s);
    } else {
        if (a.head_dim <= 32) return p.few ? launch<T, 32, 1, 4>(a, p, s) : launch<T, 32, 4, 1>(a, p, s);
        if (a.head_dim <= 64) return p.few ? launch<T, 64, 1, 4>(a, p, s) : launch<T, 64, 4, 1>(a, p, s);
        return p.few ? launch<T, 128, 1, 4>(a, p, s) : launch<T, 128, 4, 1>(a, p, s);
    }
}

int TODE_ATT_NAME(attention_forward)(const tode_cross_attention_args &a, hipStream_t s) { return forward<TODE_ATT_TYPE>(a, s); }
int64_t TODE_ATT_NAME(attention_forward_bytes)(const tode_cross_attention_args &a) { return plan_forward(a).bytes; }

}  // namespace tode

#endif
