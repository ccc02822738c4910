// Cross attention, backward.  With p = 2^(c q.k - lse) recomputed from the forward pass's lse and D = sum_d do o of every row:
//   dv = p^T do,  ds = p (do v^T - D),  dq = scale ds k,  dk = scale ds^T q
// (p and ds rounded to 16 bits ahead of their products where the data have them, as forward: gradients are off by 0.0024 in bfloat16, where
// their own rounding is 0.0017; in float16 both are taken times powers of two that keep them within its range)
// in two kernels, so that every sum is taken by one wavefront in one order: the first keeps 32 queries and goes over the keys (dq, and D
// for the second), the second keeps 32 keys and goes over the rows of all heads that share them.
#include "tode_attention.h"

#ifdef TODE_ATT_TYPE

namespace tode {

template <int WS, int NT> __device__ __forceinline__ bool join_waves(float *s_out, acc16 *out, int ws, int lane) {
    if (WS == 1) return true;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s_out[((ws * NT + t) * 16 + r) * 64 + lane] = out[t][r];
    __syncthreads();
    if (ws) return false;
    for (int w = 1; w < WS; ++w)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[t][r] += s_out[((w * NT + t) * 16 + r) * 64 + lane];
    return true;
}

// sum_d do o of a row, with what rounding took off o where it was kept
template <typename T, int DP> __device__ __forceinline__ float row_total(const Group<T> &p, int row, const Operand<T, DP> &g, int h) {
    typedef Tile<T, DP> L;
    const T *const o = p.output(row, p.a.out), *const low = p.output(row, p.a.out_low);
    float total = 0;
#pragma unroll
    for (int i = 0; i < L::NC; ++i) {
        float x[L::N], y[L::N], z[L::N];
        unpack(row_part(o, (2 * i + h) * L::N, p.D), x);
        unpack(row_part(low, (2 * i + h) * L::N, p.D), z);
        unpack(g.c[i], y);
#pragma unroll
        for (int e = 0; e < L::N; ++e) total = fmaf(x[e] + z[e], y[e], total);
    }
    return total + other_half(total);
}

template <typename T, int DP, int WC, int WS>
__global__ void __launch_bounds__(64 * WC * WS) attention_dq_kernel(tode_cross_attention_args a, int tiles, int splits, float *row_sums, float *partial) {
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
    const bool there = row < p.rows;
    Operand<T, DP> q, g;
    q.load(p.query(row), p.D, h);
    g.load(p.cotangent(row), p.D, h);
    const float total = row_total<T, DP>(p, row, g, h);
    const float lse = there ? a.lse[p.flat(row)] : INFINITY, c = (float)a.scale * LOG2E;
    if (there && split == 0 && ws == 0 && h == 0) row_sums[p.flat(row)] = total;

    if (a.dq) {
        acc16 out[L::NT];
#pragma unroll
        for (int t = 0; t < L::NT; ++t) out[t] = zero16();
        ColumnUnit<T, L::NT> unit;
        const int key_tiles = p.scores_matter(lane) ? (p.length + 31) / 32 : 0, per_split = (key_tiles + splits - 1) / splits;
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
            const acc16 s = rows_times<T, DP>(k_tile, q, lane), dp = rows_times<T, DP>(v_tile, g, lane);
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse));
                ds[r] = bits >> row_of(r, h) & 1 ? w * (dp[r] - total) : 0;
            }
            unit.fit(ds, out);
            transposed_times<DP>(k_tile, ds, out, lane);
        }
        const float undo = unit.undo();
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[t][r] *= undo;
        if (!join_waves<WS, L::NT>((float *)lds, out, ws, lane) || !there) return;
        const float f = splits > 1 ? 1 : (float)a.scale;
#pragma unroll
        for (int t = 0; t < L::NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[t][r] *= f;
        if (splits > 1)
            store_column<float, L::NT>(partial + split * (a.batch * a.queries * a.heads * p.D) + p.flat(row) * p.D, out, p.D, h);
        else
            store_column<T, L::NT>((T *)a.dq + p.flat(row) * p.D, out, p.D, h);
    }
}

template <typename T, int DP, int WC, int WS>
__global__ void __launch_bounds__(64 * WC * WS) attention_dkv_kernel(tode_cross_attention_args a, int tiles, int splits, const float *row_sums, float *partial) {
    typedef Tile<T, DP> L;
    extern __shared__ __align__(16) char lds[];
    long long group;
    int tile;
    if (!place(a, block_number(), tiles * splits, group, tile)) return;
    const int split = tile % splits;
    tile /= splits;
    const Group<T> p(a, group);
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32, wc = wave % WC, ws = wave / WC;
    T *const q_tile = (T *)lds + (WS > 1 ? ws * 2 * L::VALUES : 0), *const g_tile = q_tile + L::VALUES;
    float *const s_lse = (float *)((T *)lds + WS * 2 * L::VALUES) + (WS > 1 ? ws * 64 : 0), *const s_sum = s_lse + 32;
    const int key = (tile * WC + wc) * 32 + lane % 32;
    const bool allowed = key < p.keys && p.allowed(key), matter = p.scores_matter(lane);
    Operand<T, DP> k, v;
    const int there = min(key, p.keys - 1);
    k.load_if(p.key(there), p.D, h, allowed);
    v.load_if(p.value(there), p.D, h, allowed);
    const float c = (float)a.scale * LOG2E;
    acc16 dk[L::NT], dv[L::NT];
#pragma unroll
    for (int t = 0; t < L::NT; ++t) dk[t] = zero16(), dv[t] = zero16();
    ColumnUnit<T, L::NT> unit;
    const int row_tiles = tile * WC * 32 < p.length ? (p.rows + 31) / 32 : 0, per_split = (row_tiles + splits - 1) / splits;
    const int first = split * per_split, last = min(first + per_split, row_tiles);
    for (int t = first; t < last; t += WS) {
        const int at = 32 * (t + (WS > 1 ? ws : 0));
        if (WS > 1)
            wave_sync();
        else
            __syncthreads();
        const int end = t + (WS > 1 ? ws : 0) < last ? p.rows : 0;
        auto q_row = [&](int i) { return at + i < end ? p.query(at + i) : (const T *)nullptr; };
        auto g_row = [&](int i) { return at + i < end ? p.cotangent(at + i) : (const T *)nullptr; };
        const int member = WS > 1 ? lane : thread, members = WS > 1 ? 64 : 64 * WC;
        stage<T, DP>(q_tile, member, members, p.D, q_row);
        stage<T, DP>(g_tile, member, members, p.D, g_row);
        if (member < 32) {
            const bool there = at + member < end;
            s_lse[member] = there ? a.lse[p.flat(at + member)] - WEIGHT_BITS<T> : INFINITY;
            s_sum[member] = there ? row_sums[p.flat(at + member)] * WEIGHT_UNIT<T> : 0;
        }
        if (WS > 1)
            wave_sync();
        else
            __syncthreads();
        const acc16 s = rows_times<T, DP>(q_tile, k, lane), dp = rows_times<T, DP>(g_tile, v, lane);
        float w[16], ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = row_of(r, h);
            w[r] = allowed ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -s_lse[i])) : 0;
            ds[r] = allowed && matter ? w[r] * fmaf(dp[r], WEIGHT_UNIT<T>, -s_sum[i]) : 0;
        }
        transposed_times<DP>(g_tile, w, dv, lane);
        unit.fit(ds, dk);
        transposed_times<DP>(q_tile, ds, dk, lane);
    }
    const float undo = unit.undo();
#pragma unroll
    for (int t = 0; t < L::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[t][r] *= undo;
    join_waves<WS, L::NT>((float *)lds, dk, ws, lane);
    if (!join_waves<WS, L::NT>((float *)lds, dv, ws, lane) || key >= p.keys) return;
    const float f = splits > 1 ? 1 : (float)a.scale;
#pragma unroll
    for (int t = 0; t < L::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[t][r] = allowed ? dk[t][r] * f : 0, dv[t][r] = allowed ? dv[t][r] * WEIGHT_UNIT<T> : 0;
    const long long at = ((p.b * a.keys + key) * a.kv_heads + p.head) * p.D;
    if (splits > 1) {
        const long long n = a.batch * a.keys * a.kv_heads * p.D;
        store_column<float, L::NT>(partial + 2 * split * n + at, dk, p.D, h);
        store_column<float, L::NT>(partial + (2 * split + 1) * n + at, dv, p.D, h);
    } else {
        store_column<T, L::NT>((T *)a.dk + at, dk, p.D, h);
        store_column<T, L::NT>((T *)a.dv + at, dv, p.D, h);
    }
}

// The same for 16-bit types and many keys: the next tile of rows is loaded into registers while one is worked on, and lies in one of two
// places in LDS, so that one barrier a tile is enough.  Nothing is masked on the way: a key that may not be looked at has sums of its own, which
// are dropped at the end.  dk and dv have workgroups of their own: the scores are computed twice, five products in place of four, but the sums
// of both leave registers for one wavefront a SIMD only (D = 128; 8 samples of 1024 queries of 16 heads over 787 keys of 4: 371 us in one, 303 apart; 282 with a fetch that adds a fixed way).
template <typename T, int DP, bool KEYS>
__device__ __forceinline__ void dkv_tiles(const tode_cross_attention_args &a, const Group<T> &p, int tile, int split, int splits, const float *row_sums, float *partial, char *lds) {
    typedef Tile<T, DP> L;
    constexpr int ROWS = 64, PARTS = DP / L::N, LOADS = ROWS * PARTS / 256;
    static_assert(ROWS * PARTS % 256 == 0, "whole loads");
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32, key = (tile * 4 + wave) * 32 + lane % 32;
    T *const buffer = (T *)lds;                              // [2][q, g][64][STRIDE]
    float *const s_rows = (float *)(buffer + 8 * L::VALUES);  // [2][lse, sum][64]
    const bool matter = !KEYS || p.scores_matter(lane), allowed = key < p.keys && p.allowed(key);
    Operand<T, DP> k, v;
    k.load(allowed ? p.key(key) : nullptr, p.D, h);
    if (KEYS) v.load(allowed ? p.value(key) : nullptr, p.D, h);
    const float c = (float)a.scale * LOG2E;
    acc16 sum[L::NT];
#pragma unroll
    for (int t = 0; t < L::NT; ++t) sum[t] = zero16();
    ColumnUnit<T, L::NT> unit;
    const int row_tiles = tile * 128 < p.length && matter ? (p.rows + ROWS - 1) / ROWS : 0, per_split = (row_tiles + splits - 1) / splits;
    const int first = split * per_split, last = min(first + per_split, row_tiles);
    Raw<T> q_next[LOADS], g_next[LOADS];
    float row_next = 0;
    // Where a tile's rows are whole queries, the next one's lie a fixed way behind them: a thread keeps its places in the first tile.
    int q_offset[LOADS], g_offset[LOADS], inside = 0;
    const int queries = p.shift >= 0 ? ROWS >> p.shift : 0;
    const bool simple = queries > 0 && p.D % L::N == 0 && a.q_strides[1] < (1 << 24) && a.grad_strides[1] < (1 << 24) && a.q_strides[2] < (1 << 22) && a.grad_strides[2] < (1 << 22);
    const T *const q_rows = (const T *)a.q + p.b * a.q_strides[0] + (long long)p.head * p.G * a.q_strides[2];
    const T *const g_rows = (const T *)a.grad_out + p.b * a.grad_strides[0] + (long long)p.head * p.G * a.grad_strides[2];
    const long long flat_rows = p.b * a.queries * a.heads + p.head * p.G;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int n = thread + 256 * i, row = n / PARTS, part = n % PARTS * L::N, query = simple ? row >> p.shift : 0, member = row - query * p.G;
        q_offset[i] = query * (int)a.q_strides[1] + member * (int)a.q_strides[2] + part;
        g_offset[i] = query * (int)a.grad_strides[1] + member * (int)a.grad_strides[2] + part;
        inside |= (part < p.D) << i;
        q_next[i].zero(), g_next[i].zero();
    }
    const int row0 = thread % ROWS, query0 = simple ? row0 >> p.shift : 0, flat_offset = query0 * a.heads + row0 - query0 * p.G;
    const float *const of_rows = KEYS && thread >= ROWS ? row_sums : a.lse;
    auto fetch = [&](int t) {
        if (simple && ROWS * (t + 1) <= p.rows) {
            const T *const q_from = q_rows + (long long)t * queries * a.q_strides[1], *const g_from = g_rows + (long long)t * queries * a.grad_strides[1];
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (inside >> i & 1) q_next[i].load(q_from + q_offset[i]), g_next[i].load(g_from + g_offset[i]);
            if (thread < 2 * ROWS) {
                row_next = of_rows[flat_rows + (long long)t * queries * a.heads + flat_offset];
                row_next = thread < ROWS ? row_next - WEIGHT_BITS<T> : row_next * WEIGHT_UNIT<T>;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int n = thread + 256 * i, row = ROWS * t + n / PARTS, part = n % PARTS * L::N;
            q_next[i] = row_part(p.query(row), part, p.D), g_next[i] = row_part(p.cotangent(row), part, p.D);
        }
        if (thread < 2 * ROWS) {
            const int row = ROWS * t + thread % ROWS;
            if (thread < ROWS)
                row_next = row < p.rows ? a.lse[p.flat(row)] - WEIGHT_BITS<T> : INFINITY;
            else if (KEYS)
                row_next = row < p.rows ? row_sums[p.flat(row)] * WEIGHT_UNIT<T> : 0;
        }
    };
    if (first < last) fetch(first);
    for (int t = first; t < last; ++t) {
        T *const q_tile = buffer + (t & 1) * 4 * L::VALUES, *const g_tile = q_tile + 2 * L::VALUES;
        float *const s_lse = s_rows + (t & 1) * 2 * ROWS, *const s_sum = s_lse + ROWS;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int n = thread + 256 * i, at = n / PARTS * L::STRIDE + n % PARTS * L::N;
            *(uint4 *)(q_tile + at) = make_uint4(q_next[i].w[0], q_next[i].w[1], q_next[i].w[2], q_next[i].w[3]);
            *(uint4 *)(g_tile + at) = make_uint4(g_next[i].w[0], g_next[i].w[1], g_next[i].w[2], g_next[i].w[3]);
        }
        if (thread < 2 * ROWS) s_lse[thread] = row_next;
        __syncthreads();
        if (t + 1 < last) fetch(t + 1);
#pragma unroll
        for (int sub = 0; sub < ROWS / 32; ++sub) {
            const T *const q_sub = q_tile + sub * L::VALUES, *const g_sub = g_tile + sub * L::VALUES;
            const acc16 s = rows_times<T, DP>(q_sub, k, lane);
            float w[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -s_lse[32 * sub + row_of(r, h)]));
            if (KEYS) {
                const acc16 dp = rows_times<T, DP>(g_sub, v, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) w[r] *= fmaf(dp[r], WEIGHT_UNIT<T>, -s_sum[32 * sub + row_of(r, h)]);
                unit.fit(w, sum);
            }
            transposed_times<DP>(KEYS ? q_sub : g_sub, w, sum, lane);
        }
    }
    if (key >= p.keys) return;
    const float f = KEYS ? unit.undo() * (splits > 1 ? 1 : (float)a.scale) : WEIGHT_UNIT<T>;
#pragma unroll
    for (int t = 0; t < L::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[t][r] = allowed ? sum[t][r] * f : 0;
    const long long at = ((p.b * a.keys + key) * a.kv_heads + p.head) * p.D;
    if (splits > 1)
        store_column<float, L::NT>(partial + (2 * split + !KEYS) * (a.batch * a.keys * a.kv_heads * p.D) + at, sum, p.D, h);
    else
        store_column<T, L::NT>((T *)(KEYS ? a.dk : a.dv) + at, sum, p.D, h);
}
template <typename T, int DP>
__global__ void __launch_bounds__(256, 2) attention_dkv_tiles_kernel(tode_cross_attention_args a, int tiles, int splits, const float *row_sums, float *partial) {
    extern __shared__ __align__(16) char lds[];
    long long group;
    int n;
    if (!place(a, block_number(), 2 * tiles * splits, group, n)) return;
    const Group<T> p(a, group);
    if (n % 2)
        dkv_tiles<T, DP, false>(a, p, n / 2 / splits, n / 2 % splits, splits, row_sums, partial, lds);
    else
        dkv_tiles<T, DP, true>(a, p, n / 2 / splits, n / 2 % splits, splits, row_sums, partial, lds);
}

// And of the first kernel: tiles of 32 keys fetched ahead.
template <typename T, int DP>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) attention_dq_tiles_kernel(tode_cross_attention_args a, int tiles, int splits, float *row_sums, float *partial) {
    typedef Tile<T, DP> L;
    constexpr int PARTS = DP / L::N, LOADS = (32 * PARTS + 255) / 256;
    extern __shared__ __align__(16) char lds[];
    long long group;
    int tile;
    if (!place(a, block_number(), tiles * splits, group, tile)) return;
    const int split = tile % splits;
    tile /= splits;
    const Group<T> p(a, group);
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, h = lane / 32, row = (tile * 4 + wave) * 32 + lane % 32;
    T *const buffer = (T *)lds;  // [2][k, v][32][STRIDE]
    const bool there = row < p.rows;
    Operand<T, DP> q, g;
    q.load(p.query(row), p.D, h);
    g.load(p.cotangent(row), p.D, h);
    const float total = row_total<T, DP>(p, row, g, h);
    const float lse = there ? a.lse[p.flat(row)] : INFINITY, c = (float)a.scale * LOG2E;
    if (there && split == 0 && h == 0) row_sums[p.flat(row)] = total;
    if (!a.dq) return;
    acc16 out[L::NT];
#pragma unroll
    for (int t = 0; t < L::NT; ++t) out[t] = zero16();
    ColumnUnit<T, L::NT> unit;
    const int key_tiles = p.scores_matter(lane) ? (p.length + 31) / 32 : 0, per_split = (key_tiles + splits - 1) / splits;
    const int first = split * per_split, last = min(first + per_split, key_tiles);
    const T *const keys = p.key(0), *const values = p.value(0);
    Raw<T> k_next[LOADS], v_next[LOADS];
    int k_offset[LOADS], v_offset[LOADS], inside = 0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int n = thread + 256 * i, j = n / PARTS, part = n % PARTS * L::N;
        k_offset[i] = j * (int)a.k_strides[1] + part, v_offset[i] = j * (int)a.v_strides[1] + part;
        inside |= (n < 32 * PARTS && part < p.D) << i;
        k_next[i].zero(), v_next[i].zero();
    }
    const bool simple = !a.mask && p.D % L::N == 0 && a.k_strides[1] < (1 << 24) && a.v_strides[1] < (1 << 24);
    auto fetch = [&](int t) {
        if (simple && 32 * (t + 1) <= p.length) {
            const T *const k_from = keys + 32ll * t * a.k_strides[1], *const v_from = values + 32ll * t * a.v_strides[1];
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (inside >> i & 1) k_next[i].load(k_from + k_offset[i]), v_next[i].load(v_from + v_offset[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int n = thread + 256 * i, j = 32 * t + n / PARTS, part = n % PARTS * L::N;
            if (32 * PARTS % 256 != 0 && n >= 32 * PARTS) break;
            const bool one = p.allowed(j);
            k_next[i] = row_part(one ? keys + j * a.k_strides[1] : (const T *)nullptr, part, p.D);
            v_next[i] = row_part(one ? values + j * a.v_strides[1] : (const T *)nullptr, part, p.D);
        }
    };
    if (first < last) fetch(first);
    for (int t = first; t < last; ++t) {
        T *const k_tile = buffer + (t & 1) * 2 * L::VALUES, *const v_tile = k_tile + L::VALUES;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int n = thread + 256 * i, at = n / PARTS * L::STRIDE + n % PARTS * L::N;
            if (32 * PARTS % 256 != 0 && n >= 32 * PARTS) break;
            *(uint4 *)(k_tile + at) = make_uint4(k_next[i].w[0], k_next[i].w[1], k_next[i].w[2], k_next[i].w[3]);
            *(uint4 *)(v_tile + at) = make_uint4(v_next[i].w[0], v_next[i].w[1], v_next[i].w[2], v_next[i].w[3]);
        }
        __syncthreads();
        if (t + 1 < last) fetch(t + 1);
        const acc16 s = rows_times<T, DP>(k_tile, q, lane), dp = rows_times<T, DP>(v_tile, g, lane);
        float ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (dp[r] - total);
        if (a.mask || 32 * (t + 1) > p.length) {
            const unsigned bits = p.allowed_bits(32 * t, lane) >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = bits >> row_of(r, 0) & 1 ? ds[r] : 0;
        }
        unit.fit(ds, out);
        transposed_times<DP>(k_tile, ds, out, lane);
    }
    if (!there) return;
    const float f = unit.undo() * (splits > 1 ? 1 : (float)a.scale);
#pragma unroll
    for (int t = 0; t < L::NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) out[t][r] *= f;
    if (splits > 1)
        store_column<float, L::NT>(partial + split * (a.batch * a.queries * a.heads * p.D) + p.flat(row) * p.D, out, p.D, h);
    else
        store_column<T, L::NT>((T *)a.dq + p.flat(row) * p.D, out, p.D, h);
}

// out[i] = f * (the sum of `splits` pieces, `step` values apart)
template <typename T> __global__ void __launch_bounds__(256) attention_add_kernel(long long n, int splits, long long step, const float *partial, float f, T *out) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) v += partial[s * step + i];
    out[i] = (T)(f * v);
}

struct BackwardPlan {
    bool few_rows, few_keys;
    int row_tiles, row_splits;  // of the first kernel: tiles of queries, pieces of the keys
    int key_tiles, key_splits;  // of the second one: tiles of keys, pieces of the queries
    long long groups, sums, bytes;
};
static BackwardPlan plan_backward(const tode_cross_attention_args &a) {
    BackwardPlan p;
    const long long rows = a.queries * (a.heads / a.kv_heads);
    p.groups = a.batch * a.kv_heads;
    // four wavefronts on 32 rows where there are no more, and in float32 where there are few tiles of 128: as forward, here (us of the whole backward
    // pass, 128 rows over 200 keys) with heads of 32 values 192 groups 52 either way, 256 groups 63 and 54; of 64, 64 groups 54 and 69, 96 groups 78 and 71; of
    // 128, 64 groups 98 and 133, 96 groups 149 and 138.  (The second kernel is slower that way.)
    const long long tiles = p.groups * ((rows + 127) / 128);
    p.few_rows = rows <= 32 || (a.dtype == TODE_F32 && a.keys > 64 && tiles <= (a.head_dim <= 32 ? 192 : 64));
    p.few_keys = a.keys <= 32;
    p.row_tiles = (int)((rows + (p.few_rows ? 31 : 127)) / (p.few_rows ? 32 : 128));
    p.key_tiles = (int)((a.keys + (p.few_keys ? 31 : 127)) / (p.few_keys ? 32 : 128));
    // Pieces where there are fewer than three workgroups a compute unit: their sums go through memory in float32 and take a launch of their own.
    auto splits = [&](long long tiles, long long length) {
        const long long there = p.groups * tiles, most = (length + 511) / 512, wanted = there > 0 ? 1280 / there : 1;
        return (int)(wanted < 1 || most < 1 ? 1 : wanted < most ? wanted : most);
    };
    p.row_splits = a.dq ? splits(p.row_tiles, a.keys) : 1;
    p.key_splits = a.dk ? splits(a.dtype != TODE_F32 && a.head_dim <= 128 && !p.few_keys ? 2 * p.key_tiles : p.key_tiles, rows) : 1;
    p.sums = (a.batch * a.queries * a.heads * 4 + 255) / 256 * 256;
    const long long q = p.row_splits > 1 ? p.row_splits * a.batch * a.queries * a.heads * a.head_dim * 4 : 0;
    const long long kv = p.key_splits > 1 ? 2 * p.key_splits * a.batch * a.keys * a.kv_heads * a.head_dim * 4 : 0;
    p.bytes = p.sums + (q > kv ? q : kv);  // (one after the other)
    return p;
}

template <typename T, int DP, int WC, int WS> static int launch_dq(const tode_cross_attention_args &a, const BackwardPlan &p, hipStream_t s) {
    typedef Tile<T, DP> L;
    float *const sums = (float *)a.workspace, *const partial = (float *)((char *)a.workspace + p.sums);
    const dim3 grid = grid_line(placed(a, p.row_tiles * p.row_splits));
    if constexpr (sizeof(T) == 2 && WC == 4) {
        constexpr int bytes = 4 * L::VALUES * (int)sizeof(T);
        static_assert(bytes <= 160 * 1024, "LDS");
        if (int rc = allow_lds((const void *)attention_dq_tiles_kernel<T, DP>, bytes)) return rc;
        hipLaunchKernelGGL((attention_dq_tiles_kernel<T, DP>), grid, dim3(256), bytes, s, a, p.row_tiles, p.row_splits, sums, partial);
    } else {
        constexpr int tile_bytes = WS * 2 * L::VALUES * (int)sizeof(T), join_bytes = WS > 1 ? WS * L::NT * 16 * 64 * 4 : 0;
        constexpr int bytes = tile_bytes > join_bytes ? tile_bytes : join_bytes;
        static_assert(bytes <= 160 * 1024, "LDS");
        if (int rc = allow_lds((const void *)attention_dq_kernel<T, DP, WC, WS>, bytes)) return rc;
        hipLaunchKernelGGL((attention_dq_kernel<T, DP, WC, WS>), grid, dim3(64 * WC * WS), bytes, s, a, p.row_tiles, p.row_splits, sums, partial);
    }
    if (p.row_splits > 1) {
        const long long n = a.batch * a.queries * a.heads * a.head_dim;
        hipLaunchKernelGGL((attention_add_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, n, p.row_splits, n, (const float *)partial, (float)a.scale, (T *)a.dq);
    }
    return check_hip(hipGetLastError(), "tode_cross_attention_backward launch");
}

template <typename T, int DP, int WC, int WS> static int launch_dkv(const tode_cross_attention_args &a, const BackwardPlan &p, hipStream_t s) {
    typedef Tile<T, DP> L;
    float *const sums = (float *)a.workspace, *const partial = (float *)((char *)a.workspace + p.sums);
    if constexpr (sizeof(T) == 2 && WC == 4 && DP <= 128) {
        constexpr int bytes = 8 * L::VALUES * (int)sizeof(T) + 1024;
        static_assert(bytes <= 160 * 1024, "LDS");
        if (int rc = allow_lds((const void *)attention_dkv_tiles_kernel<T, DP>, bytes)) return rc;
        hipLaunchKernelGGL((attention_dkv_tiles_kernel<T, DP>), grid_line(placed(a, 2 * p.key_tiles * p.key_splits)), dim3(256), bytes, s, a, p.key_tiles, p.key_splits, (const float *)sums,
                           partial);
    } else {
        constexpr int tile_bytes = WS * (2 * L::VALUES * (int)sizeof(T) + 64 * 4), join_bytes = WS > 1 ? WS * L::NT * 16 * 64 * 4 : 0;
        constexpr int bytes = tile_bytes > join_bytes ? tile_bytes : join_bytes;
        static_assert(bytes <= 160 * 1024, "LDS");
        if (int rc = allow_lds((const void *)attention_dkv_kernel<T, DP, WC, WS>, bytes)) return rc;
        hipLaunchKernelGGL((attention_dkv_kernel<T, DP, WC, WS>), grid_line(placed(a, p.key_tiles * p.key_splits)), dim3(64 * WC * WS), bytes, s, a, p.key_tiles, p.key_splits, (const float *)sums,
                           partial);
    }
    if (p.key_splits > 1) {
        const long long n = a.batch * a.keys * a.kv_heads * a.head_dim;
        hipLaunchKernelGGL((attention_add_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, n, p.key_splits, 2 * n, (const float *)partial, (float)a.scale, (T *)a.dk);
        hipLaunchKernelGGL((attention_add_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, n, p.key_splits, 2 * n, (const float *)(partial + n), 1.0f, (T *)a.dv);
    }
    return check_hip(hipGetLastError(), "tode_cross_attention_backward launch");
}

template <typename T, int DP> static int backward_as(const tode_cross_attention_args &a, hipStream_t s) {
    const BackwardPlan p = plan_backward(a);
    if (a.queries > 0)
        if (int rc = p.few_rows ? launch_dq<T, DP, 1, 4>(a, p, s) : launch_dq<T, DP, 4, 1>(a, p, s)) return rc;
    if (!a.dk || a.keys == 0) return TODE_OK;
    return p.few_keys ? launch_dkv<T, DP, 1, 4>(a, p, s) : launch_dkv<T, DP, 4, 1>(a, p, s);
}

template <typename T> static int backward(const tode_cross_attention_args &a, hipStream_t s) {
    if (a.head_dim <= 32) return backward_as<T, 32>(a, s);
    if (a.head_dim <= 64) return backward_as<T, 64>(a, s);
    if (a.head_dim <= 128) return backward_as<T, 128>(a, s);
    if constexpr (sizeof(T) == 2) return backward_as<T, 256>(a, s);
    return fail(TODE_E_UNSUPPORTED, "head_dim %d", a.head_dim);
}

int TODE_ATT_NAME(attention_backward)(const tode_cross_attention_args &a, hipStream_t s) { return backward<TODE_ATT_TYPE>(a, s); }
int64_t TODE_ATT_NAME(attention_backward_bytes)(const tode_cross_attention_args &a) { return plan_backward(a).bytes; }

}  // namespace tode

#endif
