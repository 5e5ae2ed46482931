// paged_attention.hip -- attention of one new token per row over a paged key-value cache (layout: csrc/paged_cache.hip).
//   o[n, h] = sum_j softmax_j(scale * q[n, h] . K_j) V_j     over the keys j < lengths[n] of head h / (Hq / Hkv), key j in page block_table[n, j / s]
// A key whose page number lies outside [0, P) does not exist, and no key at all, or none with a score above -inf, leaves a row of zeros.  What a page holds
// behind a row's length does not reach the result, NaN included: the scores of such keys are replaced by -inf, their values zeroed before the product.
//
// Every key and value is read once for up to 16 query heads (a key head with more of them is walked once per 16, and all but the first walk find it in the
// caches: 8 rows of 8000 keys, 1 key head of 128 bf16 columns, 32 query heads 28.2 us, 64 34.7): the operator is bound by the bandwidth of
// the cache, and by the latency of one pass where that is short.  One
// workgroup of four waves serves the (up to 16) query heads of one key head over one stretch of one row's keys; the waves take consecutive tiles of
// the stretch and run an online softmax over them (running maximum m and sum l per query, base 2), so the cache is walked in one pass.
//   * both products run on the matrix unit with the KEYS as the wide operand: S^T = K Q^T and O^T = V^T P^T.  A lane then owns ONE query (its
//     column, lane % 16) throughout: the scores it gets are the probabilities it feeds back (same registers), its m, l and rescale factor are its
//     own, and only the maximum crosses lanes (two swaps per tile).  With fewer than 16 queries the other columns idle; the unit is far from
//     its limit all the same: a tile of 32 keys x 128 columns is 24 instructions, 0.16 us of a SIMD, and its 16 KB are 3.2 us of a SIMD's share
//     of the bandwidth.
//   * K goes straight from memory into the matrix unit's registers (16 B a lane, no LDS): the order in which the contraction visits the columns is
//     free as long as Q uses the same.  V is needed with the keys along the contraction, 8 (bf16) or 4 (fp32) keys per lane; its rows are loaded
//     as they lie, consecutive columns a lane, and a pair of keys is interleaved with one byte permute (bf16; fp32 needs none).
//   * the head's run inside a page is contiguous and a 16-key subtile never leaves its page, so a subtile's address is one scalar base (its page
//     number, fetched 64 subtiles ahead into a register) plus offsets that no lane ever recomputes.
//   * two tiles per wave in registers: the next one is requested before the current one is used, and nothing in the walk is loaded behind a condition
//     (a load in a branch makes the compiler wait for everything in flight).  Worth 6 % at 128 columns.
//   * heads above 128 columns have no registers for two tiles: K of the next tile is requested once this one's scores are there, V once it is added
//     up, so one of the two is always in flight (32 rows up to 4000, 4 key heads of 256 columns: 65 us against 72, fp32 121 against 172).
//   * a head that fills its tile (32, 64, 96, 128, 192, 256 columns) has its size compiled in: every address is one base and constants (fp32 128 columns: 200
//     registers against 256 and 44 spilled ones; 48 rows up to 8192 289 us against 415).
//   * long rows are split over workgroups (``splits``); partial (m, l, O) in fp32 go to a workspace and a second launch joins them.  Each row is
//     split by its OWN length, so the table's width decides only how many workgroups start.
// Measured: 48 rows of 0 .. 8192 keys, 32 query and 8 key heads of 128 bf16 columns (810 MB of cache): 150 us with the join, 5.4 TB/s (a large copy: 5.2); in fp32 289;
// one row of 40001 keys, the same heads: 32 us, 5.1 TB/s; 256 rows of up to 128 keys, 12 heads of 64 fp32 columns: 25 us, 4.2 TB/s (short rows: a
// wave's few tiles do not cover the latency of its first); 64 rows of them in bf16: 7.4 us, three dependent trips to memory and a merge.
#include "common.h"
#include <algorithm>

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t pa_u3 __attribute__((ext_vector_type(3), aligned(4)));
// 16 bytes of the cache, marked as read once (a step's other data keeps its place in the caches; 153 -> 148 us for 0.8 GB).  Right also where blocks of query heads
// read them again: without the mark 8 rows of 8000 keys and 32 heads on one 32.6 us against 28.2, 64 heads 36.2 against 34.7, fp32 45.6 against 38.5.
__device__ __forceinline__ uint4_t pa_ld(const void* p) { return __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p)); }

struct PagedAttnArgs {
    const void* q; int64_t q_row, q_head; const void* k; const void* v; const int32_t* table; int64_t ld_table; const int32_t* lengths; void* o;
    float* part_o; float* part_ml; int N, Hq, Hk, G, qblocks, dh, P, shift, M, splits, q_wide; float scale_log2;
    int first;                 // workgroup number of this launch's first one
};
#define PA_WAVES 4             // of a workgroup that shares a row with others
__device__ __forceinline__ void pa_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void pa_store(bf16_t* p, float v) { *p = f32_to_bf16(v); }

__device__ __forceinline__ float pa_col_max(float v) {          // over the four lanes of a column (lane ^ 16, lane ^ 32)
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pa_col_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// DK columns of K and Q (a multiple of 32), W columns of V per lane (16 W >= dh; one load takes VC of them, side by side over
// the lanes: a multiple of VC is where a head may end), SUB 16-key subtiles per tile
template <typename T, int W, int DK> struct PaTile;

template <int W, int DK> struct PaTile<bf16_t, W, DK> {
    static constexpr int SUB = 2, KC = DK / 32;                  // K fragments of 32 columns: 8 per lane
    static constexpr int VD = W / 2;                              // dwords of V per lane and key
    static constexpr int VC = W < 8 ? W : W == 12 ? 4 : 8;                    // columns of V per load: a wave's 16 lanes lie side by side in it
    struct Q { uint4 q[KC]; };
    uint4 k[SUB][KC];
    uint32_t v[SUB][4][VD];
    static __device__ __forceinline__ void load_q(Q& x, const bf16_t* row, int g, int dh, bool live, bool wide) {      // any stride and alignment
        if (wide) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                x.q[c] = make_uint4(0, 0, 0, 0);
                if (live && c * 32 + g * 8 < dh) x.q[c] = *reinterpret_cast<const uint4*>(row + c * 32 + g * 8);
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = c * 32 + g * 8 + 2 * i;
                w[i] = live && d < dh ? (uint32_t)row[d] | ((uint32_t)row[d + 1] << 16) : 0u;
            }
            x.q[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    // base: the subtile's first key row; r = lane % 16, g = lane / 16.  Columns that the head does not have (dh < 16 W) are read from its last ones
    // instead, so that no load hangs on a condition: Q is zero there, and such columns of O are not stored.
    __device__ __forceinline__ void load_k(int u, const bf16_t* base, int r, int g, int dh) {
#pragma unroll
        for (int c = 0; c < KC; ++c) k[u][c] = __builtin_bit_cast(uint4, pa_ld(base + r * dh + min(c * 32 + g * 8, dh - 8)));
    }
    __device__ __forceinline__ void load_v(int u, const bf16_t* base, int r, int g, int dh) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16_t* p = base + (g * 4 + i) * dh;
            if constexpr (VD == 1) v[u][i][0] = *reinterpret_cast<const uint32_t*>(p + min(r * W, dh - W));
            else if constexpr (VD == 3) { const pa_u3 x = *reinterpret_cast<const pa_u3*>(p + min(r * W, dh - W)); v[u][i][0] = x[0]; v[u][i][1] = x[1]; v[u][i][2] = x[2]; }
            else if constexpr (VD == 2) { const uint2 x = *reinterpret_cast<const uint2*>(p + min(r * W, dh - W)); v[u][i][0] = x.x; v[u][i][1] = x.y; }
            else if constexpr (VD == 6) {
#pragma unroll
                for (int d = 0; d < VD; d += 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(p + min(32 * d + r * 4, dh - 4));
                    v[u][i][d] = x.x; v[u][i][d + 1] = x.y;
                }
            } else {
#pragma unroll
                for (int d = 0; d < VD; d += 4) {
                    const uint4_t x = pa_ld(p + min(32 * d + r * 8, dh - 8));
                    v[u][i][d] = x.x; v[u][i][d + 1] = x.y; v[u][i][d + 2] = x.z; v[u][i][d + 3] = x.w;
                }
            }
        }
    }
    // ... and zeroed before they meet that zero: an infinity among the head's last columns would make it NaN
    __device__ __forceinline__ void trim_k(int g, int dh) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const bool in = c * 32 + g * 8 < dh;
                k[u][c] = make_uint4(in ? k[u][c].x : 0u, in ? k[u][c].y : 0u, in ? k[u][c].z : 0u, in ? k[u][c].w : 0u);
            }
    }
    __device__ __forceinline__ void drop_v(int u, int i, bool ok) {
#pragma unroll
        for (int d = 0; d < VD; ++d) v[u][i][d] = ok ? v[u][i][d] : 0u;
    }
    __device__ __forceinline__ void scores(const Q& x, float4_t (&s)[SUB]) const {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            s[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c)
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k[u][c]), __builtin_bit_cast(bf16x8_t, x.q[c]), s[u], 0, 0, 0);
        }
    }
    // O^T += V^T P^T.  A probability goes in as two bf16 parts, hi (truncated) + lo: one bf16 would cost 2^-8 of every probability; the second
    // product is free next to the loads.  hi is the truncation of p less 128 steps of fp32 (2^-16 .. 2^-17 of p), so that lo is positive wherever p is: an
    // infinite V then stays infinite (0 * inf would make it NaN).  With p in [1, 2) lo lies below 2^-7 + 2^-16; under 2^-7 its own rounding is at
    // most 2^-16, above it goes to 2^-7: what is left out is at most 2^-16 of p.
    __device__ __forceinline__ void accumulate(const float4_t (&p)[SUB], float4_t (&o)[W]) const {
        uint4 hi, lo;
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = p[e >> 1][2 * (e & 1)], b = p[e >> 1][2 * (e & 1) + 1];
            const uint32_t ah = __builtin_elementwise_sub_sat(__float_as_uint(a), 0x80u) & 0xffff0000u, bh = __builtin_elementwise_sub_sat(__float_as_uint(b), 0x80u) & 0xffff0000u;
            h[e] = (ah >> 16) | bh;
            l[e] = pack_bf16x2(a - __uint_as_float(ah), b - __uint_as_float(bh));
        }
        hi = make_uint4(h[0], h[1], h[2], h[3]); lo = make_uint4(l[0], l[1], l[2], l[3]);
        const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, hi), pl = __builtin_bit_cast(bf16x8_t, lo);
#pragma unroll
        for (int d = 0; d < VD; ++d) {                            // the dword holds columns 2 d (low half) and 2 d + 1
            uint32_t a[4], b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = v[e >> 1][2 * (e & 1)][d], y = v[e >> 1][2 * (e & 1) + 1][d];
                a[e] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                b[e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            }
            const bf16x8_t va = __builtin_bit_cast(bf16x8_t, make_uint4(a[0], a[1], a[2], a[3])), vb = __builtin_bit_cast(bf16x8_t, make_uint4(b[0], b[1], b[2], b[3]));
            o[2 * d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, ph, o[2 * d], 0, 0, 0);
            o[2 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, ph, o[2 * d + 1], 0, 0, 0);
            o[2 * d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pl, o[2 * d], 0, 0, 0);
            o[2 * d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, pl, o[2 * d + 1], 0, 0, 0);
        }
    }
};

// fp32: exact products on the f32 matrix instruction (4 columns / 4 keys per step; element j of a lane's 16 B feeds step j)
template <int W, int DK> struct PaTile<float, W, DK> {
    static constexpr int SUB = 1, KC = DK / 16;
    static constexpr int VC = W % 4 ? 2 : 4;
    struct Q { float4_t q[KC]; };
    float4_t k[SUB][KC];
    float v[SUB][4][W];
    static __device__ __forceinline__ void load_q(Q& x, const float* row, int g, int dh, bool live, bool wide) {
        if (wide) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                x.q[c] = float4_t{0.f, 0.f, 0.f, 0.f};
                if (live && c * 16 + g * 4 < dh) x.q[c] = *reinterpret_cast<const float4_t*>(row + c * 16 + g * 4);
            }
            return;
        }
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) x.q[c][i] = live && c * 16 + g * 4 + i < dh ? row[c * 16 + g * 4 + i] : 0.f;
    }
    __device__ __forceinline__ void load_k(int u, const float* base, int r, int g, int dh) {
#pragma unroll
        for (int c = 0; c < KC; ++c) k[u][c] = __builtin_bit_cast(float4_t, pa_ld(base + r * dh + min(c * 16 + g * 4, dh - 4)));
    }
    __device__ __forceinline__ void load_v(int u, const float* base, int r, int g, int dh) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* p = base + (g * 4 + i) * dh;
            if constexpr (W == 2 || W == 6) {
#pragma unroll
                for (int d = 0; d < W; d += 2) { const float2 x = *reinterpret_cast<const float2*>(p + min(16 * d + r * 2, dh - 2)); v[u][i][d] = x.x; v[u][i][d + 1] = x.y; }
            } else {
#pragma unroll
                for (int d = 0; d < W; d += 4) {
                    const float4_t x = __builtin_bit_cast(float4_t, pa_ld(p + min(16 * d + r * 4, dh - 4)));
                    v[u][i][d] = x[0]; v[u][i][d + 1] = x[1]; v[u][i][d + 2] = x[2]; v[u][i][d + 3] = x[3];
                }
            }
        }
    }
    __device__ __forceinline__ void trim_k(int g, int dh) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) k[u][c][i] = c * 16 + g * 4 < dh ? k[u][c][i] : 0.f;
    }
    __device__ __forceinline__ void drop_v(int u, int i, bool ok) {
#pragma unroll
        for (int d = 0; d < W; ++d) v[u][i][d] = ok ? v[u][i][d] : 0.f;
    }
    __device__ __forceinline__ void scores(const Q& x, float4_t (&s)[SUB]) const {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            s[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u][c][i], x.q[c][i], s[u], 0, 0, 0);
        }
    }
    __device__ __forceinline__ void accumulate(const float4_t (&p)[SUB], float4_t (&o)[W]) const {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < W; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[u][i][d], p[u][i], o[d], 0, 0, 0);
    }
};

// tiles [t0, t1) of a row for (wave) part ``w`` of ``parts``
__device__ __forceinline__ void pa_range(int tiles, int parts, int w, int& t0, int& t1) {
    const int per = (tiles + parts - 1) / parts;
    t0 = min(w * per, tiles);
    t1 = min(t0 + per, tiles);
}
template <typename T> constexpr int pa_tile_keys() { return 16 * PaTile<T, 2, 32>::SUB; }

template <typename T, int W, int DK, bool WHOLE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, W <= 8 ? 2 : 1) void paged_attention_kernel(const PagedAttnArgs p) {
    const int dh = WHOLE ? DK : p.dh;
    extern __shared__ __attribute__((aligned(16))) float pa_sm[];      // [waves][16][2] (m, l) | [waves][queries][dh] O
    constexpr int SUB = PaTile<T, W, DK>::SUB, TK = 16 * SUB;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    int b = p.first + blockIdx.x;
    const int split = b % p.splits; b /= p.splits;
    const int qb = b % p.qblocks; b /= p.qblocks;
    const int kv = b % p.Hk, n = b / p.Hk;
    const int h0 = kv * p.G + qb * 16, nq = min(16, p.G - qb * 16);    // this workgroup's query heads
    const int32_t* row = p.table + n * p.ld_table;
    // page numbers of 64 subtiles from subtile ``first`` on, one per lane; a row that has no more of them is fetched at once, along with its
    // length and the queries (entries behind the length are never used)
    const int cap = p.M << p.shift;
    // (a number outside the pool becomes -1 here, in the branch that fetches it: the walk below then never waits for a load it did not ask for)
    int first = cap <= 64 * 16 ? 0 : -64, pages = -1;
    auto fetch = [&](int limit) {
        const int key = first * 16 + lane * 16;
        if (key < limit) { const int page = row[key >> p.shift]; pages = page >= 0 && page < p.P ? page : -1; }
    };
    if (first == 0) fetch(cap);
    using Tile = PaTile<T, W, DK>;
    typename Tile::Q q;
    Tile::load_q(q, (const T*)p.q + n * p.q_row + (h0 + min(r, nq - 1)) * p.q_head, g, dh, r < nq, p.q_wide);
    const int len = min(max(p.lengths[n], 0), cap), tiles = (len + TK - 1) / TK;
    const bool only = p.splits == 1;
    int t0, t1;
    pa_range(tiles, p.splits * WAVES, split * WAVES, t0, t1);
    if (t0 >= t1 && !only) return;                                    // (workgroup-uniform; the join counts the stretches by the same rule)
    pa_range(tiles, p.splits * WAVES, split * WAVES + wave, t0, t1);
    float m = -INFINITY, l = 0.f;
    float4_t o[W];
#pragma unroll
    for (int d = 0; d < W; ++d) o[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int64_t head = (int64_t)kv << p.shift, page_rows = (int64_t)p.Hk << p.shift;
    const int mask = (1 << p.shift) - 1;
    auto place = [&](int64_t (&at)[SUB], bool (&good)[SUB], int t) {
        if (t * SUB >= first + 64) { first = t * SUB; pages = -1; fetch(len); }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int key = t * TK + u * 16, page = __builtin_amdgcn_readlane(pages, (t * SUB - first + u) & 63);
            good[u] = key < len && page >= 0;
            at[u] = ((int64_t)(good[u] ? page : 0) * page_rows + head + (key & mask)) * dh;
        }
    };
    auto load_k = [&](Tile& x, const int64_t (&at)[SUB]) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) x.load_k(u, (const T*)p.k + at[u], r, g, dh);
    };
    auto load_v = [&](Tile& x, const int64_t (&at)[SUB]) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) x.load_v(u, (const T*)p.v + at[u], r, g, dh);
    };
    auto load = [&](Tile& x, bool (&good)[SUB], int t) {
        int64_t at[SUB];
        place(at, good, t);
#pragma unroll
        for (int u = 0; u < SUB; ++u) { x.load_k(u, (const T*)p.k + at[u], r, g, dh); x.load_v(u, (const T*)p.v + at[u], r, g, dh); }
    };
    auto score = [&](Tile& x, float4_t (&s)[SUB]) {
        if (!WHOLE) x.trim_k(g, dh);
        x.scores(q, s);
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] *= p.scale_log2;
    };
    auto weigh = [&](Tile& x, float4_t (&s)[SUB], const bool (&good)[SUB], int t) {
        bool whole = (t + 1) * TK <= len;
#pragma unroll
        for (int u = 0; u < SUB; ++u) whole = whole && good[u];
        float mx = m;
        if (!whole) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool ok = good[u] && t * TK + u * 16 + g * 4 + i < len;
                    s[u][i] = ok ? s[u][i] : -INFINITY;
                    x.drop_v(u, i, ok);
                }
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[u][i]);
        mx = pa_col_max(mx);
        const float base = mx == -INFINITY ? 0.f : mx;
        const float f = __builtin_amdgcn_exp2f(m - base);             // 0 the first time (m = -inf)
        if (__any(mx > m)) {
            l *= f;
#pragma unroll
            for (int d = 0; d < W; ++d) o[d] *= f;
        }
        m = mx;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) { s[u][i] = __builtin_amdgcn_exp2f(s[u][i] - base); l += s[u][i]; }
        x.accumulate(s, o);
    };
    auto use = [&](Tile& x, const bool (&good)[SUB], int t) {
        float4_t s[SUB];
        score(x, s);
        weigh(x, s, good, t);
    };
    if (t0 < t1) {
        Tile a;
        bool ga[SUB];
        int t = t0;
        if constexpr (W <= 8) {                              // the next tile is on its way while this one is worked on
            Tile b;
            bool gb[SUB];
            load(a, ga, t);
            for (; t + 2 < t1; t += 2) {
                load(b, gb, t + 1);
                use(a, ga, t);
                load(a, ga, t + 2);
                use(b, gb, t + 1);
            }
            if (t + 1 < t1) {
                load(b, gb, t + 1);
                use(a, ga, t);
                use(b, gb, t + 1);
            } else {
                use(a, ga, t);
            }
        } else {                                                 // K of the next tile while V of this one is worked on, and the other way round
            load(a, ga, t);
            for (; t + 1 < t1; ++t) {
                float4_t s[SUB];
                int64_t at[SUB];
                bool gb[SUB];
                score(a, s);
                place(at, gb, t + 1);
                load_k(a, at);
                weigh(a, s, ga, t);
                load_v(a, at);
#pragma unroll
                for (int u = 0; u < SUB; ++u) ga[u] = gb[u];
            }
            use(a, ga, t);
        }
    }
    l = pa_col_sum(l);
    float* ml = pa_sm + wave * 32;
    float* so = pa_sm + WAVES * 32 + wave * nq * dh;
    if (g == 0) { ml[2 * r] = m; ml[2 * r + 1] = l; }
    if (r < nq) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < W; ++d) {
                const int c = (d / Tile::VC * 16 + g * 4 + i) * Tile::VC + d % Tile::VC;
                if (c < dh) so[r * dh + c] = o[d][i];
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nq * dh; e += 64 * WAVES) {
        const int qi = e / dh, c = e - qi * dh;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, pa_sm[w * 32 + 2 * qi]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float acc = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(pa_sm[w * 32 + 2 * qi] - base);
            acc = fmaf(f, pa_sm[WAVES * 32 + (w * nq + qi) * dh + c], acc);
            sum = fmaf(f, pa_sm[w * 32 + 2 * qi + 1], sum);
        }
        const int64_t out = (int64_t)n * p.Hq + h0 + qi;
        if (only) {
            pa_store((T*)p.o + out * dh + c, sum == 0.f ? 0.f : acc / sum);
        } else {
            p.part_o[(out * p.splits + split) * dh + c] = acc;
            if (c == 0) { p.part_ml[2 * (out * p.splits + split)] = mm; p.part_ml[2 * (out * p.splits + split) + 1] = sum; }
        }
    }
}

// one workgroup per (row, query head): the stretches' partial results, rescaled to their common maximum.  The stretches' weights go to LDS first (one
// trip to memory for all of them), then the workgroup's groups of dh / 4 threads walk every groups-th stretch, 16 B a thread, and are added in LDS.
#define PA_MAX_SPLITS 2048
template <typename T>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const PagedAttnArgs p, int tile_keys) {
    __shared__ float weight[PA_MAX_SPLITS];
    __shared__ float4_t sums[256];
    __shared__ float red[8];
    const int64_t out = blockIdx.x;
    const int n = blockIdx.x / p.Hq, tid = threadIdx.x;
    const int len = min(max(p.lengths[n], 0), p.M << p.shift), tiles = (len + tile_keys - 1) / tile_keys;
    const int per = (tiles + p.splits * PA_WAVES - 1) / (p.splits * PA_WAVES), used = per ? (tiles + per * PA_WAVES - 1) / (per * PA_WAVES) : 0;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + out * p.splits;
    float m = -INFINITY;
    for (int s = tid; s < used; s += 256) m = fmaxf(m, ml[s].x);
    m = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = tid; s < used; s += 256) { const float2 x = ml[s]; const float f = __builtin_amdgcn_exp2f(x.x - base); weight[s] = f; l = fmaf(f, x.y, l); }
    l = wave_sum(l);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    const int lanes = p.dh / 4, groups = 256 / lanes, grp = tid / lanes, c = tid - grp * lanes;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
        const float* po = p.part_o + out * p.splits * p.dh + 4 * c;
#pragma unroll 4
        for (int s = grp; s < used; s += groups) acc += weight[s] * *reinterpret_cast<const float4_t*>(po + (int64_t)s * p.dh);
    }
    sums[tid] = acc;
    __syncthreads();
    if (grp == 0) {
        for (int j = 1; j < groups; ++j) acc += sums[j * lanes + c];
        T* o = (T*)p.o + out * p.dh + 4 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) pa_store(o + i, l == 0.f ? 0.f : acc[i] / l);
    }
}

// How many workgroups share a row's keys.  The chip's 256 CUs are fed evenly by 256, 512, ... workgroups: one 40001-token row with 8 key heads took 33 us on
// 160 workgroups, 38 on 320 (64 CUs have twice the work of the others) and 40 on 632.  So: as many rounds of 256 as leave a workgroup 1024 keys of a
// full row (fewer keys where the rows are short and few: at least 256), shared by the rows.  Several rows are rarely all full, they get 512 (16 rows up to
// 18000 with 2 key heads 42 -> 38 us, 2 rows up to 20000 with 12 41 -> 36; 256 keys lose again), and the number of rounds is the nearest one where they are
// split in any case (4 rows up to 8000 with 8 key heads, 1.95 rounds: 25 -> 22; where a nearest second round would be what brings the join, 360 workgroups
// of 1024 keys 17 -> 20).  At most 8 rounds (48 rows up to 8192 with 8 key heads 150 us; 5: 158, 16: 154), 12 of heads up to 64 columns, whose keys
// are half the bytes (64 rows up to 2000 with 12 key heads 49 -> 45, fp32 86 -> 79).
static int pa_splits(int N, int Hq, int Hkv, int dh, int M, int page_size) {
    const int64_t blocks = (int64_t)N * Hkv * ((Hq / Hkv + 15) / 16);
    const int64_t keys = (int64_t)M * page_size, most = (keys + 255) / 256;
    const int64_t round = 256 * (N > 1 ? 512 : 1024);
    int64_t rounds = (keys * blocks + (blocks <= 128 && N > 1 ? round / 2 : 0)) / round;
    const int most_rounds = dh <= 64 ? 12 : 8;
    rounds = rounds < 1 ? 1 : (rounds > most_rounds ? most_rounds : rounds);
    int64_t s = 256 * rounds / blocks;
    if (s > most) s = most;
    if (s > PA_MAX_SPLITS) s = PA_MAX_SPLITS;
    return (int)(s < 1 ? 1 : s);
}
extern "C" size_t vm_paged_attention_ws(int N, int Hq, int Hkv, int dh, int M, int page_size, int dtype) {
    (void)dtype;
    if (N <= 0 || Hq <= 0 || Hkv <= 0 || M <= 0 || page_size <= 0 || dh <= 0 || Hq % Hkv) return 0;
    const int s = pa_splits(N, Hq, Hkv, dh, M, page_size);
    return s == 1 ? 0 : (size_t)N * Hq * s * (dh + 2) * sizeof(float);
}

template <typename T, int W, int DK, bool WHOLE, int WAVES>
static void pa_launch_waves(PagedAttnArgs a, hipStream_t s) {
    const int nq = a.G < 16 ? a.G : 16;
    const size_t lds = sizeof(float) * (WAVES * 32 + (size_t)WAVES * nq * a.dh);
    if (lds > 65536) hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_attention_kernel<T, W, DK, WHOLE, WAVES>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    const int64_t blocks = (int64_t)a.N * a.Hk * a.qblocks * a.splits;
    for (int64_t first = 0; first < blocks; first += VM_MAX_BLOCKS) {
        a.first = (int)first;
        hipLaunchKernelGGL((paged_attention_kernel<T, W, DK, WHOLE, WAVES>), dim3((unsigned)std::min<int64_t>(blocks - first, VM_MAX_BLOCKS)), dim3(64 * WAVES), lds, s, a);
    }
}
// One wave per row and head, without the merge of four, where that alone fills the chip (12 waves for each of its 256 CUs): 256 rows x 12 heads of up to 128
// fp32 keys 27.8 us against 30.0; 64 rows the other way round, 9.6 us against 7.6.
#define PA_ONE (256 * 12)
template <typename T, int W, int DK, bool WHOLE>
static void pa_launch(const PagedAttnArgs& a, hipStream_t s) {
    if (a.splits == 1 && (int64_t)a.N * a.Hk * a.qblocks >= PA_ONE) return pa_launch_waves<T, W, DK, WHOLE, 1>(a, s);
    pa_launch_waves<T, W, DK, WHOLE, PA_WAVES>(a, s);
    if (a.splits > 1) hipLaunchKernelGGL(paged_attention_join_kernel<T>, dim3(a.N * a.Hq), dim3(256), 0, s, a, pa_tile_keys<T>());
}
template <typename T>
static void pa_launch_w(const PagedAttnArgs& a, hipStream_t s) {
    if (a.dh == 32) pa_launch<T, 2, 32, true>(a, s);
    else if (a.dh < 32) pa_launch<T, 2, 32, false>(a, s);
    else if (a.dh == 64) pa_launch<T, 4, 64, true>(a, s);
    else if (a.dh < 64) pa_launch<T, 4, 64, false>(a, s);
    else if (a.dh == 96) pa_launch<T, 6, 96, true>(a, s);
    else if (a.dh < 96) {
        if constexpr (sizeof(T) == 2)
            if (a.dh % 6) return pa_launch<T, 8, 96, false>(a, s);        // 80, 88: a bf16 load of 6 columns would straddle the head's end
        pa_launch<T, 6, 96, false>(a, s);
    } else if (a.dh == 128) pa_launch<T, 8, 128, true>(a, s);
    else if (a.dh < 128) pa_launch<T, 8, 128, false>(a, s);
    else if (a.dh == 192) pa_launch<T, 12, 192, true>(a, s);
    else if (a.dh < 192) pa_launch<T, 12, 192, false>(a, s);
    else if (a.dh == 256) pa_launch<T, 16, 256, true>(a, s);
    else pa_launch<T, 16, 256, false>(a, s);
}

extern "C" int vm_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k_pages, const void* v_pages,
                                  const int32_t* block_table, int64_t ld_table, const int32_t* lengths, void* o, int N, int Hq, int Hkv, int dh, int P,
                                  int page_size, int M, float scale, int dtype, void* ws, size_t ws_bytes, void* stream) {
    VM_REQUIRE(q && k_pages && v_pages && block_table && lengths && o, "vm_paged_attention: null pointer");
    VM_REQUIRE(N > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && P > 0 && M > 0 && ld_table >= M, "vm_paged_attention: bad shape");
    VM_REQUIRE(dh >= 8 && dh <= 256 && dh % 8 == 0, "vm_paged_attention: dh = %d: a multiple of 8 up to 256 is required", dh);
    VM_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0 && (int64_t)M * page_size < (1ll << 31) - 2048,
               "vm_paged_attention: page_size must be a power of two from 16 on, M * page_size below 2^31 - 2048");
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "vm_paged_attention: dtype must be VM_F32 or VM_BF16");
    VM_REQUIRE(((uintptr_t)k_pages % 16) == 0 && ((uintptr_t)v_pages % 16) == 0, "vm_paged_attention: pages must be 16-byte aligned");
    const int splits = pa_splits(N, Hq, Hkv, dh, M, page_size), qblocks = (Hq / Hkv + 15) / 16;
    VM_REQUIRE((int64_t)N * Hq < (1ll << 31) && (int64_t)N * Hkv * qblocks * splits < (1ll << 31), "vm_paged_attention: too many rows x heads");
    const size_t need = vm_paged_attention_ws(N, Hq, Hkv, dh, M, page_size, dtype);
    VM_REQUIRE(need == 0 || (ws && ((uintptr_t)ws % 16) == 0 && ws_bytes >= need), "vm_paged_attention: 16-byte aligned workspace of %zu bytes required", need);
    const int e = dtype == VM_F32 ? 4 : 2;
    PagedAttnArgs a = {q, q_row_stride, q_head_stride, k_pages, v_pages, block_table, ld_table, lengths, o, (float*)ws,
                       (float*)ws + (size_t)N * Hq * splits * dh, N, Hq, Hkv, Hq / Hkv, qblocks, dh, P, __builtin_ctz(page_size), M, splits,
                       (((uintptr_t)q | (uintptr_t)(q_row_stride * e) | (uintptr_t)(q_head_stride * e)) % 16) == 0, scale * 1.4426950408889634f, 0};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_ATTN, 0.0, s, "paged_attn_n%d_h%d_k%d_d%d", N, Hq, Hkv, dh);
    if (dtype == VM_F32) pa_launch_w<float>(a, s);
    else pa_launch_w<bf16_t>(a, s);
    return vm_check_launch("vm_paged_attention");
}
