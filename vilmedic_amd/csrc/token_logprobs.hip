// token_logprobs.hip -- log probabilities of given tokens with the entropy of their distribution and its best alternatives, and the gradient of all
// three with respect to the logits.  Per row x of V logits, target t:
//   z = log sum exp(x)      logp = x_t - z      H = log s - (sum_c e_c d_c) / s   with d_c = x_c - m, e_c = exp(d_c), s = sum e_c, m = max x
//   top: the n largest logits, largest first, equal ones by ascending column (a NaN counts as the largest, as torch.topk has it), as x_c - z
// A target < 0 is no token (logp 0, no gradient from it); a target >= V makes its logp NaN.  A column at -inf has p = 0: its gradient is that of a logp or an
// alternative of its own, if any (as log_softmax has it).  A row without a logit above -inf has logp -inf, entropy 0, alternatives -inf, gradient 0.
//
// Forward: ONE pass over the row with a running maximum per thread (sums rescaled when it grows: sum e d becomes f (sum e d + delta sum e) with
// delta = m_old - m_new, f = exp(delta)), 4 x 16 B per thread in flight; m and log s leave the kernel apart, because m + log s in one float loses
// log s where the logits sit far from 0.  Backward: one streaming pass, p recomputed from them.
// Alternatives: the n-th largest of the per-thread maxima, L, is a lower bound of the row's n-th largest logit (n logits >= it exist).  All logits >= L
// belong to the n threads whose own maximum reaches it: only those threads' pieces are read again, dealt out to the whole workgroup (n of 256 threads
// hold n / 256 of the row; with the weaker bound of one wave's maxima 3 n of them did: 8192 x 30522 bf16, n = 8: 103 us against 114).  The
// candidates are ranked by (value, column) in LDS, so the order in which they were collected does not matter.  Rows where that fails (fewer than n logits
// above the bound: -inf columns; thousands of equal logits; NaN) take n exact passes instead.
// Backward writes the gradient with streaming stores and walks the rows from the last one, which the forward pass has just read: the logits' tail is still in
// the 256 MB cache, and the gradient does not push the next step's data out of it.
// Measured, 8192 x 30522 bf16 (500 MB): forward 92 us (5.4 TB/s), with 8 alternatives 100; backward 157 us for 1 GB (6.4 TB/s).  1021 x 50001 fp32
// (204 MB): forward with 4 alternatives 42 us (4.9 TB/s), backward 69 us (5.9 TB/s).  64 x 30522 fp32 with 5 alternatives: 10.5 us, 64 workgroups
// whose rows come through one CU each.  The arithmetic (6 operations and an exponential per logit) takes about three quarters of the memory's time.
#include "common.h"
#include <float.h>
#include <algorithm>

// ascending unsigned order of the values; -0 and +0 are one value, every NaN the largest
__device__ __forceinline__ uint32_t lp_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
#define LP_LOG2E 1.4426950408889634f
#define LP_FLOOR -200.f          // exp of anything below is 0: d is cut here where it meets a factor of 0 (0 * -inf would be NaN)
#define LP_CAND 512
#define LP_U 4                   // 16-byte pieces per thread in flight (2, 3 and 8 measured the same within 3 %, 16 a third slower: fewer waves)

// 16 bytes of a row, whatever its alignment (rows of an odd width start anywhere; the loads stay 16 bytes wide)
typedef uint32_t lp_u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t lp_u4a4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct LpVec;
template <> struct LpVec<bf16_t> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float at(const bf16_t* p) { return bf16_to_f32(*p); }
    static __device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }
    static __device__ __forceinline__ uint4 load(const bf16_t* p) { return __builtin_bit_cast(uint4, *reinterpret_cast<const lp_u4a2*>(p)); }
    static __device__ __forceinline__ void unpack(const uint4 v, float* f) { unpack8(v, f); }
    static __device__ __forceinline__ void store(bf16_t* p, const float* f) { __builtin_nontemporal_store(__builtin_bit_cast(lp_u4a2, pack8(f)), reinterpret_cast<lp_u4a2*>(p)); }
};
// (what a thread without a piece works on: logits of -inf, which change no sum)
template <typename T> __device__ __forceinline__ uint4 lp_none();
template <> __device__ __forceinline__ uint4 lp_none<bf16_t>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
template <> __device__ __forceinline__ uint4 lp_none<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <> struct LpVec<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ float at(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ uint4 load(const float* p) { return __builtin_bit_cast(uint4, *reinterpret_cast<const lp_u4a4*>(p)); }
    static __device__ __forceinline__ void unpack(const uint4 v, float* f) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ void store(float* p, const float* f) { __builtin_nontemporal_store(lp_u4a4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}, reinterpret_cast<lp_u4a4*>(p)); }
};

// descending sort of a wave's 64 values (bitonic; every merge starts with a mirrored step, so that all steps keep the larger value in the lower
// lane): 21 steps of a DPP move or a row swap, a max, a min and a select
template <int CTRL> __device__ __forceinline__ float lp_keep(float v, bool lower) { const float o = dpp_f32<CTRL>(v); return lower ? fmaxf(v, o) : fminf(v, o); }
__device__ __forceinline__ float lp_pick(float v, float o, bool lower) { return lower ? fmaxf(v, o) : fminf(v, o); }
__device__ __forceinline__ float lp_xor16(float v, bool lower) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lower ? a[1] : a[0]);
}
__device__ __forceinline__ float lp_xor32(float v, bool lower) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lower ? a[1] : a[0]);
}
__device__ __forceinline__ float lp_sort_wave(float v) {
    const int lane = threadIdx.x & 63;
    const bool l1 = !(lane & 1), l2 = !(lane & 2), l4 = !(lane & 4), l8 = !(lane & 8), l16 = !(lane & 16), l32 = !(lane & 32);
    auto x4 = [&](float a) { return lp_pick(a, dpp_f32<0x1B>(dpp_f32<0x141>(a)), l4); };       // lane ^ 7, then ^ 3
    auto tail4 = [&](float a) { return lp_keep<0xB1>(lp_keep<0x4E>(a, l2), l1); };              // lane ^ 2, ^ 1
    v = lp_keep<0xB1>(v, l1);
    v = lp_keep<0xB1>(lp_keep<0x1B>(v, l2), l1);                                                // ^ 3, ^ 1
    v = tail4(lp_keep<0x141>(v, l4));                                                           // ^ 7, ^ 2, ^ 1
    v = tail4(x4(lp_keep<0x140>(v, l8)));                                                       // ^ 15, ^ 4, ..
    v = lp_pick(v, lp_xor16(dpp_f32<0x140>(v), l16), l16);                                      // ^ 31
    v = tail4(x4(lp_keep<0x128>(v, l8)));                                                       // ^ 8, ^ 4, ..
    v = lp_pick(v, lp_xor32(lp_xor16(dpp_f32<0x140>(v), l16), l32), l32);                       // ^ 63
    v = lp_pick(v, lp_xor16(v, l16), l16);                                                      // ^ 16
    return tail4(x4(lp_keep<0x128>(v, l8)));
}

struct LogprobArgs {
    const void* x; int64_t ld_outer, ld_inner; int inner;      // row r starts at (r / inner) * ld_outer + (r % inner) * ld_inner
    const int64_t* target; int V, top; float* logp; float* ent; float* stats; float* top_logp; int64_t* top_ids;
    int first;                                                 // this launch's first row
};

// running (maximum, sum e, sum e d) of a thread
struct LpSum {
    float m = -FLT_MAX, s = 0.f, w = 0.f;                      // (not -inf: -inf - -inf; a logit of -FLT_MAX itself still counts)
    __device__ __forceinline__ void rise(float to) {
        const float d = m - to, f = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        w = f * fmaf(fmaxf(d, LP_FLOOR), s, w);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        const float d = x - m, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        s += e;
        w = fmaf(e, fmaxf(d, LP_FLOOR), w);
    }
};

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(const LogprobArgs p) {
    using Vec = LpVec<T>;
    constexpr int E = Vec::E, WAVES = THREADS / 64;
    __shared__ float sh[3][WAVES];
    __shared__ float s_tops[WAVES * VM_MAX_TOP_LOGPROBS];
    __shared__ float s_bound;
    __shared__ uint64_t s_best[WAVES];
    __shared__ float2 cand[LP_CAND];                            // (value, column as bits)
    __shared__ int s_list[THREADS];
    __shared__ int s_n, s_owners;
    const int r = p.first + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* x = (const T*)p.x + (r / p.inner) * p.ld_outer + (r % p.inner) * p.ld_inner;
    // whole pieces, and single logits behind them; a row whose pieces would leave too few threads with a maximum for the alternatives' bound is read in
    // single logits altogether (1000000 x 100 bf16, n = 16: 3.0 ms in pieces, all 100 logits candidates, against 0.77)
    const int full = p.V / E >= min(THREADS, 2 * p.top) ? p.V / E : 0, single = p.V - full * E;
    if (tid == 0) s_n = s_owners = 0;
    LpSum a;
    uint4 raw[LP_U];                                            // (a lone wave's row of one turn stays here for the alternatives)
    float el[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int c = full * E + tid + j * THREADS;
        el[j] = -INFINITY;
        if (j * THREADS >= single) continue;
        if (c < p.V) el[j] = Vec::at(x + c);
    }
    for (int c0 = 0; c0 < full; c0 += LP_U * THREADS) {
        const int ch = c0 + tid;
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            raw[u] = lp_none<T>();
            if (ch + u * THREADS < full) raw[u] = Vec::load(x + (int64_t)(ch + u * THREADS) * E);
        }
        float f[LP_U][E], mx = -FLT_MAX;
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            if (c0 + u * THREADS >= full) break;                // (the same for the whole workgroup: short rows pay for the pieces they have)
            Vec::unpack(raw[u], f[u]);
#pragma unroll
            for (int j = 0; j < E; ++j) mx = fmaxf(mx, f[u][j]);
        }
        if (mx > a.m) a.rise(mx);
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            if (c0 + u * THREADS >= full) break;
#pragma unroll
            for (int j = 0; j < E; ++j) a.add(f[u][j]);
        }
    }
    {
        float mx = -FLT_MAX;
#pragma unroll
        for (int j = 0; j < E; ++j) mx = fmaxf(mx, el[j]);
        if (mx > a.m) a.rise(mx);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (j * THREADS >= single) break;
            a.add(el[j]);
        }
    }
    const float mine = a.m;                                     // this thread's own maximum
    // the row's sums
    float m = wave_max(a.m);
    if (lane == 0) sh[0][wave] = m;
    __syncthreads();
    m = sh[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) m = fmaxf(m, sh[0][i]);
    a.rise(m);
    const float ws = wave_sum(a.s), ww = wave_sum(a.w);
    if (lane == 0) { sh[1][wave] = ws; sh[2][wave] = ww; }
    // (the alternatives' bound in the same round: the wave's largest maxima in order)
    if (p.top > 0) {
        float sorted;
        if (p.top == 1) sorted = wave_max(mine);
        else sorted = lp_sort_wave(mine);
        if (WAVES == 1) { if (lane == p.top - 1) s_bound = sorted; }
        else if (lane < p.top) s_tops[wave * p.top + lane] = sorted;
    }
    __syncthreads();
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) { s += sh[1][i]; w += sh[2][i]; }
    const float ls = logf(s);
    if (tid == 0) {
        const int64_t t = p.target[r];
        if (p.stats) { p.stats[2 * (int64_t)r] = m; p.stats[2 * (int64_t)r + 1] = ls; }
        p.ent[r] = s == 0.f ? 0.f : ls - w / s;
        p.logp[r] = t < 0 ? 0.f : (t >= p.V ? NAN : (s == 0.f ? -INFINITY : (Vec::at(x + t) - m) - ls));
    }
    if (p.top == 0) return;
    if (WAVES > 1) {                                            // the n-th largest of the waves' lists
        for (int i = tid; i < WAVES * p.top; i += THREADS) {
            const float v = s_tops[i];
            int above = 0;
#pragma unroll 8
            for (int q = 0; q < WAVES * p.top; ++q) { const float o = s_tops[q]; above += o > v || (o == v && q < i) ? 1 : 0; }
            if (above == p.top - 1) s_bound = v;
        }
        __syncthreads();
    }
    const float L = s_bound;
    int found = 0;                                              // of a lone wave; several count in s_n
    auto look = [&](int c, float v) {
        const uint64_t hits = __ballot(v >= L);
        if (hits == 0) return;
        const int leader = __ffsll((unsigned long long)hits) - 1, count = __popcll(hits);
        int at = found;
        if (WAVES == 1) found += count;
        else {
            if (lane == leader) at = atomicAdd(&s_n, count);
            at = __builtin_amdgcn_readlane(at, leader);
        }
        at += __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0));
        if (v >= L && at < LP_CAND) cand[at] = make_float2(v, __int_as_float(c));
    };
    auto look_piece = [&](int ch, const uint4 piece) {           // (every lane takes part, so that a wave's count stays one number; L > -inf)
        float f[E], mx = -INFINITY;
        Vec::unpack(piece, f);
#pragma unroll
        for (int j = 0; j < E; ++j) mx = fmaxf(mx, f[j]);
        if (__any(mx >= L)) {
#pragma unroll
            for (int j = 0; j < E; ++j) look(ch * E + j, f[j]);
        }
    };
#pragma unroll
    for (int j = 0; j < E; ++j) {
        if (j * THREADS >= single) break;
        const int c = full * E + tid + j * THREADS;
        if (WAVES > 1) el[j] = c < p.V ? Vec::at(x + c) : -INFINITY;       // (again: registers held through the pass would cost it waves)
        look(c, el[j]);
    }
    if (WAVES == 1 && full <= LP_U * THREADS) {                               // the pieces are still in the registers
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            if (u * THREADS >= full) break;
            look_piece(tid + u * THREADS, raw[u]);
        }
    } else {                                                    // the owners' pieces once more, dealt out to all threads
        if (mine >= L) s_list[atomicAdd(&s_owners, 1)] = tid;
        __syncthreads();
        const int owners = s_owners, pieces = owners * ((full + THREADS - 1) / THREADS);
        for (int i0 = 0; i0 < pieces; i0 += THREADS) {
            const int i = i0 + tid, turn = i / owners, ch = i < pieces ? s_list[i - turn * owners] + turn * THREADS : full;
            look_piece(ch, ch < full ? Vec::load(x + (int64_t)ch * E) : lp_none<T>());
        }
    }
    __syncthreads();
    const int n = WAVES == 1 ? __builtin_amdgcn_readfirstlane(found) : s_n;
    float* out = p.top_logp + (int64_t)r * p.top;
    int64_t* ids = p.top_ids + (int64_t)r * p.top;
    if (n >= p.top && n <= LP_CAND && s == s) {
        for (int i = tid; i < n; i += THREADS) {
            const float v = cand[i].x; const int c = __float_as_int(cand[i].y);
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) { const float2 o = cand[j]; above += (o.x > v || (o.x == v && __float_as_int(o.y) < c)) ? 1 : 0; }
            if (above < p.top) { ids[above] = c; out[above] = (v - m) - ls; }
        }
        return;
    }
    uint64_t last = ~0ull;                                      // (value key, V - 1 - column): descending order of it is the wanted order
    for (int k = 0; k < p.top; ++k) {
        uint64_t b = 0;
        for (int c = tid; c < p.V; c += THREADS) {
            const uint64_t key = ((uint64_t)lp_key(Vec::at(x + c)) << 32) | (uint32_t)(p.V - 1 - c);
            if (key < last && key > b) b = key;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const uint32_t lo = __shfl_xor((int)(uint32_t)b, d), hi = __shfl_xor((int)(b >> 32), d);
            const uint64_t o = ((uint64_t)hi << 32) | lo;
            b = o > b ? o : b;
        }
        if (lane == 0) s_best[wave] = b;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) b = s_best[i] > b ? s_best[i] : b;
        __syncthreads();
        last = b;
        if (tid == 0) {
            const int c = p.V - 1 - (int)(uint32_t)b;
            ids[k] = c;
            out[k] = s == 0.f ? -INFINITY : (Vec::at(x + c) - m) - ls;
        }
    }
}

// dx_c = -p_c (g_l + sum_k g_k + g_h (log p_c + H))  + g_l [c = t] + sum_k g_k [c = id_k]
struct LogprobGradArgs {
    const void* x; int64_t ld_outer, ld_inner; int inner; const int64_t* target; int V, top; const float* stats; const float* ent; const int64_t* top_ids;
    const float* g_logp; const float* g_ent; const float* g_top; void* dx; int64_t ld_dx;
    int first;
};
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprobs_bwd_kernel(const LogprobGradArgs p) {
    using Vec = LpVec<T>;
    constexpr int E = Vec::E;
    const int r = p.first + (gridDim.x - 1 - blockIdx.x), tid = threadIdx.x;
    const T* x = (const T*)p.x + (r / p.inner) * p.ld_outer + (r % p.inner) * p.ld_inner;
    T* dx = (T*)p.dx + r * p.ld_dx;
    const int64_t t = p.target[r];
    const float m = p.stats[2 * (int64_t)r], ls = p.stats[2 * (int64_t)r + 1], H = p.ent[r];
    const int full = p.V / E, rest = full * E + tid;
    const bool empty = ls == -INFINITY;                         // nothing in the row: its outputs are constants
    const float gl = !p.g_logp || t < 0 || empty ? 0.f : (t < p.V ? p.g_logp[r] : NAN), gh = p.g_ent && !empty ? p.g_ent[r] : 0.f;
    const int top = p.g_top && !empty ? p.top : 0;
    float g0 = gl;
    for (int k = 0; k < top; ++k) g0 += p.g_top[(int64_t)r * p.top + k];
    g0 = fmaf(gh, H, g0);
    auto grad = [&](float v) {                                  // without the single columns' own terms
        const float lp = (v - m) - ls, e = __builtin_amdgcn_exp2f(lp * LP_LOG2E);
        return empty ? 0.f : -e * fmaf(gh, fmaxf(lp, LP_FLOOR), g0);
    };
    for (int ch = tid; ch < full; ch += LP_U * THREADS) {
        uint4 raw[LP_U];
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            raw[u] = lp_none<T>();
            if (ch + u * THREADS < full) raw[u] = Vec::load(x + (int64_t)(ch + u * THREADS) * E);
        }
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            if (ch + u * THREADS >= full) break;
            float f[E];
            Vec::unpack(raw[u], f);
#pragma unroll
            for (int j = 0; j < E; ++j) f[j] = grad(f[j]);
            Vec::store(dx + (int64_t)(ch + u * THREADS) * E, f);
        }
    }
    if (rest < p.V) Vec::put(dx + rest, grad(Vec::at(x + rest)));
    // the target's and the alternatives' columns once more, with their own terms (whole values, not added to the rounded ones)
    __syncthreads();
    if (tid <= top) {
        const int64_t c = tid < top ? p.top_ids[(int64_t)r * p.top + tid] : t;
        if (c >= 0 && c < p.V) {
            float d = grad(Vec::at(x + c)) + (c == t ? gl : 0.f);
            for (int k = 0; k < top; ++k) d += p.top_ids[(int64_t)r * p.top + k] == c ? p.g_top[(int64_t)r * p.top + k] : 0.f;
            Vec::put(dx + c, d);
        }
    }
}

static int logprob_check(const void* x, int R, int inner, int V, int top, int dtype, const char* what) {
    VM_REQUIRE(x && R > 0 && inner > 0 && V > 0, "%s: bad arguments", what);
    VM_REQUIRE(top >= 0 && top <= VM_MAX_TOP_LOGPROBS && top <= V, "%s: top = %d: at most %d and at most V alternatives", what, top, VM_MAX_TOP_LOGPROBS);
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "%s: dtype must be VM_F32 or VM_BF16", what);
    return VM_OK;
}
// Threads per row, by the 16-byte pieces of a row.  Forward: one wave where a row is short and there are rows enough to fill the chip with waves (no
// barriers, many rows in flight): 100000 x 1000 bf16 with 5 alternatives 96 us with 64 threads, 195 with 128, 292 with 256; 20000 x 8832 bf16 86 / 102 / 103;
// longer rows the other way round: 10000 x 8832 fp32 82 / 76 / 71, 8192 x 30522 bf16 - / 123 / 115.  Backward (no reduction): about one batch of
// LP_U pieces per thread: 100000 x 1000 bf16 106 us with 64 threads, 144 with 128, 176 with 256, 676 with 1024; 20000 x 8832 bf16 111 with 256, 118 with 512, 184
// with 1024; 10000 x 8832 fp32 116 / 108 / 120; 8192 x 30522 bf16 169 / 164 / 157.
#define LP_LAUNCH(KERNEL, THREADS)                                                                                          \
    for (int64_t first = 0; first < R; first += VM_MAX_BLOCKS) {                                                            \
        const dim3 grid((unsigned)std::min<int64_t>(R - first, VM_MAX_BLOCKS));                                             \
        a.first = (int)first;                                                                                               \
        if (dtype == VM_F32) hipLaunchKernelGGL((KERNEL<float, THREADS>), grid, dim3(THREADS), 0, s, a);                    \
        else hipLaunchKernelGGL((KERNEL<bf16_t, THREADS>), grid, dim3(THREADS), 0, s, a);                                   \
    }

extern "C" int vm_token_logprobs_fwd(const void* logits, int64_t ld_outer, int64_t ld_inner, int inner, const int64_t* targets, int R, int V, int top,
                                     float* logp, float* entropy, float* stats, float* top_logp, int64_t* top_ids, int dtype, void* stream) {
    if (int rc = logprob_check(logits, R, inner, V, top, dtype, "vm_token_logprobs_fwd")) return rc;
    VM_REQUIRE(targets && logp && entropy && (top == 0 || (top_logp && top_ids)), "vm_token_logprobs_fwd: null pointer");
    LogprobArgs a = {logits, ld_outer, ld_inner, inner, targets, V, top, logp, entropy, stats, top_logp, top_ids, 0};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_LOSS, (dtype == VM_F32 ? 4.0 : 2.0) * R * (double)V, s, "token_logprobs_r%d_V%d_k%d", R, V, top);
    if (V / (dtype == VM_F32 ? 4 : 8) <= 1536 && R >= 2048) { LP_LAUNCH(token_logprobs_kernel, 64) }
    else { LP_LAUNCH(token_logprobs_kernel, 256) }
    return vm_check_launch("vm_token_logprobs_fwd");
}
extern "C" int vm_token_logprobs_bwd(const void* logits, int64_t ld_outer, int64_t ld_inner, int inner, const int64_t* targets, int R, int V, int top,
                                     const float* stats, const float* entropy, const int64_t* top_ids, const float* g_logp, const float* g_entropy,
                                     const float* g_top, void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
    if (int rc = logprob_check(logits, R, inner, V, top, dtype, "vm_token_logprobs_bwd")) return rc;
    VM_REQUIRE(targets && stats && entropy && dlogits && ld_dlogits >= V && (!g_top || top == 0 || top_ids), "vm_token_logprobs_bwd: bad arguments");
    LogprobGradArgs a = {logits, ld_outer, ld_inner, inner, targets, V, top, stats, entropy, top_ids, g_logp, g_entropy, top ? g_top : nullptr, dlogits, ld_dlogits, 0};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_LOSS, (dtype == VM_F32 ? 8.0 : 4.0) * R * (double)V, s, "token_logprobs_bwd_r%d_V%d_k%d", R, V, top);
    const int want = V / (dtype == VM_F32 ? 4 : 8) / LP_U;
    if (want <= 96) { LP_LAUNCH(token_logprobs_bwd_kernel, 64) }
    else if (want <= 384) { LP_LAUNCH(token_logprobs_bwd_kernel, 256) }
    else if (want <= 704) { LP_LAUNCH(token_logprobs_bwd_kernel, 512) }
    else { LP_LAUNCH(token_logprobs_bwd_kernel, 1024) }
    return vm_check_launch("vm_token_logprobs_bwd");
}
