// paged_cache.hip -- the bookkeeping of a paged key-value cache on the device: page allocation, block tables and slot maps from request
// lengths (vm_paged_plan), and the write of new keys / values through a slot map (vm_paged_kv_write).
//
// Cache layout: k_pages, v_pages [P, Hkv, page_size, dh], so the keys of one head inside one page are ONE contiguous run of page_size * dh
// elements (2 KB for 16 x 64 bf16): the attention kernel reads whole runs, whatever the number of heads.  A token's slot is
// page * page_size + offset; slots are int64, everything inside a row of the table is int32.
#include "common.h"
#include <algorithm>

// ------------------------------------------------------------------ plan
// Integers only and deterministic.  With s = page_size, L_i = clamp(lengths[i], 0, M s), t_i = max(new_tokens[i], 0):
//   end_i  = t_0 + ... + t_i                            the packed token order of the batch
//   want_i = ceil((L_i + t_i) / s) - ceil(L_i / s)      if t_i > 0, L_i + t_i <= M s and end_i <= max_tokens, else refused
//   row i is accepted iff want_i = 0 or want_0 + ... + want_i <= free pages: the accepted rows that need pages are a PREFIX of the rows that
//   need pages, so one scan decides everything and their pages are consecutive places of the free ring;
//   new_tokens[i] < 0 releases row i: its pages go to the end of the ring in (row, column) order.
// The free pages are a ring (first in, first out), not a stack: what is taken (from the head) and what is returned (behind the tail) never
// share a place while the pool holds P pages in all, so the rows can be served in parallel without a hand-over.
//
// Phase A, one workgroup: two scans over the rows (tokens; wanted and returned pages).  Phase B: table rows and ring places by wave, slots by token
// (binary search of the row in the token offsets).  A step of a running batch does both in ONE launch of one workgroup, with everything that B needs
// in LDS; with more rows or tokens B is a launch of its own over the chip.  Bound by latency everywhere: 64 rows, one more token each: 3.6 us; 500 rows
// admitted with 450000 tokens: 6.0 + 7.0 us for the two launches (7.2 MB written).
struct PlanRow { int len, ofs, cnt, kind; };       // kind 0 refused / nothing, 1 accepted (cnt pages from ring place head + ofs), 2 released (cnt pages back)
struct PlanRing { int head, count, returned, more; };      // more: rows that take several pages or return some
struct PlanArgs {
    int32_t* lengths; const int32_t* new_tokens; int32_t* table; int64_t ld_table; int N, M; int32_t* free_pages; int32_t* ring; int P, s;
    int64_t* slots; int64_t* positions; int max_tokens; int32_t* cu; int32_t* granted; PlanRow* rows; PlanRing* snap;
};
#define PLAN_THREADS 1024
#define PLAN_FUSED_ROWS 1024
#define PLAN_FUSED_TOKENS 4096
#define PLAN_FUSED_TABLE 65536
#define PLAN_FULL ((1u << 30) + 1)                // token sums stop here: past every max_tokens, and two of them fit into 32 bits

// inclusive scan over the wave: rows of 16 lanes first (row_shr 1, 2, 4, 8), then lane 15 of each row into the next (row_bcast15, row_bcast31)
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t plan_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ uint32_t plan_add(uint32_t a, uint32_t b, bool capped) { const uint32_t s = a + b; return capped ? min(s, PLAN_FULL) : s; }
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, bool capped) {
    v = plan_add(v, plan_dpp<0x111, 0xf>(v), capped);
    v = plan_add(v, plan_dpp<0x112, 0xf>(v), capped);
    v = plan_add(v, plan_dpp<0x114, 0xf>(v), capped);
    v = plan_add(v, plan_dpp<0x118, 0xf>(v), capped);
    v = plan_add(v, plan_dpp<0x142, 0xa>(v), capped);
    return plan_add(v, plan_dpp<0x143, 0xc>(v), capped);
}
// inclusive scan over the workgroup out of the wave scans and the waves' sums in `sh`; `before` (the sum of earlier calls) is added and moved on
template <int WAVES> __device__ __forceinline__ uint32_t plan_join(uint32_t v, const uint32_t* sh, uint32_t& before, bool capped) {
    const int wave = threadIdx.x >> 6;
    uint32_t mine = before, all = before;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) { const uint32_t x = sh[w]; if (w < wave) mine = plan_add(mine, x, capped); all = plan_add(all, x, capped); }
    before = all;
    return plan_add(mine, v, capped);
}

// FUSED: rows and cu are LDS arrays (cu is written to memory as well)
template <int THREADS, bool FUSED>
__device__ __forceinline__ void plan_scan(const PlanArgs& p, PlanRow* rows, int* cu, PlanRing* snap) {
    constexpr int WAVES = THREADS / 64;
    __shared__ uint32_t sh[3][WAVES];
    __shared__ int s_taken, s_more;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int turned = p.ring[0] % p.P, head = turned < 0 ? turned + p.P : turned;            // (no sum above P: two pools of more than 2^30 pages pass 31 bits)
    const int count = min(max(p.ring[1], 0), p.P);                                            // (outside: the caller's error, and no way out of the ring)
    const int64_t cap = (int64_t)p.M * p.s;
    uint32_t tok_before = 0, want_before = 0, back_before = 0;
    if (tid == 0) s_taken = s_more = 0;
    for (int base = 0; base < p.N; base += THREADS) {
        const int i = base + tid;
        int64_t L = 0; int n = 0;
        if (i < p.N) {
            L = p.lengths[i]; n = p.new_tokens[i];
            L = L < 0 ? 0 : (L > cap ? cap : L);
        }
        const int64_t t = n > 0 ? n : 0;
        __syncthreads();                                                   // (sh is free again, s_taken is set)
        const uint32_t tok = wave_scan((uint32_t)min(t, (int64_t)PLAN_FULL), true);
        if (lane == 63) sh[0][wave] = tok;
        __syncthreads();
        const uint32_t end = plan_join<WAVES>(tok, sh[0], tok_before, true);
        const int have = (int)((L + p.s - 1) / p.s);
        const bool fits = n > 0 && L + t <= cap && end <= (uint32_t)p.max_tokens;
        const int want = fits ? (int)((L + t + p.s - 1) / p.s) - have : 0;
        const int back = n < 0 ? have : 0;
        const uint32_t ws = wave_scan((uint32_t)want, false), bs = wave_scan((uint32_t)back, false);       // (sums below 2^31: the host checks N * M)
        if (lane == 63) { sh[1][wave] = ws; sh[2][wave] = bs; }
        __syncthreads();
        const uint32_t upto = plan_join<WAVES>(ws, sh[1], want_before, false), back_upto = plan_join<WAVES>(bs, sh[2], back_before, false);
        const bool ok = fits && (want == 0 || (int)upto <= count);
        const bool last = ok && want > 0;                                  // the accepted rows that need pages are a prefix: the largest upto is their sum
        if (last) atomicMax(&s_taken, (int)upto);
        if (i < p.N) {
            PlanRow r;
            r.len = (int)L;
            r.kind = n < 0 ? 2 : (ok ? 1 : 0);
            r.cnt = n < 0 ? back : (ok ? want : 0);
            r.ofs = n < 0 ? (int)back_upto - back : (int)upto - want;
            rows[i] = r;
            if (r.kind == 2 || r.cnt > 1) s_more = 1;
            p.lengths[i] = n < 0 ? 0 : (int)(L + (ok ? t : 0));
            p.granted[i] = ok ? (int)t : 0;
            const int e = (int)min(end, (uint32_t)p.max_tokens);
            cu[i + 1] = e;
            if constexpr (FUSED) p.cu[i + 1] = e;
        }
    }
    __syncthreads();
    if (tid == 0) {
        cu[0] = 0;
        if constexpr (FUSED) p.cu[0] = 0;
        const int returned = min((int)back_before, p.P - count);           // (more than fits: pages returned twice, the caller's error)
        PlanRing g = {head, count, returned, s_more};
        *snap = g;
        p.ring[0] = (int)(((int64_t)head + s_taken) % p.P);
        p.ring[1] = count - s_taken + returned;
    }
}
// pages of `len` tokens (len, s < 2^31: their sum passes 31 bits where s is no power of two)
__device__ __forceinline__ int plan_pages(int len, int s) { return (int)(((uint32_t)len + (uint32_t)s - 1) / (uint32_t)s); }
// head + something below 2 P, taken around the ring (no division: a 64-bit one costs more than everything around it)
__device__ __forceinline__ int ring_place(int64_t at, int P) { at -= at >= P ? P : 0; return (int)(at - (at >= P ? P : 0)); }

// table rows and ring places, thread `tid` of `threads`: rows that take one page (a decode step's) one thread each, the others by groups of lanes that
// cover a table row (a wave where it is longer)
__device__ __forceinline__ void plan_rows(const PlanArgs& p, const PlanRow* rows, const PlanRing g, int tid, int threads) {
    for (int i = tid; i < p.N; i += threads) {
        const PlanRow r = rows[i];
        if (r.kind == 1 && r.cnt == 1) p.table[(int64_t)i * p.ld_table + plan_pages(r.len, p.s)] = p.free_pages[ring_place((int64_t)g.head + r.ofs, p.P)];
    }
    if (!g.more) return;
    int lanes = 64;
    while (lanes > 8 && lanes / 2 >= p.M) lanes >>= 1;
    const int lane = tid & (lanes - 1);
    for (int i = tid / lanes; i < p.N; i += threads / lanes) {
        const PlanRow r = rows[i];
        int32_t* row = p.table + (int64_t)i * p.ld_table;
        if (r.kind == 1 && r.cnt > 1) {
            const int have = plan_pages(r.len, p.s);
            for (int j = lane; j < r.cnt; j += lanes) row[have + j] = p.free_pages[ring_place((int64_t)g.head + r.ofs + j, p.P)];
        } else if (r.kind == 2) {
            for (int j = lane; j < p.M; j += lanes) {
                if (j < r.cnt && r.ofs + j < g.returned) p.free_pages[ring_place((int64_t)g.head + g.count + r.ofs + j, p.P)] = row[j];
                row[j] = -1;
            }
        }
    }
}
// the slot and position of token `t`
__device__ __forceinline__ void plan_token(const PlanArgs& p, const PlanRow* rows, const int* cu, const PlanRing g, int t) {
    int64_t slot = -1, pos = 0;
    if (t < cu[p.N]) {
        int lo = 0, hi = p.N;                                             // the last row whose first token is <= t
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (cu[mid] <= t) lo = mid; else hi = mid; }
        const PlanRow r = rows[lo];
        if (r.kind == 1) {
            const int at = r.len + (t - cu[lo]), have = plan_pages(r.len, p.s), col = at / p.s;
            // a page taken in this call is read from the ring: the row of the table may be under construction
            const int page = col >= have ? p.free_pages[ring_place((int64_t)g.head + r.ofs + (col - have), p.P)] : p.table[(int64_t)lo * p.ld_table + col];
            pos = at;
            if (page >= 0 && page < p.P) slot = (int64_t)page * p.s + (at - col * p.s);
        }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_plan_step_kernel(const PlanArgs p) {
    __shared__ PlanRow rows[PLAN_FUSED_ROWS];
    __shared__ int cu[PLAN_FUSED_ROWS + 1];
    __shared__ PlanRing snap;
    plan_scan<THREADS, true>(p, rows, cu, &snap);
    __syncthreads();
    const PlanRing g = snap;
    plan_rows(p, rows, g, threadIdx.x, THREADS);
    for (int t = threadIdx.x; t < p.max_tokens; t += THREADS) plan_token(p, rows, cu, g, t);
}
__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_scan_kernel(const PlanArgs p) { plan_scan<PLAN_THREADS, false>(p, p.rows, p.cu, p.snap); }
__global__ __launch_bounds__(256) void paged_plan_fill_kernel(const PlanArgs p) {
    const PlanRing g = *p.snap;
    plan_rows(p, p.rows, g, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
    for (int t = blockIdx.x * 256 + threadIdx.x; t < p.max_tokens; t += gridDim.x * 256) plan_token(p, p.rows, p.cu, g, t);
}

// One launch while one workgroup can do the step: its rows fit into LDS, and the tokens do not keep it busy for long.  500 rows x 128 columns: one more token for
// each in one launch 6.3 us, in two 8.5 us and 5 us more of the host; releasing all of them at once 24 us against 8.5, which is rarer.
static bool plan_fused(int N, int M, int max_tokens) { return N <= PLAN_FUSED_ROWS && max_tokens <= PLAN_FUSED_TOKENS && (int64_t)N * M <= PLAN_FUSED_TABLE; }
extern "C" size_t vm_paged_plan_ws(int N, int M, int max_tokens) { return N <= 0 || plan_fused(N, M, max_tokens) ? 0 : (size_t)N * sizeof(PlanRow) + sizeof(PlanRing); }

extern "C" int vm_paged_plan(int32_t* lengths, const int32_t* new_tokens, int32_t* block_table, int64_t ld_table, int N, int M, int32_t* free_pages,
                             int32_t* ring, int P, int page_size, int64_t* slots, int64_t* positions, int max_tokens, int32_t* cu_tokens,
                             int32_t* granted, void* ws, size_t ws_bytes, void* stream) {
    VM_REQUIRE(lengths && new_tokens && block_table && free_pages && ring && cu_tokens && granted, "vm_paged_plan: null pointer");
    VM_REQUIRE(N > 0 && M > 0 && P > 0 && page_size > 0 && max_tokens >= 0 && ld_table >= M, "vm_paged_plan: bad shape");
    VM_REQUIRE(max_tokens == 0 || (slots && positions), "vm_paged_plan: slots and positions of max_tokens entries required");
    VM_REQUIRE(max_tokens <= (1 << 30) && N <= (1 << 30), "vm_paged_plan: max_tokens and N must be at most 2^30");       // (the strides of the loops over them stay in 31 bits)
    VM_REQUIRE((int64_t)N * M < (1ll << 31) && (int64_t)M * page_size < (1ll << 31), "vm_paged_plan: N * M and M * page_size must stay below 2^31");
    const size_t need = vm_paged_plan_ws(N, M, max_tokens);
    VM_REQUIRE(need == 0 || (ws && ((uintptr_t)ws % 16) == 0 && ws_bytes >= need), "vm_paged_plan: 16-byte aligned workspace of %zu bytes required", need);
    PlanRow* rows = reinterpret_cast<PlanRow*>(ws);
    PlanArgs a = {lengths, new_tokens, block_table, ld_table, N, M, free_pages, ring, P, page_size, slots, positions, max_tokens, cu_tokens, granted,
                  rows, reinterpret_cast<PlanRing*>(rows + N)};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_DECODE, 16.0 * N + 16.0 * max_tokens, s, "paged_plan_n%d_t%d", N, max_tokens);
    if (plan_fused(N, M, max_tokens)) {
        if (N <= 256 && max_tokens <= 1024) hipLaunchKernelGGL(paged_plan_step_kernel<256>, dim3(1), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(paged_plan_step_kernel<1024>, dim3(1), dim3(1024), 0, s, a);
        return vm_check_launch("vm_paged_plan");
    }
    hipLaunchKernelGGL(paged_plan_scan_kernel, dim3(1), dim3(PLAN_THREADS), 0, s, a);
    int blocks = max_tokens > N * 64ll ? (max_tokens + 255) / 256 : (N + 3) / 4;
    if (blocks > 2048) blocks = 2048;
    if (blocks < 1) blocks = 1;
    hipLaunchKernelGGL(paged_plan_fill_kernel, dim3(blocks), dim3(256), 0, s, a);
    return vm_check_launch("vm_paged_plan");
}

// ------------------------------------------------------------------ write
// k_pages[slot / s, h, slot % s, :] = k[t, h, :] and v likewise, for every token with 0 <= slot < P s.  A pure copy (HBM-bound; every value moves
// as it is, so no type but the storage size matters): one workgroup per token, a 16-byte piece per thread where the new rows are aligned.
// Measured: 16000 tokens x 8 heads x 128 bf16 columns (128 MB read and written) 24.6 us, 5.2 TB/s, the rate of a large copy; 64 tokens x 12 heads x 64
// columns 2.7 us, a launch's latency.
struct KvWriteArgs {
    const char* k; const char* v; int64_t k_tok, k_head, v_tok, v_head;      // strides in BYTES
    char* k_pages; char* v_pages; const int64_t* slots; int H, dh, s, esize; int64_t n_slots, first;
};
template <int PIECE>        // bytes a thread moves: 16, or one element
__global__ __launch_bounds__(256) void paged_kv_write_kernel(const KvWriteArgs p) {
    const int64_t t = p.first + blockIdx.x;
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= p.n_slots) return;
    const int64_t page = slot / p.s;
    const int off = (int)(slot - page * p.s);
    const int row_bytes = p.dh * p.esize, ppr = row_bytes / PIECE, total = p.H * ppr;
    for (int c = threadIdx.x; c < 2 * total; c += 256) {
        const bool is_v = c >= total;
        const int cc = is_v ? c - total : c;
        const int h = cc / ppr, b = (cc - h * ppr) * PIECE;
        const char* src = is_v ? p.v + t * p.v_tok + h * p.v_head + b : p.k + t * p.k_tok + h * p.k_head + b;
        char* dst = (is_v ? p.v_pages : p.k_pages) + ((page * p.H + h) * p.s + off) * (int64_t)row_bytes + b;
        if constexpr (PIECE == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
        else if constexpr (PIECE == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
        else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
    }
}

extern "C" int vm_paged_kv_write(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                 void* k_pages, void* v_pages, const int64_t* slots, int T, int Hkv, int dh, int P, int page_size, int dtype, void* stream) {
    VM_REQUIRE(k && v && k_pages && v_pages && slots, "vm_paged_kv_write: null pointer");
    VM_REQUIRE(T > 0 && Hkv > 0 && P > 0 && page_size > 0 && dh > 0 && dh % 8 == 0, "vm_paged_kv_write: bad shape (dh must be a multiple of 8)");
    VM_REQUIRE((int64_t)Hkv * dh < (1ll << 29), "vm_paged_kv_write: Hkv * dh must stay below 2^29");              // (a token's pieces are counted in 31 bits)
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "vm_paged_kv_write: dtype must be VM_F32 or VM_BF16");
    VM_REQUIRE(((uintptr_t)k_pages % 16) == 0 && ((uintptr_t)v_pages % 16) == 0, "vm_paged_kv_write: pages must be 16-byte aligned");
    const int e = dtype == VM_F32 ? 4 : 2;
    KvWriteArgs a = {(const char*)k, (const char*)v, k_token_stride * e, k_head_stride * e, v_token_stride * e, v_head_stride * e, (char*)k_pages, (char*)v_pages,
                     slots, Hkv, dh, page_size, e, (int64_t)P * page_size, 0};
    const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)a.k_tok | (uintptr_t)a.k_head | (uintptr_t)a.v_tok | (uintptr_t)a.v_head) % 16) == 0;
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_DECODE, 4.0 * T * Hkv * (double)dh * e, s, "paged_kv_write_t%d_h%d_d%d", T, Hkv, dh);
    for (int64_t first = 0; first < T; first += VM_MAX_BLOCKS) {
        const dim3 grid((unsigned)std::min<int64_t>(T - first, VM_MAX_BLOCKS));
        a.first = first;
        if (wide) hipLaunchKernelGGL(paged_kv_write_kernel<16>, grid, dim3(256), 0, s, a);
        else if (e == 4) hipLaunchKernelGGL(paged_kv_write_kernel<4>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(paged_kv_write_kernel<2>, grid, dim3(256), 0, s, a);
    }
    return vm_check_launch("vm_paged_kv_write");
}
