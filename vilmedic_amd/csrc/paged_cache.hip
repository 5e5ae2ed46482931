// paged_cache.hip -- the bookkeeping of a paged key-value cache on the device: page allocation, block tables and slot maps from request
// lengths (vm_paged_plan), and the write of new keys / values through a slot map (vm_paged_kv_write).
//
// Cache layout: k_pages, v_pages [P, Hkv, page_size, dh], so the keys of one head inside one page are ONE contiguous run of page_size * dh
// elements (2 KB for 16 x 64 bf16): the attention kernel reads whole runs, whatever the number of heads.  A token's slot is
// page * page_size + offset; slots are int64, everything inside a row of the table is int32.
#include "common.h"

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
// Phase A, one workgroup: two scans over the rows (tokens; wanted and returned pages packed into one 64-bit scan).  Phase B, any grid: table
// rows and ring places by wave, slots by token (binary search of the row in cu_tokens).
struct PlanRow { int len, ofs, cnt, kind; };       // kind 0 refused / nothing, 1 accepted (cnt pages from ring place head + ofs), 2 released (cnt pages back)
struct PlanRing { int head, count, returned, pad; };
struct PlanArgs {
    int32_t* lengths; const int32_t* new_tokens; int32_t* table; int64_t ld_table; int N, M; int32_t* free_pages; int32_t* ring; int P, s;
    int64_t* slots; int64_t* positions; int max_tokens; int32_t* cu; int32_t* granted; PlanRow* rows; PlanRing* snap;
};
#define PLAN_THREADS 1024

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) {
    const int lo = __shfl_up((int)(uint32_t)v, d), hi = __shfl_up((int)(v >> 32), d);
    return ((int64_t)hi << 32) | (uint32_t)lo;
}
// inclusive scan over the workgroup's 1024 threads; total of all threads in `total`
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int64_t o = shfl_up64(v, d); if (lane >= d) v += o; }
    if (lane == 63) sh[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < PLAN_THREADS / 64; ++w) { const int64_t x = sh[w]; if (w < wave) before += x; total += x; }
    __syncthreads();
    return v + before;
}

__device__ __forceinline__ void plan_scan(const PlanArgs& p) {
    __shared__ int64_t sh[PLAN_THREADS / 64];
    const int tid = threadIdx.x;
    const int head = p.ring[0], count = p.ring[1];
    const int64_t cap = (int64_t)p.M * p.s;
    int64_t tok_before = 0;
    int64_t want_before = 0, back_before = 0, taken_all = 0;
    for (int base = 0; base < p.N; base += PLAN_THREADS) {
        const int i = base + tid;
        int64_t L = 0; int n = 0;
        if (i < p.N) {
            L = p.lengths[i]; n = p.new_tokens[i];
            L = L < 0 ? 0 : (L > cap ? cap : L);
        }
        const int64_t t = n > 0 ? n : 0;
        int64_t tot;
        const int64_t end = tok_before + block_scan(t, sh, tot);
        tok_before += tot;
        const int have = (int)((L + p.s - 1) / p.s);
        const bool fits = n > 0 && L + t <= cap && end <= p.max_tokens;
        const int want = fits ? (int)((L + t + p.s - 1) / p.s) - have : 0;
        const int back = n < 0 ? have : 0;
        const int64_t both = block_scan(((int64_t)want << 32) | (uint32_t)back, sh, tot);      // (sums below 2^31 each: the host checks N * M)
        const int64_t upto = want_before + (both >> 32);
        const int64_t back_upto = back_before + (both & 0xffffffff);
        want_before += tot >> 32; back_before += tot & 0xffffffff;
        const bool ok = fits && (want == 0 || upto <= count);
        block_scan(ok ? want : 0, sh, tot);
        taken_all += tot;
        if (i < p.N) {
            PlanRow r;
            r.len = (int)L;
            r.kind = n < 0 ? 2 : (ok ? 1 : 0);
            r.cnt = n < 0 ? back : (ok ? want : 0);
            r.ofs = n < 0 ? (int)(back_upto - back) : (int)(upto - want);
            p.rows[i] = r;
            p.lengths[i] = n < 0 ? 0 : (int)(L + (ok ? t : 0));
            p.granted[i] = ok ? (int)t : 0;
            p.cu[i + 1] = (int)(end < p.max_tokens ? end : p.max_tokens);
        }
    }
    if (tid == 0) {
        p.cu[0] = 0;
        const int64_t room = (int64_t)p.P - count;                        // (a count that lies outside [0, P] is the caller's error; nothing is read or written outside)
        const int returned = (int)(back_before < room ? back_before : (room > 0 ? room : 0));
        PlanRing g = {head, count, returned, 0};
        *p.snap = g;
        p.ring[0] = (int)(((int64_t)head + taken_all) % p.P);
        p.ring[1] = (int)(count - taken_all + returned);
    }
}
__device__ __forceinline__ int ring_place(int64_t at, int P) { const int r = (int)(at % P); return r < 0 ? r + P : r; }

// table rows and ring places: wave `wave` of `waves`
__device__ __forceinline__ void plan_rows(const PlanArgs& p, int wave, int waves) {
    const PlanRing g = *p.snap;
    const int lane = threadIdx.x & 63;
    for (int i = wave; i < p.N; i += waves) {
        const PlanRow r = p.rows[i];
        int32_t* row = p.table + (int64_t)i * p.ld_table;
        if (r.kind == 1) {
            const int have = (r.len + p.s - 1) / p.s;
            for (int j = lane; j < r.cnt; j += 64) row[have + j] = p.free_pages[ring_place((int64_t)g.head + r.ofs + j, p.P)];
        } else if (r.kind == 2) {
            for (int j = lane; j < p.M; j += 64) {
                if (j < r.cnt && r.ofs + j < g.returned) p.free_pages[ring_place((int64_t)g.head + g.count + r.ofs + j, p.P)] = row[j];
                row[j] = -1;
            }
        }
    }
}
// the slot and position of token `t`
__device__ __forceinline__ void plan_token(const PlanArgs& p, const PlanRing& g, int t) {
    int64_t slot = -1, pos = 0;
    if (t < p.cu[p.N]) {
        int lo = 0, hi = p.N;                                             // the last row whose first token is <= t
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (p.cu[mid] <= t) lo = mid; else hi = mid; }
        const PlanRow r = p.rows[lo];
        if (r.kind == 1) {
            pos = r.len + (t - p.cu[lo]);
            const int have = (r.len + p.s - 1) / p.s, col = (int)(pos / p.s);
            // a page taken in this call is read from the ring: the row of the table may be under construction
            const int page = col >= have ? p.free_pages[ring_place((int64_t)g.head + r.ofs + (col - have), p.P)] : p.table[(int64_t)lo * p.ld_table + col];
            if (page >= 0 && page < p.P) slot = (int64_t)page * p.s + (pos - (int64_t)col * p.s);
        }
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
}

__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_scan_kernel(const PlanArgs p) { plan_scan(p); }
__global__ __launch_bounds__(256) void paged_plan_fill_kernel(const PlanArgs p) {
    plan_rows(p, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4);
    const PlanRing g = *p.snap;
    for (int t = blockIdx.x * 256 + threadIdx.x; t < p.max_tokens; t += gridDim.x * 256) plan_token(p, g, t);
}

extern "C" size_t vm_paged_plan_ws(int N) { return N > 0 ? (size_t)N * sizeof(PlanRow) + sizeof(PlanRing) : 0; }

extern "C" int vm_paged_plan(int32_t* lengths, const int32_t* new_tokens, int32_t* block_table, int64_t ld_table, int N, int M, int32_t* free_pages,
                             int32_t* ring, int P, int page_size, int64_t* slots, int64_t* positions, int max_tokens, int32_t* cu_tokens,
                             int32_t* granted, void* ws, size_t ws_bytes, void* stream) {
    VM_REQUIRE(lengths && new_tokens && block_table && free_pages && ring && cu_tokens && granted && ws, "vm_paged_plan: null pointer");
    VM_REQUIRE(N > 0 && M > 0 && P > 0 && page_size > 0 && max_tokens >= 0 && ld_table >= M, "vm_paged_plan: bad shape");
    VM_REQUIRE(max_tokens == 0 || (slots && positions), "vm_paged_plan: slots and positions of max_tokens entries required");
    VM_REQUIRE(max_tokens <= (1 << 30), "vm_paged_plan: max_tokens must be at most 2^30");
    VM_REQUIRE((int64_t)N * M < (1ll << 31) && (int64_t)M * page_size < (1ll << 31), "vm_paged_plan: N * M and M * page_size must stay below 2^31");
    VM_REQUIRE(((uintptr_t)ws % 16) == 0 && ws_bytes >= vm_paged_plan_ws(N), "vm_paged_plan: 16-byte aligned workspace of vm_paged_plan_ws(N) bytes required");
    PlanRow* rows = reinterpret_cast<PlanRow*>(ws);
    PlanArgs a = {lengths, new_tokens, block_table, ld_table, N, M, free_pages, ring, P, page_size, slots, positions, max_tokens, cu_tokens, granted,
                  rows, reinterpret_cast<PlanRing*>(rows + N)};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_DECODE, 16.0 * N + 16.0 * max_tokens, s, "paged_plan_n%d_t%d", N, max_tokens);
    hipLaunchKernelGGL(paged_plan_scan_kernel, dim3(1), dim3(PLAN_THREADS), 0, s, a);
    int blocks = max_tokens > N * 64 ? (max_tokens + 255) / 256 : (N + 3) / 4;
    if (blocks > 2048) blocks = 2048;
    if (blocks < 1) blocks = 1;
    hipLaunchKernelGGL(paged_plan_fill_kernel, dim3(blocks), dim3(256), 0, s, a);
    return vm_check_launch("vm_paged_plan");
}

// ------------------------------------------------------------------ write
// k_pages[slot / s, h, slot % s, :] = k[t, h, :] and v likewise, for every token with 0 <= slot < P s.  A pure copy (HBM-bound; every value moves
// as it is, so no type but the storage size matters): one workgroup per token, a 16-byte piece per thread where the new rows are aligned.
struct KvWriteArgs {
    const char* k; const char* v; int64_t k_tok, k_head, v_tok, v_head;      // strides in BYTES
    char* k_pages; char* v_pages; const int64_t* slots; int H, dh, s, esize; int64_t n_slots;
};
template <int PIECE>        // bytes a thread moves: 16, or one element
__global__ __launch_bounds__(256) void paged_kv_write_kernel(const KvWriteArgs p) {
    const int64_t t = blockIdx.x;
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
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "vm_paged_kv_write: dtype must be VM_F32 or VM_BF16");
    VM_REQUIRE(((uintptr_t)k_pages % 16) == 0 && ((uintptr_t)v_pages % 16) == 0, "vm_paged_kv_write: pages must be 16-byte aligned");
    const int e = dtype == VM_F32 ? 4 : 2;
    KvWriteArgs a = {(const char*)k, (const char*)v, k_token_stride * e, k_head_stride * e, v_token_stride * e, v_head_stride * e, (char*)k_pages, (char*)v_pages,
                     slots, Hkv, dh, page_size, e, (int64_t)P * page_size};
    const bool wide = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)a.k_tok | (uintptr_t)a.k_head | (uintptr_t)a.v_tok | (uintptr_t)a.v_head) % 16) == 0;
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_DECODE, 4.0 * T * Hkv * (double)dh * e, s, "paged_kv_write_t%d_h%d_d%d", T, Hkv, dh);
    if (wide) hipLaunchKernelGGL(paged_kv_write_kernel<16>, dim3(T), dim3(256), 0, s, a);
    else if (e == 4) hipLaunchKernelGGL(paged_kv_write_kernel<4>, dim3(T), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(paged_kv_write_kernel<2>, dim3(T), dim3(256), 0, s, a);
    return vm_check_launch("vm_paged_kv_write");
}
