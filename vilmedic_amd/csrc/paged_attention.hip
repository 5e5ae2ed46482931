// paged_attention.hip -- attention of one new token per row over a paged key-value cache (layout: csrc/paged_cache.hip).
//   o[n, h] = sum_j softmax_j(scale * q[n, h] . K_j) V_j     over the keys j < lengths[n] of head h / (Hq / Hkv), key j in page block_table[n, j / s]
// A key whose page number lies outside [0, P) does not exist, and no key at all leaves a row of zeros; what a page holds behind a row's length is
// never multiplied (stale values, NaN included, do not reach the result).
#include "common.h"

struct PagedAttnArgs {
    const void* q; int64_t q_row, q_head; const void* k; const void* v; const int32_t* table; int64_t ld_table; const int32_t* lengths; void* o;
    int N, Hq, Hk, G, dh, P, s, M; float scale_log2;
};
template <typename T> __device__ __forceinline__ float ld1(const T* p);
template <> __device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ld1<bf16_t>(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16_t* p, float v) { *p = f32_to_bf16(v); }

// one wave per (row, query head): a lane scores one key, then the lanes split the head's columns
template <typename T>
__global__ __launch_bounds__(64) void paged_attention_kernel(const PagedAttnArgs p) {
    __shared__ float qs[256];
    __shared__ float ps[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x, n = blockIdx.x / p.Hq, h = blockIdx.x - n * p.Hq, kv = h / p.G;
    const T* q = (const T*)p.q + n * p.q_row + h * p.q_head;
    for (int d = lane; d < p.dh; d += 64) qs[d] = ld1(q + d) * p.scale_log2;
    int64_t len = p.lengths[n];
    const int64_t cap = (int64_t)p.M * p.s;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    for (int64_t j0 = 0; j0 < len; j0 += 64) {
        const int64_t j = j0 + lane;
        int64_t row = -1;
        float sc = -INFINITY;
        if (j < len) {
            const int page = p.table[n * p.ld_table + j / p.s];
            if (page >= 0 && page < p.P) {
                row = (((int64_t)page * p.Hk + kv) * p.s + j % p.s) * p.dh;
                const T* k = (const T*)p.k + row;
                sc = 0.f;
                for (int d = 0; d < p.dh; ++d) sc = fmaf(qs[d], ld1(k + d), sc);
            }
        }
        const float mn = fmaxf(m, wave_max(sc));
        const float base = mn == -INFINITY ? 0.f : mn;
        const float e = exp2f(sc - base), f = exp2f(m - base);
        l = l * f + wave_sum(e);
        m = mn;
        __syncthreads();
        ps[lane] = e; at[lane] = row;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d < p.dh) {
                float a = acc[i] * f;
                for (int u = 0; u < 64; ++u) if (at[u] >= 0) a = fmaf(ps[u], ld1((const T*)p.v + at[u] + d), a);
                acc[i] = a;
            }
        }
    }
    T* o = (T*)p.o + ((int64_t)n * p.Hq + h) * p.dh;
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (lane + 64 * i < p.dh) st1(o + lane + 64 * i, l == 0.f ? 0.f : acc[i] * inv);
}

extern "C" size_t vm_paged_attention_ws(int N, int Hq, int Hkv, int dh, int M, int page_size, int dtype) { return 0; }

extern "C" int vm_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k_pages, const void* v_pages,
                                  const int32_t* block_table, int64_t ld_table, const int32_t* lengths, void* o, int N, int Hq, int Hkv, int dh, int P,
                                  int page_size, int M, float scale, int dtype, void* ws, size_t ws_bytes, void* stream) {
    VM_REQUIRE(q && k_pages && v_pages && block_table && lengths && o, "vm_paged_attention: null pointer");
    VM_REQUIRE(N > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && P > 0 && M > 0 && ld_table >= M, "vm_paged_attention: bad shape");
    VM_REQUIRE(dh >= 8 && dh <= 256 && dh % 8 == 0, "vm_paged_attention: dh = %d: a multiple of 8 up to 256 is required", dh);
    VM_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0 && (int64_t)M * page_size < (1ll << 31),
               "vm_paged_attention: page_size must be a power of two from 16 on, M * page_size below 2^31");
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "vm_paged_attention: dtype must be VM_F32 or VM_BF16");
    VM_REQUIRE(((uintptr_t)k_pages % 16) == 0 && ((uintptr_t)v_pages % 16) == 0, "vm_paged_attention: pages must be 16-byte aligned");
    VM_REQUIRE((int64_t)N * Hq < (1ll << 31), "vm_paged_attention: N * Hq must stay below 2^31");
    PagedAttnArgs a = {q, q_row_stride, q_head_stride, k_pages, v_pages, block_table, ld_table, lengths, o, N, Hq, Hkv, Hq / Hkv, dh, P, page_size, M,
                       scale * 1.4426950408889634f};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_ATTN, 0.0, s, "paged_attn_n%d_h%d_k%d_d%d", N, Hq, Hkv, dh);
    if (dtype == VM_F32) hipLaunchKernelGGL(paged_attention_kernel<float>, dim3(N * Hq), dim3(64), 0, s, a);
    else hipLaunchKernelGGL(paged_attention_kernel<bf16_t>, dim3(N * Hq), dim3(64), 0, s, a);
    return vm_check_launch("vm_paged_attention");
}
