// token_logprobs.hip -- log probabilities of given tokens with the entropy of their distribution and its best alternatives, and the gradient of all
// three with respect to the logits.  Per row x of V logits, target t:
//   z = log sum exp(x)      logp = x_t - z      H = z - sum_c p_c x_c  (p = exp(x - z); p_c = 0 adds nothing, also where x_c = -inf)
//   top: the n largest logits, largest first, equal ones by ascending column (a NaN counts as the largest, as torch.topk has it), as x_c - z
// A target < 0 is no token (logp 0, no gradient from it); a target >= V makes its logp NaN.  A row without a finite logit (all -inf) has
// z = -inf: logp -inf, entropy 0, alternatives -inf, gradient 0.
#include "common.h"

template <typename T> __device__ __forceinline__ float lp_ld(const T* p);
template <> __device__ __forceinline__ float lp_ld<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float lp_ld<bf16_t>(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void lp_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_st(bf16_t* p, float v) { *p = f32_to_bf16(v); }

// ascending unsigned order of the values; -0 and +0 are one value, every NaN the largest
__device__ __forceinline__ uint32_t lp_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct LogprobArgs {
    const void* x; int64_t ld_outer, ld_inner; int inner;      // row r starts at (r / inner) * ld_outer + (r % inner) * ld_inner
    const int64_t* target; int V, top; float* logp; float* ent; float* stats; float* top_logp; int64_t* top_ids;
};

#define LP_THREADS 256
__device__ __forceinline__ float lp_block(float v, float* sh, bool is_max) {
    v = is_max ? wave_max(v) : wave_sum(v);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (int i = 1; i < LP_THREADS / 64; ++i) r = is_max ? fmaxf(r, sh[i]) : r + sh[i];
    __syncthreads();
    return r;
}

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void token_logprobs_kernel(const LogprobArgs p) {
    __shared__ float sh[LP_THREADS / 64];
    __shared__ uint64_t best[LP_THREADS / 64];
    const int r = blockIdx.x, tid = threadIdx.x;
    const T* x = (const T*)p.x + (r / p.inner) * p.ld_outer + (r % p.inner) * p.ld_inner;
    float m = -INFINITY;
    for (int c = tid; c < p.V; c += LP_THREADS) m = fmaxf(m, lp_ld(x + c));
    m = lp_block(m, sh, true);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, w = 0.f;
    for (int c = tid; c < p.V; c += LP_THREADS) {
        const float d = lp_ld(x + c) - base, e = expf(d);
        s += e;
        if (e != 0.f) w = fmaf(e, d, w);
    }
    s = lp_block(s, sh, false);
    w = lp_block(w, sh, false);
    const float ls = logf(s);
    if (tid == 0) {
        const int64_t t = p.target[r];
        p.stats[2 * (int64_t)r] = base;                          // z in two parts: base + ls would round away log s where the logits are far from 0
        p.stats[2 * (int64_t)r + 1] = ls;
        p.ent[r] = s == 0.f ? 0.f : ls - w / s;
        p.logp[r] = t < 0 ? 0.f : (t >= p.V ? NAN : (s == 0.f ? -INFINITY : (lp_ld(x + t) - base) - ls));
    }
    uint64_t last = ~0ull;                                      // (value key, V - 1 - column): descending order of it is the wanted order
    for (int k = 0; k < p.top; ++k) {
        uint64_t b = 0;
        for (int c = tid; c < p.V; c += LP_THREADS) {
            const uint64_t key = ((uint64_t)lp_key(lp_ld(x + c)) << 32) | (uint32_t)(p.V - 1 - c);
            if (key < last && key > b) b = key;
        }
        for (int d = 32; d; d >>= 1) {
            const uint32_t lo = __shfl_xor((int)(uint32_t)b, d), hi = __shfl_xor((int)(b >> 32), d);
            const uint64_t o = ((uint64_t)hi << 32) | lo;
            b = o > b ? o : b;
        }
        if ((tid & 63) == 0) best[tid >> 6] = b;
        __syncthreads();
        for (int i = 0; i < LP_THREADS / 64; ++i) b = best[i] > b ? best[i] : b;
        __syncthreads();
        last = b;
        if (tid == 0) {
            const int c = p.V - 1 - (int)(uint32_t)b;
            p.top_ids[(int64_t)r * p.top + k] = c;
            p.top_logp[(int64_t)r * p.top + k] = s == 0.f ? -INFINITY : (lp_ld(x + c) - base) - ls;
        }
    }
}

// dx_c = -(g_l + sum_k g_k) p_c - g_h p_c (log p_c + H)  + g_l [c = t] + sum_k g_k [c = id_k]
struct LogprobGradArgs {
    const void* x; int64_t ld_outer, ld_inner; int inner; const int64_t* target; int V, top; const float* stats; const float* ent; const int64_t* top_ids;
    const float* g_logp; const float* g_ent; const float* g_top; void* dx; int64_t ld_dx;
};
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void token_logprobs_bwd_kernel(const LogprobGradArgs p) {
    const int r = blockIdx.x, tid = threadIdx.x;
    const T* x = (const T*)p.x + (r / p.inner) * p.ld_outer + (r % p.inner) * p.ld_inner;
    T* dx = (T*)p.dx + r * p.ld_dx;
    const int64_t t = p.target[r];
    const float base = p.stats[2 * (int64_t)r], ls = p.stats[2 * (int64_t)r + 1], H = p.ent[r];
    if (ls == -INFINITY) {                                       // nothing in the row: its outputs are constants
        for (int c = tid; c < p.V; c += LP_THREADS) lp_st(dx + c, 0.f);
        return;
    }
    const float gl = p.g_logp && t >= 0 ? (t < p.V ? p.g_logp[r] : NAN) : 0.f, gh = p.g_ent ? p.g_ent[r] : 0.f;
    float gt = gl;
    for (int k = 0; k < p.top; ++k) gt += p.g_top ? p.g_top[(int64_t)r * p.top + k] : 0.f;
    for (int c = tid; c < p.V; c += LP_THREADS) {
        const float lp = (lp_ld(x + c) - base) - ls, e = expf(lp);
        float d = e == 0.f ? 0.f : -e * (gt + gh * (lp + H));
        if (c == t) d += gl;
        if (p.g_top) for (int k = 0; k < p.top; ++k) if (p.top_ids[(int64_t)r * p.top + k] == c) d += p.g_top[(int64_t)r * p.top + k];
        lp_st(dx + c, d);
    }
}

static int logprob_check(const void* x, int R, int inner, int V, int top, int dtype, const char* what) {
    VM_REQUIRE(x && R > 0 && inner > 0 && V > 0, "%s: bad arguments", what);
    VM_REQUIRE(top >= 0 && top <= VM_MAX_TOP_LOGPROBS && top <= V, "%s: top = %d: at most %d and at most V alternatives", what, top, VM_MAX_TOP_LOGPROBS);
    VM_REQUIRE(dtype == VM_F32 || dtype == VM_BF16, "%s: dtype must be VM_F32 or VM_BF16", what);
    return VM_OK;
}
extern "C" int vm_token_logprobs_fwd(const void* logits, int64_t ld_outer, int64_t ld_inner, int inner, const int64_t* targets, int R, int V, int top,
                                     float* logp, float* entropy, float* stats, float* top_logp, int64_t* top_ids, int dtype, void* stream) {
    if (int rc = logprob_check(logits, R, inner, V, top, dtype, "vm_token_logprobs_fwd")) return rc;
    VM_REQUIRE(targets && logp && entropy && stats && (top == 0 || (top_logp && top_ids)), "vm_token_logprobs_fwd: null pointer");
    LogprobArgs a = {logits, ld_outer, ld_inner, inner, targets, V, top, logp, entropy, stats, top_logp, top_ids};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_LOSS, (dtype == VM_F32 ? 4.0 : 2.0) * R * (double)V, s, "token_logprobs_r%d_V%d_k%d", R, V, top);
    if (dtype == VM_F32) hipLaunchKernelGGL(token_logprobs_kernel<float>, dim3(R), dim3(LP_THREADS), 0, s, a);
    else hipLaunchKernelGGL(token_logprobs_kernel<bf16_t>, dim3(R), dim3(LP_THREADS), 0, s, a);
    return vm_check_launch("vm_token_logprobs_fwd");
}
extern "C" int vm_token_logprobs_bwd(const void* logits, int64_t ld_outer, int64_t ld_inner, int inner, const int64_t* targets, int R, int V, int top,
                                     const float* stats, const float* entropy, const int64_t* top_ids, const float* g_logp, const float* g_entropy,
                                     const float* g_top, void* dlogits, int64_t ld_dlogits, int dtype, void* stream) {
    if (int rc = logprob_check(logits, R, inner, V, top, dtype, "vm_token_logprobs_bwd")) return rc;
    VM_REQUIRE(targets && stats && entropy && dlogits && ld_dlogits >= V && (!g_top || top == 0 || top_ids), "vm_token_logprobs_bwd: bad arguments");
    LogprobGradArgs a = {logits, ld_outer, ld_inner, inner, targets, V, top, stats, entropy, top_ids, g_logp, g_entropy, top ? g_top : nullptr, dlogits, ld_dlogits};
    hipStream_t s = (hipStream_t)stream;
    VmProfScope prof(VM_FAM_LOSS, (dtype == VM_F32 ? 8.0 : 4.0) * R * (double)V, s, "token_logprobs_bwd_r%d_V%d_k%d", R, V, top);
    if (dtype == VM_F32) hipLaunchKernelGGL(token_logprobs_bwd_kernel<float>, dim3(R), dim3(LP_THREADS), 0, s, a);
    else hipLaunchKernelGGL(token_logprobs_bwd_kernel<bf16_t>, dim3(R), dim3(LP_THREADS), 0, s, a);
    return vm_check_launch("vm_token_logprobs_bwd");
}
