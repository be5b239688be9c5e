// Log probabilities of given tokens, the entropy of their distributions and the most likely alternatives, from logits;
// and the gradient of the logits.  With M a row's largest logit and d = (logit - M) / temperature:
//   S = sum exp d      log p = d - log S      logprob = log p[target]      entropy = log S - sum exp(d) d / S
//   d_logits[v] = (g (1[v = target] - p_v) - g_H p_v (log p_v + entropy)) / temperature
// A logit of minus infinity is a token that is ruled out: p 0, no part in the entropy, gradient 0.  M and log S stay apart
// for the backward: where M is large (a row of the type's lowest value, say) their sum would round log S away, and M / temperature
// rounded once would be off by more than the differences that count.
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxTop = 32;

struct FwdParams {
    const void* logits;
    const int* targets;
    float *lse, *entropy, *logprob;
    int* top_ids;
    float* top_logprobs;
    long long ld, rows;
    int V, top;
    float inv_temp;
};

// m: largest logit; s = sum of 2^d, s1 = sum of 2^d d with d = (logit - m) c.
struct Sums {
    float m, s, s1;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s, a.s1 + b.s1};  // (nothing yet, or NaN)
    // (below 2^-256 there is nothing left: a term of 0 times minus infinity would be NaN)
    const float da = fmaxf((a.m - m) * c, -256.0f), db = fmaxf((b.m - m) * c, -256.0f);
    const float ea = ex2(da), eb = ex2(db);
    Sums r;
    r.m = m;
    r.s = a.s * ea + b.s * eb;
    r.s1 = (a.m == -INFINITY ? a.s1 : ea * fmaf(a.s, da, a.s1)) + (b.m == -INFINITY ? b.s1 : eb * fmaf(b.s, db, b.s1));
    return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const FwdParams p) {
    __shared__ Sums part[kWarps];
    __shared__ float best_v[kWarps];
    __shared__ int best_i[kWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = p.inv_temp * kLog2e;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* row = static_cast<const T*>(p.logits) + r * p.ld;
        Sums a{-INFINITY, 0.0f, 0.0f};
        for (int i = tid; i < p.V; i += kThreads) {
            const float l = to_f(row[i]);
            if (l == -INFINITY) continue;
            a = join(a, {l, 1.0f, 0.0f}, c);
            if (l != l || l == INFINITY) a.s = NAN;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.s1, o)};
            a = join(a, b, c);
        }
        __syncthreads();
        if (lane == 0) part[warp] = a;
        __syncthreads();
        a = part[0];
        for (int w = 1; w < kWarps; ++w) a = join(a, part[w], c);
        // (an infinite logit leaves no distribution: everything of the row is NaN)
        const float log_s = lg2(a.s) * kLn2;
        const bool none = a.m == -INFINITY && a.s == a.s;
        if (tid == 0) {
            if (p.lse) {
                p.lse[r] = a.s == a.s ? a.m : a.s;
                p.lse[p.rows + r] = none ? 0.0f : log_s;
            }
            if (p.entropy) p.entropy[r] = none ? 0.0f : log_s - a.s1 / a.s * kLn2;
            if (p.targets && p.logprob) {
                const int t = p.targets[r];
                const bool ok = t >= 0 && t < p.V;
                p.logprob[r] = !ok ? 0.0f : none ? -INFINITY : (to_f(row[t]) - a.m) * p.inv_temp - log_s;
            }
        }
        // the most likely tokens, one after the other: the largest below the last one's (value, index)
        float last_v = INFINITY;
        int last_i = -1;
        for (int k = 0; k < p.top; ++k) {
            float v = -INFINITY;
            int at = 0x7fffffff;
            for (int i = tid; i < p.V; i += kThreads) {
                float l = to_f(row[i]);
                if (l != l) l = -INFINITY;
                const bool after = l < last_v || (l == last_v && i > last_i);
                if (after && (at == 0x7fffffff || l > v)) {
                    v = l;
                    at = i;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float v2 = __shfl_xor_sync(0xffffffffu, v, o);
                const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
                if (at2 != 0x7fffffff && (at == 0x7fffffff || v2 > v || (v2 == v && at2 < at))) {
                    v = v2;
                    at = at2;
                }
            }
            __syncthreads();
            if (lane == 0) {
                best_v[warp] = v;
                best_i[warp] = at;
            }
            __syncthreads();
            v = best_v[0];
            at = best_i[0];
            for (int w = 1; w < kWarps; ++w)
                if (best_i[w] != 0x7fffffff && (at == 0x7fffffff || best_v[w] > v || (best_v[w] == v && best_i[w] < at))) {
                    v = best_v[w];
                    at = best_i[w];
                }
            last_v = v;
            last_i = at;
            if (tid == 0) {
                p.top_ids[r * p.top + k] = at;
                p.top_logprobs[r * p.top + k] = none ? -INFINITY : (v - a.m) * p.inv_temp - log_s;
            }
        }
    }
}

struct BwdParams {
    const void* logits;
    const int* targets;
    const float *lse, *entropy, *d_logprob, *d_entropy;
    void* dlogits;
    long long ld, ld_d, rows;
    int V;
    float inv_temp;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const BwdParams p) {
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* row = static_cast<const T*>(p.logits) + r * p.ld;
        T* out = static_cast<T*>(p.dlogits) + r * p.ld_d;
        const float m = p.lse[r], log_s = p.lse[p.rows + r];
        const int t = p.targets ? p.targets[r] : -1;
        const bool none = m == -INFINITY;
        const float g = t >= 0 && t < p.V && p.d_logprob && !none ? p.d_logprob[r] : 0.0f;
        const float gh = p.d_entropy && !none ? p.d_entropy[r] : 0.0f;
        const float k0 = (g + gh * (p.d_entropy ? p.entropy[r] : 0.0f)) * p.inv_temp, k1 = gh * p.inv_temp;
        for (int i = threadIdx.x; i < p.V; i += kThreads) {
            const float lq = fmaf(to_f(row[i]) - m, p.inv_temp, -log_s);  // log p
            const float q = ex2(lq * kLog2e);
            float d = none || q == 0.0f ? 0.0f : -q * fmaf(k1, lq, k0);
            if (i == t) d += g * p.inv_temp;
            out[i] = from_f<T>(d);
        }
    }
}

}  // namespace lp
}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API int mamba_b200_token_logprobs(void* handle, void* stream, int dtype, const void* logits, long long ld,
                                                        const int* targets, float temperature, float* lse, float* entropy,
                                                        float* logprob, int top, int* top_ids, float* top_logprobs, long long rows,
                                                        int V) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: bad dtype %d", dtype);
    if (rows < 0 || V <= 0 || ld < V) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: bad dims");
    if (!(temperature > 0.0f) || temperature > 3e38f || 1.0f / temperature > 3e38f) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: temperature %g", temperature);
    if (top < 0 || top > lp::kMaxTop || top > V)
        return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs: %d alternatives of %d tokens (at most %d)", top, V, lp::kMaxTop);
    if (rows == 0) return MAMBA_B200_OK;
    if (rows > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs: too many rows");
    if (!logits || (logprob && !targets) || (top && (!top_ids || !top_logprobs)))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: null pointer");
    const lp::FwdParams p{logits, targets, lse, entropy, logprob, top_ids, top_logprobs, ld, rows, V, top, 1.0f / temperature};
    const int grid = static_cast<int>(rows < 65536 ? rows : 65536);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) lp::token_logprobs_kernel<float><<<grid, lp::kThreads, 0, st>>>(p);
    else if (dtype == MAMBA_B200_F16) lp::token_logprobs_kernel<__half><<<grid, lp::kThreads, 0, st>>>(p);
    else lp::token_logprobs_kernel<__nv_bfloat16><<<grid, lp::kThreads, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

extern "C" MAMBA_B200_API int mamba_b200_token_logprobs_bwd(void* handle, void* stream, int dtype, const void* logits, long long ld,
                                                            const int* targets, float temperature, const float* lse,
                                                            const float* entropy, const float* d_logprob, const float* d_entropy,
                                                            void* dlogits, long long ld_d, long long rows, int V) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: bad dtype %d", dtype);
    if (rows < 0 || V <= 0 || ld < V || ld_d < V) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: bad dims");
    if (!(temperature > 0.0f) || temperature > 3e38f || 1.0f / temperature > 3e38f) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: temperature %g", temperature);
    if (rows == 0) return MAMBA_B200_OK;
    if (rows > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs_bwd: too many rows");
    if (!logits || !lse || !dlogits || (d_logprob && !targets) || (d_entropy && !entropy))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: null pointer");
    const lp::BwdParams p{logits, targets, lse, entropy, d_logprob, d_entropy, dlogits, ld, ld_d, rows, V, 1.0f / temperature};
    const int grid = static_cast<int>(rows < 65536 ? rows : 65536);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) lp::token_logprobs_bwd_kernel<float><<<grid, lp::kThreads, 0, st>>>(p);
    else if (dtype == MAMBA_B200_F16) lp::token_logprobs_bwd_kernel<__half><<<grid, lp::kThreads, 0, st>>>(p);
    else lp::token_logprobs_bwd_kernel<__nv_bfloat16><<<grid, lp::kThreads, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}
