// Log probabilities of given tokens, the entropy of their distributions and the most likely alternatives, from logits;
// and the gradient of the logits.  With M a row's largest logit and d = (logit - M) / temperature:
//   S = sum exp d      log p = d - log S      logprob = log p[target]      entropy = log S - sum exp(d) d / S
//   d_logits[v] = (g (1[v = target] - p_v) - g_H p_v (log p_v + entropy)) / temperature
// A logit of minus infinity is a token that is ruled out: p 0, no part in the entropy, gradient 0.  M and log S stay apart
// for the backward: where M is large (a row of the type's lowest value, say) their sum would round log S away, and M / temperature
// rounded once would be off by more than the differences that count.
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxTop = 32, kGroups = 128, kRoom = 1024, kUnroll = 4;
constexpr float kNothing = -256.0f;  // 2^-256 is 0 in f32

// max that a NaN passes through.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A 16-byte piece of a row.
template <typename T>
struct Piece {
    static constexpr int W = 16 / sizeof(T);
    uint4 q;
    __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void fill(uint32_t w) { q = make_uint4(w, w, w, w); }
    __device__ __forceinline__ float2 pair(int j) const {
        if constexpr (sizeof(T) == 2) {
            return unpack2<T>(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w);
        } else {
            return j == 0 ? make_float2(__uint_as_float(q.x), __uint_as_float(q.y)) : make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
        }
    }
    // The largest (NaN aside).
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 *h = reinterpret_cast<const __half2*>(&q), m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(__low2float(m), __high2float(m));
        } else {
            const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162*>(&q), m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(__low2float(m), __high2float(m));
        }
    }
};
template <typename T> __device__ __forceinline__ uint32_t minus_inf();
template <> __device__ __forceinline__ uint32_t minus_inf<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t minus_inf<__half>() { return 0xfc00fc00u; }
template <> __device__ __forceinline__ uint32_t minus_inf<__nv_bfloat16>() { return 0xff80ff80u; }

// A row in 16-byte pieces: `head` elements before the first aligned one, `pieces`, and a tail of less than one.
template <typename T>
struct Row {
    const T* p;
    int head, pieces, V;
    __device__ __forceinline__ Row(const T* row, int n) : p(row), V(n) {
        head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
        head = min(head, n);
        pieces = (n - head) / Piece<T>::W;
    }
    __device__ __forceinline__ int tail() const { return head + pieces * Piece<T>::W; }
};

struct FwdParams {
    const void* logits;
    const int* targets;
    float *lse, *entropy, *logprob;
    int* top_ids;
    float* top_logprobs;
    long long ld, rows;
    int V, top, split;
    float inv_temp;
};

// m: largest logit; s = sum of 2^d, s1 = sum of 2^d d with d = (logit - m) c.  Nothing yet: m is the lowest finite value, s 0
// (so a row has something left if and only if its s is not 0).
struct Sums {
    float m, s, s1;
    __device__ __forceinline__ void raise(float to, float c) {
        const float d = max_nan((m - to) * c, kNothing), e = ex2(d);
        s1 = e * fmaf(s, d, s1);
        s *= e;
        m = to;
    }
    __device__ __forceinline__ void add(float v, float c) {
        const float d = max_nan((v - m) * c, kNothing), e = ex2(d);
        s += e;
        s1 = fmaf(e, d, s1);
    }
};
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ bool before(float v, int i, float v2, int i2) { return v > v2 || (v == v2 && i < i2); }
__device__ __forceinline__ float ranked(float v) { return v == v ? v : -INFINITY; }

// The alternatives of [lo, hi) pieces (and the ends) of a row, in order, in sel_v / sel_i[0 .. top); beyond what is there, index
// 0x7fffffff.  Two threads' elements form a group.  tau, the top-th largest of the groups' maxima, is a lower bound of the
// top-th largest element, so only groups that reach it are read again (from L2); what reaches it in them is ranked by counting.
struct TopRoom {
    float group[kGroups], v[kRoom], sel_v[kMaxTop];
    int i[kRoom], sel_i[kMaxTop], n, best_i[kWarps];
    float tau, best_v[kWarps];
};

template <typename T>
__device__ __noinline__ void pick_top(TopRoom& t, const Row<T>& row, int lo, int hi, bool first, bool last, int top) {
    constexpr int W = Piece<T>::W;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // (the groups' maxima are there; a barrier lies behind them)
    if (tid < kGroups) {
        const float mine = t.group[tid];
        int rank = 0;
        for (int j = 0; j < kGroups; ++j) rank += before(t.group[j], j, mine, tid);
        if (rank == top - 1) t.tau = mine;
    }
    if (tid == 0) t.n = 0;
    if (tid < kMaxTop) t.sel_v[tid] = -INFINITY, t.sel_i[tid] = 0x7fffffff;
    __syncthreads();
    const float tau = t.tau;
    auto offer = [&](float v, int i) {
        v = ranked(v);
        if (v > -INFINITY && v >= tau) {
            const int at = atomicAdd(&t.n, 1);
            if (at < kRoom) t.v[at] = v, t.i[at] = i;
        }
    };
    for (int g = warp; g < kGroups; g += kWarps) {
        if (!(t.group[g] >= tau) || t.group[g] == -INFINITY) continue;
        // the pieces of threads 2 g and 2 g + 1: lane l has every 16th of one of them
        for (int j = lo + 2 * g + (lane & 1) + (lane >> 1) * kThreads; j < hi; j += 16 * kThreads) {
            Piece<T> q;
            q.load(row.p + row.head + j * W);
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const float2 v = q.pair(e / 2);
                offer(v.x, row.head + j * W + e);
                offer(v.y, row.head + j * W + e + 1);
            }
        }
        if (lane < 2) {
            const int i = 2 * g + lane;
            if (first && i < row.head) offer(to_f(row.p[i]), i);
            if (last && row.tail() + i < row.V) offer(to_f(row.p[row.tail() + i]), row.tail() + i);
        }
    }
    __syncthreads();
    int n = t.n;
    const int begin = first ? 0 : row.head + lo * W, end = last ? row.V : row.head + hi * W;
    if (n > kRoom) {
        // More reach tau than there is room for: those above it one after the other, until tau itself is met.
        __syncthreads();
        float last_v = INFINITY;
        int last_i = -1, k = 0;
        for (; k < top; ++k) {
            float v = -INFINITY;
            int at = 0x7fffffff;
            for (int i = begin + tid; i < end; i += kThreads) {
                const float l = ranked(to_f(row.p[i]));
                if (before(last_v, last_i, l, i) && before(l, i, v, at)) v = l, at = i;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float v2 = __shfl_xor_sync(0xffffffffu, v, o);
                const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
                if (before(v2, at2, v, at)) v = v2, at = at2;
            }
            if (lane == 0) t.best_v[warp] = v, t.best_i[warp] = at;
            __syncthreads();
            v = t.best_v[0], at = t.best_i[0];
            for (int w = 1; w < kWarps; ++w)
                if (before(t.best_v[w], t.best_i[w], v, at)) v = t.best_v[w], at = t.best_i[w];
            __syncthreads();
            if (v <= tau) break;
            last_v = v, last_i = at;
            if (tid == 0) t.v[k] = v, t.i[k] = at;
        }
        n = k;
        __syncthreads();
    }
    // in order by counting who comes before; each warp's lanes share a candidate's count
    const int kept = n < top ? n : top;
    for (int a = warp; a < n; a += kWarps) {
        int rank = 0;
        for (int b = lane; b < n; b += 32) rank += before(t.v[b], t.i[b], t.v[a], t.i[a]);
        rank = __reduce_add_sync(0xffffffffu, rank);
        if (lane == 0 && rank < top) t.sel_v[rank] = t.v[a], t.sel_i[rank] = t.i[a];
    }
    if (kept < top) {
        // what is left are equals: tau where there was no room, else tokens that are ruled out.  The lowest indices.
        const float equal = t.n > kRoom ? tau : -INFINITY;
        if (warp == 0) {
            int found = kept;
            for (int i0 = begin; i0 < end && found < top; i0 += 8 * 32) {
                bool hit[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int i = i0 + 32 * u + lane;
                    hit[u] = i < end && ranked(to_f(row.p[i])) == equal;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const unsigned hits = __ballot_sync(0xffffffffu, hit[u]);
                    const int at = found + __popc(hits & ((1u << lane) - 1));
                    if (hit[u] && at < top) t.sel_v[at] = equal, t.sel_i[at] = i0 + 32 * u + lane;
                    found += __popc(hits);
                }
            }
        }
    }
    __syncthreads();
}

// A CTA has a row, or with SPLIT the CTAs of a cluster have a piece of one each and the first joins what they found.
template <typename T, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const FwdParams p) {
    constexpr int W = Piece<T>::W;
    __shared__ Sums part[kWarps], mine;
    __shared__ TopRoom room;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = p.inv_temp * kLog2e;
    const int R = SPLIT ? p.split : 1, rank = SPLIT ? static_cast<int>(blockIdx.x) % R : 0;
    const long long r = SPLIT ? blockIdx.x / R : blockIdx.x;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    const int lo = static_cast<int>(static_cast<long long>(row.pieces) * rank / R), hi = static_cast<int>(static_cast<long long>(row.pieces) * (rank + 1) / R);
    const bool first = rank == 0, last = rank == R - 1;
    Sums a{kLowest, 0.0f, 0.0f};
    float top_v = -INFINITY;
    float2 s2 = splat2(0.0f), s12 = splat2(0.0f);
    const float2 cc = splat2(c);
    for (int j0 = lo + tid; j0 < hi; j0 += kThreads * kUnroll) {
        Piece<T> q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int j = j0 + u * kThreads;
            if (j < hi) q[u].load(row.p + row.head + j * W);
            else q[u].fill(minus_inf<T>());
        }
        float m = q[0].top();
#pragma unroll
        for (int u = 1; u < kUnroll; ++u) m = fmaxf(m, q[u].top());
        top_v = fmaxf(top_v, m);
        const float to = fmaxf(a.m, m), d = fmaxf((a.m - to) * c, kNothing), e = ex2(d);
        a.m = to;
        s12 = mul2(splat2(e), fma2(s2, splat2(d), s12));
        s2 = mul2(s2, splat2(e));
        const float2 neg = splat2(-to);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int k = 0; k < W / 2; ++k) {
                float2 t = mul2(add2(q[u].pair(k), neg), cc);
                t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
                const float2 x = make_float2(ex2(t.x), ex2(t.y));
                s2 = add2(s2, x);
                s12 = fma2(x, t, s12);
            }
    }
    a.s = s2.x + s2.y, a.s1 = s12.x + s12.y;
    // the ends
    auto end = [&](int i) {
        const float v = to_f(row.p[i]);
        top_v = fmaxf(top_v, v);
        a.raise(fmaxf(a.m, v), c);
        a.add(v, c);
    };
    if (first && tid < row.head) end(tid);
    if (last && row.tail() + tid < p.V) end(row.tail() + tid);
    if (TOP) {
        const float other = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, 1));
        if ((lane & 1) == 0) room.group[tid >> 1] = other;
    }
    auto join_lanes = [&](int from) {
        float m = a.m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o <= from) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        a.raise(m, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o <= from) {
                a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
                a.s1 += __shfl_xor_sync(0xffffffffu, a.s1, o);
            }
    };
    join_lanes(16);
    if (lane == 0) part[warp] = a;
    __syncthreads();
    a = part[lane % kWarps];
    join_lanes(kWarps / 2);
    if (TOP) pick_top<T>(room, row, lo, hi, first, last, p.top);
    if (SPLIT) {
        if (tid == 0) mine = a;
        cluster_sync();
        if (rank == 0) {
            const uint32_t at = smem_u32(&mine);
            a = Sums{kLowest, 0.0f, 0.0f};
            if (lane < R) {
                const uint32_t far = cluster_addr(at, lane);
                a = Sums{ld_cluster1(far), ld_cluster1(far + 4), ld_cluster1(far + 8)};
            }
            join_lanes(16);
            if (TOP) {  // every piece's alternatives, in order by counting
                const int n = R * p.top;
                for (int i = tid; i < n; i += kThreads) {
                    const int from = i / p.top, k = i - from * p.top;
                    room.v[i] = ld_cluster1(cluster_addr(smem_u32(room.sel_v + k), from));
                    room.i[i] = __float_as_int(ld_cluster1(cluster_addr(smem_u32(room.sel_i + k), from)));
                }
                __syncthreads();
            }
        }
        cluster_sync();
        if (rank != 0) return;
        if (TOP) {
            const int n = R * p.top;
            for (int i = warp; i < n; i += kWarps) {
                int k = 0;
                for (int b = lane; b < n; b += 32) k += before(room.v[b], room.i[b], room.v[i], room.i[i]);
                k = __reduce_add_sync(0xffffffffu, k);
                if (lane == 0 && k < p.top && room.i[i] != 0x7fffffff) room.sel_v[k] = room.v[i], room.sel_i[k] = room.i[i];
            }
            __syncthreads();
        }
    }
    const float log_s = lg2(a.s) * kLn2;
    const bool none = a.s == 0.0f;
    if (tid == 0) {
        if (p.lse) {
            p.lse[r] = none ? -INFINITY : a.s == a.s ? a.m : a.s;
            p.lse[p.rows + r] = none ? 0.0f : log_s;
        }
        if (p.entropy) p.entropy[r] = none ? 0.0f : log_s - a.s1 / a.s * kLn2;
    }
    if (tid == 32 && p.targets && p.logprob) {
        const int t = p.targets[r];
        const bool ok = t >= 0 && t < p.V;
        p.logprob[r] = !ok ? 0.0f : none ? -INFINITY : (to_f(row.p[t]) - a.m) * p.inv_temp - log_s;
    }
    if (TOP && tid < p.top) {
        p.top_ids[r * p.top + tid] = room.sel_i[tid];
        p.top_logprobs[r * p.top + tid] = none ? -INFINITY : (room.sel_v[tid] - a.m) * p.inv_temp - log_s;
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

// With t = log2 p: d_logits = -p (k0 + k1 t), plus the target's share.  One read and one write; ALIGNED: rows of both tensors
// start at the same place of 16 bytes.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_bwd_kernel(const BwdParams p) {
    constexpr int W = Piece<T>::W;
    const int tid = threadIdx.x;
    const long long r = blockIdx.x;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    T* out = static_cast<T*>(p.dlogits) + r * p.ld_d;
    const float m = p.lse[r], log2_s = p.lse[p.rows + r] * kLog2e;
    const int tgt = p.targets ? p.targets[r] : -1;
    const bool none = m == -INFINITY;
    const float g = tgt >= 0 && tgt < p.V && p.d_logprob && !none ? p.d_logprob[r] * p.inv_temp : 0.0f;
    const float gh = p.d_entropy && !none ? p.d_entropy[r] * p.inv_temp : 0.0f;
    const float k0 = -fmaf(gh, p.d_entropy ? p.entropy[r] : 0.0f, g), k1 = -gh * kLn2, c = p.inv_temp * kLog2e;
    auto one = [&](float v, int i) {
        const float t = none ? kNothing : max_nan(fmaf(v - m, c, -log2_s), kNothing);
        const float d = ex2(t) * fmaf(k1, t, k0);
        return i == tgt ? d + g : d;
    };
    if (!ALIGNED) {
        for (int i = tid; i < p.V; i += kThreads) out[i] = from_f<T>(one(to_f(row.p[i]), i));
        return;
    }
    const float2 neg = splat2(none ? 0.0f : -m), cc = splat2(c), ls = splat2(-log2_s), kk0 = splat2(k0), kk1 = splat2(k1);
    for (int j0 = tid; j0 < row.pieces; j0 += kThreads * kUnroll) {
        Piece<T> q[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (j0 + u * kThreads < row.pieces) q[u].load(row.p + row.head + (j0 + u * kThreads) * W);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = row.head + (j0 + u * kThreads) * W;
            if (j0 + u * kThreads >= row.pieces) break;
            float2 d[W / 2];
#pragma unroll
            for (int k = 0; k < W / 2; ++k) {
                float2 t = fma2(add2(q[u].pair(k), neg), cc, ls);
                t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
                d[k] = mul2(make_float2(ex2(t.x), ex2(t.y)), fma2(kk1, t, kk0));
                if (none) d[k] = splat2(0.0f);
            }
            const int at = tgt - i;
            if (static_cast<unsigned>(at) < W) {
#pragma unroll
                for (int k = 0; k < W / 2; ++k) {
                    if (at == 2 * k) d[k].x += g;
                    if (at == 2 * k + 1) d[k].y += g;
                }
            }
            uint4 o;
            if constexpr (sizeof(T) == 2)
                o = make_uint4(pack2<T>(d[0].x, d[0].y), pack2<T>(d[1].x, d[1].y), pack2<T>(d[2].x, d[2].y), pack2<T>(d[3].x, d[3].y));
            else
                o = make_uint4(__float_as_uint(d[0].x), __float_as_uint(d[0].y), __float_as_uint(d[1].x), __float_as_uint(d[1].y));
            *reinterpret_cast<uint4*>(out + i) = o;
        }
    }
    if (tid < row.head) out[tid] = from_f<T>(one(to_f(row.p[tid]), tid));
    const int i = row.tail() + tid;
    if (i < p.V) out[i] = from_f<T>(one(to_f(row.p[i]), i));
}

// How many CTAs share a row: as many as find room beside one another (four on an SM), each with 2048 logits or more.
static int pick_split(int sms, long long rows, int V) {
    int s = 1;
    while (s < 16 && rows * 2 * s <= 4ll * sms && V >= 2 * s * 2048) s *= 2;
    return s;
}

template <typename T, bool TOP>
static int launch_fwd(Ctx* c, FwdParams& p, cudaStream_t st) {
    p.split = pick_split(c->sm_count, p.rows, p.V);
    const dim3 grid(static_cast<unsigned>(p.rows * p.split));
    if (p.split == 1) {
        token_logprobs_kernel<T, TOP, false><<<grid, kThreads, 0, st>>>(p);
    } else {
        void* args[] = {&p};
        MB200_CUDA_CHECK(c, launch_cluster(reinterpret_cast<const void*>(token_logprobs_kernel<T, TOP, true>), grid, dim3(kThreads), 0, st, p.split, args));
    }
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}
template <typename T>
static int launch_fwd(Ctx* c, FwdParams& p, cudaStream_t st) {
    return p.top ? launch_fwd<T, true>(c, p, st) : launch_fwd<T, false>(c, p, st);
}

template <typename T>
static int launch_bwd(Ctx* c, const BwdParams& p, cudaStream_t st) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p.logits), y = reinterpret_cast<uintptr_t>(p.dlogits);
    const bool aligned = (x - y) % 16 == 0 && (p.rows == 1 || (p.ld - p.ld_d) * static_cast<long long>(sizeof(T)) % 16 == 0);
    const unsigned grid = static_cast<unsigned>(p.rows);
    if (aligned) token_logprobs_bwd_kernel<T, true><<<grid, kThreads, 0, st>>>(p);
    else token_logprobs_bwd_kernel<T, false><<<grid, kThreads, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

}  // namespace lp

int logprobs_configure(Ctx* c) {
    const void* fns[] = {reinterpret_cast<const void*>(lp::token_logprobs_kernel<float, true, true>),
                         reinterpret_cast<const void*>(lp::token_logprobs_kernel<float, false, true>),
                         reinterpret_cast<const void*>(lp::token_logprobs_kernel<__half, true, true>),
                         reinterpret_cast<const void*>(lp::token_logprobs_kernel<__half, false, true>),
                         reinterpret_cast<const void*>(lp::token_logprobs_kernel<__nv_bfloat16, true, true>),
                         reinterpret_cast<const void*>(lp::token_logprobs_kernel<__nv_bfloat16, false, true>)};
    for (const void* fn : fns) MB200_CUDA_CHECK(c, cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return MAMBA_B200_OK;
}

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
    if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: misaligned logits");
    lp::FwdParams p{logits, targets, lse, entropy, logprob, top_ids, top_logprobs, ld, rows, V, top, 1, 1.0f / temperature};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) return lp::launch_fwd<float>(c, p, st);
    if (dtype == MAMBA_B200_F16) return lp::launch_fwd<__half>(c, p, st);
    return lp::launch_fwd<__nv_bfloat16>(c, p, st);
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
    if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dlogits)) % dtype_size(dtype))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: misaligned logits");
    const lp::BwdParams p{logits, targets, lse, entropy, d_logprob, d_entropy, dlogits, ld, ld_d, rows, V, 1.0f / temperature};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) return lp::launch_bwd<float>(c, p, st);
    if (dtype == MAMBA_B200_F16) return lp::launch_bwd<__half>(c, p, st);
    return lp::launch_bwd<__nv_bfloat16>(c, p, st);
}
