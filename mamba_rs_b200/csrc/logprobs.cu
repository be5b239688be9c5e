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

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxTop = 32, kRoom = 1024, kUnroll = 4;
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
    __device__ __forceinline__ void put(int i, T v) {  // (i known to the compiler)
        if constexpr (sizeof(T) == 4) {
            (i == 0 ? q.x : q.y) = *reinterpret_cast<uint32_t*>(&v);
        } else {
            const uint32_t w = *reinterpret_cast<unsigned short*>(&v);
            q.x = i == 0 ? (q.x & 0xffff0000u) | w : (q.x & 0xffffu) | (w << 16);
        }
    }
    // The largest of kUnroll pieces (NaN aside).
    __device__ __forceinline__ static float top(const Piece* q) {
        if constexpr (sizeof(T) == 4) {
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 v = q[u].pair(k);
                    m = fmaxf(m, fmaxf(v.x, v.y));
                }
            return m;
        } else {
            using H2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            H2 m = *reinterpret_cast<const H2*>(&q[0].q.x);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const H2* h = reinterpret_cast<const H2*>(&q[u].q);
#pragma unroll
                for (int k = 0; k < 4; ++k) m = __hmax2(m, h[k]);
            }
            return fmaxf(__low2float(m), __high2float(m));
        }
    }
    // No value below `lowest` (NaN stays).
    __device__ __forceinline__ static void floor(Piece* q, float lowest) {
        using H2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const uint32_t w = pack2<T>(lowest, lowest);
        const H2 lo = *reinterpret_cast<const H2*>(&w);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            H2* h = reinterpret_cast<H2*>(&q[u].q);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = __hmax2_nan(h[k], lo);
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

// top: largest logit.  With rho a reference near top c (c = log2 e / temperature; the product is rounded, but the same rho meets
// every term): s = sum of 2^t, s1 = sum of 2^t t, t = logit c - rho in one rounding.  Then log2 S = log2 s - (top c - rho) and, in
// base 2, the entropy = log2 s - s1 / s whatever rho is.
struct Sums {
    float top, rho, s, s1;
    __device__ __forceinline__ void raise(float to) {
        const float d = max_nan(rho - to, kNothing), e = ex2(d);
        s1 = e * fmaf(s, d, s1);
        s *= e;
        rho = to;
    }
};
constexpr float kFarDown = -1e37f;  // below any reference
__device__ __forceinline__ Sums no_sums() { return {-INFINITY, kFarDown, 0.0f, 0.0f}; }
// Where rho cannot follow the largest logit (a row of the type's lowest value: the product with c overflows, or 16-bit logits of
// minus infinity cannot be told from it), the pass shows it by these and the row is summed again.
__device__ __forceinline__ bool in_doubt(const Sums& a) { return a.top > -INFINITY && (a.s == 0.0f || (a.s == a.s && a.s1 != a.s1)); }

// Sums over the lanes that differ in the bits below `lanes`, the same in each of them.
__device__ __forceinline__ void join_lanes(Sums& a, int lanes) {
    float rho = a.rho;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < lanes) {
            a.top = fmaxf(a.top, __shfl_xor_sync(0xffffffffu, a.top, o));
            rho = fmaxf(rho, __shfl_xor_sync(0xffffffffu, rho, o));
        }
    a.raise(rho);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < lanes) {
            a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
            a.s1 += __shfl_xor_sync(0xffffffffu, a.s1, o);
        }
}
__device__ __forceinline__ void join_block(Sums& a, Sums* part) {
    join_lanes(a, 32);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = a;
    __syncthreads();
    a = part[threadIdx.x % kWarps];
    join_lanes(a, kWarps);
}

// The sums of a whole row relative to its largest logit, term by term.
template <typename T>
__device__ __noinline__ Sums sum_again(const Row<T>& row, float top, float c, Sums* part) {
    Sums a{top, 0.0f, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < row.V; i += kThreads) {
        const float t = max_nan((to_f(row.p[i]) - top) * c, kNothing), e = ex2(t);
        a.s += e;
        a.s1 = fmaf(e, t, a.s1);
    }
    __syncthreads();
    join_block(a, part);
    return a;
}

// Order of the alternatives: by falling logit (NaN as minus infinity), equal ones by rising index, as one number; 0 is none.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    const uint32_t b = __float_as_uint((v == v ? v : -INFINITY) + 0.0f);  // (-0 is 0)
    return (static_cast<uint64_t>(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int key_index(uint64_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct TopRoom {
    float group[32];
    uint64_t key[kRoom], sel[kMaxTop], best[kWarps];
    int n;
};

// The alternatives of [lo, hi) pieces (and the ends) of a row, in order, in sel[0 .. top).  Eight threads' elements form a group.
// tau, the top-th largest of the 32 groups' maxima, is a lower bound of the top-th largest element: only what threads whose own
// maximum reaches it have seen is read again (from L2), and what reaches it there is ranked by counting.
template <typename T>
__device__ __noinline__ void pick_top(TopRoom& t, const Row<T>& row, int lo, int hi, bool first, bool last, int top, float own_top) {
    constexpr int W = Piece<T>::W;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // (the groups' maxima and n = 0 are there; a barrier lies behind them)
    float tau = t.group[lane];
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, tau, o);
            tau = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(tau, other) : fminf(tau, other);
        }
    tau = __shfl_sync(0xffffffffu, tau, top - 1);
    if (tid < kMaxTop) t.sel[tid] = 0;
    auto offer = [&](float v, int i) {
        if (v >= tau && v > -INFINITY) {
            const int at = atomicAdd(&t.n, 1);
            if (at < kRoom) t.key[at] = key_of(v, i);
        }
    };
    // half a warp for each such thread: a lane has every 16th of its pieces
    unsigned reach = __ballot_sync(0xffffffffu, own_top >= tau && own_top > -INFINITY);
    while (reach) {
        const int one = __ffs(reach) - 1;
        reach &= reach - 1;
        const int two = reach ? __ffs(reach) - 1 : -1;
        reach &= reach - 1;
        const int who = lane < 16 ? one : two;
        if (who < 0) continue;
        const int x = warp * 32 + who;
        for (int j = lo + x + (lane & 15) * kThreads; j < hi; j += 16 * kThreads) {
            Piece<T> q;
            q.load(row.p + row.head + j * W);
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const float2 v = q.pair(e / 2);
                offer(v.x, row.head + j * W + e);
                offer(v.y, row.head + j * W + e + 1);
            }
        }
        if ((lane & 15) == 0 && first && x < row.head) offer(to_f(row.p[x]), x);
        if ((lane & 15) == 1 && last && row.tail() + x < row.V) offer(to_f(row.p[row.tail() + x]), row.tail() + x);
    }
    __syncthreads();
    int n = t.n;
    const bool crowded = n > kRoom;
    const int begin = first ? 0 : row.head + lo * W, end = last ? row.V : row.head + hi * W;
    if (crowded) {
        // More reach tau than there is room for: those above it one after the other, until tau itself is met.
        __syncthreads();
        uint64_t below = ~0ull;
        for (n = 0; n < top; ++n) {
            uint64_t k = 0;
            for (int i = begin + tid; i < end; i += kThreads) {
                const uint64_t k2 = key_of(to_f(row.p[i]), i);
                if (k2 < below && k2 > k) k = k2;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const uint64_t k2 = __shfl_xor_sync(0xffffffffu, k, o);
                if (k2 > k) k = k2;
            }
            if (lane == 0) t.best[warp] = k;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w)
                if (t.best[w] > k) k = t.best[w];
            __syncthreads();
            if (key_value(k) <= tau) break;
            below = k;
            if (tid == 0) t.key[n] = k;
        }
        __syncthreads();
    }
    for (int a = tid; a < n; a += kThreads) {
        const uint64_t mine = t.key[a];
        int rank = 0;
        for (int b = 0; b < n; ++b) rank += t.key[b] > mine;
        if (rank < top) t.sel[rank] = mine;
    }
    if (n < top && warp == 0) {
        // what is left are equals: tau where there was no room, else tokens that are ruled out.  The lowest indices.
        const float equal = crowded ? tau : -INFINITY;
        int found = n;
        for (int i0 = begin; i0 < end && found < top; i0 += 8 * 32) {
            bool hit[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + 32 * u + lane;
                const float v = i < end ? to_f(row.p[i]) : 0.0f;
                hit[u] = i < end && (v == v ? v : -INFINITY) == equal;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const unsigned hits = __ballot_sync(0xffffffffu, hit[u]);
                const int at = found + __popc(hits & ((1u << lane) - 1));
                if (hit[u] && at < top) t.sel[at] = key_of(equal, i0 + 32 * u + lane);
                found += __popc(hits);
            }
        }
    }
    __syncthreads();
}

// A CTA has a row, or with SPLIT the CTAs of a cluster have a part of one each and the first joins what they found.
template <typename T, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const FwdParams p) {
    constexpr int W = Piece<T>::W;
    __shared__ Sums part[kWarps];
    __shared__ __align__(16) Sums mine;
    __shared__ TopRoom room;
    const int tid = threadIdx.x, lane = tid & 31;
    const float c = p.inv_temp * kLog2e;
    const int R = SPLIT ? p.split : 1, rank = SPLIT ? static_cast<int>(blockIdx.x) % R : 0;
    const long long r = SPLIT ? blockIdx.x / R : blockIdx.x;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    const int lo = static_cast<int>(static_cast<long long>(row.pieces) * rank / R), hi = static_cast<int>(static_cast<long long>(row.pieces) * (rank + 1) / R);
    const bool first = rank == 0, last = rank == R - 1;
    Sums a = no_sums();
    float2 s2 = splat2(0.0f), s12 = splat2(0.0f);
    const float2 cc = splat2(c);
    const float margin = 200.0f / c;
    auto take = [&](Piece<T>* q) {
        a.top = fmaxf(a.top, Piece<T>::top(q));
        if constexpr (sizeof(T) == 2) {
            if (a.top == -INFINITY) {  // nothing but ruled out tokens (or NaN) yet
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                    for (int k = 0; k < W / 2; ++k) {
                        const float2 v = q[u].pair(k);
                        if (v.x != v.x || v.y != v.y) s2.x = NAN;
                    }
                return;
            }
        }
        const float to = fmaxf(a.rho, a.top * c), d = fmaxf(a.rho - to, kNothing), e = ex2(d);
        a.rho = to;
        s12 = mul2(splat2(e), fma2(s2, splat2(d), s12));
        s2 = mul2(s2, splat2(e));
        const float2 neg = splat2(-to);
        // 16-bit logits far below are brought to a finite one whose exponential is still 0, two at a time; f32 ones after the product
        if constexpr (sizeof(T) == 2) Piece<T>::floor(q, a.top - margin - fabsf(a.top) * 0.015625f);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int k = 0; k < W / 2; ++k) {
                float2 t = fma2(q[u].pair(k), cc, neg);
                if constexpr (sizeof(T) == 4) t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
                const float2 x = make_float2(ex2(t.x), ex2(t.y));
                s2 = add2(s2, x);
                s12 = fma2(x, t, s12);
            }
    };
    const T* base = row.p + row.head;
    int j0 = lo + tid;
    Piece<T> q[kUnroll], next[kUnroll];
    const int whole = j0 < hi ? (hi - j0 + kThreads * kUnroll - 1 - (kUnroll - 1) * kThreads) / (kThreads * kUnroll) : 0;  // full rounds
    if (whole > 0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) next[u].load(base + static_cast<long long>(j0 + u * kThreads) * W);
    }
    for (int k = 0; k < whole; ++k) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = next[u];
        j0 += kThreads * kUnroll;
        if (k + 1 < whole) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) next[u].load(base + static_cast<long long>(j0 + u * kThreads) * W);
        }
        take(q);
    }
    // what is left of the thread's pieces, and the ends
    const bool head = first && tid < row.head, tail = last && row.tail() + tid < p.V;
    if (j0 < hi || head || tail) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            q[u].fill(minus_inf<T>());
            if (u < kUnroll - 1 && j0 + u * kThreads < hi) q[u].load(base + static_cast<long long>(j0 + u * kThreads) * W);
        }
        if (head) q[kUnroll - 1].put(0, row.p[tid]);
        if (tail) q[kUnroll - 1].put(1, row.p[row.tail() + tid]);
        take(q);
    }
    a.s = s2.x + s2.y, a.s1 = s12.x + s12.y;
    const float own_top = a.top;
    if (TOP) {
        float g = own_top;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (lane % 8 == 0) room.group[tid / 8] = g;
        if (tid == 0) room.n = 0;
    }
    join_block(a, part);
    if (TOP) pick_top<T>(room, row, lo, hi, first, last, p.top, own_top);
    if (SPLIT) {
        if (tid == 0) mine = a;
        cluster_sync();
        if (rank == 0) {
            const uint32_t at = smem_u32(&mine);
            a = no_sums();
            if (lane < R) {
                const float4 v = ld_cluster4(cluster_addr(at, lane));
                a = Sums{v.x, v.y, v.z, v.w};
            }
            join_lanes(a, 32);
            if (TOP) {
                for (int i = tid; i < R * p.top; i += kThreads) {
                    const int from = i / p.top, k = i - from * p.top;
                    uint64_t v;
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(smem_u32(room.sel + k), from)));
                    room.key[i] = v;
                }
                __syncthreads();
            }
        }
        cluster_sync();
        if (rank != 0) return;
        if (TOP) {
            // each part's alternatives are in order: a token's place is the sum of its places in the parts
            for (int i = tid; i < R * p.top; i += kThreads) {
                const uint64_t v = room.key[i];
                int place = 0;
                for (int f = 0; f < R; ++f) {
                    const uint64_t* list = room.key + f * p.top;
                    int at = 0;
#pragma unroll
                    for (int step = 32; step > 0; step >>= 1)
                        if (at + step <= p.top && list[at + step - 1] > v) at += step;
                    place += at;
                }
                if (v != 0 && place < p.top) room.sel[place] = v;
            }
            __syncthreads();
        }
    }
    if (in_doubt(a)) a = sum_again(row, a.top, c, part);  // (alike in all threads)
    else a.rho = fmaf(a.top, c, -a.rho);                  // top c - rho
    const float log_s = (lg2(a.s) - a.rho) * kLn2;
    const bool none = a.s == 0.0f;
    if (tid == 0) {
        if (p.lse) {
            p.lse[r] = a.s == a.s ? a.top : a.s;
            p.lse[p.rows + r] = none ? 0.0f : log_s;
        }
        if (p.entropy) p.entropy[r] = none ? 0.0f : (lg2(a.s) - a.s1 / a.s) * kLn2;
    }
    if (tid == 32 && p.targets && p.logprob) {
        const int t = p.targets[r];
        const bool ok = t >= 0 && t < p.V;
        p.logprob[r] = !ok ? 0.0f : none ? -INFINITY : (to_f(row.p[t]) - a.top) * p.inv_temp - log_s;
    }
    if (TOP && tid < p.top) {
        const uint64_t k = room.sel[tid];
        p.top_ids[r * p.top + tid] = key_index(k);
        p.top_logprobs[r * p.top + tid] = none ? -INFINITY : (key_value(k) - a.top) * p.inv_temp - log_s;
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
