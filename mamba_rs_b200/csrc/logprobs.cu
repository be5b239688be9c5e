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
#include "m3_tc.cuh"

namespace mb200 {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxTop = 32, kRoom = 1024, kUnroll = 4, kCtas = 3;
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
    __device__ __forceinline__ void ruled_out() {
        const uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        q = make_uint4(w, w, w, w);
    }
    __device__ __forceinline__ float2 pair(int j) const {
        if constexpr (sizeof(T) == 2) {
            return unpack2<T>(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w);
        } else {
            return j == 0 ? make_float2(__uint_as_float(q.x), __uint_as_float(q.y)) : make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
        }
    }
    // The largest of N pieces' even elements and of their odd ones (NaN aside).
    template <int N> __device__ __forceinline__ static float2 tops(const Piece* q) {
        if constexpr (sizeof(T) == 4) {
            float2 m = make_float2(-INFINITY, -INFINITY);
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 v = q[u].pair(k);
                    m.x = fmaxf(m.x, v.x), m.y = fmaxf(m.y, v.y);
                }
            return m;
        } else {
            using H2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            H2 m = *reinterpret_cast<const H2*>(&q[0].q.x);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const H2* h = reinterpret_cast<const H2*>(&q[u].q);
#pragma unroll
                for (int k = 0; k < 4; ++k) m = __hmax2(m, h[k]);
            }
            return make_float2(__low2float(m), __high2float(m));
        }
    }
    template <int N> __device__ __forceinline__ static float top(const Piece* q) {
        const float2 m = tops<N>(q);
        return fmaxf(m.x, m.y);
    }
};
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

// top: largest logit.  With rho a reference near top c (c = log2 e / temperature; the product is rounded, and rho may lie up to
// kSlack below, but the same rho meets every term): s = sum of 2^t, s1 = sum of 2^t t, t = logit c - rho in one rounding.  With
// r = top c - rho the sums relative to the largest logit are S = s 2^-r and S1 = (s1 - r s) 2^-r, the entropy is, in base 2,
// log2 S - S1 / S.
struct Sums {
    float top, rho, s, s1;
    __device__ __forceinline__ void raise(float to) {
        const float d = rho == to ? 0.0f : max_nan(rho - to, kNothing), e = ex2(d);  // (both may be infinite)
        s1 = e * fmaf(s, d, s1);
        s *= e;
        rho = to;
    }
};
constexpr float kFarDown = -1e37f;  // below any reference
// A term may be 2^8.  The exponent of a token that is all but certain is rounded at that size (2^-21), and log S and the entropy, which
// are near 0 then, are off by as much: with 60 they were off by 2.6e-6 and 5.1e-6 and came out below 0.  A raise is one thread's, in
// rows with a logit that stands out; 4096 x 50280 takes no longer than with 60 (72.8 us without alternatives).
constexpr float kSlack = 8.0f;
// The reference of a largest logit.  The product is rounded up: a term's exponent, which is exact but for its own rounding, is then
// never far above kSlack, however large the product.  (To nearest, a thread that had met nothing but a mask's -1e10 had terms of
// 2^440, and made its row NaN.)
__device__ __forceinline__ float reference(float top, float c) { return __fmul_ru(top, c); }
__device__ __forceinline__ Sums no_sums() { return {-INFINITY, kFarDown, 0.0f, 0.0f}; }
// Where rho cannot follow the largest logit (products beyond 2^27 are 8 or more apart, or overflow to either side: a row of a mask's
// value, a logit of the type's largest, a tiny temperature; or 16-bit logits of minus infinity cannot be told from it), the row is
// summed again.  A logit of plus infinity is not in doubt: its own term is NaN.
constexpr float kFarProduct = 134217728.0f;
__device__ __forceinline__ bool in_doubt(const Sums& a, float c) {
    return a.top > -INFINITY && a.top < INFINITY && (fabsf(a.top * c) >= kFarProduct || a.s == 0.0f || (a.s == a.s && a.s1 != a.s1));
}

// A thread's running sums over pieces of a row, two chains.
template <typename T>
struct Running {
    float top, rho;
    float2 s, s1;
    bool masked;  // logits of minus infinity have been met
    __device__ __forceinline__ Running() : top(-INFINITY), rho(kFarDown), s(splat2(0.0f)), s1(splat2(0.0f)), masked(false) {}
    __device__ __forceinline__ Sums sums() const { return {top, rho, s.x + s.y, s1.x + s1.y}; }

    // N pieces, kThreads apart, from `at`.
    template <int N>
    __device__ __forceinline__ void take(const T* at, float c) {
        constexpr int W = Piece<T>::W;
        Piece<T> q[N];
#pragma unroll
        for (int u = 0; u < N; ++u) q[u].load(at + u * kThreads * W);
        top = fmaxf(top, Piece<T>::template top<N>(q));
        if (const float at_top = reference(top, c); at_top > rho + kSlack) raise(at_top);  // (the first time, and where a row rises steeply)
        const float2 cc = splat2(c), neg = splat2(-rho), was = s1;
        if (masked) {
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int k = 0; k < W / 2; ++k) {
                    float2 t = fma2(q[u].pair(k), cc, neg);
                    t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
                    const float2 x = make_float2(ex2(t.x), ex2(t.y));
                    s = add2(s, x);
                    s1 = fma2(x, t, s1);
                }
            return;
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int k = 0; k < W / 2; ++k) {
                const float2 t = fma2(q[u].pair(k), cc, neg), x = make_float2(ex2(t.x), ex2(t.y));
                s = add2(s, x);
                s1 = fma2(x, t, s1);
            }
        // A logit of minus infinity has made 0 times minus infinity of its term (unless the sum is NaN already, and stays so).
        if (!(s1.x + s1.y == s1.x + s1.y)) {
            s1 = again<N>(at, c, was);
            masked = true;
        }
    }
    template <int N>
    __device__ __noinline__ float2 again(const T* at, float c, float2 sum) const {
#pragma unroll 1
        for (int u = 0; u < N; ++u) {
            Piece<T> q;
            q.load(at + u * kThreads * Piece<T>::W);
#pragma unroll
            for (int k = 0; k < Piece<T>::W / 2; ++k) {
                float2 t = fma2(q.pair(k), splat2(c), splat2(-rho));
                t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
                sum = fma2(make_float2(ex2(t.x), ex2(t.y)), t, sum);
            }
        }
        return sum;
    }
    __device__ __forceinline__ void raise(float to) {
        const float d = fmaxf(rho - to, kNothing), e = ex2(d);
        rho = to;
        s1 = mul2(splat2(e), fma2(s, splat2(d), s1));
        s = mul2(s, splat2(e));
    }
    __device__ __forceinline__ void end(float v, float c) {
        top = fmaxf(top, v);
        if (const float at_top = reference(top, c); at_top > rho + kSlack) raise(at_top);
        const float t = max_nan(fmaf(v, c, -rho), kNothing), x = ex2(t);
        s.x += x;
        s1.x = fmaf(x, t, s1.x);
    }
};

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
// The sums of a whole row relative to its largest logit, term by term, by one warp.  (4096 x 50280 bf16 with every row summed
// again: 257 us; an element at a time 589.)
template <typename T>
__device__ __noinline__ Sums sum_again(const Row<T>& row, float top, float c) {
    constexpr int N = 4;
    const int lane = threadIdx.x % 32;
    const float2 neg = splat2(-top), cc = splat2(c);
    float2 s = splat2(0.0f), s1 = splat2(0.0f);
    auto term = [&](float2 v) {
        float2 t = mul2(add2(v, neg), cc);
        t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
        const float2 e = make_float2(ex2(t.x), ex2(t.y));
        s = add2(s, e);
        s1 = fma2(e, t, s1);
    };
    for (int j0 = lane; j0 - lane < row.pieces; j0 += 32 * N) {
        Piece<T> q[N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (j0 + 32 * u < row.pieces) q[u].load(row.p + row.head + static_cast<long long>(j0 + 32 * u) * Piece<T>::W);
            else q[u].ruled_out();
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int k = 0; k < Piece<T>::W / 2; ++k) term(q[u].pair(k));
    }
    term(make_float2(lane < row.head ? to_f(row.p[lane]) : -INFINITY, row.tail() + lane < row.V ? to_f(row.p[row.tail() + lane]) : -INFINITY));
    Sums a{top, 0.0f, s.x + s.y, s1.x + s1.y};
    join_lanes(a, 32);
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

constexpr int kGroup = kThreads / 64;  // threads of a group
constexpr int kMaxSplit = 16;
static_assert(kRoom >= kMaxSplit * kMaxTop, "the parts' alternatives are joined in key");
static_assert(kRoom >= kMaxTop * 4 * 8, "neighbouring tokens that are fewer than the groups they would need fit");
struct TopRoom {
    float group[64];
    uint64_t key[kRoom], sel[kMaxTop], best[kWarps];
    int n;
};
__device__ __forceinline__ void group_max(TopRoom& t, float own_top) {
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) own_top = fmaxf(own_top, __shfl_xor_sync(0xffffffffu, own_top, o));
    if (threadIdx.x % kGroup == 0) t.group[threadIdx.x / kGroup] = own_top;
}
__device__ __forceinline__ void sync_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

// The n-th largest of the lanes' values (of their two values), in every lane.
__device__ __forceinline__ float ordered(float v, int o, bool falling) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    return ((threadIdx.x & o) == 0) == falling ? fmaxf(v, other) : fminf(v, other);
}
__device__ __forceinline__ float nth_of_32(float v, int n) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) v = ordered(v, o, (threadIdx.x % 32 & size) == 0);
    return __shfl_sync(0xffffffffu, v, n - 1);
}
__device__ __forceinline__ float first_of_64(float a, float b) {  // the 32 largest in falling order
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const bool falling = (threadIdx.x % 32 & size) == 0;
            a = ordered(a, o, falling);
            b = ordered(b, o, size == 32 ? false : falling);
        }
    a = fmaxf(a, b);  // the larger half; it falls and rises, one more pass puts it in order
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = ordered(a, o, true);
    return a;
}
__device__ __forceinline__ float nth_of_64(float a, float b, int n) { return __shfl_sync(0xffffffffu, first_of_64(a, b), n - 1); }  // n <= 32

// The alternatives of [lo, hi) pieces (and the ends) of a row.  Four threads' elements form a group.  tau, the top-th largest of
// the 64 groups' maxima (of 32 groups': 32 alternatives of 8 rows 16.8 us instead of 10.6, 20 alternatives 10.1 instead of 9.0), is a lower bound of the top-th largest element: only what threads whose own maximum reaches it have seen
// is read again (from L2), and what reaches it there goes to key[0 .. n) in any order.  Called by kThreads threads behind a
// barrier that the groups' maxima and n = 0 have passed; a barrier ends it.  Returns how many keys there are: all that reach tau,
// or where there was no room the largest (what is left equals tau then); or kInOrder, when sel is complete.
constexpr int kInOrder = -1;
template <typename T>
__device__ __noinline__ int reach(TopRoom& t, const Row<T>& row, int lo, int hi, bool first, bool last, int top, float own_top, float* equals) {
    constexpr int W = Piece<T>::W;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float tau = nth_of_64(t.group[lane], t.group[lane + 32], top);
    auto offer = [&](float v, int i) {
        if (v >= tau && v > -INFINITY) {
            const int at = atomicAdd(&t.n, 1);
            if (at < kRoom) t.key[at] = key_of(v, i);
        }
    };
    // half a warp for each such thread: a lane has every 16th of its pieces
    unsigned who = __ballot_sync(0xffffffffu, own_top >= tau && own_top > -INFINITY);
    while (who) {
        const int one = __ffs(who) - 1;
        who &= who - 1;
        const int two = who ? __ffs(who) - 1 : -1;
        who &= who - 1;
        const int x = lane < 16 ? one : two;
        if (x < 0) continue;
        const int y = warp * 32 + x;
        for (int j = lo + y + (lane & 15) * kThreads; j < hi; j += 16 * kThreads) {
            Piece<T> q;
            q.load(row.p + row.head + static_cast<long long>(j) * W);
            if (Piece<T>::template top<1>(&q) < tau) continue;
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const float2 v = q.pair(e / 2);
                offer(v.x, row.head + j * W + e);
                offer(v.y, row.head + j * W + e + 1);
            }
        }
        if ((lane & 15) == 0 && first && y < row.head) offer(to_f(row.p[y]), y);
        if ((lane & 15) == 1 && last && row.tail() + y < row.V) offer(to_f(row.p[row.tail() + y]), row.tail() + y);
    }
    sync_consumers();
    const int n = t.n;
    *equals = -INFINITY;
    if (n <= 64) return n;
    if (n <= kRoom) {  // (many equals: one warp alone would take long)
        for (int a = tid; a < n; a += kThreads) {
            const uint64_t mine = t.key[a];
            int rank = 0;
            for (int b = 0; b < n; ++b) rank += t.key[b] > mine;
            if (rank < top) t.sel[rank] = mine;
        }
        sync_consumers();
        return kInOrder;
    }
    // More reach tau than there is room for: those above it one after the other, until tau itself is met.
    sync_consumers();
    *equals = tau;
    const int begin = first ? 0 : row.head + lo * W, end = last ? row.V : row.head + hi * W;
    uint64_t below = ~0ull;
    int k = 0;
    for (; k < top; ++k) {
        uint64_t best = 0;
        for (int i = begin + tid; i < end; i += kThreads) {
            const uint64_t k2 = key_of(to_f(row.p[i]), i);
            if (k2 < below && k2 > best) best = k2;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t k2 = __shfl_xor_sync(0xffffffffu, best, o);
            if (k2 > best) best = k2;
        }
        if (lane == 0) t.best[warp] = best;
        sync_consumers();
        for (int w = 0; w < kWarps; ++w)
            if (t.best[w] > best) best = t.best[w];
        sync_consumers();
        if (key_value(best) <= tau) break;
        below = best;
        if (tid == 0) t.key[k] = best;
    }
    sync_consumers();
    return k;
}

// One warp puts the n keys in order into sel[0 .. top) and fills up with the lowest indices of what equals `equals`.
template <typename T>
__device__ __forceinline__ void rank_keys(const uint64_t* key, uint64_t* sel, int n, float equals, const Row<T>& row, int begin, int end, int top) {
    const int lane = threadIdx.x % 32;
    if (n == kInOrder) return;
    sel[lane] = 0;
    __syncwarp();
    for (int a = lane; a < n; a += 32) {
        const uint64_t mine = key[a];
        int rank = 0;
        for (int b = 0; b < n; ++b) rank += key[b] > mine;
        if (rank < top) sel[rank] = mine;
    }
    int found = n;
    for (int i0 = begin; i0 < end && found < top; i0 += 8 * 32) {
        bool hit[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + 32 * u + lane;
            const float v = i < end ? to_f(row.p[i]) : 0.0f;
            hit[u] = i < end && (v == v ? v : -INFINITY) == equals;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const unsigned hits = __ballot_sync(0xffffffffu, hit[u]);
            const int at = found + __popc(hits & ((1u << lane) - 1));
            if (hit[u] && at < top) sel[at] = key_of(equals, i0 + 32 * u + lane);
            found += __popc(hits);
        }
    }
    __syncwarp();
}

// Sums relative to a row's largest logit from those relative to rho.
template <typename T>
__device__ __forceinline__ void settle(Sums& a, const Row<T>& row, float c) {
    if (in_doubt(a, c)) {
        a = sum_again(row, a.top, c);
    } else if (a.top > -INFINITY) {
        const float r = fmaf(a.top, c, -a.rho), e = exp2f(-r);
        a.s1 = e * fmaf(-r, a.s, a.s1);
        a.s *= e;
    }
}
// One warp writes a row's results from its sums (alike in all lanes, relative to the largest logit), the target's logit and the
// alternatives in order.  The largest logit's own term is 1, so S is no less, a log probability no more than 0 and an entropy no less.
template <typename T>
__device__ __forceinline__ void write_row(const FwdParams& p, long long r, const Sums& a, int target, float logit, const uint64_t* sel) {
    const int lane = threadIdx.x % 32;
    const float S = max_nan(a.s, 1.0f), log_s = logf(S);  // (lg2 near 1 is good to 2^-22 alone)
    const bool none = a.s == 0.0f;
    if (lane == 0) {
        if (p.lse) {
            p.lse[r] = a.s == a.s ? a.top : a.s;
            p.lse[p.rows + r] = none ? 0.0f : log_s;
        }
        if (p.entropy) p.entropy[r] = none ? 0.0f : max_nan(fmaf(-a.s1 / S, kLn2, log_s), 0.0f);
        if (p.logprob) {
            const bool ok = target >= 0 && target < p.V;
            p.logprob[r] = !ok ? 0.0f : none ? -INFINITY : (logit - a.top) * p.inv_temp - log_s;
        }
    }
    if (sel && lane < p.top) {
        const uint64_t k = sel[lane];
        p.top_ids[r * p.top + lane] = key_index(k);
        p.top_logprobs[r * p.top + lane] = none ? -INFINITY : (key_value(k) - a.top) * p.inv_temp - log_s;
    }
}
__device__ __forceinline__ int target_of(const FwdParams& p, long long r) { return p.targets && p.logprob ? p.targets[r] : -1; }

// Rows one after another, by eight warps that do nothing but read: a ninth brings the rows to shared memory by bulk copies of
// 16 KB, three more make the results of rows while the next ones are read, so the memory is never idle.  HBM would be 12 logits a cycle
// and SM in 16 bits: with 16 exponentials a cycle and some 5 instructions a logit (of 128) the arithmetic is close behind, so the
// pass has one fma and one exponential a logit, no clamp, and no test but two in 32 logits.  4096 x 50280 bf16 without alternatives
// 72 us, 87 % of the copy rate.
constexpr int kRound = kThreads * kUnroll, kStages = 3;
constexpr int kMakers = 3, kMakerRoom = 256;  // warps that make results
struct __align__(16) Maker {  // a row's, while the next rows' are found
    float thread_top[kThreads];
    Sums part[kWarps];
    uint64_t key[kMakerRoom], sel[kMaxTop], full, empty;
    int piece[kMakerRoom], n;
    unsigned char threads[kThreads];
};
struct RowsRoom {
    Maker maker[kMakers];
    uint64_t full[kStages], empty[kStages];
};
static_assert(sizeof(Maker) % 16 == 0 && kThreads <= 256, "float4 reads of thread_top; threads are bytes");
constexpr int kRowsSmem = kStages * kRound * 16 + static_cast<int>(sizeof(RowsRoom)) + 128;
static_assert(kCtas * (kRowsSmem + 1024) <= 228 * 1024, "CTAs on an SM");

// The alternatives of a row in order into sel, by one warp.  Four threads' elements form a group.  tau, the top-th largest of
// the 64 groups' maxima, is a lower bound of the top-th largest element: only what threads whose own maximum reaches it have seen
// is read again (from L2), and what reaches it there is ranked by counting.  Some 37 us a row and warp with 20 alternatives, while nine
// such warps share an SM with the readers: 4096 x 50280 takes 110 us, with 5 alternatives 77, with none 72.  (Three threads' pieces at
// once; with four, registers spill and 20 alternatives take 115, with two they take 115 to 131.)
template <typename T>
__device__ __noinline__ void find_top(Maker& t, const Row<T>& row, float row_top, int top) {
    constexpr int W = Piece<T>::W, kEach = kThreads / 32, kAtOnce = 3;
    static_assert(kEach == 8, "two groups of four threads a lane");
    const int lane = threadIdx.x % 32;
    float mine[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(t.thread_top + lane * kEach + i);
        mine[i] = v.x, mine[i + 1] = v.y, mine[i + 2] = v.z, mine[i + 3] = v.w;
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&t.empty);
    const float a = fmaxf(fmaxf(mine[0], mine[1]), fmaxf(mine[2], mine[3])), b = fmaxf(fmaxf(mine[4], mine[5]), fmaxf(mine[6], mine[7]));
    float tau = top <= 8 ? nth_of_32(fmaxf(a, b), top) : nth_of_64(a, b, top);
    int threads = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const bool hit = mine[i] >= tau && mine[i] > -INFINITY;
        const unsigned hits = __ballot_sync(0xffffffffu, hit);
        if (hit) t.threads[threads + __popc(hits & ((1u << lane) - 1))] = static_cast<unsigned char>(lane * kEach + i);
        threads += __popc(hits);
    }
    if (lane == 0) t.n = 0;
    __syncwarp();
    // their pieces that reach tau (where tau is the largest logit and many threads have it, the first of its equals are enough)
    const bool level = tau == row_top && threads > 64;
    int pieces = level ? kMakerRoom + 1 : 0;
    for (int x = 0; x < threads && !level; x += kAtOnce)
        for (int j0 = 0; j0 < row.pieces; j0 += 32 * kThreads) {
            Piece<T> q[kAtOnce];
            int j[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                j[u] = x + u < threads ? j0 + lane * kThreads + t.threads[x + u] : row.pieces;
                if (j[u] < row.pieces) q[u].load(row.p + row.head + static_cast<long long>(j[u]) * W);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float best = j[u] < row.pieces ? Piece<T>::template top<1>(q + u) : -INFINITY;
                const bool hit = best >= tau && best > -INFINITY;
                const unsigned hits = __ballot_sync(0xffffffffu, hit);
                const int at = pieces + __popc(hits & ((1u << lane) - 1));
                if (hit && at < kMakerRoom) t.piece[at] = j[u];
                pieces += __popc(hits);
            }
        }
    __syncwarp();
    auto offer = [&](float v, int i) {
        if (v >= tau && v > -INFINITY) {
            const int at = atomicAdd(&t.n, 1);
            if (at < kMakerRoom) t.key[at] = key_of(v, i);
        }
    };
    auto piece = [&](int x) {
        Piece<T> q;
        q.load(row.p + row.head + static_cast<long long>(t.piece[x]) * W);
        return q;
    };
    auto offer_all = [&]() {
        for (int x = lane; x < pieces; x += 32) {
            const Piece<T> q = piece(x);
            const int i = row.head + t.piece[x] * W;
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const float2 v = q.pair(e / 2);
                offer(v.x, i + e);
                offer(v.y, i + e + 1);
            }
        }
        if (lane < row.head) offer(to_f(row.p[lane]), lane);
        if (row.tail() + lane < row.V) offer(to_f(row.p[row.tail() + lane]), row.tail() + lane);
        __syncwarp();
    };
    if (pieces <= kMakerRoom) offer_all();
    if (t.n > kMakerRoom) {
        // Many in few threads' places (neighbouring tokens, when all others are ruled out): the top-th largest of the pieces' own
        // largest is a closer bound.
        float first = -INFINITY;
        for (int x = lane; x - lane < pieces; x += 32) {
            float best = -INFINITY;
            if (x < pieces) {
                const Piece<T> q = piece(x);
                best = Piece<T>::template top<1>(&q);
            }
            first = first_of_64(first, best);
        }
        tau = fmaxf(tau, __shfl_sync(0xffffffffu, first, top - 1));
        __syncwarp();
        if (lane == 0) t.n = 0;
        __syncwarp();
        offer_all();
    }
    int n = max(t.n, pieces);
    if (n <= kMakerRoom) n = t.n;
    float equals = -INFINITY;
    if (n > kMakerRoom) {
        // More reach tau than there is room for: those above it one after the other, until tau itself is met.
        equals = tau;
        n = 0;
        uint64_t below = ~0ull;
        if (row_top > tau)
            for (; n < top; ++n) {
                uint64_t best = 0;
                for (int i0 = lane; i0 < row.V; i0 += 8 * 32) {
                    float v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) v[u] = i0 + 32 * u < row.V ? to_f(row.p[i0 + 32 * u]) : -INFINITY;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const uint64_t k = key_of(v[u], i0 + 32 * u);
                        if (k < below && k > best) best = k;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
                    if (k > best) best = k;
                }
                if (key_value(best) <= tau) break;
                below = best;
                if (lane == 0) t.key[n] = best;
            }
        __syncwarp();
    }
    rank_keys<T>(t.key, t.sel, n, equals, row, 0, row.V, top);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads + 32 + 32 * kMakers, kCtas) token_logprobs_rows_kernel(const FwdParams p, int* status) {
    constexpr int W = Piece<T>::W;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    RowsRoom& room = *reinterpret_cast<RowsRoom*>(sm + kStages * kRound * 16);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&room.full[s], 1);
            mbar_init(&room.empty[s], kWarps);
        }
        for (int m = 0; m < kMakers; ++m) {
            mbar_init(&room.maker[m].full, kWarps);
            mbar_init(&room.maker[m].empty, 1);
        }
        fence_barrier_init();
    }
    __syncthreads();
    const float c = p.inv_temp * kLog2e;
    bool alive = true;
    if (warp == kWarps) {  // brings the rows
        if (lane != 0) return;
        int s = 0;
        uint32_t parity = 1;  // (the first round of the ring waits for nobody)
        for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
            const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
            for (int j = 0; j < row.pieces; j += kRound) {
                alive = alive && mbar_wait(&room.empty[s], parity, status);
                const uint32_t bytes = 16u * min(kRound, row.pieces - j);
                mbar_expect_tx(&room.full[s], bytes);
                bulk_load(sm + s * kRound * 16, row.p + row.head + static_cast<long long>(j) * W, bytes, &room.full[s]);
                if (++s == kStages) s = 0, parity ^= 1;
            }
        }
        return;
    }
    if (warp > kWarps) {  // makes the results of every kMakers-th row
        Maker& t = room.maker[warp - kWarps - 1];
        uint32_t flips = 0;
        for (long long r = blockIdx.x + static_cast<long long>(warp - kWarps - 1) * gridDim.x; r < p.rows; r += static_cast<long long>(kMakers) * gridDim.x, flips ^= 1) {
            const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
            const int target = target_of(p, r);
            const float logit = target >= 0 && target < p.V ? to_f(row.p[target]) : 0.0f;
            alive = alive && mbar_wait(&t.full, flips, status);
            Sums a = t.part[lane % kWarps];
            join_lanes(a, kWarps);
            if (TOP) {
                find_top<T>(t, row, a.top, p.top);
            } else {
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&t.empty);
            }
            settle(a, row, c);
            write_row<T>(p, r, a, target, logit, TOP ? t.sel : nullptr);
        }
        return;
    }
    int maker = 0;
    uint32_t flips = 1;
    int s = 0;
    uint32_t parity = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
        const bool head = tid < row.head, tail = row.tail() + tid < p.V;
        const T head_v = head ? row.p[tid] : from_f<T>(0.0f), tail_v = tail ? row.p[row.tail() + tid] : from_f<T>(0.0f);
        Running<T> run;
        for (int j = 0; j < row.pieces; j += kRound) {
            alive = alive && mbar_wait(&room.full[s], parity, status);
            const T* stage = reinterpret_cast<const T*>(sm + s * kRound * 16) + tid * W;
            if (j + kRound <= row.pieces) {
                run.template take<kUnroll>(stage, c);
            } else {
#pragma unroll 1
                for (int u = 0; j + u * kThreads + tid < row.pieces; ++u) run.template take<1>(stage + u * kThreads * W, c);
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&room.empty[s]);
            if (++s == kStages) s = 0, parity ^= 1;
        }
        if (head) run.end(to_f(head_v), c);
        if (tail) run.end(to_f(tail_v), c);
        const float own_top = run.top;
        Sums a = run.sums();
        join_lanes(a, 32);
        Maker& t = room.maker[maker];
        alive = alive && mbar_wait(&t.empty, flips, status);  // (its last row is done with)
        if (TOP) t.thread_top[tid] = own_top;
        if (lane == 0) t.part[warp] = a;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&t.full);
        if (++maker == kMakers) maker = 0, flips ^= 1;
    }
}

// Short rows: a warp has one in registers, so the largest logit is known before the sums and nothing is read twice.  Up to
// 32 P pieces; kShortPieces 32 are 8192 logits in 16 bits, and half of that where there are alternatives.  tau, a lower bound of the top-th largest logit, comes from the largest
// of each lane's even and odd elements (of each lane's alone, 32 alternatives of 4096 x 4000 were 374 us and not 26: the smallest of
// 32 lanes lets too many through); up to 8 alternatives the lanes' suffice and cost less.
constexpr int kShortPieces = 32, kShortWarps = 4, kShortRoom = 128;
template <typename T, bool TOP, int P>
__global__ void __launch_bounds__(kShortWarps * 32) token_logprobs_short_kernel(const FwdParams p) {
    constexpr int W = Piece<T>::W;
    __shared__ uint64_t keys[TOP ? kShortWarps : 1][kShortRoom], sels[TOP ? kShortWarps : 1][kMaxTop];
    __shared__ int counts[kShortWarps];
    __shared__ Piece<T> found[TOP ? kShortWarps : 1][kShortRoom];
    __shared__ short which[TOP ? kShortWarps : 1][kShortRoom];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long r = blockIdx.x * static_cast<long long>(kShortWarps) + warp;
    if (r >= p.rows) return;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    Piece<T> q[P];
#pragma unroll
    for (int u = 0; u < P; ++u) {
        if (u * 32 + lane < row.pieces) q[u].load(row.p + row.head + (u * 32 + lane) * W);
        else q[u].ruled_out();
    }
    const float head = lane < row.head ? to_f(row.p[lane]) : -INFINITY, tail = row.tail() + lane < p.V ? to_f(row.p[row.tail() + lane]) : -INFINITY;
    const int target = target_of(p, r);
    const float logit = target >= 0 && target < p.V ? to_f(row.p[target]) : 0.0f;
    float2 own = Piece<T>::template tops<P>(q);
    // (A lane that has met nothing but NaN: minus infinity.  As NaN it took the other lane's value in the search for the n-th largest,
    // and the bound came out too high.)
    own.x = fmaxf(fmaxf(own.x, head), -INFINITY), own.y = fmaxf(fmaxf(own.y, tail), -INFINITY);
    const float c = p.inv_temp * kLog2e, own_top = fmaxf(own.x, own.y);
    Sums a{own_top, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a.top = fmaxf(a.top, __shfl_xor_sync(0xffffffffu, a.top, o));
    const float from = a.top == -INFINITY ? 0.0f : a.top;  // (nothing left: every term is 0, but for NaN)
    const float2 cc = splat2(c), neg = splat2(-from);
    float2 s = splat2(0.0f), s1 = splat2(0.0f);
    auto term = [&](float2 v) {
        float2 t = mul2(add2(v, neg), cc);
        t.x = max_nan(t.x, kNothing), t.y = max_nan(t.y, kNothing);
        const float2 x = make_float2(ex2(t.x), ex2(t.y));
        s = add2(s, x);
        s1 = fma2(x, t, s1);
    };
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u * 32 < row.pieces)
#pragma unroll
            for (int k = 0; k < W / 2; ++k) term(q[u].pair(k));
    term(make_float2(head, tail));
    a.s = s.x + s.y, a.s1 = s1.x + s1.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.s1 += __shfl_xor_sync(0xffffffffu, a.s1, o);
    }
    uint64_t* sel = sels[TOP ? warp : 0];
    if (TOP) {
        uint64_t* key = keys[TOP ? warp : 0];
        const float tau = p.top == 1 ? a.top : p.top <= 8 ? nth_of_32(own_top, p.top) : nth_of_64(own.x, own.y, p.top);
        // The pieces that reach it go to shared memory first: looked through where they are, in registers, they are as much code as there
        // are registers, fetched from L2 by every CTA (20 alternatives of 4096 x 4000 22.1 us, 15.7 like this).
        if (lane == 0) counts[warp] = 0;
        int pieces = 0;
#pragma unroll
        for (int u = 0; u < P; ++u) {
            const float best = Piece<T>::template top<1>(q + u);
            const bool hit = best >= tau && best > -INFINITY;
            const unsigned hits = __ballot_sync(0xffffffffu, hit);
            const int at = pieces + __popc(hits & ((1u << lane) - 1));
            if (hit && at < kShortRoom) found[warp][at] = q[u], which[warp][at] = static_cast<short>(u * 32 + lane);
            pieces += __popc(hits);
        }
        __syncwarp();
        auto offer = [&](float v, int i) {
            if (v >= tau && v > -INFINITY) {
                const int at = atomicAdd(&counts[warp], 1);
                if (at < kShortRoom) key[at] = key_of(v, i);
            }
        };
#pragma unroll 1
        for (int x = lane; x < min(pieces, kShortRoom); x += 32) {
            const Piece<T> piece = found[warp][x];
            const int i = row.head + which[warp][x] * W;
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const float2 v = piece.pair(e / 2);
                offer(v.x, i + e);
                offer(v.y, i + e + 1);
            }
        }
        offer(head, lane);
        offer(tail, row.tail() + lane);
        __syncwarp();
        const int n = max(counts[warp], pieces > kShortRoom ? pieces : 0);
        if (n <= kShortRoom) {
            rank_keys<T>(key, sel, n, -INFINITY, row, 0, p.V, p.top);
        } else {
            // crowded by what equals tau: those above it one after the other
            uint64_t below = ~0ull;
            int k = 0;
            if (a.top > tau)
                for (; k < p.top; ++k) {
                    uint64_t best = 0;
                    for (int i = lane; i < p.V; i += 32) {
                        const uint64_t k2 = key_of(to_f(row.p[i]), i);
                        if (k2 < below && k2 > best) best = k2;
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const uint64_t k2 = __shfl_xor_sync(0xffffffffu, best, o);
                        if (k2 > best) best = k2;
                    }
                    if (key_value(best) <= tau) break;
                    below = best;
                    if (lane == 0) key[k] = best;
                }
            __syncwarp();
            rank_keys<T>(key, sel, k, tau, row, 0, p.V, p.top);
        }
    }
    write_row<T>(p, r, a, target, logit, TOP ? sel : nullptr);
}

// Few rows: the CTAs of a cluster have a part of one each, and the first joins what they found.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_split_kernel(const FwdParams p) {
    constexpr int W = Piece<T>::W;
    __shared__ Sums part[kWarps];
    __shared__ __align__(16) Sums mine;
    __shared__ TopRoom room;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = p.inv_temp * kLog2e;
    const int R = p.split, rank = static_cast<int>(blockIdx.x) % R;
    const long long r = blockIdx.x / R;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    const int lo = static_cast<int>(static_cast<long long>(row.pieces) * rank / R), hi = static_cast<int>(static_cast<long long>(row.pieces) * (rank + 1) / R);
    const bool first = rank == 0, last = rank == R - 1;
    const T* base = row.p + row.head;
    int target = -1;
    float logit = 0.0f;
    if (first && tid == 0) {
        target = target_of(p, r);
        if (target >= 0 && target < p.V) logit = to_f(row.p[target]);
        room.n = 0;
    }
    if (!first && tid == 0) room.n = 0;
    Running<T> run;
    int j = lo + tid;
    for (; j + (kUnroll - 1) * kThreads < hi; j += kRound) run.template take<kUnroll>(base + static_cast<long long>(j) * W, c);
    for (; j < hi; j += kThreads) run.template take<1>(base + static_cast<long long>(j) * W, c);
    if (first && tid < row.head) run.end(to_f(row.p[tid]), c);
    if (last && row.tail() + tid < p.V) run.end(to_f(row.p[row.tail() + tid]), c);
    if (TOP) group_max(room, run.top);
    Sums a = run.sums();
    join_lanes(a, 32);
    if (lane == 0) part[warp] = a;
    sync_consumers();
    int n = 0;
    float equals = 0.0f;
    if (TOP) n = reach<T>(room, row, lo, hi, first, last, p.top, run.top, &equals);
    if (warp == 0) {
        a = part[lane % kWarps];
        join_lanes(a, kWarps);
        if (lane == 0) mine = a;
        if (TOP) rank_keys<T>(room.key, room.sel, n, equals, row, first ? 0 : row.head + lo * W, last ? p.V : row.head + hi * W, p.top);
    }
    cluster_sync();
    if (first) {
        if (warp == 0) {
            a = no_sums();
            if (lane < R) {
                const float4 v = ld_cluster4(cluster_addr(smem_u32(&mine), lane));
                a = Sums{v.x, v.y, v.z, v.w};
            }
            join_lanes(a, 32);
        }
        if (TOP)
            for (int i = tid; i < R * p.top; i += kThreads) {
                const int from = i / p.top, k = i - from * p.top;
                uint64_t v;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(smem_u32(room.sel + k), from)));
                room.key[i] = v;
            }
    }
    cluster_sync();
    if (!first) return;
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
        sync_consumers();
    }
    if (warp == 0) {
        settle(a, row, c);
        write_row<T>(p, r, a, target, logit, TOP ? room.sel : nullptr);
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
// start at the same place of 16 bytes.  A row has G threads, each with four loads in flight, the first ones asked for before
// anything else of the row: a short one is over as soon as they are there.
constexpr int kBwdThreads = 256, kBwdUnroll = 4;
template <typename T, bool ALIGNED, int G>
__global__ void __launch_bounds__(kBwdThreads, 4) token_logprobs_bwd_kernel(const BwdParams p) {
    constexpr int W = Piece<T>::W;
    const int tid = threadIdx.x % G;
    const long long r = blockIdx.x * static_cast<long long>(kBwdThreads / G) + threadIdx.x / G;
    if (r >= p.rows) return;
    const Row<T> row(static_cast<const T*>(p.logits) + r * p.ld, p.V);
    T* out = static_cast<T*>(p.dlogits) + r * p.ld_d;
    Piece<T> q[kBwdUnroll];
    float head = 0.0f, tail = 0.0f;
    if constexpr (ALIGNED) {
#pragma unroll
        for (int u = 0; u < kBwdUnroll; ++u)
            if (tid + u * G < row.pieces) q[u].load(row.p + row.head + (tid + u * G) * W);
        if (tid < row.head) head = to_f(row.p[tid]);
        if (row.tail() + tid < p.V) tail = to_f(row.p[row.tail() + tid]);
    }
    const float m = p.lse[r], log2_s = p.lse[p.rows + r] * kLog2e, dl = p.d_logprob ? p.d_logprob[r] : 0.0f, dh = p.d_entropy ? p.d_entropy[r] : 0.0f;
    const float entropy = p.d_entropy ? p.entropy[r] : 0.0f;
    const int tgt = p.targets ? p.targets[r] : -1;
    const bool none = m == -INFINITY;
    const float g = tgt >= 0 && tgt < p.V && !none ? dl * p.inv_temp : 0.0f, gh = none ? 0.0f : dh * p.inv_temp;
    const float k0 = -fmaf(gh, entropy, g), k1 = -gh * kLn2, c = p.inv_temp * kLog2e;
    auto one = [&](float v, int i) {
        const float t = none ? kNothing : max_nan(fmaf(v - m, c, -log2_s), kNothing);
        const float d = ex2(t) * fmaf(k1, t, k0);
        return i == tgt ? d + g : d;
    };
    if constexpr (!ALIGNED) {
        for (int i = tid; i < p.V; i += G) out[i] = from_f<T>(one(to_f(row.p[i]), i));
        return;
    }
    const float2 neg = splat2(none ? 0.0f : -m), cc = splat2(c), ls = splat2(-log2_s), kk0 = splat2(k0), kk1 = splat2(k1);
    for (int j0 = tid; j0 < row.pieces; j0 += G * kBwdUnroll) {
#pragma unroll
        for (int u = 0; u < kBwdUnroll; ++u) {
            const int j = j0 + u * G, i = row.head + j * W;
            if (j >= row.pieces) break;
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
        // (four at once: one for each that is done mixes reads and writes, 150 us for 4096 x 50280 against 129.5)
#pragma unroll
        for (int u = 0; u < kBwdUnroll; ++u) {
            const int j = j0 + (u + kBwdUnroll) * G;
            if (j < row.pieces) q[u].load(row.p + row.head + j * W);
        }
    }
    if (tid < row.head) out[tid] = from_f<T>(one(head, tid));
    const int i = row.tail() + tid;
    if (i < p.V) out[i] = from_f<T>(one(tail, i));
}

// How many CTAs share a row: as many as find room beside one another (four on an SM), each with 2048 logits or more.  Joining the
// parts' alternatives costs more than reading them faster gains: 8 rows of 50280 with 20 alternatives 15.6 us over 16 CTAs, 10.6 over
// 8, 9.9 over 4; without alternatives 4.1, 4.8 and 4.8.
static int pick_split(int sms, long long rows, int V, bool top) {
    int s = 1;
    while (s < (top ? 4 : kMaxSplit) && rows * 2 * s <= 4ll * sms && V >= 2 * s * 2048) s *= 2;
    return s;
}

template <typename T, bool TOP>
static int launch_fwd(Ctx* c, FwdParams& p, cudaStream_t st) {
    constexpr int W = Piece<T>::W;
    if (p.V <= 32 * W * (TOP ? kShortPieces / 2 : kShortPieces)) {
        const unsigned blocks = static_cast<unsigned>((p.rows + kShortWarps - 1) / kShortWarps);
        if (p.V <= 32 * W * 4) token_logprobs_short_kernel<T, TOP, 4><<<blocks, kShortWarps * 32, 0, st>>>(p);
        else if (p.V <= 32 * W * 8) token_logprobs_short_kernel<T, TOP, 8><<<blocks, kShortWarps * 32, 0, st>>>(p);
        else if (TOP || p.V <= 32 * W * 16) token_logprobs_short_kernel<T, TOP, 16><<<blocks, kShortWarps * 32, 0, st>>>(p);
        else if constexpr (!TOP) token_logprobs_short_kernel<T, TOP, kShortPieces><<<blocks, kShortWarps * 32, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        return MAMBA_B200_OK;
    }
    p.split = pick_split(c->sm_count, p.rows, p.V, TOP);
    if (p.split == 1) {
        const long long most = static_cast<long long>(kCtas) * c->sm_count;
        token_logprobs_rows_kernel<T, TOP><<<static_cast<unsigned>(p.rows < most ? p.rows : most), kThreads + 32 + 32 * kMakers, kRowsSmem, st>>>(p, c->d_status);
    } else {
        void* args[] = {&p};
        MB200_CUDA_CHECK(c, launch_cluster(reinterpret_cast<const void*>(token_logprobs_split_kernel<T, TOP>), dim3(static_cast<unsigned>(p.rows * p.split)),
                                           dim3(kThreads), 0, st, p.split, args));
    }
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}
template <typename T, bool TOP>
static int configure(Ctx* c) {
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(token_logprobs_rows_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem));
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(token_logprobs_split_kernel<T, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return MAMBA_B200_OK;
}
template <typename T>
static int launch_fwd(Ctx* c, FwdParams& p, cudaStream_t st) {
    return p.top ? launch_fwd<T, true>(c, p, st) : launch_fwd<T, false>(c, p, st);
}

// A warp for each row where that fills the SMs and a row is no more than eight pieces a lane; a CTA otherwise.  us, warps and CTAs: 8192
// rows of 637 in 16 bits 5.3 and 14.5, 2630 of 1872 5.0 and 6.5, 64 of 4000 5.3 and 2.2; f32: 5180 of 3144 34 and 23.
template <typename T>
static int launch_bwd(Ctx* c, const BwdParams& p, cudaStream_t st) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p.logits), y = reinterpret_cast<uintptr_t>(p.dlogits);
    const bool aligned = (x - y) % 16 == 0 && (p.rows == 1 || (p.ld - p.ld_d) * static_cast<long long>(sizeof(T)) % 16 == 0);
    const unsigned grid = static_cast<unsigned>(p.rows), few = static_cast<unsigned>((p.rows + kBwdThreads / 32 - 1) / (kBwdThreads / 32));
    const bool narrow = p.V <= 256 * Piece<T>::W && p.rows >= 4ll * c->sm_count;
    if (aligned && narrow) token_logprobs_bwd_kernel<T, true, 32><<<few, kBwdThreads, 0, st>>>(p);
    else if (aligned) token_logprobs_bwd_kernel<T, true, kBwdThreads><<<grid, kBwdThreads, 0, st>>>(p);
    else if (narrow) token_logprobs_bwd_kernel<T, false, 32><<<few, kBwdThreads, 0, st>>>(p);
    else token_logprobs_bwd_kernel<T, false, kBwdThreads><<<grid, kBwdThreads, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

}  // namespace lp

int logprobs_configure(Ctx* c) {
    int rc = lp::configure<float, true>(c);
    if (!rc) rc = lp::configure<float, false>(c);
    if (!rc) rc = lp::configure<__half, true>(c);
    if (!rc) rc = lp::configure<__half, false>(c);
    if (!rc) rc = lp::configure<__nv_bfloat16, true>(c);
    if (!rc) rc = lp::configure<__nv_bfloat16, false>(c);
    return rc;
}

}  // namespace mb200

using namespace mb200;

// The kernels multiply by log2(e) / temperature.
static bool temperature_ok(float temperature) { return temperature > 0.0f && temperature <= 3e38f && kLog2e / temperature <= 3e38f; }

extern "C" MAMBA_B200_API int mamba_b200_token_logprobs(void* handle, void* stream, int dtype, const void* logits, long long ld,
                                                        const int* targets, float temperature, float* lse, float* entropy,
                                                        float* logprob, int top, int* top_ids, float* top_logprobs, long long rows,
                                                        int V) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: bad dtype %d", dtype);
    if (rows < 0 || V <= 0 || ld < V) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: bad dims");
    if (!temperature_ok(temperature)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: temperature %g", temperature);
    if (top < 0 || top > lp::kMaxTop || top > V)
        return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs: %d alternatives of %d tokens (at most %d)", top, V, lp::kMaxTop);
    if (rows == 0) return MAMBA_B200_OK;
    if (rows > 2147483647ll || V > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs: too many rows or tokens");
    if (!aligned_to(dtype_size(dtype), {logits}) || !aligned_to(4, {targets, lse, entropy, logprob, top_ids, top_logprobs}))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: misaligned pointer");
    if (!logits || (logprob && !targets) || (top && (!top_ids || !top_logprobs)))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs: null pointer");
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
    if (!temperature_ok(temperature)) return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: temperature %g", temperature);
    if (rows == 0) return MAMBA_B200_OK;
    if (rows > 2147483647ll || V > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "token_logprobs_bwd: too many rows or tokens");
    if (!aligned_to(dtype_size(dtype), {logits, dlogits}) || !aligned_to(4, {targets, lse, entropy, d_logprob, d_entropy}))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: misaligned pointer");
    if (!logits || !lse || !dlogits || (d_logprob && !targets) || (d_entropy && !entropy))
        return fail(c, MAMBA_B200_ERR_ARG, "token_logprobs_bwd: null pointer");
    const lp::BwdParams p{logits, targets, lse, entropy, d_logprob, d_entropy, dlogits, ld, ld_d, rows, V, 1.0f / temperature};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) return lp::launch_bwd<float>(c, p, st);
    if (dtype == MAMBA_B200_F16) return lp::launch_bwd<__half>(c, p, st);
    return lp::launch_bwd<__nv_bfloat16>(c, p, st);
}
