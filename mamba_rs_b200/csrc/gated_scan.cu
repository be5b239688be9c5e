// Gated linear recurrence, elementwise over channels:
//   u_t = sigmoid(-f_t)      h_t = h_{t-1} + u_t (x_t - h_{t-1})      y_t = h_t * SiLU(z_t)
// that is h_t = a_t h_{t-1} + (1 - a_t) x_t with the forget gate a = sigmoid(f) = 1 - u.
//   backward  g_t = dy_t SiLU(z_t) + (1 - u_{t+1}) g_{t+1}
//             d_x = u g      d_f = g (h_{t-1} - x) u (1 - u)      d_z = dy h SiLU'(z)
// A channel that forgets slowly has u near 0, and 1 - u rounded would lose it; one that forgets fast has 1 - u near 0, and loses
// that where only u is kept (6 % of it at f = -16, all at -17: a d_f of 0, and an error of 2^-25 of any earlier state in every
// later one).  So both are made, and a gate in one number is the smaller one, with a sign that says which it is: c = -u or 1 - u.
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace gs {

constexpr int kTile = MAMBA_B200_GATED_SCAN_SAVE;  // steps of a CTA's tile: one saved state each

// One or two neighbouring channels of a lane.
template <int V> struct Ch;
template <> struct Ch<1> {
    float a;
    __device__ __forceinline__ static Ch splat(float v) { return {v}; }
    template <typename T> __device__ __forceinline__ static Ch load(const T* p) { return {to_f(*p)}; }
    template <typename T> __device__ __forceinline__ void store(T* p) const { *p = from_f<T>(a); }
    template <typename F> __device__ __forceinline__ Ch map(F f) const { return {f(a)}; }
};
template <> struct Ch<2> {
    float2 a;
    __device__ __forceinline__ static Ch splat(float v) { return {splat2(v)}; }
    template <typename T> __device__ __forceinline__ static Ch load(const T* p) { return {ld_pair(p)}; }
    template <typename T> __device__ __forceinline__ void store(T* p) const { st_pair(p, a); }
    template <typename F> __device__ __forceinline__ Ch map(F f) const { return {make_float2(f(a.x), f(a.y))}; }
};
__device__ __forceinline__ Ch<1> fma(Ch<1> a, Ch<1> b, Ch<1> c) { return {fmaf(a.a, b.a, c.a)}; }
__device__ __forceinline__ Ch<2> fma(Ch<2> a, Ch<2> b, Ch<2> c) { return {fma2(a.a, b.a, c.a)}; }
__device__ __forceinline__ Ch<1> mul(Ch<1> a, Ch<1> b) { return {a.a * b.a}; }
__device__ __forceinline__ Ch<2> mul(Ch<2> a, Ch<2> b) { return {mul2(a.a, b.a)}; }
__device__ __forceinline__ Ch<1> add(Ch<1> a, Ch<1> b) { return {a.a + b.a}; }
__device__ __forceinline__ Ch<2> add(Ch<2> a, Ch<2> b) { return {add2(a.a, b.a)}; }
// a - b; the packed instructions have no signs of their own, so it is a product with -1.
template <int V> __device__ __forceinline__ Ch<V> sub(Ch<V> a, Ch<V> b) { return fma(b, Ch<V>::splat(-1.0f), a); }

template <int V> __device__ __forceinline__ Ch<V> sigmoid(Ch<V> v) {
    return add(mul(v, Ch<V>::splat(-kLog2e)).map(ex2), Ch<V>::splat(1.0f)).map(rcp);
}
// By a sign (-0 has one).
__device__ __forceinline__ float pick(float sign, float minus, float plus) { return __float_as_int(sign) < 0 ? minus : plus; }
__device__ __forceinline__ Ch<1> pick(Ch<1> sign, Ch<1> minus, Ch<1> plus) { return {pick(sign.a, minus.a, plus.a)}; }
__device__ __forceinline__ Ch<2> pick(Ch<2> sign, Ch<2> minus, Ch<2> plus) {
    return {make_float2(pick(sign.a.x, minus.a.x, plus.a.x), pick(sign.a.y, minus.a.y, plus.a.y))};
}
// u and p = 1 - u, each to its own last places, from f (t = 2^(f log2 e), u = 1 / (1 + t), p = t u or, where t is above 1, 1 - u) or
// from c.
template <int V> struct Gate {
    Ch<V> u, p;
    __device__ __forceinline__ static Gate of(Ch<V> f) {
        const Ch<V> one = Ch<V>::splat(1.0f), t = mul(f, Ch<V>::splat(kLog2e)).map(ex2), u = add(t, one).map(rcp);
        return {u, pick(f, mul(t, u), sub(one, u))};
    }
    __device__ __forceinline__ static Gate from(Ch<V> c) {
        const Ch<V> s = c.map([](float v) { return fabsf(v); }), rest = sub(Ch<V>::splat(1.0f), s);
        return {pick(c, s, rest), pick(c, rest, s)};
    }
    // (A channel that keeps everything is -0.)
    __device__ __forceinline__ Ch<V> small() const {
        if constexpr (V == 1) return {u.a < 0.5f ? -u.a : p.a};
        else return {make_float2(u.a.x < 0.5f ? -u.a.x : p.a.x, u.a.y < 0.5f ? -u.a.y : p.a.y)};
    }
    // The gate of this span of steps and one more, or another span, behind it: u is a sum of positive terms, so it keeps its relative
    // precision as p does.
    __device__ __forceinline__ void grow(const Gate& next) {
        u = fma(next.u, p, u);
        p = mul(p, next.p);
    }
};
template <int V> __device__ __forceinline__ Gate<V> no_steps() { return {Ch<V>::splat(0.0f), Ch<V>::splat(1.0f)}; }
// h + u (x - h) = x + p (h - x).  (p h + u x would round p, the same way at every step: a state that lives for a million steps
// would drift by 3 %.  Over the 16 steps of a span that is 2^-21, and spans are joined by over.)
template <int V> __device__ __forceinline__ Ch<V> step(Ch<V> c, Ch<V> h, Ch<V> x) { return fma(c, sub(h, x), pick(c, h, x)); }
// A span of steps acts on a state as h -> p h + A; its gate is written by c too: h - u h or p h.
template <int V> __device__ __forceinline__ Ch<V> over(Ch<V> c, Ch<V> a, Ch<V> h) { return add(fma(c, h, pick(c, h, Ch<V>::splat(0.0f))), a); }
template <int V> __device__ __forceinline__ Ch<V> both(Ch<V> c, Ch<V> d) {
    Gate<V> g = Gate<V>::from(c);
    g.grow(Gate<V>::from(d));
    return g.small();
}
constexpr float kKeeps = -0.0f;  // the gate of no steps

template <int V> __device__ __forceinline__ Ch<V> get(const float* row, int c, int D, float none = 0.0f) {
    if constexpr (V == 1) return {c < D ? row[c] : none};
    else return {make_float2(c < D ? row[c] : none, c + 1 < D ? row[c + 1] : none)};
}
__device__ __forceinline__ void put(float* row, int c, int D, Ch<1> v) {
    if (c < D) row[c] = v.a;
}
__device__ __forceinline__ void put(float* row, int c, int D, Ch<2> v) {
    if (c < D) row[c] = v.a.x;
    if (c + 1 < D) row[c + 1] = v.a.y;
}
struct Params {
    mamba_b200_gated_scan_args a;
    int* status;
    float* sums;  // [B, segments, 2, D]: what each segment does to the state (or gradient) that enters it: its gate, and what it adds
    int tiles, segments, per_segment, tma_out, stages;
};

// ---------------------------------------------------------------------------------------------------
// Tiles of 64 steps x 32 V channels.  A warp has 16 consecutive steps of them, a lane V channels: it finds what its span does
// to a state, the four warps join their spans in order, and each walks its steps again from the state that is really there.
// Gates and inputs stay in registers between the two walks, so everything is read once; results take the place of the inputs
// in shared memory and leave by TMA, which also clips what lies outside the tensor.  Where there are few strips of channels,
// time is cut into segments: a first kernel finds what each does to a state, and a CTA starts from what the earlier ones leave.
// ---------------------------------------------------------------------------------------------------
constexpr int kFwdWarps = 4, kBwdWarps = 4;
constexpr int kFwdCtas = 3, kFwdStages = 3;
// The gradient writes over its inputs, so a stage is asked for again only when its results have been read: with two CTAs or one on an
// SM two stages leave the memory idle meanwhile, and three are used.  us with two and three: 135 strips x 49 tiles 106 and 89, 144 x 64
// 136 and 116, 168 x 64 165 and 157, 192 x 32 87 and 82, 288 x 32 99 and 96; but three CTAs with two stages are 384 x 32 121, two with
// three 158.
constexpr int kFewStages = 3;
static bool few_ctas(int sms, long long ctas) { return 2 * ctas <= 3ll * sms; }

template <typename T, int V, int NIN, bool BWD>
struct Layout {
    static constexpr int CH = 32 * V, kStages = BWD ? 2 : kFwdStages, kWarps = BWD ? kBwdWarps : kFwdWarps, L = kTile / kWarps;
    static constexpr uint32_t kIn = kTile * CH * sizeof(T);  // one input's tile
    // backward: the warps' three sums (the forward's two lie in the place of f, which is done with) | barriers | stages of inputs
    static constexpr uint32_t oBar = BWD ? 3 * kWarps * CH * sizeof(float) : 0, oIn = oBar + 128;
    static constexpr uint32_t bytes(int stages) { return oIn + stages * NIN * kIn + 128; }
    static_assert((BWD ? 3 : kFwdCtas) * (bytes(kStages) + 1024) <= 228 * 1024, "CTAs on an SM");
    static_assert(!BWD || 2 * (bytes(kFewStages) + 1024) <= 228 * 1024, "two CTAs on an SM");
    static_assert(L * CH * sizeof(T) >= 2 * CH * sizeof(float), "two sums in a warp's rows of f");
};

template <typename T, int V, int NIN, bool BWD, bool PLAIN>
struct Tiles {
    using Lay = Layout<T, V, NIN, BWD>;
    const Params& p;
    unsigned char* sm;
    uint64_t* bars;
    int b, c0, warp, lane;
    bool alive;
    static constexpr int L = Lay::L;

    __device__ __forceinline__ T* at(int s, int i) const { return reinterpret_cast<T*>(sm + Lay::oIn + (s * NIN + i) * Lay::kIn); }
    // The warp's first row, this lane's first channel.
    __device__ __forceinline__ T* mine(int s, int i) const { return at(s, i) + warp * L * Lay::CH + lane * V; }
    // Asks for tile k in stage s, once what was written from that stage has been read.
    __device__ __forceinline__ void ask(int s, int k, const CUtensorMap* const* map) {
        if (threadIdx.x != 0) return;
        if (p.tma_out) tma_wait_read0();
        if (PLAIN) return;
        mbar_expect_tx(&bars[s], NIN * Lay::kIn);
#pragma unroll
        for (int i = 0; i < NIN; ++i) tma_load_3d(at(s, i), map[i], &bars[s], c0, k * kTile, b);
    }
    // The warp's rows of tile k are in stage s from here on; steps behind the end have gates that change nothing.
    __device__ __forceinline__ void wait(int s, int k, uint32_t parity) {
        alive = alive && mbar_wait(&bars[s], parity, p.status);
        for (int j = max(0, p.a.T - k * kTile - warp * L); j < L; ++j) Ch<V>::splat(INFINITY).store(mine(s, 0) + j * Lay::CH);
    }
    // Rows that TMA cannot describe: a lane fetches its own channels of the warp's rows, a tile ahead, and hands them over in shared
    // memory.  (Fetched when they were needed, a tile took 4 us.)
    struct __align__(sizeof(T) * V) Word { T v[V]; };
    __device__ __forceinline__ void fetch(Word (*to)[L], int k, const void* const* src, const long long* ld) const {
        const int c = c0 + lane * V, t0 = k * kTile + warp * L;
        const bool inside = c0 + Lay::CH <= p.a.D && t0 + L <= p.a.T;
#pragma unroll
        for (int i = 0; i < NIN; ++i) {
            const T* row = static_cast<const T*>(src[i]) + (static_cast<long long>(b) * p.a.T + t0) * ld[i] + c;
            if (inside) {
#pragma unroll
                for (int j = 0; j < L; ++j) to[i][j] = *reinterpret_cast<const Word*>(row + j * ld[i]);
            } else {
#pragma unroll
                for (int j = 0; j < L; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) to[i][j].v[e] = t0 + j < p.a.T && c + e < p.a.D ? row[j * ld[i] + e] : from_f<T>(i == 0 ? INFINITY : 0.0f);
            }
        }
    }
    __device__ __forceinline__ void hand_over(const Word (*from)[L], int s) {
#pragma unroll
        for (int i = 0; i < NIN; ++i)
#pragma unroll
            for (int j = 0; j < L; ++j) *reinterpret_cast<Word*>(mine(s, i) + j * Lay::CH) = from[i][j];
    }
    // Writes input i's place in stage s to a tensor, row by row, where TMA cannot.
    __device__ __forceinline__ void plain_out(int s, int i, int k, void* dst, long long ld) const {
        const T* from = mine(s, i);
        const int t0 = k * kTile + warp * L, c = c0 + lane * V, n = p.a.T - t0;
        T* to = static_cast<T*>(dst) + (static_cast<long long>(b) * p.a.T + t0) * ld + c;
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (j < n && c + e < p.a.D) to[j * ld + e] = from[j * Lay::CH + e];
    }
};

// What enters a segment: the state (or gradient) that enters the call, of which the first kernel kept a copy in the place of the
// sums that nobody needs (`copy`; the call may write its result over the original), through segments from, from + step, ...
// before `to`, which the warps share.
template <int V, int kWarps>
__device__ __forceinline__ Ch<V> enter(const Params& p, float* part, int b, int c, int copy, int from, int to, int step) {
    using C = Ch<V>;
    constexpr int CH = 32 * V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = (to - from) * step, per = (n + kWarps - 1) / kWarps;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    C N = C::splat(kKeeps), A = C::splat(0.0f);
    for (int i0 = warp * per; i0 < min(n, (warp + 1) * per); i0 += 8) {
        C m[8], a[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool ok = i0 + i < min(n, (warp + 1) * per);
            const float* row = p.sums + (static_cast<long long>(b) * p.segments + (ok ? from + (i0 + i) * step : 0)) * 2 * p.a.D;
            m[i] = get<V>(row, ok ? c : p.a.D, p.a.D, kKeeps);
            a[i] = get<V>(row + p.a.D, ok ? c : p.a.D, p.a.D);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            A = over(m[i], a[i], A);
            N = both(N, m[i]);
        }
    }
    N.store(part + warp * CH + lane * V);
    A.store(part + (kWarps + warp) * CH + lane * V);
    C v = get<V>(p.sums + (static_cast<long long>(b) * p.segments + copy) * 2 * p.a.D, c, p.a.D);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v = over(C::load(part + w * CH + lane * V), C::load(part + (kWarps + w) * CH + lane * V), v);
    fence_proxy_async();  // (a tile may come here)
    __syncthreads();
    return v;
}

template <typename T, int V, bool GATE, bool PLAIN>
__global__ void __launch_bounds__(kFwdWarps * 32, kFwdCtas)
    gated_scan_fwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx,
                          const __grid_constant__ CUtensorMap mz, const __grid_constant__ CUtensorMap my, const __grid_constant__ Params p) {
    constexpr int NIN = GATE ? 3 : 2;
    using Lay = Layout<T, V, NIN, false>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH, S = Lay::kStages, W = Lay::kWarps, L = Lay::L;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seg = static_cast<int>(blockIdx.x) % p.segments;
    const int strip = static_cast<int>(blockIdx.x) / p.segments, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c0 = (strip - b * per_b) * CH, c = c0 + lane * V, D = p.a.D;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
        fence_barrier_init();
    }
    __syncthreads();
    using In = Tiles<T, V, NIN, false, PLAIN>;
    In in{p, sm, bars, b, c0, warp, lane, true};
    const CUtensorMap* maps[3] = {&mf, &mx, &mz};
    const void* src[3] = {p.a.f, p.a.x, p.a.z};
    const long long ld[3] = {p.a.ld_f, p.a.ld_x, p.a.ld_z};
    const int first = seg * p.per_segment, rounds = min(p.per_segment, p.tiles - first);
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (i < rounds) in.ask(i, first + i, maps);
    typename In::Word next_rows[PLAIN ? NIN : 1][L];
    if (PLAIN && rounds > 0) in.fetch(next_rows, first, src, ld);
    C carry = C::splat(0.0f);
    if (p.segments > 1) carry = enter<V, W>(p, reinterpret_cast<float*>(in.at(S - 1, 0)), b, c, p.segments - 1, 0, seg, 1);
    else if (p.a.h0) carry = get<V>(p.a.h0 + static_cast<long long>(b) * D, c, D);
    int s = 0;
    uint32_t parity = 0;
    for (int it = 0; it < rounds; ++it) {
        const int k = first + it;
        // what each step keeps and adds, the output gates, and what the span does to the state that enters it
        C kept[L], added[L], q[GATE ? L : 1], A = C::splat(0.0f);
        Gate<V> span = no_steps<V>();
        if constexpr (PLAIN) {
            in.hand_over(next_rows, s);
            if (it + 1 < rounds) in.fetch(next_rows, k + 1, src, ld);
        } else {
            in.wait(s, k, parity);
        }
        const T *sf = in.mine(s, 0), *sx = in.mine(s, 1), *sz = in.mine(s, NIN - 1);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const Gate<V> g = Gate<V>::of(C::load(sf + j * CH));
            kept[j] = g.p;
            added[j] = mul(g.u, C::load(sx + j * CH));
            A = fma(g.p, A, added[j]);
            span.grow(g);
            if constexpr (GATE) {
                const C z = C::load(sz + j * CH);
                q[j] = mul(z, sigmoid(z));  // SiLU(z)
            }
        }
        // the sums go where the warp's rows of f were: two rows of 4-byte channels
        float* part = reinterpret_cast<float*>(in.at(s, 0));
        constexpr int kStep = L * CH * sizeof(T) / sizeof(float);
        __syncwarp();
        span.small().store(part + warp * kStep + lane * V);
        A.store(part + warp * kStep + CH + lane * V);
        __syncthreads();
        C h = carry;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w == warp) carry = h;  // (what enters this warp's span)
            h = over(C::load(part + w * kStep + lane * V), C::load(part + w * kStep + CH + lane * V), h);
        }
        if (p.a.chunk_states && warp == 0) put(p.a.chunk_states + (static_cast<long long>(b) * p.tiles + k) * D, c, D, carry);
        T* sy = in.mine(s, 1);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            carry = fma(kept[j], carry, added[j]);
            if constexpr (GATE) mul(carry, q[j]).store(sy + j * CH);
            else carry.store(sy + j * CH);
        }
        carry = h;
        fence_proxy_async();
        if (!p.tma_out) in.plain_out(s, 1, k, p.a.y, p.a.ld_y);
        __syncthreads();
        // the stage of the tile before: what was written from it has long been read
        if (it + S - 1 < rounds) in.ask(s == 0 ? S - 1 : s - 1, k + S - 1, maps);
        if (p.tma_out && threadIdx.x == 0) {
            tma_store_3d(&my, in.at(s, 1), c0, k * kTile, b);
            tma_commit();
        }
        if (++s == S) s = 0, parity ^= 1;
    }
    if (p.a.h_last && seg == p.segments - 1 && warp == 0) put(p.a.h_last + static_cast<long long>(b) * D, c, D, carry);
    if (p.tma_out && threadIdx.x == 0) tma_wait_read0();
}

// The gradient walks the tiles from the last to the first.  The states inside a tile come from the saved one that enters it, by
// the same two walks; g is joined over the warps the same way in the other direction: over a span of steps (1 - u) g at its first
// step = P g_behind + G, with the forward's P.
template <typename T, int V, bool GATE, bool PLAIN>
__global__ void __launch_bounds__(kBwdWarps * 32, 3)
    gated_scan_bwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap me,
                          const __grid_constant__ CUtensorMap mz, const __grid_constant__ CUtensorMap mdf, const __grid_constant__ CUtensorMap mdx,
                          const __grid_constant__ CUtensorMap mdz, const __grid_constant__ Params p) {
    constexpr int NIN = GATE ? 4 : 3;
    using Lay = Layout<T, V, NIN, true>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH, W = Lay::kWarps, L = Lay::L;
    const int S = p.stages;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    float* part = reinterpret_cast<float*>(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seg = static_cast<int>(blockIdx.x) % p.segments;
    const int strip = static_cast<int>(blockIdx.x) / p.segments, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c0 = (strip - b * per_b) * CH, c = c0 + lane * V, D = p.a.D;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(&bars[i], 1);
        fence_barrier_init();
    }
    __syncthreads();
    using In = Tiles<T, V, NIN, true, PLAIN>;
    In in{p, sm, bars, b, c0, warp, lane, true};
    const CUtensorMap* maps[4] = {&mf, &mx, &me, &mz};
    const void* src[4] = {p.a.f, p.a.x, p.a.dy, p.a.z};
    const long long ld[4] = {p.a.ld_f, p.a.ld_x, p.a.ld_dy, p.a.ld_z};
    const int first = min((seg + 1) * p.per_segment, p.tiles) - 1, rounds = first + 1 - seg * p.per_segment;
    const C one = C::splat(1.0f), minus = C::splat(-1.0f);
    for (int i = 0; i < min(S - 1, rounds); ++i) in.ask(i, first - i, maps);
    typename In::Word next_rows[PLAIN ? NIN : 1][L];
    if (PLAIN && rounds > 0) in.fetch(next_rows, first, src, ld);
    C carry = C::splat(0.0f);
    if (p.segments > 1) carry = enter<V, W>(p, part, b, c, 0, p.segments - 1, seg, -1);
    else if (p.a.d_last) carry = get<V>(p.a.d_last + static_cast<long long>(b) * D, c, D);
    const float* states = p.a.chunk_states + static_cast<long long>(b) * p.tiles * D;
    auto state = [&](int k) { return k >= 0 ? get<V>(states + static_cast<long long>(k) * D, c, D) : C::splat(0.0f); };
    C next = state(first);
    int s = 0;
    uint32_t parity = 0;
    for (int it = 0; it < rounds; ++it) {
        const int k = first - it;
        C h = next;
        next = state(k - 1);
        C n[L], x[L], e[L], q[L], A = C::splat(0.0f), G = C::splat(0.0f);
        Gate<V> span = no_steps<V>();
        if constexpr (PLAIN) {
            in.hand_over(next_rows, s);
            if (it + 1 < rounds) in.fetch(next_rows, k - 1, src, ld);
        } else {
            in.wait(s, k, parity);
        }
        const T *sf = in.mine(s, 0), *sx = in.mine(s, 1), *se = in.mine(s, 2), *sz = in.mine(s, NIN - 1);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const C f = C::load(sf + j * CH);
            const Gate<V> gate = Gate<V>::of(f);
            n[j] = pick(f, gate.p, mul(gate.u, minus));
            x[j] = C::load(sx + j * CH);
            e[j] = C::load(se + j * CH);
            if constexpr (GATE) {
                const C z = C::load(sz + j * CH), m = sigmoid(z), dm = mul(e[j], m);
                q[j] = mul(dm, fma(z, fma(m, minus, one), one));  // dy SiLU'(z) = dy sigmoid (1 + z (1 - sigmoid))
                e[j] = mul(dm, z);                                // dy SiLU(z)
            }
            A = fma(gate.p, A, mul(gate.u, x[j]));
            span.grow(gate);
            G = fma(span.p, e[j], G);
        }
        span.small().store(part + warp * CH + lane * V);
        A.store(part + (W + warp) * CH + lane * V);
        G.store(part + (2 * W + warp) * CH + lane * V);
        __syncthreads();
        if (it + S - 1 < rounds) in.ask(s == 0 ? S - 1 : s - 1, k - (S - 1), maps);
        C g = carry, start = carry;
#pragma unroll
        for (int w = 0; w < W - 1; ++w)
            if (w < warp) h = over(C::load(part + w * CH + lane * V), C::load(part + (W + w) * CH + lane * V), h);
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            if (w == warp) start = g;
            g = over(C::load(part + w * CH + lane * V), C::load(part + (2 * W + w) * CH + lane * V), g);
        }
        carry = g;
        T *df = in.mine(s, 0), *dx = in.mine(s, 1), *dz = in.mine(s, NIN - 1);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const C to = pick(n[j], h, x[j]);
            x[j] = sub(h, x[j]);  // h_{t-1} - x_t
            h = fma(n[j], x[j], to);
            if constexpr (GATE) mul(q[j], h).store(dz + j * CH);
        }
        g = start;
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            const Gate<V> gate = Gate<V>::from(n[j]);
            g = add(g, e[j]);
            mul(gate.u, g).store(dx + j * CH);
            g = mul(gate.p, g);
            mul(x[j], mul(gate.u, g)).store(df + j * CH);
        }
        fence_proxy_async();
        if (!p.tma_out) {
            in.plain_out(s, 0, k, p.a.d_f, p.a.ld_df);
            in.plain_out(s, 1, k, p.a.d_x, p.a.ld_dx);
            if constexpr (GATE) in.plain_out(s, 3, k, p.a.d_z, p.a.ld_dz);
        }
        __syncthreads();
        if (p.tma_out && threadIdx.x == 0) {
            tma_store_3d(&mdf, in.at(s, 0), c0, k * kTile, b);
            tma_store_3d(&mdx, in.at(s, 1), c0, k * kTile, b);
            if constexpr (GATE) tma_store_3d(&mdz, in.at(s, 3), c0, k * kTile, b);
            tma_commit();
        }
        if (++s == S) s = 0, parity ^= 1;
    }
    if (p.a.d_h0 && seg == 0 && warp == 0) put(p.a.d_h0 + static_cast<long long>(b) * D, c, D, carry);
    if (p.tma_out && threadIdx.x == 0) tma_wait_read0();
}

// What each segment of time does to a state (forward) or to the gradient that comes from behind it, without results: f and x
// (dy and z) are read once more than the floor.  A warp has an eighth of the segment, 16 steps at a time, all their loads in
// flight; it ends where the kernel above begins, so that what it read last is still in L2 then.
constexpr int kSumWarps = 8;  // (4: 62.0 us for one sequence of 32749 x 768, 8: 57.9, 16: 65.4)
template <typename T, int V, bool GATE, bool BWD>
__global__ void __launch_bounds__(kSumWarps * 32) gated_scan_sums_kernel(const __grid_constant__ Params p) {
    using C = Ch<V>;
    constexpr int CH = 32 * V, kWarps = kSumWarps, L = 16, M = kTile / L;
    __shared__ __align__(8) float part[2 * kWarps * CH];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = p.segments - 1;
    const int seg = static_cast<int>(blockIdx.x) % parts + (BWD ? 1 : 0), strip = static_cast<int>(blockIdx.x) / parts;
    const int D = p.a.D, per_b = (D + CH - 1) / CH, b = strip / per_b, c = (strip - b * per_b) * CH + lane * V;
    const int first = seg * p.per_segment * M, n = min(p.per_segment, p.tiles - seg * p.per_segment) * M, per = (n + kWarps - 1) / kWarps;
    const int lo = first + min(n, warp * per), hi = first + min(n, (warp + 1) * per);  // pieces of L steps
    const bool inside = (strip - b * per_b + 1) * CH <= D;
    struct __align__(sizeof(T) * V) Word { T v[V]; };
    // L steps from t0; behind the end, and beside the last channel, `none`.
    auto fetch = [&](Word* to, const void* src, long long ld, int t0, float none) {
        const T* row = static_cast<const T*>(src) + (static_cast<long long>(b) * p.a.T + t0) * ld + c;
        if (inside && t0 + L <= p.a.T) {
#pragma unroll
            for (int j = 0; j < L; ++j) to[j] = *reinterpret_cast<const Word*>(row + j * ld);
        } else {
#pragma unroll
            for (int j = 0; j < L; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) to[j].v[e] = t0 + j < p.a.T && c + e < D ? row[j * ld + e] : from_f<T>(none);
        }
    };
    C N = C::splat(kKeeps), A = C::splat(0.0f);
    for (int i = 0; i < hi - lo; ++i) {
        const int t0 = (BWD ? lo + i : hi - 1 - i) * L;
        Word fw[L], xw[L], zw[L];
        fetch(fw, p.a.f, p.a.ld_f, t0, INFINITY);
        fetch(xw, BWD ? p.a.dy : p.a.x, BWD ? p.a.ld_dy : p.a.ld_x, t0, 0.0f);
        if constexpr (BWD && GATE) fetch(zw, p.a.z, p.a.ld_z, t0, 0.0f);
        C a1 = C::splat(0.0f);
        Gate<V> span = no_steps<V>();
#pragma unroll
        for (int jj = 0; jj < L; ++jj) {
            const int j = BWD ? L - 1 - jj : jj;
            const Gate<V> gate = Gate<V>::of(C::load(fw[j].v));
            C x = C::load(xw[j].v);
            if constexpr (BWD) {
                if constexpr (GATE) {
                    const C z = C::load(zw[j].v);
                    x = mul(x, mul(z, sigmoid(z)));
                }
                a1 = mul(gate.p, add(x, a1));
            } else {
                a1 = fma(gate.p, a1, mul(gate.u, x));
            }
            span.grow(gate);
        }
        A = over(N, A, a1);  // this piece is met before those that are there
        N = both(span.small(), N);
    }
    N.store(part + warp * CH + lane * V);
    A.store(part + (kWarps + warp) * CH + lane * V);
    __syncthreads();
    if (warp != 0) return;
    N = C::splat(kKeeps), A = C::splat(0.0f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const int w = BWD ? kWarps - 1 - i : i;
        const C m = C::load(part + w * CH + lane * V);
        A = over(m, C::load(part + (kWarps + w) * CH + lane * V), A);
        N = both(N, m);
    }
    // From here on the other kernel's CTAs may start; they wait for this one's end before they read the sums.  (Let in at the
    // beginning they could take the room of CTAs that are still to come; 48 strips, 9 segments 58.6 us then, 59.5 like this, 59.8 without.)
    asm volatile("griddepcontrol.launch_dependents;");
    float* row = p.sums + (static_cast<long long>(b) * p.segments + seg) * 2 * D;
    put(row, c, D, N);
    put(row + D, c, D, A);
    if (seg == (BWD ? 1 : 0)) {
        const float* from = BWD ? p.a.d_last : p.a.h0;
        const C v = from ? get<V>(from + static_cast<long long>(b) * D, c, D) : C::splat(0.0f);
        put(p.sums + (static_cast<long long>(b) * p.segments + (BWD ? 0 : p.segments - 1)) * 2 * D, c, D, v);
    }
}

// Windows of a few steps (decoding: one): a thread has one channel and walks it, its loads in flight together.
constexpr int kShort = 8;
template <typename T>
__global__ void __launch_bounds__(128) gated_scan_short_kernel(const mamba_b200_gated_scan_args p) {
    const long long i = blockIdx.x * 128ll + threadIdx.x;
    if (i >= static_cast<long long>(p.B) * p.D) return;
    const long long b = i / p.D;
    const int d = static_cast<int>(i - b * p.D);
    const T *x = static_cast<const T*>(p.x) + b * p.T * p.ld_x + d, *f = static_cast<const T*>(p.f) + b * p.T * p.ld_f + d;
    const T* z = p.z ? static_cast<const T*>(p.z) + b * p.T * p.ld_z + d : nullptr;
    T* y = static_cast<T*>(p.y) + b * p.T * p.ld_y + d;
    float h = p.h0 ? p.h0[i] : 0.0f, xv[kShort], fv[kShort], zv[kShort];
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.T) break;
        xv[t] = to_f(x[t * p.ld_x]);
        fv[t] = to_f(f[t * p.ld_f]);
        zv[t] = z ? to_f(z[t * p.ld_z]) : 0.0f;
    }
    if (p.chunk_states && p.T) p.chunk_states[i] = h;
#pragma unroll
    for (int t = 0; t < kShort; ++t) {
        if (t >= p.T) break;
        h = step(Gate<1>::of({fv[t]}).small(), {h}, {xv[t]}).a;
        y[t * p.ld_y] = from_f<T>(z ? h * siluf_fast(zv[t]) : h);
    }
    if (p.h_last) p.h_last[i] = h;
}

static int check(Ctx* c, const mamba_b200_gated_scan_args* a, bool bwd) {
    const char* fn = bwd ? "gated_scan_bwd" : "gated_scan_fwd";
    if (!dtype_ok(a->dtype)) return fail(c, MAMBA_B200_ERR_ARG, "%s: bad dtype %d", fn, a->dtype);
    if (a->B < 0 || a->T < 0 || a->D <= 0) return fail(c, MAMBA_B200_ERR_ARG, "%s: bad dims", fn);
    if (a->T > kMaxSize || a->D > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: too many steps or channels", fn);
    if (a->ld_x < a->D || a->ld_f < a->D || (a->z && a->ld_z < a->D)) return fail(c, MAMBA_B200_ERR_ARG, "%s: row stride below D", fn);
    if (a->B == 0) return MAMBA_B200_OK;
    const size_t n = dtype_size(a->dtype);
    const bool aligned = aligned_to(n, {a->x, a->f, a->z}) && aligned_to(4, {a->chunk_states}) &&
                         (bwd ? aligned_to(n, {a->dy, a->d_x, a->d_f, a->d_z}) && aligned_to(4, {a->d_last, a->d_h0})
                              : aligned_to(n, {a->y}) && aligned_to(4, {a->h0, a->h_last}));
    if (!aligned) return fail(c, MAMBA_B200_ERR_ARG, "%s: misaligned pointer", fn);
    if (a->T && (!a->x || !a->f)) return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", fn);
    if (!bwd) {
        if (a->ld_y < a->D) return fail(c, MAMBA_B200_ERR_ARG, "%s: row stride below D", fn);
        if (a->T && !a->y) return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", fn);
    } else {
        if (a->ld_dy < a->D || a->ld_dx < a->D || a->ld_df < a->D || (a->z && a->ld_dz < a->D))
            return fail(c, MAMBA_B200_ERR_ARG, "%s: row stride below D", fn);
        if (a->T && (!a->dy || !a->d_x || !a->d_f || !a->chunk_states || (a->z && !a->d_z)))
            return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", fn);
    }
    return MAMBA_B200_OK;
}


// Segments of time, so that every SM has its three CTAs.  Cut, f and x (dy and z) are read twice; whole, a CTA's tiles follow one
// another at 1.1 us (backward 1.8).  Below 3/4 of a strip an SM there is room for four segments or more.  us, whole and cut: 168 strips
// x 64 tiles 96 and 103 (backward 157 and 167), 120 x 64 70 and 75 (116 and 118), 112 x 64 71 and 80 (117 and 137), 108 x 64 70 and 62
// (116 and 111), 96 x 64 70 and 57 (116 and 92), 72 x 64 69 and 46 (116 and 81), 12 x 128 132 and 21 (224 and 32); 12 x 4 5.9 and 5.9.
constexpr int kMaxSegments = 128;
static int pick_segments(int sms, long long strips, int tiles) {
    if (strips * 4 > 3ll * sms || tiles <= 4) return 1;
    const long long want = 3ll * sms / (strips > 0 ? strips : 1);
    const int most = static_cast<int>(want < kMaxSegments ? want : kMaxSegments);
    return most < tiles ? most : tiles;
}

template <typename T, int V, bool GATE, bool BWD, bool PLAIN>
static const void* kernel() {
    if constexpr (BWD) return reinterpret_cast<const void*>(gated_scan_bwd_kernel<T, V, GATE, PLAIN>);
    else return reinterpret_cast<const void*>(gated_scan_fwd_kernel<T, V, GATE, PLAIN>);
}

template <typename T, int V, bool GATE, bool BWD, bool PLAIN>
static int launch_tiled(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    using Lay = Layout<T, V, (GATE ? 3 : 2) + (BWD ? 1 : 0), BWD>;
    Params p{a, c->d_status};
    const long long strips = static_cast<long long>(a.B) * ((a.D + Lay::CH - 1) / Lay::CH);
    if (strips > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "gated_scan: too many channels");
    p.tiles = (a.T + kTile - 1) / kTile;
    int segments = pick_segments(c->sm_count, strips, p.tiles);
    if (reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) return fail(c, MAMBA_B200_ERR_ARG, "gated_scan: the workspace is 16-byte aligned");
    const long long row = static_cast<long long>(a.B) * a.D * 2 * sizeof(float);  // a segment's sums
    if (!a.workspace || a.workspace_bytes < 0) segments = 1;
    else if (segments * row > a.workspace_bytes) segments = a.workspace_bytes / row > 1 ? static_cast<int>(a.workspace_bytes / row) : 1;
    p.per_segment = (p.tiles + segments - 1) / segments;
    p.segments = p.tiles ? (p.tiles + p.per_segment - 1) / p.per_segment : 1;
    p.sums = static_cast<float*>(a.workspace);
    CUtensorMap mf{}, mx{}, me{}, mz{}, o0{}, o1{}, o2{};
    auto map = [&](CUtensorMap* m, const void* base, long long ld) { return make_tmap_3d(c, m, a.dtype, base, ld, a.D, a.T, a.B, Lay::CH, kTile); };
    const void* fn = kernel<T, V, GATE, BWD, PLAIN>();
    if (!PLAIN && !(map(&mf, a.f, a.ld_f) && map(&mx, a.x, a.ld_x) && (!BWD || map(&me, a.dy, a.ld_dy)) && (!GATE || map(&mz, a.z, a.ld_z))))
        return fail(c, MAMBA_B200_ERR_CUDA, "gated_scan: a tensor map was refused");
    p.tma_out = BWD ? map(&o0, a.d_f, a.ld_df) && map(&o1, a.d_x, a.ld_dx) && (!GATE || map(&o2, a.d_z, a.ld_dz)) : map(&o0, a.y, a.ld_y);
    void* fwd_args[] = {&mf, &mx, &mz, &o0, &p};
    void* bwd_args[] = {&mf, &mx, &me, &mz, &o0, &o1, &o2, &p};
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    const long long ctas = strips * p.segments;
    p.stages = BWD && few_ctas(c->sm_count, ctas) ? kFewStages : Lay::kStages;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(Lay::kWarps * 32);
    cfg.dynamicSmemBytes = Lay::bytes(p.stages);
    cfg.stream = st;
    cudaLaunchAttribute early;
    memset(&early, 0, sizeof(early));
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    if (p.segments > 1) {  // the second kernel asks for its first tiles while the first one ends
        gated_scan_sums_kernel<T, V, GATE, BWD><<<static_cast<unsigned>(strips * (p.segments - 1)), kSumWarps * 32, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        cfg.attrs = &early;
        cfg.numAttrs = 1;
    }
    MB200_CUDA_CHECK(c, cudaLaunchKernelExC(&cfg, fn, BWD ? bwd_args : fwd_args));
    return MAMBA_B200_OK;
}

template <typename T, int V, bool GATE, bool BWD, bool PLAIN>
static int configure(Ctx* c) {
    using Lay = Layout<T, V, (GATE ? 3 : 2) + (BWD ? 1 : 0), BWD>;
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(kernel<T, V, GATE, BWD, PLAIN>(), cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::bytes(BWD ? kFewStages : Lay::kStages)));
    return MAMBA_B200_OK;
}

// A lane has two channels in 16 bits and one in f32: rows of 128 bytes, brought by TMA.  Rows that it cannot describe (odd channel
// counts or starts) take one channel a lane: 16 x 2048 x 769 and x 770 are 109 us, the gradient 232.  Two of their 2-byte columns a lane
// were slower, 140 and 414.
template <bool GATE, bool BWD>
static int launch_typed(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    const int cols = a.dtype == MAMBA_B200_F32 ? 32 : 64;
    auto fits = [&](const void* q, long long ld) { return tmap_3d_fits(c, a.dtype, q, ld, a.D, a.T, cols, kTile); };
    const bool tma = a.T > 0 && fits(a.f, a.ld_f) && fits(a.x, a.ld_x) && (!BWD || fits(a.dy, a.ld_dy)) && (!GATE || fits(a.z, a.ld_z));
    if (a.dtype == MAMBA_B200_F32) return tma ? launch_tiled<float, 1, GATE, BWD, false>(c, a, st) : launch_tiled<float, 1, GATE, BWD, true>(c, a, st);
    if (a.dtype == MAMBA_B200_F16) return tma ? launch_tiled<__half, 2, GATE, BWD, false>(c, a, st) : launch_tiled<__half, 1, GATE, BWD, true>(c, a, st);
    return tma ? launch_tiled<__nv_bfloat16, 2, GATE, BWD, false>(c, a, st) : launch_tiled<__nv_bfloat16, 1, GATE, BWD, true>(c, a, st);
}

}  // namespace gs

int gated_scan_configure(Ctx* c) {
    int rc = MAMBA_B200_OK;
#define MB200_GS(T, V, PLAIN)                                             \
    if (!rc) rc = gs::configure<T, V, true, true, PLAIN>(c);              \
    if (!rc) rc = gs::configure<T, V, false, true, PLAIN>(c);             \
    if (!rc) rc = gs::configure<T, V, true, false, PLAIN>(c);             \
    if (!rc) rc = gs::configure<T, V, false, false, PLAIN>(c);
    MB200_GS(float, 1, false) MB200_GS(float, 1, true) MB200_GS(__half, 2, false) MB200_GS(__half, 1, true)
    MB200_GS(__nv_bfloat16, 2, false) MB200_GS(__nv_bfloat16, 1, true)
#undef MB200_GS
    return rc;
}

}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API long long mamba_b200_gated_scan_workspace_bytes(int B, int T, int D) {
    if (B <= 0 || T <= gs::kShort || D <= 0 || T > kMaxSize || D > kMaxSize) return 0;
    // (strips of 64 channels, or of 32: the more segments of the two; sized for 148 SMs, and a launch that would take more takes what fits)
    const int segments = gs::pick_segments(148, static_cast<long long>(B) * ((D + 63) / 64), (T + gs::kTile - 1) / gs::kTile);
    return segments > 1 ? static_cast<long long>(segments) * B * D * 2 * sizeof(float) : 0;
}

extern "C" MAMBA_B200_API int mamba_b200_gated_scan_fwd(void* handle, void* stream, const mamba_b200_gated_scan_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gs::check(c, args, false);
    if (rc || args->B == 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (args->T > gs::kShort) return args->z ? gs::launch_typed<true, false>(c, *args, st) : gs::launch_typed<false, false>(c, *args, st);
    const long long blocks = (static_cast<long long>(args->B) * args->D + 127) / 128;
    if (blocks > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "gated_scan_fwd: too many channels");
    const unsigned grid = static_cast<unsigned>(blocks);
    if (args->dtype == MAMBA_B200_F32) gs::gated_scan_short_kernel<float><<<grid, 128, 0, st>>>(*args);
    else if (args->dtype == MAMBA_B200_F16) gs::gated_scan_short_kernel<__half><<<grid, 128, 0, st>>>(*args);
    else gs::gated_scan_short_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(*args);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

extern "C" MAMBA_B200_API int mamba_b200_gated_scan_bwd(void* handle, void* stream, const mamba_b200_gated_scan_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gs::check(c, args, true);
    if (rc || args->B == 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return args->z ? gs::launch_typed<true, true>(c, *args, st) : gs::launch_typed<false, true>(c, *args, st);
}
