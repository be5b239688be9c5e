// Gated linear recurrence, elementwise over channels:
//   u_t = sigmoid(-f_t)      h_t = h_{t-1} + u_t (x_t - h_{t-1})      y_t = h_t * SiLU(z_t)
// that is h_t = a_t h_{t-1} + (1 - a_t) x_t with the forget gate a = sigmoid(f) = 1 - u.  Written with u, a channel that
// forgets slowly (u near 0) keeps u's relative precision; a rounded to 1 - 2^-24 would not.
//   backward  g_t = dy_t SiLU(z_t) + (1 - u_{t+1}) g_{t+1}
//             d_x = u g      d_f = g (h_{t-1} - x) u (1 - u)      d_z = dy h SiLU'(z)
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

// -1 / (1 + 2^(v k)): with k = log2 e the negative of u = sigmoid(-v), with -log2 e that of sigmoid(v).  The negative, because
// everything it meets is then one packed fma: h - u (h - x) = fma(-u, h - x, h).
template <int V> __device__ __forceinline__ Ch<V> neg_gate(Ch<V> v, float k) {
    const Ch<V> t = mul(v, Ch<V>::splat(k)).map(ex2), m = Ch<V>::splat(-1.0f);
    return fma(t, m, m).map(rcp);
}
// A span of steps acts on a state as h -> h - U h + A.  span(h) with n = -U:
template <int V> __device__ __forceinline__ Ch<V> over(Ch<V> n, Ch<V> a, Ch<V> h) { return add(fma(n, h, h), a); }
// n of a span and one that follows it.
template <int V> __device__ __forceinline__ Ch<V> both(Ch<V> n, Ch<V> m) { return fma(m, add(Ch<V>::splat(1.0f), n), n); }

template <int V> __device__ __forceinline__ Ch<V> get(const float* row, int c, int D) {
    if constexpr (V == 1) return {c < D ? row[c] : 0.0f};
    else return {make_float2(c < D ? row[c] : 0.0f, c + 1 < D ? row[c + 1] : 0.0f)};
}
__device__ __forceinline__ void put(float* row, int c, int D, Ch<1> v) {
    if (c < D) row[c] = v.a;
}
__device__ __forceinline__ void put(float* row, int c, int D, Ch<2> v) {
    if (c < D) row[c] = v.a.x;
    if (c + 1 < D) row[c + 1] = v.a.y;
}
template <int V> __device__ __forceinline__ Ch<V> ld_remote(uint32_t at) {
    if constexpr (V == 1) {
        return {ld_cluster1(at)};
    } else {
        float2 v;
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
        return {v};
    }
}

struct Params {
    mamba_b200_gated_scan_args a;
    int* status;
    int tiles, ranks, tma_in, tma_out;
};

// ---------------------------------------------------------------------------------------------------
// Tiles of 64 steps x 32 V channels.  A warp has 16 consecutive steps of them, a lane V channels: it finds what its span does
// to a state, the four warps join their spans in order, and each walks its steps again from the state that is really there.
// Gates and inputs stay in registers between the two walks, so everything is read once; results take the place of the inputs
// in shared memory and leave by TMA, which also clips what lies outside the tensor.  Where there are few strips of channels,
// the CTAs of a cluster take consecutive tiles of one strip and join their spans through distributed shared memory.
// ---------------------------------------------------------------------------------------------------
constexpr int kWarps = 4, L = kTile / kWarps;

template <typename T, int V, int NIN>
struct Layout {
    static constexpr int CH = 32 * V;
    static constexpr uint32_t kIn = kTile * CH * sizeof(T);  // one input's tile
    // two stages of inputs | the warps' sums (three each, the forward uses two) | barriers | (clusters) two buffers of the CTA's
    // two sums
    static constexpr uint32_t oPart = 2 * NIN * kIn, oBar = oPart + 3 * kWarps * CH * sizeof(float), oTot = oBar + 16;
    static constexpr uint32_t kBytes = oTot + 128;
    static constexpr uint32_t kMore = 4 * CH * sizeof(float);
};

template <typename T, int V, int NIN>
struct Tiles {
    using Lay = Layout<T, V, NIN>;
    const Params& p;
    unsigned char* sm;
    uint64_t* bars;
    int b, c0, warp, lane;
    bool alive;

    __device__ __forceinline__ bool exists(int k) const { return k >= 0 && k < p.tiles; }
    __device__ __forceinline__ T* at(int s, int i) const { return reinterpret_cast<T*>(sm + (s * NIN + i) * Lay::kIn); }
    // The warp's first row, this lane's first channel.
    __device__ __forceinline__ T* mine(int s, int i) const { return at(s, i) + warp * L * Lay::CH + lane * V; }
    // Asks for tile k in stage s, once what was written from that stage has been read.
    __device__ __forceinline__ void ask(int s, int k, const CUtensorMap* const* map) {
        if (threadIdx.x != 0 || !exists(k)) return;
        if (p.tma_out) tma_wait_read0();
        if (!p.tma_in) return;
        mbar_expect_tx(&bars[s], NIN * Lay::kIn);
#pragma unroll
        for (int i = 0; i < NIN; ++i) tma_load_3d(sm + (s * NIN + i) * Lay::kIn, map[i], &bars[s], c0, k * kTile, b);
    }
    // The warp's rows of tile k are in stage s from here on; steps behind the end have gates that change nothing.
    __device__ __forceinline__ void wait(int s, int k, uint32_t parity, const void* const* src, const long long* ld) {
        if (p.tma_in) {
            alive = alive && mbar_wait(&bars[s], parity, p.status);
        } else {
#pragma unroll 1
            for (int i = 0; i < NIN; ++i)
                plain_channels<Lay::CH>(at(s, i) + warp * L * Lay::CH, static_cast<const T*>(src[i]), ld[i],
                                        static_cast<long long>(b) * p.a.T, k * kTile + warp * L, L, p.a.T, c0, p.a.D, lane);
            __syncwarp();
        }
        for (int j = max(0, p.a.T - k * kTile - warp * L); j < L; ++j) Ch<V>::splat(INFINITY).store(mine(s, 0) + j * Lay::CH);
    }
    // Writes input i's place in stage s to a tensor, row by row, where TMA cannot.
    __device__ __forceinline__ void plain_out(int s, int i, int k, void* dst, long long ld) const {
        const T* from = at(s, i) + warp * L * Lay::CH;
        const int t0 = k * kTile + warp * L;
        for (int j = 0; j < L && t0 + j < p.a.T; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = e * 32 + lane;
                if (c0 + c < p.a.D) static_cast<T*>(dst)[(static_cast<long long>(b) * p.a.T + t0 + j) * ld + c0 + c] = from[j * Lay::CH + c];
            }
    }
};

// The CTA's two sums, joined over the cluster: what was there before this CTA's tile, and behind the last one's.
template <int V>
__device__ __forceinline__ Ch<V> join_cluster(float* tot, int it, int rank, int R, int lane, Ch<V>& carry) {
    constexpr int CH = 32 * V;
    Ch<V> h = carry;
    const uint32_t base = smem_u32(tot + (it & 1) * (2 * CH) + lane * V);
    for (int r = 0; r < R; ++r) {
        const uint32_t far = cluster_addr(base, r);
        const Ch<V> n = ld_remote<V>(far), a = ld_remote<V>(far + CH * 4);
        if (r == rank) h = carry;
        carry = over(n, a, carry);
    }
    return h;
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(kWarps * 32, 3)
    gated_scan_fwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx,
                          const __grid_constant__ CUtensorMap mz, const __grid_constant__ CUtensorMap my, const __grid_constant__ Params p) {
    constexpr int NIN = GATE ? 3 : 2;
    using Lay = Layout<T, V, NIN>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    float *part = reinterpret_cast<float*>(sm + Lay::oPart), *tot = reinterpret_cast<float*>(sm + Lay::oTot);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = p.ranks, rank = R == 1 ? 0 : static_cast<int>(blockIdx.x) % R;
    const int strip = static_cast<int>(blockIdx.x) / R, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c0 = (strip - b * per_b) * CH, c = c0 + lane * V, D = p.a.D;
    if (threadIdx.x == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        fence_barrier_init();
    }
    __syncthreads();
    Tiles<T, V, NIN> in{p, sm, bars, b, c0, warp, lane, true};
    const CUtensorMap* maps[3] = {&mf, &mx, &mz};
    const void* src[3] = {p.a.f, p.a.x, p.a.z};
    const long long ld[3] = {p.a.ld_f, p.a.ld_x, p.a.ld_z};
    in.ask(0, rank, maps);
    C carry = p.a.h0 ? get<V>(p.a.h0 + static_cast<long long>(b) * D, c, D) : C::splat(0.0f);
    const int rounds = (p.tiles + R - 1) / R;
    for (int it = 0; it < rounds; ++it) {
        const int k = it * R + rank, s = it & 1;
        const bool here = in.exists(k);
        C n[L], x[L], N = C::splat(0.0f), A = C::splat(0.0f);
        if (here) {
            in.wait(s, k, (it >> 1) & 1, src, ld);
            const T *sf = in.mine(s, 0), *sx = in.mine(s, 1);
#pragma unroll
            for (int j = 0; j < L; ++j) {
                n[j] = neg_gate(C::load(sf + j * CH), kLog2e);
                x[j] = C::load(sx + j * CH);
                A = fma(n[j], sub(A, x[j]), A);
                N = both(N, n[j]);
            }
        }
        N.store(part + warp * CH + lane * V);
        A.store(part + (kWarps + warp) * CH + lane * V);
        __syncthreads();
        in.ask(s ^ 1, k + R, maps);
        C h = carry, start = carry;
        if (R > 1) {
            if (warp == 0) {
                N = C::splat(0.0f), A = C::splat(0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const C m = C::load(part + w * CH + lane * V);
                    A = over(m, C::load(part + (kWarps + w) * CH + lane * V), A);
                    N = both(N, m);
                }
                N.store(tot + (it & 1) * (2 * CH) + lane * V);
                A.store(tot + (it & 1) * (2 * CH) + CH + lane * V);
            }
            cluster_sync();
            h = join_cluster<V>(tot, it, rank, R, lane, carry);
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) start = h;
            h = over(C::load(part + w * CH + lane * V), C::load(part + (kWarps + w) * CH + lane * V), h);
        }
        if (R == 1) carry = h;
        if (here) {
            if (p.a.chunk_states && warp == 0) put(p.a.chunk_states + (static_cast<long long>(b) * p.tiles + k) * D, c, D, start);
            h = start;
            T* sy = in.mine(s, 1);
            const T* sz = in.mine(s, NIN - 1);
#pragma unroll
            for (int j = 0; j < L; ++j) {
                h = fma(n[j], sub(h, x[j]), h);
                if constexpr (GATE) {
                    const C z = C::load(sz + j * CH);
                    mul(mul(h, z), mul(neg_gate(z, -kLog2e), C::splat(-1.0f))).store(sy + j * CH);
                } else {
                    h.store(sy + j * CH);
                }
            }
            fence_proxy_async();
            if (!p.tma_out) {
                __syncwarp();
                in.plain_out(s, 1, k, p.a.y, p.a.ld_y);
            }
        }
        __syncthreads();
        if (p.tma_out && threadIdx.x == 0 && here) {
            tma_store_3d(&my, in.at(s, 1), c0, k * kTile, b);
            tma_commit();
        }
    }
    if (p.a.h_last && rank == 0 && warp == 0) put(p.a.h_last + static_cast<long long>(b) * D, c, D, carry);
    if (p.tma_out && threadIdx.x == 0) tma_wait_read0();
    if (R > 1) cluster_sync();  // the others may still read this CTA's sums
}

// The gradient walks the tiles from the last to the first.  The states inside a tile come from the saved one that enters it, by
// the same two walks; g is joined over the warps (and the cluster) the same way in the other direction: over a span of steps
// (1 - u) g at its first step = g_behind - U g_behind + G, with the forward's U.  g runs with its sign turned, like the gates.
template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(kWarps * 32, 3)
    gated_scan_bwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap me,
                          const __grid_constant__ CUtensorMap mz, const __grid_constant__ CUtensorMap mdf, const __grid_constant__ CUtensorMap mdx,
                          const __grid_constant__ CUtensorMap mdz, const __grid_constant__ Params p) {
    constexpr int NIN = GATE ? 4 : 3;
    using Lay = Layout<T, V, NIN>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    float *part = reinterpret_cast<float*>(sm + Lay::oPart), *tot = reinterpret_cast<float*>(sm + Lay::oTot);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = p.ranks, rank = R == 1 ? 0 : static_cast<int>(blockIdx.x) % R;
    const int strip = static_cast<int>(blockIdx.x) / R, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c0 = (strip - b * per_b) * CH, c = c0 + lane * V, D = p.a.D;
    if (threadIdx.x == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        fence_barrier_init();
    }
    __syncthreads();
    Tiles<T, V, NIN> in{p, sm, bars, b, c0, warp, lane, true};
    const CUtensorMap* maps[4] = {&mf, &mx, &me, &mz};
    const void* src[4] = {p.a.f, p.a.x, p.a.dy, p.a.z};
    const long long ld[4] = {p.a.ld_f, p.a.ld_x, p.a.ld_dy, p.a.ld_z};
    const int last = p.tiles - 1 - rank;
    const C minus = C::splat(-1.0f);
    in.ask(0, last, maps);
    C carry = p.a.d_last ? mul(get<V>(p.a.d_last + static_cast<long long>(b) * D, c, D), minus) : C::splat(0.0f);
    const float* states = p.a.chunk_states + static_cast<long long>(b) * p.tiles * D;
    auto state = [&](int k) { return k >= 0 ? get<V>(states + static_cast<long long>(k) * D, c, D) : C::splat(0.0f); };
    C next = state(last);
    const int rounds = (p.tiles + R - 1) / R;
    for (int it = 0; it < rounds; ++it) {
        const int k = last - it * R, s = it & 1;
        const bool here = k >= 0;
        C h = next;
        next = state(k - R);
        C n[L], x[L], e[L], q[L], N = C::splat(0.0f), A = C::splat(0.0f), G = C::splat(0.0f);
        if (here) {
            in.wait(s, k, (it >> 1) & 1, src, ld);
            const T *sf = in.mine(s, 0), *sx = in.mine(s, 1), *se = in.mine(s, 2), *sz = in.mine(s, NIN - 1);
#pragma unroll
            for (int j = 0; j < L; ++j) {
                n[j] = neg_gate(C::load(sf + j * CH), kLog2e);
                x[j] = C::load(sx + j * CH);
                const C dy = C::load(se + j * CH);
                if constexpr (GATE) {
                    const C z = C::load(sz + j * CH), m = neg_gate(z, -kLog2e);  // -sigmoid(z)
                    q[j] = mul(dy, mul(m, fma(z, fma(m, minus, minus), minus)));  // dy SiLU'(z) = dy sigmoid (1 + z (1 - sigmoid))
                    e[j] = mul(dy, mul(z, m));                                    // -dy SiLU(z)
                } else {
                    e[j] = mul(dy, minus);
                }
                A = fma(n[j], sub(A, x[j]), A);
                N = both(N, n[j]);
            }
#pragma unroll
            for (int j = L - 1; j >= 0; --j) {
                const C g = add(e[j], G);
                G = fma(n[j], g, g);
            }
        }
        N.store(part + warp * CH + lane * V);
        A.store(part + (kWarps + warp) * CH + lane * V);
        G.store(part + (2 * kWarps + warp) * CH + lane * V);
        __syncthreads();
        in.ask(s ^ 1, k - R, maps);
        C g = carry, start = carry;
        if (R > 1) {
            if (warp == 0) {
                N = C::splat(0.0f), G = C::splat(0.0f);
#pragma unroll
                for (int w = kWarps - 1; w >= 0; --w) {
                    const C m = C::load(part + w * CH + lane * V);
                    G = over(m, C::load(part + (2 * kWarps + w) * CH + lane * V), G);
                    N = both(N, m);
                }
                N.store(tot + (it & 1) * (2 * CH) + lane * V);
                G.store(tot + (it & 1) * (2 * CH) + CH + lane * V);
            }
            cluster_sync();
            g = join_cluster<V>(tot, it, rank, R, lane, carry);
        }
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w)
            if (w < warp) h = over(C::load(part + w * CH + lane * V), C::load(part + (kWarps + w) * CH + lane * V), h);
#pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) {
            if (w == warp) start = g;
            g = over(C::load(part + w * CH + lane * V), C::load(part + (2 * kWarps + w) * CH + lane * V), g);
        }
        if (R == 1) carry = g;
        if (here) {
            T *df = in.mine(s, 0), *dx = in.mine(s, 1), *dz = in.mine(s, NIN - 1);
#pragma unroll
            for (int j = 0; j < L; ++j) {
                x[j] = sub(h, x[j]);  // h_{t-1} - x_t
                h = fma(n[j], x[j], h);
                if constexpr (GATE) mul(q[j], h).store(dz + j * CH);
            }
            g = start;
#pragma unroll
            for (int j = L - 1; j >= 0; --j) {
                g = add(g, e[j]);
                mul(g, n[j]).store(dx + j * CH);
                g = fma(n[j], g, g);
                mul(x[j], mul(n[j], g)).store(df + j * CH);
            }
            fence_proxy_async();
            if (!p.tma_out) {
                __syncwarp();
                in.plain_out(s, 0, k, p.a.d_f, p.a.ld_df);
                in.plain_out(s, 1, k, p.a.d_x, p.a.ld_dx);
                if constexpr (GATE) in.plain_out(s, 3, k, p.a.d_z, p.a.ld_dz);
            }
        }
        __syncthreads();
        if (p.tma_out && threadIdx.x == 0 && here) {
            tma_store_3d(&mdf, in.at(s, 0), c0, k * kTile, b);
            tma_store_3d(&mdx, in.at(s, 1), c0, k * kTile, b);
            if constexpr (GATE) tma_store_3d(&mdz, in.at(s, 3), c0, k * kTile, b);
            tma_commit();
        }
    }
    if (p.a.d_h0 && rank == 0 && warp == 0) put(p.a.d_h0 + static_cast<long long>(b) * D, c, D, mul(carry, minus));
    if (p.tma_out && threadIdx.x == 0) tma_wait_read0();
    if (R > 1) cluster_sync();
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
        h = fmaf(rcp(1.0f + ex2(fv[t] * kLog2e)), xv[t] - h, h);
        y[t * p.ld_y] = from_f<T>(z ? h * siluf_fast(zv[t]) : h);
    }
    if (p.h_last) p.h_last[i] = h;
}

static int check(Ctx* c, const mamba_b200_gated_scan_args* a, bool bwd) {
    const char* fn = bwd ? "gated_scan_bwd" : "gated_scan_fwd";
    if (!dtype_ok(a->dtype)) return fail(c, MAMBA_B200_ERR_ARG, "%s: bad dtype %d", fn, a->dtype);
    if (a->B < 0 || a->T < 0 || a->D <= 0) return fail(c, MAMBA_B200_ERR_ARG, "%s: bad dims", fn);
    if (a->ld_x < a->D || a->ld_f < a->D || (a->z && a->ld_z < a->D)) return fail(c, MAMBA_B200_ERR_ARG, "%s: row stride below D", fn);
    if (a->B == 0) return MAMBA_B200_OK;
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


// How many CTAs of a cluster share a strip: as many as keep every CTA resident, up to 16, when strips are few.
static int pick_ranks(int strips, int tiles, int slots) {
    int r = 1;
    while (r < 16 && 2 * r <= tiles && strips * 2 * r <= slots) r *= 2;
    return r;
}

template <typename T, int V, bool GATE, bool BWD>
static const void* kernel() {
    if constexpr (BWD) return reinterpret_cast<const void*>(gated_scan_bwd_kernel<T, V, GATE>);
    else return reinterpret_cast<const void*>(gated_scan_fwd_kernel<T, V, GATE>);
}

template <typename T, int V, bool GATE, bool BWD>
static int launch_tiled(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    using Lay = Layout<T, V, (GATE ? 3 : 2) + (BWD ? 1 : 0)>;
    const void* fn = kernel<T, V, GATE, BWD>();
    Params p{a, c->d_status};
    const long long strips = static_cast<long long>(a.B) * ((a.D + Lay::CH - 1) / Lay::CH);
    if (strips > 2147483647ll / 16) return fail(c, MAMBA_B200_ERR_SHAPE, "gated_scan: too many channels");
    p.tiles = (a.T + kTile - 1) / kTile;
    p.ranks = pick_ranks(static_cast<int>(strips), p.tiles, c->sm_count * 3);
    CUtensorMap mf{}, mx{}, me{}, mz{}, o0{}, o1{}, o2{};
    auto map = [&](CUtensorMap* m, const void* base, long long ld) { return make_tmap_3d(c, m, a.dtype, base, ld, a.D, a.T, a.B, Lay::CH, kTile); };
    p.tma_in = map(&mf, a.f, a.ld_f) && map(&mx, a.x, a.ld_x) && (!BWD || map(&me, a.dy, a.ld_dy)) && (!GATE || map(&mz, a.z, a.ld_z));
    p.tma_out = BWD ? map(&o0, a.d_f, a.ld_df) && map(&o1, a.d_x, a.ld_dx) && (!GATE || map(&o2, a.d_z, a.ld_dz)) : map(&o0, a.y, a.ld_y);
    void* fwd_args[] = {&mf, &mx, &mz, &o0, &p};
    void* bwd_args[] = {&mf, &mx, &me, &mz, &o0, &o1, &o2, &p};
    const dim3 grid(static_cast<unsigned>(strips * p.ranks)), block(kWarps * 32);
    void** args = BWD ? bwd_args : fwd_args;
    if (p.ranks == 1) MB200_CUDA_CHECK(c, cudaLaunchKernel(fn, grid, block, args, Lay::kBytes, st));
    else MB200_CUDA_CHECK(c, launch_cluster(fn, grid, block, Lay::kBytes + Lay::kMore, st, p.ranks, args));
    return MAMBA_B200_OK;
}

template <typename T, int V, bool GATE, bool BWD>
static int configure(Ctx* c) {
    using Lay = Layout<T, V, (GATE ? 3 : 2) + (BWD ? 1 : 0)>;
    const void* fn = kernel<T, V, GATE, BWD>();
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::kBytes + Lay::kMore));
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return MAMBA_B200_OK;
}

// f32 rows of 32 channels and 16-bit rows of 64 are both 128 bytes; where 16-bit strips are few, they are halved.
template <bool GATE, bool BWD>
static int launch_typed(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    const bool few = static_cast<long long>(a.B) * ((a.D + 63) / 64) * 16 < 2 * c->sm_count;
    if (a.dtype == MAMBA_B200_F32) return launch_tiled<float, 1, GATE, BWD>(c, a, st);
    if (a.dtype == MAMBA_B200_F16) return few ? launch_tiled<__half, 1, GATE, BWD>(c, a, st) : launch_tiled<__half, 2, GATE, BWD>(c, a, st);
    return few ? launch_tiled<__nv_bfloat16, 1, GATE, BWD>(c, a, st) : launch_tiled<__nv_bfloat16, 2, GATE, BWD>(c, a, st);
}

}  // namespace gs

int gated_scan_configure(Ctx* c) {
    int rc = MAMBA_B200_OK;
#define MB200_GS(T, V)                                                    \
    if (!rc) rc = gs::configure<T, V, true, true>(c);                  \
    if (!rc) rc = gs::configure<T, V, false, true>(c);                 \
    if (!rc) rc = gs::configure<T, V, true, false>(c);                 \
    if (!rc) rc = gs::configure<T, V, false, false>(c);
    MB200_GS(float, 1) MB200_GS(__half, 1) MB200_GS(__half, 2) MB200_GS(__nv_bfloat16, 1) MB200_GS(__nv_bfloat16, 2)
#undef MB200_GS
    return rc;
}

}  // namespace mb200

using namespace mb200;

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
