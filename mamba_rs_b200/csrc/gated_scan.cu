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

__device__ __forceinline__ float gate_u(float f) { return rcp(1.0f + ex2(f * kLog2e)); }

// One or two neighbouring channels of a lane.
template <int V> struct Ch;
template <> struct Ch<1> {
    float a;
    __device__ __forceinline__ static Ch splat(float v) { return {v}; }
    template <typename T> __device__ __forceinline__ static Ch load(const T* p) { return {to_f(*p)}; }
    template <typename F> __device__ __forceinline__ Ch map(F f) const { return {f(a)}; }
};
template <> struct Ch<2> {
    float2 a;
    __device__ __forceinline__ static Ch splat(float v) { return {splat2(v)}; }
    template <typename T> __device__ __forceinline__ static Ch load(const T* p) { return {ld_pair(p)}; }
    template <typename F> __device__ __forceinline__ Ch map(F f) const { return {make_float2(f(a.x), f(a.y))}; }
};
__device__ __forceinline__ Ch<1> fma(Ch<1> a, Ch<1> b, Ch<1> c) { return {fmaf(a.a, b.a, c.a)}; }
__device__ __forceinline__ Ch<2> fma(Ch<2> a, Ch<2> b, Ch<2> c) { return {fma2(a.a, b.a, c.a)}; }
__device__ __forceinline__ Ch<1> mul(Ch<1> a, Ch<1> b) { return {a.a * b.a}; }
__device__ __forceinline__ Ch<2> mul(Ch<2> a, Ch<2> b) { return {mul2(a.a, b.a)}; }
__device__ __forceinline__ Ch<1> add(Ch<1> a, Ch<1> b) { return {a.a + b.a}; }
__device__ __forceinline__ Ch<2> add(Ch<2> a, Ch<2> b) { return {add2(a.a, b.a)}; }
__device__ __forceinline__ Ch<1> sub(Ch<1> a, Ch<1> b) { return {a.a - b.a}; }
__device__ __forceinline__ Ch<2> sub(Ch<2> a, Ch<2> b) { return {add2(a.a, make_float2(-b.a.x, -b.a.y))}; }
// v - u v in one rounding: the state that is left after a span that replaced the share u.
template <int V> __device__ __forceinline__ Ch<V> left(Ch<V> u, Ch<V> v) { return fma(u, v.map([](float x) { return -x; }), v); }

// Writes a lane's channels c, c + 1 < D of a row; pairs only where the rows allow.
template <typename T> __device__ __forceinline__ void put(T* row, int c, int D, bool, Ch<1> v) {
    if (c < D) row[c] = from_f<T>(v.a);
}
template <typename T> __device__ __forceinline__ void put(T* row, int c, int D, bool pairs, Ch<2> v) {
    if (pairs && c + 1 < D) {
        st_pair(row + c, v.a);
    } else {
        if (c < D) row[c] = from_f<T>(v.a.x);
        if (c + 1 < D) row[c + 1] = from_f<T>(v.a.y);
    }
}
__device__ __forceinline__ Ch<1> get(const float* row, int c, int D, Ch<1>*) { return {c < D ? row[c] : 0.0f}; }
__device__ __forceinline__ Ch<2> get(const float* row, int c, int D, Ch<2>*) {
    return {make_float2(c < D ? row[c] : 0.0f, c + 1 < D ? row[c + 1] : 0.0f)};
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
    int strips, tiles, ranks, tma, pairs;
};

// ---------------------------------------------------------------------------------------------------
// Tiles of 64 steps x 32 V channels.  A warp has L = 64 / W consecutive steps of them, a lane V channels.  A span of steps
// acts on the state that enters it as h -> h - U h + C: a warp finds its span's U and C from zero, the CTA's warps join them
// in order, and each walks its steps again from the state that is really there.  The gates stay in registers between the two
// walks, the inputs in shared memory, so everything is read once.  Where there are few strips of channels, the CTAs of a
// cluster take consecutive tiles of one strip and join their spans through distributed shared memory.
// ---------------------------------------------------------------------------------------------------
template <typename T, int V, int W, int NIN>
struct Layout {
    static constexpr int CH = 32 * V, L = kTile / W, kStages = 3;
    static constexpr uint32_t kIn = kTile * CH * sizeof(T);  // one input's tile
    // inputs | the warps' sums (backward: three each) | two buffers of the CTA's two sums | barriers
    static constexpr uint32_t oPart = kStages * NIN * kIn, oTot = oPart + 3 * W * CH * sizeof(float);
    static constexpr uint32_t oBar = oTot + 4 * CH * sizeof(float);
    static constexpr uint32_t kBytes = oBar + kStages * 8 + 128;
};

template <typename T, int V, int NIN, typename Lay>
struct Feed {
    const CUtensorMap* map[NIN];
    const T* src[NIN];
    long long ld[NIN];
    unsigned char* sm;
    uint64_t* bars;
    const Params& p;
    int b, c0;
    bool alive;

    // Stage s is to hold tile k.
    __device__ __forceinline__ void ask(int s, int k) {
        if (!p.tma || threadIdx.x != 0 || k < 0 || k >= p.tiles) return;
        mbar_expect_tx(&bars[s], NIN * Lay::kIn);
#pragma unroll
        for (int i = 0; i < NIN; ++i) tma_load_3d(sm + (s * NIN + i) * Lay::kIn, map[i], &bars[s], c0, k * kTile, b);
    }
    // The warp's rows of tile k are in stage s from here on.
    __device__ __forceinline__ void wait(int s, int k, uint32_t parity, int warp, int lane) {
        if (k < 0 || k >= p.tiles) return;
        if (p.tma) {
            alive = alive && mbar_wait(&bars[s], parity, p.status);
        } else {
#pragma unroll
            for (int i = 0; i < NIN; ++i)
                plain_channels<Lay::CH>(at(s, i) + warp * Lay::L * Lay::CH, src[i], ld[i], static_cast<long long>(b) * p.a.T,
                                        k * kTile + warp * Lay::L, Lay::L, p.a.T, c0, p.a.D, lane);
            __syncwarp();
        }
    }
    __device__ __forceinline__ T* at(int s, int i) { return reinterpret_cast<T*>(sm + (s * NIN + i) * Lay::kIn); }
};

template <typename T, int V, int W, bool GATE>
__global__ void __launch_bounds__(W * 32) gated_scan_fwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx,
                                                                const __grid_constant__ CUtensorMap mz, const Params p) {
    constexpr int NIN = GATE ? 3 : 2;
    using Lay = Layout<T, V, W, NIN>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH, L = Lay::L, S = Lay::kStages;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    float *part = reinterpret_cast<float*>(sm + Lay::oPart), *tot = reinterpret_cast<float*>(sm + Lay::oTot);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = p.ranks, rank = R == 1 ? 0 : static_cast<int>(blockIdx.x) % R;
    const int strip = static_cast<int>(blockIdx.x) / R, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c = (strip - b * per_b) * CH + lane * V, D = p.a.D, Tn = p.a.T;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&bars[s], 1);
        fence_barrier_init();
    }
    __syncthreads();
    Feed<T, V, NIN, Lay> in{{&mf, &mx}, {static_cast<const T*>(p.a.f), static_cast<const T*>(p.a.x)}, {p.a.ld_f, p.a.ld_x}, sm, bars, p,
                            b, c - lane * V, true};
    if constexpr (GATE) {
        in.map[2] = &mz;
        in.src[2] = static_cast<const T*>(p.a.z);
        in.ld[2] = p.a.ld_z;
    }
#pragma unroll
    for (int s = 0; s < S - 1; ++s) in.ask(s, s * R + rank);
    C carry = p.a.h0 ? get(p.a.h0 + static_cast<long long>(b) * D, c, D, static_cast<C*>(nullptr)) : C::splat(0.0f);
    const int rounds = (p.tiles + R - 1) / R;
    const C one = C::splat(1.0f);
    int s = 0;
    uint32_t parity = 0;
    for (int it = 0; it < rounds; ++it) {
        const int k = it * R + rank, t0 = k * kTile + warp * L;
        in.ask(s == 0 ? S - 1 : s - 1, k + (S - 1) * R);
        in.wait(s, k, parity, warp, lane);
        const T *sf = in.at(s, 0) + warp * L * CH + lane * V, *sx = in.at(s, 1) + warp * L * CH + lane * V;
        C u[L], U = C::splat(0.0f), A = C::splat(0.0f);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const bool ok = t0 + j < Tn;
            u[j] = C::load(sf + j * CH).map([ok](float f) { return ok ? gate_u(f) : 0.0f; });
            const C x = C::load(sx + j * CH).map([ok](float f) { return ok ? f : 0.0f; });
            A = fma(u[j], sub(x, A), A);
            U = fma(u[j], sub(one, U), U);
        }
        float* mine = part;
        *reinterpret_cast<C*>(mine + warp * CH + lane * V) = U;
        *reinterpret_cast<C*>(mine + (W + warp) * CH + lane * V) = A;
        __syncthreads();
        C h = carry, start = carry;
        if (R > 1) {
            float* own = tot + (it & 1) * (2 * CH);
            if (warp == 0) {
                U = C::splat(0.0f), A = C::splat(0.0f);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const C u2 = C::load(mine + w * CH + lane * V);
                    A = add(left(u2, A), C::load(mine + (W + w) * CH + lane * V));
                    U = fma(u2, sub(one, U), U);
                }
                *reinterpret_cast<C*>(own + lane * V) = U;
                *reinterpret_cast<C*>(own + CH + lane * V) = A;
            }
            cluster_sync();
            const uint32_t base = smem_u32(own + lane * V);
            for (int r = 0; r < R; ++r) {
                const uint32_t far = cluster_addr(base, r);
                const C u2 = ld_remote<V>(far), a2 = ld_remote<V>(far + CH * 4);
                if (r == rank) h = carry;
                carry = add(left(u2, carry), a2);
            }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w == warp) start = h;
            h = add(left(C::load(mine + w * CH + lane * V), h), C::load(mine + (W + w) * CH + lane * V));
        }
        if (R == 1) carry = h;
        if (p.a.chunk_states && warp == 0 && k < p.tiles) {
            float* row = p.a.chunk_states + (static_cast<long long>(b) * p.tiles + k) * D;
            put(row, c, D, false, start);
        }
        h = start;
        T* y = static_cast<T*>(p.a.y) + (static_cast<long long>(b) * Tn + t0) * p.a.ld_y;
        const T* sz = GATE ? in.at(s, NIN - 1) + warp * L * CH + lane * V : nullptr;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            h = fma(u[j], sub(C::load(sx + j * CH), h), h);
            C o = h;
            if constexpr (GATE) o = mul(h, C::load(sz + j * CH).map(siluf_fast));
            if (t0 + j < Tn) put(y, c, D, p.pairs, o);
            y += p.a.ld_y;
        }
        __syncthreads();  // the stage may be filled again
        if (++s == S) s = 0, parity ^= 1;
    }
    if (p.a.h_last && rank == 0 && warp == 0) put(p.a.h_last + static_cast<long long>(b) * D, c, D, false, carry);
    if (R > 1) cluster_sync();  // the others may still read this CTA's sums
}

// The gradient walks the tiles from the last to the first.  The states inside a tile come from the saved one that enters it, by
// the same two walks; g is joined over the warps (and the cluster) the same way in the other direction: over a span,
// (1 - u) g at its first step = g_behind - U g_behind + G with the forward's U.
template <typename T, int V, int W, bool GATE>
__global__ void __launch_bounds__(W * 32, V == 2 ? 2 : 3)
    gated_scan_bwd_kernel(const __grid_constant__ CUtensorMap mf, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap me,
                          const __grid_constant__ CUtensorMap mz, const Params p) {
    constexpr int NIN = GATE ? 4 : 3;
    using Lay = Layout<T, V, W, NIN>;
    using C = Ch<V>;
    constexpr int CH = Lay::CH, L = Lay::L, S = Lay::kStages;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    float *part = reinterpret_cast<float*>(sm + Lay::oPart), *tot = reinterpret_cast<float*>(sm + Lay::oTot);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::oBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = p.ranks, rank = R == 1 ? 0 : static_cast<int>(blockIdx.x) % R;
    const int strip = static_cast<int>(blockIdx.x) / R, per_b = (p.a.D + CH - 1) / CH, b = strip / per_b;
    const int c = (strip - b * per_b) * CH + lane * V, D = p.a.D, Tn = p.a.T;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) mbar_init(&bars[s], 1);
        fence_barrier_init();
    }
    __syncthreads();
    Feed<T, V, NIN, Lay> in{{&mf, &mx, &me},
                            {static_cast<const T*>(p.a.f), static_cast<const T*>(p.a.x), static_cast<const T*>(p.a.dy)},
                            {p.a.ld_f, p.a.ld_x, p.a.ld_dy}, sm, bars, p, b, c - lane * V, true};
    if constexpr (GATE) {
        in.map[3] = &mz;
        in.src[3] = static_cast<const T*>(p.a.z);
        in.ld[3] = p.a.ld_z;
    }
    const int last = p.tiles - 1 - rank;
#pragma unroll
    for (int s = 0; s < S - 1; ++s) in.ask(s, last - s * R);
    C carry = p.a.d_last ? get(p.a.d_last + static_cast<long long>(b) * D, c, D, static_cast<C*>(nullptr)) : C::splat(0.0f);
    const float* states = p.a.chunk_states + static_cast<long long>(b) * p.tiles * D;
    auto state = [&](int k) { return k >= 0 ? get(states + static_cast<long long>(k) * D, c, D, static_cast<C*>(nullptr)) : C::splat(0.0f); };
    C next = state(last);
    const int rounds = (p.tiles + R - 1) / R;
    const C one = C::splat(1.0f);
    int s = 0;
    uint32_t parity = 0;
    for (int it = 0; it < rounds; ++it) {
        const int k = last - it * R, t0 = k * kTile + warp * L;
        in.ask(s == 0 ? S - 1 : s - 1, k - (S - 1) * R);
        C h = next;
        next = state(k - R);
        in.wait(s, k, parity, warp, lane);
        const int row = warp * L * CH + lane * V;
        const T *sf = in.at(s, 0) + row, *sx = in.at(s, 1) + row, *se = in.at(s, 2) + row, *sz = in.at(s, NIN - 1) + row;
        C u[L], e[L], q[L], U = C::splat(0.0f), A = C::splat(0.0f), G = C::splat(0.0f);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const bool ok = k >= 0 && t0 + j < Tn;
            auto in_range = [ok](float f) { return ok ? f : 0.0f; };
            u[j] = C::load(sf + j * CH).map([ok](float f) { return ok ? gate_u(f) : 0.0f; });
            const C x = C::load(sx + j * CH).map(in_range);
            e[j] = C::load(se + j * CH).map(in_range);
            if constexpr (GATE) {
                const C z = C::load(sz + j * CH).map(in_range), g = z.map(sigmoidf_fast), zg = mul(z, g);
                q[j] = mul(e[j], fma(zg, sub(one, g), g));  // dy SiLU'(z)
                e[j] = mul(e[j], zg);
            }
            A = fma(u[j], sub(x, A), A);
            U = fma(u[j], sub(one, U), U);
        }
#pragma unroll
        for (int j = L - 1; j >= 0; --j) G = left(u[j], add(e[j], G));
        float* mine = part;
        *reinterpret_cast<C*>(mine + warp * CH + lane * V) = U;
        *reinterpret_cast<C*>(mine + (W + warp) * CH + lane * V) = A;
        *reinterpret_cast<C*>(mine + (2 * W + warp) * CH + lane * V) = G;
        __syncthreads();
        C g = carry, start = carry;
        if (R > 1) {
            float* own = tot + (it & 1) * (2 * CH);
            if (warp == 0) {
                U = C::splat(0.0f), G = C::splat(0.0f);
#pragma unroll
                for (int w = W - 1; w >= 0; --w) {
                    const C u2 = C::load(mine + w * CH + lane * V);
                    G = add(left(u2, G), C::load(mine + (2 * W + w) * CH + lane * V));
                    U = fma(u2, sub(one, U), U);
                }
                *reinterpret_cast<C*>(own + lane * V) = U;
                *reinterpret_cast<C*>(own + CH + lane * V) = G;
            }
            cluster_sync();
            const uint32_t base = smem_u32(own + lane * V);
            for (int r = 0; r < R; ++r) {
                const uint32_t far = cluster_addr(base, r);
                const C u2 = ld_remote<V>(far), g2 = ld_remote<V>(far + CH * 4);
                if (r == rank) g = carry;
                carry = add(left(u2, carry), g2);
            }
        }
#pragma unroll
        for (int w = 0; w < W - 1; ++w)
            if (w < warp) h = add(left(C::load(mine + w * CH + lane * V), h), C::load(mine + (W + w) * CH + lane * V));
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            if (w == warp) start = g;
            g = add(left(C::load(mine + w * CH + lane * V), g), C::load(mine + (2 * W + w) * CH + lane * V));
        }
        if (R == 1) carry = g;
        const long long r0 = static_cast<long long>(b) * Tn + t0;
        C span[L];  // x_t - h_{t-1}
        T* dz = GATE ? static_cast<T*>(p.a.d_z) + r0 * p.a.ld_dz : nullptr;
#pragma unroll
        for (int j = 0; j < L; ++j) {
            span[j] = sub(C::load(sx + j * CH), h);
            h = fma(u[j], span[j], h);
            if constexpr (GATE) {
                if (k >= 0 && t0 + j < Tn) put(dz, c, D, p.pairs, mul(q[j], h));
                dz += p.a.ld_dz;
            }
        }
        T *dx = static_cast<T*>(p.a.d_x) + (r0 + L - 1) * p.a.ld_dx, *df = static_cast<T*>(p.a.d_f) + (r0 + L - 1) * p.a.ld_df;
        g = start;
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
            g = add(g, e[j]);
            const C gu = mul(g, u[j]), behind = left(u[j], g);
            if (k >= 0 && t0 + j < Tn) {
                put(dx, c, D, p.pairs, gu);
                put(df, c, D, p.pairs, mul(mul(span[j], u[j]), behind).map([](float v) { return -v; }));
            }
            g = behind;
            dx -= p.a.ld_dx;
            df -= p.a.ld_df;
        }
        __syncthreads();
        if (++s == S) s = 0, parity ^= 1;
    }
    if (p.a.d_h0 && rank == 0 && warp == 0) put(p.a.d_h0 + static_cast<long long>(b) * D, c, D, false, carry);
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
        h = fmaf(gate_u(fv[t]), xv[t] - h, h);
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

template <typename T, int V, int W, bool GATE, bool BWD>
static int launch_tiled(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    constexpr int NIN = (GATE ? 3 : 2) + (BWD ? 1 : 0);
    using Lay = Layout<T, V, W, NIN>;
    const void* fn;
    if constexpr (BWD) fn = reinterpret_cast<const void*>(gated_scan_bwd_kernel<T, V, W, GATE>);
    else fn = reinterpret_cast<const void*>(gated_scan_fwd_kernel<T, V, W, GATE>);
    Params p{a, c->d_status};
    const long long strips = static_cast<long long>(a.B) * ((a.D + Lay::CH - 1) / Lay::CH);
    p.tiles = (a.T + kTile - 1) / kTile;
    p.ranks = pick_ranks(static_cast<int>(strips < 1 << 20 ? strips : 1 << 20), p.tiles, c->sm_count * (BWD && V == 2 ? 2 : 3));
    if (strips > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "gated_scan: too many channels");
    p.strips = static_cast<int>(strips);
    CUtensorMap mf{}, mx{}, me{}, mz{};
    auto map = [&](CUtensorMap* m, const void* base, long long ld) { return make_tmap_3d(c, m, a.dtype, base, ld, a.D, a.T, a.B, Lay::CH, kTile); };
    p.tma = map(&mf, a.f, a.ld_f) && map(&mx, a.x, a.ld_x) && (!BWD || map(&me, a.dy, a.ld_dy)) && (!GATE || map(&mz, a.z, a.ld_z));
    auto pairs = [](const void* q, long long ld) { return reinterpret_cast<uintptr_t>(q) % (2 * sizeof(T)) == 0 && ld % 2 == 0; };
    p.pairs = BWD ? pairs(a.d_x, a.ld_dx) && pairs(a.d_f, a.ld_df) && (!GATE || pairs(a.d_z, a.ld_dz)) : pairs(a.y, a.ld_y);
    void* fwd_args[] = {&mf, &mx, &mz, &p};
    void* bwd_args[] = {&mf, &mx, &me, &mz, &p};
    const dim3 grid(static_cast<unsigned>(strips * p.ranks)), block(W * 32);
    void** args = BWD ? bwd_args : fwd_args;
    if (p.ranks == 1) MB200_CUDA_CHECK(c, cudaLaunchKernel(fn, grid, block, args, Lay::kBytes, st));
    else MB200_CUDA_CHECK(c, launch_cluster(fn, grid, block, Lay::kBytes, st, p.ranks, args));
    return MAMBA_B200_OK;
}

template <typename T, int V, int W, bool GATE, bool BWD>
static int configure(Ctx* c) {
    constexpr int NIN = (GATE ? 3 : 2) + (BWD ? 1 : 0);
    const void* fn;
    if constexpr (BWD) fn = reinterpret_cast<const void*>(gated_scan_bwd_kernel<T, V, W, GATE>);
    else fn = reinterpret_cast<const void*>(gated_scan_fwd_kernel<T, V, W, GATE>);
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T, V, W, NIN>::kBytes));
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    return MAMBA_B200_OK;
}

// f32 rows of 32 channels and 16-bit rows of 64 are both 128 bytes; where 16-bit strips are few, they are halved.
#define MB200_GS_EACH(F, ...)                                                                                        \
    switch (a.dtype) {                                                                                               \
    case MAMBA_B200_F32: return F<float, 1, 8, GATE, BWD>(__VA_ARGS__);                                              \
    case MAMBA_B200_F16: return few ? F<__half, 1, 8, GATE, BWD>(__VA_ARGS__) : F<__half, 2, 8, GATE, BWD>(__VA_ARGS__); \
    default: return few ? F<__nv_bfloat16, 1, 8, GATE, BWD>(__VA_ARGS__) : F<__nv_bfloat16, 2, 8, GATE, BWD>(__VA_ARGS__); \
    }
template <bool GATE, bool BWD>
static int launch_typed(Ctx* c, const mamba_b200_gated_scan_args& a, cudaStream_t st) {
    const bool few = static_cast<long long>(a.B) * ((a.D + 63) / 64) * 16 < 2 * c->sm_count;
    MB200_GS_EACH(launch_tiled, c, a, st)
}
#undef MB200_GS_EACH

}  // namespace gs

int gated_scan_configure(Ctx* c) {
    int rc = MAMBA_B200_OK;
#define MB200_GS(T, V)                                                    \
    if (!rc) rc = gs::configure<T, V, 8, true, true>(c);                  \
    if (!rc) rc = gs::configure<T, V, 8, false, true>(c);                 \
    if (!rc) rc = gs::configure<T, V, 8, true, false>(c);                 \
    if (!rc) rc = gs::configure<T, V, 8, false, false>(c);
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
