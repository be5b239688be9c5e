// Group norm over channels that lie last, with activation and gate, forward and backward.
//
//   v = (x - mean) * rstd * w + b,   y = act(v) * SiLU(z);   mean, var over the S rows of a sample and the channels of a group
//   dv = dy * SiLU(z) * act'(v),     d_z = dy * act(v) * SiLU'(z),     d_w = sum dv * xh,     d_b = sum dv     (xh = (x - mean) * rstd)
//   d_x = rstd * (dv * w - mean(dv * w) - xh * mean(dv * w * xh))
//
// Every element is read once or twice and written once, so HBM bounds it, with instructions close behind.  Three forms:
//  * rows: S = 1, a group fits a block.  A thread owns the same channels of row after row, the next of which are on their way to
//    shared memory; a group's sums are shuffles (and a barrier where it takes more than a warp), the variance is taken around the mean
//    from registers, and the backward's sums over rows stay in registers until the block's end.  32768 rows of 2048 channels in 32
//    groups, gated, bf16: 75 to 84 us, 75 to 84 % of the measured copy rate (where it was 79: 84 with activation and gate looked up for every
//    value, 118 without the rows on their way); backward 128 to 134, 78 to 81 %.  Calls one after another: 80 to 86 and 134 to 139.
//  * samples that fit shared memory: one kernel, every element read once.  3 samples of 1021 rows of 768 channels, f32: 13 to 14 us
//    (18.5 in two kernels), backward 31 to 33.
//  * other samples: a first kernel leaves mean and squared deviations (backward: the sums) of each block of rows and group, joined
//    pairwise around their means, and a second one joins the blocks of its groups in their order and goes over the rows again, which
//    L2 has where they fit it.  8 samples of 16384 rows of 512 channels, SiLU, bf16: 212 us, 19 % of the copy rate by the bytes of one
//    pass; backward 309.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace gn {

constexpr int kThreads = 256;
constexpr int kMaxRows = 1 << 30;  // of a sample: the end of a block of rows stays within 32 bits

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float* f) {
    const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f(v.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Vec<T, VEC>& v, float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f(v.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float* f) {
    Vec<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.v[i] = from_f<T>(f[i]);
    *reinterpret_cast<Vec<T, VEC>*>(p) = v;
}

// f32 storage keeps expf's form; 16-bit results are rounded far above the fast one's error (2^-20)
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
    if (sizeof(T) == 4) return rcp(1.0f + expf(-v));  // (expf to 1 ulp, the reciprocal too)
    return sigmoidf_fast(v);
}
// act(v), and its slope
template <typename T>
__device__ __forceinline__ float act(int kind, float v) {
    if (kind == MAMBA_B200_ACT_SILU) return v * sigmoid<T>(v);
    if (kind == MAMBA_B200_ACT_GELU) return 0.5f * v * erfcf(-v * 0.70710678118654752f);
    return v;
}
template <typename T>
__device__ __forceinline__ float act_slope(int kind, float v, float* value) {
    if (kind == MAMBA_B200_ACT_SILU) {
        const float q = sigmoid<T>(v);
        *value = v * q;
        return q * fmaf(v, 1.0f - q, 1.0f);
    }
    if (kind == MAMBA_B200_ACT_GELU) {
        const float q = 0.5f * erfcf(-v * 0.70710678118654752f);
        *value = v * q;
        return fmaf(v * 0.3989422804014327f, expf(-0.5f * v * v), q);
    }
    *value = v;
    return 1.0f;
}

struct Params {
    mamba_b200_group_norm_args a;
    int per;           // channels of a group
    // rows
    int lanes;         // of a group (a power of two)
    int vecs;          // vectors of a group
    int groups;        // of a block
    int rows;          // that a block takes at once
    int tiles;         // blocks side by side over the channels
    // samples
    int sub;           // pieces of a group's channels (1 where a group fits a block)
    int block_rows, blocks;  // rows of a block, blocks of a sample
    int side;                // samples side by side; a block takes every side-th
    float* part;       // [N][blocks * sub][G][2]: mean and squared deviations of a piece, or the backward's two sums
    float* sums;       // backward [2][parts][C]: d_w and d_b of a block
    int parts;
};

__device__ __forceinline__ float sum_lanes(float v, int lanes) {
    for (int m = lanes >> 1; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}
// 16 bytes into this thread's own place in shared memory
__device__ __forceinline__ void fetch16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// The same where a group may take several whole warps (every thread of the block calls it): `turn` alternates between two sets
// of sums, so that one barrier a sum is enough.
__device__ __forceinline__ float sum_group(float v, int lanes, float (*sums)[8], int& turn) {
    v = sum_lanes(v, lanes < 32 ? lanes : 32);
    if (lanes <= 32) return v;
    const int warp = threadIdx.x >> 5, n = lanes >> 5, first = warp / n * n;
    float* set = sums[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) set[warp] = v;
    __syncthreads();
    float s = set[first];
    for (int i = 1; i < n; ++i) s += set[first + i];
    return s;
}

// dv and d_z of a value
template <typename T>
__device__ __forceinline__ float through(int kind, float v, float dy, bool gate, float z, float* d_z) {
    float value;
    const float slope = act_slope<T>(kind, v, &value);
    float d = dy;
    if (gate) {
        const float q = sigmoid<T>(z);
        *d_z = dy * value * q * fmaf(z, 1.0f - q, 1.0f);
        d = dy * z * q;
    }
    return d * slope;
}

// The same for two values at a time, activation and gate known to the compiler (looked up for every value, they made up half of the
// instructions of a kernel that is bound by them).
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 v) {
    if constexpr (sizeof(T) == 4) {
        return make_float2(sigmoid<T>(v.x), sigmoid<T>(v.y));
    } else {
        const float2 e = mul2(v, splat2(-kLog2e)), d = add2(make_float2(ex2(e.x), ex2(e.y)), splat2(1.0f));
        return make_float2(rcp(d.x), rcp(d.y));
    }
}
template <typename T, int ACT>
__device__ __forceinline__ float2 act2(float2 v) {
    if constexpr (ACT == MAMBA_B200_ACT_NONE) return v;
    if constexpr (ACT == MAMBA_B200_ACT_SILU) return mul2(v, sigmoid2<T>(v));
    return make_float2(act<T>(ACT, v.x), act<T>(ACT, v.y));
}
// z^ = slope of z SiLU: q (1 + z (1 - q))
__device__ __forceinline__ float2 silu_slope2(float2 z, float2 q) {
    return mul2(q, fma2(z, fma2(q, splat2(-1.0f), splat2(1.0f)), splat2(1.0f)));
}
// dv of dy (and d_z, in z's place)
template <typename T, int ACT, bool GATE>
__device__ __forceinline__ float2 through2(float2 v, float2 dy, float2& z) {
    float2 value = v, slope;
    if constexpr (ACT == MAMBA_B200_ACT_SILU) {
        const float2 q = sigmoid2<T>(v);
        value = mul2(v, q);
        slope = silu_slope2(v, q);
    } else if constexpr (ACT == MAMBA_B200_ACT_GELU) {
        slope = make_float2(act_slope<T>(ACT, v.x, &value.x), act_slope<T>(ACT, v.y, &value.y));
    }
    float2 d = dy;
    if constexpr (GATE) {
        const float2 q = sigmoid2<T>(z);
        d = mul2(dy, mul2(z, q));
        z = mul2(mul2(dy, value), silu_slope2(z, q));
    }
    if constexpr (ACT != MAMBA_B200_ACT_NONE) d = mul2(d, slope);
    return d;
}
template <typename T, int VEC>
__device__ __forceinline__ void widen2(const Vec<T, VEC>& v, float2* f) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) f[i] = ld_pair(v.v + 2 * i);
}
template <typename T, int VEC>
__device__ __forceinline__ void store2(T* p, const float2* f) {
    Vec<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) st_pair(v.v + 2 * i, f[i]);
    *reinterpret_cast<Vec<T, VEC>*>(p) = v;
}

// ---------------------------------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------------------------------

// Where a thread stands: its group, and the vectors of it that it has.
template <int VEC, int VPT>
struct Seat {
    int wide, r, at, g, lane, col[VPT];
    bool mine, have[VPT];
    __device__ __forceinline__ Seat(const Params& p) {
        wide = p.groups * p.lanes;  // threads of a row
        r = threadIdx.x / wide;
        at = threadIdx.x - r * wide;
        const int g_in = at / p.lanes;
        lane = at - g_in * p.lanes;
        g = blockIdx.y * p.groups + g_in;
        mine = r < p.rows && g < p.a.G;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int k = lane + i * p.lanes;
            have[i] = mine && k < p.vecs;
            col[i] = g * p.per + k * VEC;
        }
    }
};

// A block's d_w and d_b: its rows are joined in their order, a vector of each thread at a time.
template <int VEC, int VPT>
__device__ __forceinline__ void leave_sums(const Params& p, const Seat<VEC, VPT>& t, const float* dw, const float* db, float* sm) {
    float* sw = sm;
    float* sb = sm + VEC * kThreads;
    float* out_w = p.sums + static_cast<long long>(blockIdx.x) * p.a.C;
    float* out_b = out_w + static_cast<long long>(p.parts) * p.a.C;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sw[e * kThreads + threadIdx.x] = dw[i * VEC + e];
            sb[e * kThreads + threadIdx.x] = db[i * VEC + e];
        }
        __syncthreads();
        if (t.r == 0 && t.have[i]) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float tw = 0.0f, tb = 0.0f;
                for (int k = 0; k < p.rows; ++k) {
                    tw += sw[e * kThreads + k * t.wide + t.at];
                    tb += sb[e * kThreads + k * t.wide + t.at];
                }
                out_w[t.col[i] + e] = tw;
                out_b[t.col[i] + e] = tb;
            }
        }
    }
}

// Vectors of 16 bytes.  A thread's vectors of the next rows are on their way to places of its own in shared memory (no barriers, no
// registers): HBM's latency at its rate is 35 KB an SM.
template <int VPT>
constexpr int kRowsAhead = VPT == 1 ? 4 : 2;

template <typename T, int VEC, int VPT, bool BWD, int ACT, bool GATE>
__global__ void __launch_bounds__(kThreads, VPT > 1 ? 1 : BWD ? 2 : 4) rows_kernel(const Params p) {
    constexpr int E = VEC * VPT, H = E / 2, D = kRowsAhead<VPT>, TENSORS = (BWD ? 2 : 1) + (GATE ? 1 : 0);
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float sums_sm[BWD ? 2 * VEC * kThreads : 1];
    __shared__ float warp_sums[2][8];
    int turn = 0;
    const mamba_b200_group_norm_args& a = p.a;
    const Seat<VEC, VPT> t(p);
    float2 w[H], bias[H], dw[BWD ? H : 1], db[BWD ? H : 1];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
            const int c = t.col[i] + 2 * e, k = i * VEC / 2 + e;
            w[k] = t.have[i] && a.weight ? make_float2(a.weight[c], a.weight[c + 1]) : splat2(1.0f);
            bias[k] = t.have[i] && a.bias ? make_float2(a.bias[c], a.bias[c + 1]) : splat2(0.0f);
            if (BWD) dw[k] = db[k] = splat2(0.0f);
        }
    const float inv = 1.0f / p.per;
    const long long NG = static_cast<long long>(a.N) * a.G;
    Vec<T, VEC>* own = reinterpret_cast<Vec<T, VEC>*>(ring) + threadIdx.x;
    auto in_ring = [&](int d, int tensor, int i) { return own + ((d * TENSORS + tensor) * VPT + i) * kThreads; };
    auto ask = [&](long long n, int d) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (t.have[i] && n < a.N) {
                fetch16(in_ring(d, 0, i), static_cast<const T*>(a.x) + n * a.ld_x + t.col[i]);
                if (BWD) fetch16(in_ring(d, 1, i), static_cast<const T*>(a.dy) + n * a.ld_dy + t.col[i]);
                if (GATE) fetch16(in_ring(d, TENSORS - 1, i), static_cast<const T*>(a.z) + n * a.ld_z + t.col[i]);
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const long long turn_rows = gridDim.x * static_cast<long long>(p.rows), first = blockIdx.x * static_cast<long long>(p.rows);
    float mean_next = 0.0f, rstd_next = 0.0f;
    auto ask_stats = [&](long long n) {
        if (BWD && t.mine && n < a.N) {
            mean_next = a.stats[n * a.G + t.g];
            rstd_next = a.stats[NG + n * a.G + t.g];
        }
    };
    ask_stats(first + t.r);
#pragma unroll
    for (int d = 0; d < D; ++d) ask(first + t.r + d * turn_rows, d);
    int d = 0;
    // (every thread of a warp takes every turn: the sums are shuffles)
    for (long long n0 = first; n0 < a.N; n0 += turn_rows) {
        const long long n = n0 + t.r;
        const bool on = t.mine && n < a.N;
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
        float2 x[H], z[H], dy[H];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            // (what a thread has no row for is never looked at, but for the sums)
            widen2(*in_ring(d, 0, i), x + i * VEC / 2);
            if (BWD) widen2(*in_ring(d, 1, i), dy + i * VEC / 2);
            if (GATE) widen2(*in_ring(d, TENSORS - 1, i), z + i * VEC / 2);
            if (!(on && t.have[i])) {
#pragma unroll
                for (int e = 0; e < VEC / 2; ++e) {
                    const int k = i * VEC / 2 + e;
                    x[k] = splat2(0.0f);
                    if (BWD) dy[k] = splat2(0.0f);
                    if (GATE) z[k] = splat2(0.0f);
                }
            }
        }
        const float mean_in = mean_next, rstd_in = rstd_next;
        ask_stats(n + turn_rows);
        ask(n + D * turn_rows, d);
        d = d + 1 == D ? 0 : d + 1;
        if constexpr (!BWD) {
            float2 s = x[0];
#pragma unroll
            for (int k = 1; k < H; ++k) s = add2(s, x[k]);
            const float mean = sum_group(s.x + s.y, p.lanes, warp_sums, turn) * inv;
            float2 q = splat2(0.0f);
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int e = 0; e < VEC / 2; ++e) {
                    float2& v = x[i * VEC / 2 + e];
                    v = add2(v, splat2(t.have[i] ? -mean : 0.0f));
                    q = fma2(v, v, q);
                }
            const float rstd = rsqrtf(fmaf(sum_group(q.x + q.y, p.lanes, warp_sums, turn), inv, a.eps));
            if (on && t.lane == 0 && a.stats) {
                a.stats[n * a.G + t.g] = mean;
                a.stats[NG + n * a.G + t.g] = rstd;
            }
#pragma unroll
            for (int k = 0; k < H; ++k) {
                x[k] = act2<T, ACT>(fma2(mul2(x[k], splat2(rstd)), w[k], bias[k]));
                if (GATE) x[k] = mul2(x[k], mul2(z[k], sigmoid2<T>(z[k])));
            }
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (on && t.have[i]) store2<T, VEC>(static_cast<T*>(a.y) + n * a.ld_y + t.col[i], x + i * VEC / 2);
        } else {
            // (threads without a row: x and dy are 0, and so is all they add)
            const float mean = on ? mean_in : 0.0f, rstd = on ? rstd_in : 0.0f;
            float2 s1 = splat2(0.0f), s2 = splat2(0.0f);
#pragma unroll
            for (int k = 0; k < H; ++k) {
                const float2 xh = mul2(add2(x[k], splat2(-mean)), splat2(rstd));
                const float2 dv = through2<T, ACT, GATE>(fma2(xh, w[k], bias[k]), dy[k], z[k]);
                dw[k] = fma2(dv, xh, dw[k]);
                db[k] = add2(db[k], dv);
                x[k] = xh;
                dy[k] = mul2(dv, w[k]);
                s1 = add2(s1, dy[k]);
                s2 = fma2(dy[k], xh, s2);
            }
            const float m1 = sum_group(s1.x + s1.y, p.lanes, warp_sums, turn) * inv * rstd;
            const float m2 = sum_group(s2.x + s2.y, p.lanes, warp_sums, turn) * inv * rstd;
#pragma unroll
            for (int k = 0; k < H; ++k) x[k] = fma2(x[k], splat2(-m2), fma2(dy[k], splat2(rstd), splat2(-m1)));
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (on && t.have[i]) {
                    store2<T, VEC>(static_cast<T*>(a.d_x) + n * a.ld_dx + t.col[i], x + i * VEC / 2);
                    if (GATE) store2<T, VEC>(static_cast<T*>(a.d_z) + n * a.ld_dz + t.col[i], z + i * VEC / 2);
                }
        }
    }
    if constexpr (BWD) {
        float fw[E], fb[E];
#pragma unroll
        for (int k = 0; k < H; ++k) {
            fw[2 * k] = dw[k].x; fw[2 * k + 1] = dw[k].y;
            fb[2 * k] = db[k].x; fb[2 * k + 1] = db[k].y;
        }
        leave_sums<VEC, VPT>(p, t, fw, fb, sums_sm);
    }
}

// Rows that start or end between vectors: element by element.
template <typename T, int VPT, bool BWD>
__global__ void __launch_bounds__(kThreads) odd_rows_kernel(const Params p) {
    constexpr int E = VPT;
    __shared__ float sums_sm[BWD ? 2 * kThreads : 1];
    __shared__ float warp_sums[2][8];
    int turn = 0;
    const mamba_b200_group_norm_args& a = p.a;
    const Seat<1, VPT> t(p);
    float w[E], bias[E], dw[E], db[E];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        w[i] = t.have[i] && a.weight ? a.weight[t.col[i]] : 1.0f;
        bias[i] = t.have[i] && a.bias ? a.bias[t.col[i]] : 0.0f;
        dw[i] = db[i] = 0.0f;
    }
    const float inv = 1.0f / p.per;
    const bool gate = a.z != nullptr;
    const long long NG = static_cast<long long>(a.N) * a.G;
    for (long long n0 = blockIdx.x * static_cast<long long>(p.rows); n0 < a.N; n0 += gridDim.x * static_cast<long long>(p.rows)) {
        const long long n = n0 + t.r;
        const bool on = t.mine && n < a.N;
        float x[E], z[E], dy[E];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const bool ok = on && t.have[i];
            x[i] = ok ? to_f(static_cast<const T*>(a.x)[n * a.ld_x + t.col[i]]) : 0.0f;
            z[i] = ok && gate ? to_f(static_cast<const T*>(a.z)[n * a.ld_z + t.col[i]]) : 0.0f;
            dy[i] = ok && BWD ? to_f(static_cast<const T*>(a.dy)[n * a.ld_dy + t.col[i]]) : 0.0f;
        }
        if constexpr (!BWD) {
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) s += x[i];
            const float mean = sum_group(s, p.lanes, warp_sums, turn) * inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                x[i] = t.have[i] ? x[i] - mean : 0.0f;
                q = fmaf(x[i], x[i], q);
            }
            const float rstd = 1.0f / sqrtf(sum_group(q, p.lanes, warp_sums, turn) * inv + a.eps);
            if (on && t.lane == 0 && a.stats) {
                a.stats[n * a.G + t.g] = mean;
                a.stats[NG + n * a.G + t.g] = rstd;
            }
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (on && t.have[i]) {
                    float y = act<T>(a.activation, fmaf(x[i] * rstd, w[i], bias[i]));
                    if (gate) y *= z[i] * sigmoid<T>(z[i]);
                    static_cast<T*>(a.y)[n * a.ld_y + t.col[i]] = from_f<T>(y);
                }
        } else {
            const float mean = on ? a.stats[n * a.G + t.g] : 0.0f, rstd = on ? a.stats[NG + n * a.G + t.g] : 0.0f;
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (on && t.have[i]) {
                    const float xh = (x[i] - mean) * rstd;
                    const float dv = through<T>(a.activation, fmaf(xh, w[i], bias[i]), dy[i], gate, z[i], &z[i]);
                    dw[i] = fmaf(dv, xh, dw[i]);
                    db[i] += dv;
                    x[i] = xh;
                    dy[i] = dv * w[i];
                    s1 += dy[i];
                    s2 = fmaf(dy[i], xh, s2);
                }
            s1 = sum_group(s1, p.lanes, warp_sums, turn) * inv;
            s2 = sum_group(s2, p.lanes, warp_sums, turn) * inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
                if (on && t.have[i]) {
                    static_cast<T*>(a.d_x)[n * a.ld_dx + t.col[i]] = from_f<T>(rstd * (dy[i] - s1 - x[i] * s2));
                    if (gate) static_cast<T*>(a.d_z)[n * a.ld_dz + t.col[i]] = from_f<T>(z[i]);
                }
        }
    }
    if constexpr (BWD) leave_sums<1, VPT>(p, t, dw, db, sums_sm);
}

// d_w and d_b from the blocks' sums: a warp's lanes hold 32 channels, its block's warps every eighth part, joined in order.
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ sums, int parts, int C, float* d_w, float* d_b, int accumulate) {
    __shared__ float sm[8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float* out = blockIdx.y ? d_b : d_w;
    if (!out) return;
    const float* src = sums + static_cast<long long>(blockIdx.y) * parts * C;
    float s = 0.0f;
    if (c < C)
        for (int i = k; i < parts; i += 8) s += src[static_cast<long long>(i) * C + c];
    sm[k][threadIdx.x & 31] = s;
    __syncthreads();
    if (k == 0 && c < C) {
        for (int i = 1; i < 8; ++i) s += sm[i][threadIdx.x];
        out[c] = accumulate ? out[c] + s : s;
    }
}

// ---------------------------------------------------------------------------------------------------
// samples
// ---------------------------------------------------------------------------------------------------

// What a block of the sample kernels covers: rows [rows0, rows1) of its samples, and either `groups` whole groups or the sub-th piece
// of one.  A thread has one vector of channels (col, its group gi in the block) of every rp-th row.
struct Cover {
    int rows0, rows1, rp, r, gi, g, col, first, groups, blk, sub;
    bool on;
};
template <int VEC, int NT = kThreads>
__device__ __forceinline__ Cover cover(const Params& p) {
    Cover c;
    const mamba_b200_group_norm_args& a = p.a;
    c.blk = blockIdx.x % p.blocks;
    c.rows0 = c.blk * p.block_rows;
    c.rows1 = min(a.S, c.rows0 + p.block_rows);
    const int vecs = p.vecs;  // vectors of a group
    const int wide = p.sub > 1 ? NT : p.groups * vecs;
    c.rp = NT / wide;
    c.r = threadIdx.x / wide;
    const int at = threadIdx.x - c.r * wide;
    c.sub = p.sub > 1 ? blockIdx.y % p.sub : 0;
    c.first = p.sub > 1 ? blockIdx.y / p.sub : blockIdx.y * p.groups;
    c.groups = p.sub > 1 ? 1 : min(p.groups, a.G - c.first);
    c.gi = p.sub > 1 ? 0 : at / vecs;
    const int k = p.sub > 1 ? c.sub * NT + at : at - c.gi * vecs;
    c.g = c.first + c.gi;
    c.col = c.g * p.per + k * VEC;
    c.on = c.r < c.rp && c.g < a.G && k < vecs;
    return c;
}

// mean and squared deviations of n values joined with those of m more
__device__ __forceinline__ void join(float& n, float& mean, float& dev, float m, float mean2, float dev2) {
    if (m == 0.0f) return;
    const float t = n + m, d = mean2 - mean, f = m / t;
    mean = fmaf(d, f, mean);
    dev = dev + dev2 + d * d * n * f;
    n = t;
}

// A block's threads leave their moments in shared memory, a warp for each group joins them in a fixed order.
// Joins what 32 lanes hold; all of them get the same bits.
__device__ __forceinline__ void join_lanes(float& n, float& mean, float& dev) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        const float on = __shfl_xor_sync(0xffffffffu, n, m), om = __shfl_xor_sync(0xffffffffu, mean, m), od = __shfl_xor_sync(0xffffffffu, dev, m);
        if (lane & m) {  // the lower lane's values come first in both
            float an = on, am = om, ad = od;
            join(an, am, ad, n, mean, dev);
            n = an; mean = am; dev = ad;
        } else {
            join(n, mean, dev, on, om, od);
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) moments_kernel(const Params p) {
    __shared__ float sn[kThreads], sm[kThreads], sd[kThreads];
    const mamba_b200_group_norm_args& a = p.a;
    const Cover c = cover<VEC>(p);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int vecs = p.sub > 1 ? kThreads : p.vecs, wide = p.sub > 1 ? kThreads : p.groups * p.vecs;
    for (int ns = blockIdx.x / p.blocks; ns < a.N; ns += p.side) {
        float n = 0.0f, mean = 0.0f, dev = 0.0f;
        if (c.on) {
            const T* x = static_cast<const T*>(a.x) + static_cast<long long>(ns) * a.S * a.ld_x + c.col;
            constexpr int U = 4;
            for (int s = c.rows0 + c.r; s < c.rows1; s += U * c.rp) {
                float v[U][VEC];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * c.rp < c.rows1) load<T, VEC>(x + static_cast<long long>(s + u * c.rp) * a.ld_x, v[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * c.rp < c.rows1) {
                        float m = 0.0f, d = 0.0f;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) m += v[u][e];
                        m *= 1.0f / VEC;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) d = fmaf(v[u][e] - m, v[u][e] - m, d);
                        join(n, mean, dev, VEC, m, d);
                    }
            }
        }
        __syncthreads();
        sn[threadIdx.x] = n;
        sm[threadIdx.x] = mean;
        sd[threadIdx.x] = dev;
        __syncthreads();
        for (int gi = warp; gi < c.groups; gi += kThreads / 32) {
            float tn = 0.0f, tm = 0.0f, td = 0.0f;
            for (int i = lane; i < c.rp * vecs; i += 32) {
                const int k = (i / vecs) * wide + gi * vecs + i % vecs;
                join(tn, tm, td, sn[k], sm[k], sd[k]);
            }
            join_lanes(tn, tm, td);
            if (lane == 0) {
                float* out = p.part + ((static_cast<long long>(ns) * p.blocks * p.sub + c.blk * p.sub + c.sub) * a.G + c.first + gi) * 2;
                out[0] = tm;
                out[1] = td;
            }
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) apply_kernel(const Params p) {
    __shared__ float s_mean[kThreads], s_rstd[kThreads];
    const mamba_b200_group_norm_args& a = p.a;
    const Cover c = cover<VEC>(p);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long NG = static_cast<long long>(a.N) * a.G;
    float w[VEC], bias[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        w[e] = c.on && a.weight ? a.weight[c.col + e] : 1.0f;
        bias[e] = c.on && a.bias ? a.bias[c.col + e] : 0.0f;
    }
    const bool gate = a.z != nullptr;
    for (int ns = blockIdx.x / p.blocks; ns < a.N; ns += p.side) {
        __syncthreads();
        for (int gi = warp; gi < c.groups; gi += kThreads / 32) {
            float tn = 0.0f, tm = 0.0f, td = 0.0f;
            for (int i = lane; i < p.blocks * p.sub; i += 32) {
                const int blk = i / p.sub, sub = i - blk * p.sub;
                const float* src = p.part + ((static_cast<long long>(ns) * p.blocks * p.sub + i) * a.G + c.first + gi) * 2;
                const int rows = min(a.S, (blk + 1) * p.block_rows) - blk * p.block_rows;
                const int chans = p.sub > 1 ? min(kThreads, p.vecs - sub * kThreads) * VEC : p.per;
                join(tn, tm, td, static_cast<float>(rows) * chans, src[0], src[1]);
            }
            join_lanes(tn, tm, td);
            if (lane == 0) {
                const float rstd = 1.0f / sqrtf(td / tn + a.eps);
                s_mean[gi] = tm;
                s_rstd[gi] = rstd;
                if (c.blk == 0 && c.sub == 0 && a.stats) {
                    a.stats[static_cast<long long>(ns) * a.G + c.first + gi] = tm;
                    a.stats[NG + static_cast<long long>(ns) * a.G + c.first + gi] = rstd;
                }
            }
        }
        __syncthreads();
        if (!c.on) continue;
        const float mean = s_mean[c.gi], rstd = s_rstd[c.gi];
        const long long row0 = static_cast<long long>(ns) * a.S;
        constexpr int U = 2;
        for (int s = c.rows0 + c.r; s < c.rows1; s += U * c.rp) {
            float v[U][VEC], z[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * c.rp < c.rows1) {
                    const long long row = row0 + s + u * c.rp;
                    load<T, VEC>(static_cast<const T*>(a.x) + row * a.ld_x + c.col, v[u]);
                    if (gate) load<T, VEC>(static_cast<const T*>(a.z) + row * a.ld_z + c.col, z[u]);
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * c.rp < c.rows1) {
                    const long long row = row0 + s + u * c.rp;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        v[u][e] = act<T>(a.activation, fmaf((v[u][e] - mean) * rstd, w[e], bias[e]));
                        if (gate) v[u][e] *= z[u][e] * sigmoid<T>(z[u][e]);
                    }
                    store<T, VEC>(static_cast<T*>(a.y) + row * a.ld_y + c.col, v[u]);
                }
        }
    }
}

// Backward: a block's sums over its rows, for each group (of dv w and dv w xh) and, over its samples, each channel (d_w, d_b).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) slopes_kernel(const Params p) {
    __shared__ float sw[kThreads * VEC], sb[kThreads * VEC];
    __shared__ float s1s[kThreads], s2s[kThreads];
    const mamba_b200_group_norm_args& a = p.a;
    const Cover c = cover<VEC>(p);
    const long long NG = static_cast<long long>(a.N) * a.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int vecs = p.sub > 1 ? kThreads : p.vecs, wide = p.sub > 1 ? kThreads : p.groups * p.vecs;
    const bool gate = a.z != nullptr;
    float w[VEC], bias[VEC], all_w[VEC], all_b[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        w[e] = c.on && a.weight ? a.weight[c.col + e] : 1.0f;
        bias[e] = c.on && a.bias ? a.bias[c.col + e] : 0.0f;
        all_w[e] = all_b[e] = 0.0f;
    }
    for (int ns = blockIdx.x / p.blocks; ns < a.N; ns += p.side) {
        float dw[VEC], db[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.0f;
        if (c.on) {
            const float mean = a.stats[static_cast<long long>(ns) * a.G + c.g], rstd = a.stats[NG + static_cast<long long>(ns) * a.G + c.g];
            const long long row0 = static_cast<long long>(ns) * a.S;
            for (int s = c.rows0 + c.r; s < c.rows1; s += c.rp) {
                float x[VEC], z[VEC], dy[VEC], dz;
                load<T, VEC>(static_cast<const T*>(a.x) + (row0 + s) * a.ld_x + c.col, x);
                load<T, VEC>(static_cast<const T*>(a.dy) + (row0 + s) * a.ld_dy + c.col, dy);
                if (gate) load<T, VEC>(static_cast<const T*>(a.z) + (row0 + s) * a.ld_z + c.col, z);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xh = (x[e] - mean) * rstd;
                    const float dv = through<T>(a.activation, fmaf(xh, w[e], bias[e]), dy[e], gate, gate ? z[e] : 0.0f, &dz);
                    dw[e] = fmaf(dv, xh, dw[e]);
                    db[e] += dv;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sw[e * kThreads + threadIdx.x] = dw[e];
            sb[e * kThreads + threadIdx.x] = db[e];
        }
        __syncthreads();
        float s1 = 0.0f, s2 = 0.0f;
        if (c.r == 0 && c.on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float tw = dw[e], tb = db[e];
                for (int k = 1; k < c.rp; ++k) {
                    tw += sw[e * kThreads + k * wide + threadIdx.x];
                    tb += sb[e * kThreads + k * wide + threadIdx.x];
                }
                all_w[e] += tw;
                all_b[e] += tb;
                s1 = fmaf(w[e], tb, s1);
                s2 = fmaf(w[e], tw, s2);
            }
        }
        s1s[threadIdx.x] = s1;
        s2s[threadIdx.x] = s2;
        __syncthreads();
        for (int gi = warp; gi < c.groups; gi += kThreads / 32) {
            float t1 = 0.0f, t2 = 0.0f;
            for (int i = lane; i < vecs; i += 32) {
                t1 += s1s[gi * vecs + i];
                t2 += s2s[gi * vecs + i];
            }
            t1 = sum_lanes(t1, 32);
            t2 = sum_lanes(t2, 32);
            if (lane == 0) {
                float* out = p.part + ((static_cast<long long>(ns) * p.blocks * p.sub + c.blk * p.sub + c.sub) * a.G + c.first + gi) * 2;
                out[0] = t1;
                out[1] = t2;
            }
        }
    }
    if (c.r == 0 && c.on) {
        float* out_w = p.sums + static_cast<long long>(blockIdx.x) * a.C + c.col;
        float* out_b = out_w + static_cast<long long>(p.parts) * a.C;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            out_w[e] = all_w[e];
            out_b[e] = all_b[e];
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) spread_kernel(const Params p) {
    __shared__ float s_1[kThreads], s_2[kThreads];
    const mamba_b200_group_norm_args& a = p.a;
    const Cover c = cover<VEC>(p);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float inv = 1.0f / (static_cast<float>(p.per) * a.S);
    const long long NG = static_cast<long long>(a.N) * a.G;
    const bool gate = a.z != nullptr;
    float w[VEC], bias[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        w[e] = c.on && a.weight ? a.weight[c.col + e] : 1.0f;
        bias[e] = c.on && a.bias ? a.bias[c.col + e] : 0.0f;
    }
    for (int ns = blockIdx.x / p.blocks; ns < a.N; ns += p.side) {
        __syncthreads();
        for (int gi = warp; gi < c.groups; gi += kThreads / 32) {
            float t1 = 0.0f, t2 = 0.0f;
            for (int i = lane; i < p.blocks * p.sub; i += 32) {
                const float* src = p.part + ((static_cast<long long>(ns) * p.blocks * p.sub + i) * a.G + c.first + gi) * 2;
                t1 += src[0];
                t2 += src[1];
            }
            t1 = sum_lanes(t1, 32);
            t2 = sum_lanes(t2, 32);
            if (lane == 0) {
                s_1[gi] = t1 * inv;
                s_2[gi] = t2 * inv;
            }
        }
        __syncthreads();
        if (!c.on) continue;
        const float m1 = s_1[c.gi], m2 = s_2[c.gi];
        const float mean = a.stats[static_cast<long long>(ns) * a.G + c.g], rstd = a.stats[NG + static_cast<long long>(ns) * a.G + c.g];
        const long long row0 = static_cast<long long>(ns) * a.S;
        for (int s = c.rows0 + c.r; s < c.rows1; s += c.rp) {
            float x[VEC], z[VEC], dy[VEC];
            load<T, VEC>(static_cast<const T*>(a.x) + (row0 + s) * a.ld_x + c.col, x);
            load<T, VEC>(static_cast<const T*>(a.dy) + (row0 + s) * a.ld_dy + c.col, dy);
            if (gate) load<T, VEC>(static_cast<const T*>(a.z) + (row0 + s) * a.ld_z + c.col, z);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = (x[e] - mean) * rstd;
                const float dv = through<T>(a.activation, fmaf(xh, w[e], bias[e]), dy[e], gate, gate ? z[e] : 0.0f, &z[e]);
                x[e] = rstd * (dv * w[e] - m1 - xh * m2);
            }
            store<T, VEC>(static_cast<T*>(a.d_x) + (row0 + s) * a.ld_dx + c.col, x);
            if (gate) store<T, VEC>(static_cast<T*>(a.d_z) + (row0 + s) * a.ld_dz + c.col, z);
        }
    }
}

// The same in one kernel, where a sample's rows of a block's channels fit shared memory: every element is read once.  A thread keeps
// its own vectors there, so that barriers are for sums alone.
constexpr int kSlabThreads = 512;

template <typename T, int VEC>
__device__ __forceinline__ float group_sum(const Params& p, const Cover& c, float v, float* per_thread, float* per_group) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, vecs = p.vecs, wide = p.groups * p.vecs;
    __syncthreads();
    per_thread[threadIdx.x] = v;
    __syncthreads();
    for (int gi = warp; gi < c.groups; gi += kSlabThreads / 32) {
        float t = 0.0f;
        for (int i = lane; i < c.rp * vecs; i += 32) t += per_thread[(i / vecs) * wide + gi * vecs + i % vecs];
        t = sum_lanes(t, 32);
        if (lane == 0) per_group[gi] = t;
    }
    __syncthreads();
    return c.on ? per_group[c.gi] : 0.0f;
}

template <typename T, int VEC, bool BWD>
__global__ void __launch_bounds__(kSlabThreads) slab_kernel(const Params p) {
    using V = Vec<T, VEC>;
    extern __shared__ __align__(16) unsigned char slab[];
    __shared__ float per_thread[kSlabThreads], per_group[kSlabThreads];
    __shared__ float sw[BWD ? kSlabThreads * VEC : 1], sb[BWD ? kSlabThreads * VEC : 1];
    const mamba_b200_group_norm_args& a = p.a;
    const Cover c = cover<VEC, kSlabThreads>(p);
    const int turns = (a.S + c.rp - 1) / c.rp;
    V* sx = reinterpret_cast<V*>(slab) + threadIdx.x;
    V* sd = sx + (BWD ? static_cast<size_t>(turns) * kSlabThreads : 0);
    V* sz = sd + static_cast<size_t>(turns) * kSlabThreads;
    const bool gate = a.z != nullptr;
    const float inv = 1.0f / (static_cast<float>(p.per) * a.S);
    const long long NG = static_cast<long long>(a.N) * a.G;
    float w[VEC], bias[VEC], all_w[BWD ? VEC : 1], all_b[BWD ? VEC : 1];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        w[e] = c.on && a.weight ? a.weight[c.col + e] : 1.0f;
        bias[e] = c.on && a.bias ? a.bias[c.col + e] : 0.0f;
        if (BWD) all_w[e] = all_b[e] = 0.0f;
    }
    for (int ns = blockIdx.x; ns < a.N; ns += p.side) {
        const long long row0 = static_cast<long long>(ns) * a.S;
        constexpr int U = 4;
        float s1 = 0.0f, s2 = 0.0f;
        float mean = 0.0f, rstd = 0.0f;
        if (BWD && c.on) {
            mean = a.stats[static_cast<long long>(ns) * a.G + c.g];
            rstd = a.stats[NG + static_cast<long long>(ns) * a.G + c.g];
        }
        if (c.on) {
            for (int s = c.r, k = 0; s < a.S; s += U * c.rp, k += U) {
                V v[U], d[BWD ? U : 1], g[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * c.rp < a.S) {
                        const long long row = row0 + s + u * c.rp;
                        v[u] = *reinterpret_cast<const V*>(static_cast<const T*>(a.x) + row * a.ld_x + c.col);
                        if (BWD) d[u % (BWD ? U : 1)] = *reinterpret_cast<const V*>(static_cast<const T*>(a.dy) + row * a.ld_dy + c.col);
                        if (gate) g[u] = *reinterpret_cast<const V*>(static_cast<const T*>(a.z) + row * a.ld_z + c.col);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (s + u * c.rp < a.S) {
                        sx[(k + u) * kSlabThreads] = v[u];
                        if (BWD) sd[(k + u) * kSlabThreads] = d[u % (BWD ? U : 1)];
                        if (gate) sz[(k + u) * kSlabThreads] = g[u];
                        if (!BWD) {
#pragma unroll
                            for (int e = 0; e < VEC; ++e) s1 += to_f(v[u].v[e]);
                        }
                    }
            }
        }
        if constexpr (!BWD) {
            mean = group_sum<T, VEC>(p, c, s1, per_thread, per_group) * inv;
            // deviations from that mean, and what they say it is off by: a thread's sum of values far from zero loses digits
            s1 = 0.0f;
            if (c.on)
                for (int s = c.r, k = 0; s < a.S; s += c.rp, ++k) {
                    float x[VEC];
                    widen(sx[k * kSlabThreads], x);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float d = x[e] - mean;
                        s1 += d;
                        s2 = fmaf(d, d, s2);
                    }
                }
            const float off = group_sum<T, VEC>(p, c, s1, per_thread, per_group) * inv;
            mean += off;
            const float var = fmaf(-off, off, group_sum<T, VEC>(p, c, s2, per_thread, per_group) * inv);
            rstd = rsqrtf((var < 0.0f ? 0.0f : var) + a.eps);  // (a NaN stays one)
            if (c.on && a.stats && c.r == 0 && c.col == c.g * p.per) {
                a.stats[static_cast<long long>(ns) * a.G + c.g] = mean;
                a.stats[NG + static_cast<long long>(ns) * a.G + c.g] = rstd;
            }
            if (c.on)
                for (int s = c.r, k = 0; s < a.S; s += c.rp, ++k) {
                    float x[VEC], z[VEC];
                    widen(sx[k * kSlabThreads], x);
                    if (gate) widen(sz[k * kSlabThreads], z);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        x[e] = act<T>(a.activation, fmaf((x[e] - mean) * rstd, w[e], bias[e]));
                        if (gate) x[e] *= z[e] * sigmoid<T>(z[e]);
                    }
                    store<T, VEC>(static_cast<T*>(a.y) + (row0 + s) * a.ld_y + c.col, x);
                }
        } else {
            float dw[VEC], db[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.0f;
            if (c.on)
                for (int s = c.r, k = 0; s < a.S; s += c.rp, ++k) {
                    float x[VEC], z[VEC], dy[VEC], dz;
                    widen(sx[k * kSlabThreads], x);
                    widen(sd[k * kSlabThreads], dy);
                    if (gate) widen(sz[k * kSlabThreads], z);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float xh = (x[e] - mean) * rstd;
                        const float dv = through<T>(a.activation, fmaf(xh, w[e], bias[e]), dy[e], gate, gate ? z[e] : 0.0f, &dz);
                        dw[e] = fmaf(dv, xh, dw[e]);
                        db[e] += dv;
                    }
                }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s1 = fmaf(w[e], db[e], s1);
                s2 = fmaf(w[e], dw[e], s2);
                all_w[e] += dw[e];
                all_b[e] += db[e];
            }
            s1 = group_sum<T, VEC>(p, c, s1, per_thread, per_group) * inv;
            s2 = group_sum<T, VEC>(p, c, s2, per_thread, per_group) * inv;
            if (c.on)
                for (int s = c.r, k = 0; s < a.S; s += c.rp, ++k) {
                    float x[VEC], z[VEC], dy[VEC];
                    widen(sx[k * kSlabThreads], x);
                    widen(sd[k * kSlabThreads], dy);
                    if (gate) widen(sz[k * kSlabThreads], z);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float xh = (x[e] - mean) * rstd;
                        const float dv = through<T>(a.activation, fmaf(xh, w[e], bias[e]), dy[e], gate, gate ? z[e] : 0.0f, &z[e]);
                        x[e] = rstd * (dv * w[e] - s1 - xh * s2);
                    }
                    store<T, VEC>(static_cast<T*>(a.d_x) + (row0 + s) * a.ld_dx + c.col, x);
                    if (gate) store<T, VEC>(static_cast<T*>(a.d_z) + (row0 + s) * a.ld_dz + c.col, z);
                }
        }
    }
    if constexpr (BWD) {
        const int wide = p.groups * p.vecs;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sw[e * kSlabThreads + threadIdx.x] = all_w[e];
            sb[e * kSlabThreads + threadIdx.x] = all_b[e];
        }
        __syncthreads();
        if (c.r == 0 && c.on) {
            float* out_w = p.sums + static_cast<long long>(blockIdx.x) * a.C + c.col;
            float* out_b = out_w + static_cast<long long>(p.parts) * a.C;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float tw = all_w[e], tb = all_b[e];
                for (int k = 1; k < c.rp; ++k) {
                    tw += sw[e * kSlabThreads + k * wide + threadIdx.x];
                    tb += sb[e * kSlabThreads + k * wide + threadIdx.x];
                }
                out_w[e] = tw;
                out_b[e] = tb;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------
constexpr int kRowVecs = 4 * kThreads;  // most vectors of a group in the row form
constexpr int kBlocks = 148 * 6;        // blocks that a launch is cut into where there are rows enough

inline int pow2_up(int n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

// Sample form: rows of a block and blocks of a sample (as many as fill the SMs, of 16 rows at least), samples side by side.
struct Cut {
    int block_rows, blocks, side;
};
inline Cut cut(int N, int S, long long across) {
    Cut r;
    long long want = (kBlocks + across * N - 1) / (across * N);
    const long long most = (static_cast<long long>(S) + 15) / 16;
    if (want > most) want = most;
    r.block_rows = static_cast<int>((S + want - 1) / want);
    r.blocks = (S + r.block_rows - 1) / r.block_rows;
    long long side = (2 * kBlocks + across * r.blocks - 1) / (across * r.blocks);
    r.side = static_cast<int>(side < N ? side : N);
    return r;
}

struct Room {
    long long part, sums;
};
// An upper bound over the vectors that a call may take (they go by its pointers and strides).
inline Room room(int N, int S, int C, int G, int backward) {
    Room r{0, 0};
    const int per = C / G;
    const bool rows = S == 1 && per <= kRowVecs;  // (with one element a vector)
    const Cut most = cut(N, S, 1);
    const long long sub = (per + kThreads - 1) / kThreads;
    if (!rows) r.part = (static_cast<long long>(N) * most.blocks * sub * G * 2 * 4 + 255) / 256 * 256;
    // (a wider covering has no more blocks of a sample, and no more of them side by side)
    const long long parts = rows ? kBlocks : static_cast<long long>(most.blocks) * most.side;
    if (backward) r.sums = 2 * parts * C * 4;
    return r;
}

// One kernel for a sample: the groups of a block (into p.groups) and its shared memory, or 0 where two kernels are better.  A block's
// piece of a row is at least 64 bytes where there are groups for it, and there have to be enough blocks for a third of the SMs.
constexpr size_t kSlab = 188 * 1024;  // (beside 36 KB of the backward's sums)
inline size_t slab_groups(const mamba_b200_group_norm_args& a, Params& p, size_t vec, bool bwd) {
    const int tensors = (bwd ? 2 : 1) + (a.z ? 1 : 0);
    int groups = static_cast<int>((64 + p.vecs * vec - 1) / (p.vecs * vec));
    if (groups > p.groups) groups = p.groups;
    const long long rp = kSlabThreads / (groups * p.vecs), turns = (a.S + rp - 1) / rp, across = (a.G + groups - 1) / groups;
    const unsigned long long bytes = static_cast<unsigned long long>(turns) * kSlabThreads * vec * tensors;
    if (bytes > kSlab || across > 65535 || across * a.N < 48) return 0;
    p.groups = groups;
    return bytes;
}

inline int join_sums(Ctx* c, const Params& p, bool bwd, cudaStream_t st) {
    const mamba_b200_group_norm_args& a = p.a;
    if (!bwd || (!a.d_weight && !a.d_bias)) return MAMBA_B200_OK;
    join_kernel<<<dim3(static_cast<unsigned>((a.C + 31) / 32), 2), 256, 0, st>>>(p.sums, p.parts, a.C, a.d_weight, a.d_bias, a.accumulate);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

template <typename T, int VEC, int VPT, bool BWD>
const void* rows_fn(int act, bool gate) {
    if (act == MAMBA_B200_ACT_SILU)
        return gate ? (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_SILU, true> : (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_SILU, false>;
    if (act == MAMBA_B200_ACT_GELU)
        return gate ? (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_GELU, true> : (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_GELU, false>;
    return gate ? (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_NONE, true> : (const void*)rows_kernel<T, VEC, VPT, BWD, MAMBA_B200_ACT_NONE, false>;
}

template <typename T, int VEC, int VPT, bool BWD>
int launch_rows(Ctx* c, Params& p, cudaStream_t st) {
    const long long steps = (p.a.N + static_cast<long long>(p.rows) - 1) / p.rows;
    const int tiles = (p.a.G + p.groups - 1) / p.groups;
    if (tiles > 65535) return fail(c, MAMBA_B200_ERR_SHAPE, "group_norm: too many groups (%d)", p.a.G);
    // as many blocks as are resident together (registers: two or four): each goes over its share of the rows
    long long blocks = static_cast<long long>(c->sm_count) * (BWD ? 2 : 4) / tiles;
    if (blocks > kBlocks) blocks = kBlocks;
    if (blocks > steps) blocks = steps;
    if (blocks < 1) blocks = 1;
    p.parts = static_cast<int>(blocks);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(tiles));
    if constexpr (VEC == 1) {
        odd_rows_kernel<T, VPT, BWD><<<grid, kThreads, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
    } else {
        const int tensors = (BWD ? 2 : 1) + (p.a.z ? 1 : 0);
        const size_t smem = static_cast<size_t>(kRowsAhead<VPT>) * tensors * VPT * kThreads * VEC * sizeof(T);
        void* args[] = {&p};
        MB200_CUDA_CHECK(c, cudaLaunchKernel(rows_fn<T, VEC, VPT, BWD>(p.a.activation, p.a.z != nullptr), grid, dim3(kThreads), args, smem, st));
    }
    return MAMBA_B200_OK;
}

template <typename T, int VEC>
int launch_vec(Ctx* c, const mamba_b200_group_norm_args& a, bool bwd, cudaStream_t st) {
    Params p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    p.per = a.C / a.G;
    p.vecs = p.per / VEC;
    const Room room = gn::room(a.N, a.S, a.C, a.G, bwd);
    p.part = static_cast<float*>(a.workspace);
    if (bwd) p.sums = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + room.part);
    int rc = MAMBA_B200_OK;
    if (a.S == 1 && p.per <= kRowVecs) {
        // a group stays within a warp where that takes at most two vectors a lane (four elements, where a vector is one): no barriers
        constexpr int most = VEC == 1 ? 4 : 2;
        const int vpt = p.vecs <= 32 ? 1 : p.vecs <= 64 ? 2 : most;
        p.lanes = pow2_up((p.vecs + vpt - 1) / vpt);
        p.groups = kThreads / p.lanes < a.G ? kThreads / p.lanes : a.G;
        p.rows = kThreads / (p.groups * p.lanes);
        if (vpt == 1) rc = bwd ? launch_rows<T, VEC, 1, true>(c, p, st) : launch_rows<T, VEC, 1, false>(c, p, st);
        else if (vpt == 2) rc = bwd ? launch_rows<T, VEC, 2, true>(c, p, st) : launch_rows<T, VEC, 2, false>(c, p, st);
        else rc = bwd ? launch_rows<T, VEC, most, true>(c, p, st) : launch_rows<T, VEC, most, false>(c, p, st);
        if (rc) return rc;
    } else {
        p.sub = (p.vecs + kThreads - 1) / kThreads;
        p.groups = p.sub > 1 ? 1 : kThreads / p.vecs < a.G ? kThreads / p.vecs : a.G;
        if (p.sub == 1) {
            const size_t bytes = slab_groups(a, p, sizeof(T) * VEC, bwd);
            if (bytes) {
                const int across = (a.G + p.groups - 1) / p.groups;
                p.block_rows = a.S;
                p.blocks = 1;
                // (no more blocks side by side than the two kernels' scratch has sums for)
                const long long side = (2 * kBlocks + across - 1) / across;
                p.side = p.parts = static_cast<int>(side < a.N ? side : a.N);
                const dim3 grid(static_cast<unsigned>(p.side), static_cast<unsigned>(across));
                if (bwd) slab_kernel<T, VEC, true><<<grid, kSlabThreads, bytes, st>>>(p);
                else slab_kernel<T, VEC, false><<<grid, kSlabThreads, bytes, st>>>(p);
                MB200_CUDA_CHECK(c, cudaGetLastError());
                return join_sums(c, p, bwd, st);
            }
        }
        const long long across = p.sub > 1 ? static_cast<long long>(a.G) * p.sub : (a.G + p.groups - 1) / p.groups;
        const Cut k = cut(a.N, a.S, across);
        p.block_rows = k.block_rows;
        p.blocks = k.blocks;
        p.side = k.side;
        p.parts = k.blocks * k.side;
        if (across > 65535) return fail(c, MAMBA_B200_ERR_SHAPE, "group_norm: too many groups (%d)", a.G);
        const dim3 grid(static_cast<unsigned>(p.parts), static_cast<unsigned>(across));
        if (bwd) {
            slopes_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
            MB200_CUDA_CHECK(c, cudaGetLastError());
            spread_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
        } else {
            moments_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
            MB200_CUDA_CHECK(c, cudaGetLastError());
            apply_kernel<T, VEC><<<grid, kThreads, 0, st>>>(p);
        }
        MB200_CUDA_CHECK(c, cudaGetLastError());
    }
    return join_sums(c, p, bwd, st);
}

template <typename T>
int launch_typed(Ctx* c, const mamba_b200_group_norm_args& a, bool bwd, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    long long odd = a.C / a.G;
    if (static_cast<long long>(a.N) * a.S > 1) {
        odd |= a.ld_x;
        if (a.z) odd |= a.ld_z;
        if (bwd) odd |= a.ld_dy | a.ld_dx | (a.z ? a.ld_dz : 0);
        else odd |= a.ld_y;
    }
    const bool wide = odd % W == 0 && aligned_to(16, {a.x, a.z}) && (bwd ? aligned_to(16, {a.dy, a.d_x, a.z ? a.d_z : nullptr}) : aligned_to(16, {a.y}));
    return wide ? launch_vec<T, W>(c, a, bwd, st) : launch_vec<T, 1>(c, a, bwd, st);
}

int check(Ctx* c, const mamba_b200_group_norm_args* a, bool bwd) {
    const char* what = bwd ? "group_norm_bwd" : "group_norm_fwd";
    int cur = -1;
    MB200_CUDA_CHECK(c, cudaGetDevice(&cur));
    if (cur != c->device)
        return fail(c, MAMBA_B200_ERR_DEVICE, "%s: the handle belongs to device %d but device %d is current", what, c->device, cur);
    if (!dtype_ok(a->dtype)) return fail(c, MAMBA_B200_ERR_ARG, "%s: unknown dtype %d", what, a->dtype);
    if (a->N < 0 || a->S < 0 || a->C < 1 || a->G < 1 || a->C % a->G)
        return fail(c, MAMBA_B200_ERR_SHAPE, "%s: N %d S %d C %d G %d", what, a->N, a->S, a->C, a->G);
    if (a->N > kMaxSize || a->S > kMaxRows || a->C > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: too many rows or channels", what);
    if (a->activation < 0 || a->activation > MAMBA_B200_ACT_GELU) return fail(c, MAMBA_B200_ERR_ARG, "%s: unknown activation %d", what, a->activation);
    if (!(a->eps >= 0.0f) || isinf(a->eps)) return fail(c, MAMBA_B200_ERR_ARG, "%s: eps %g", what, a->eps);
    if (a->N == 0 || a->S == 0) return MAMBA_B200_OK;
    if (!a->x || (!bwd && !a->y) || (bwd && (!a->dy || !a->d_x || !a->stats || (a->z && !a->d_z))))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", what);
    if (a->ld_x < a->C || (a->z && a->ld_z < a->C) || (!bwd && a->ld_y < a->C) ||
        (bwd && (a->ld_dy < a->C || a->ld_dx < a->C || (a->z && a->ld_dz < a->C))))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: a row stride is narrower than %d channels", what, a->C);
    const size_t es = dtype_size(a->dtype);
    if (!aligned_to(es, {a->x, a->z}) || (bwd ? !aligned_to(es, {a->dy, a->d_x, a->d_z}) : !aligned_to(es, {a->y})) ||
        !aligned_to(4, {a->weight, a->bias, a->stats}) || (bwd && !aligned_to(4, {a->d_weight, a->d_bias})))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: misaligned pointer", what);
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256) return fail(c, MAMBA_B200_ERR_ARG, "%s: misaligned workspace", what);
    // (a thread writes where it has read: with other strides it would write where others have yet to read)
    struct Rows {
        const void* p;
        long long ld;
    };
    if (static_cast<long long>(a->N) * a->S > 1)
        for (const Rows& in : {Rows{a->x, a->ld_x}, Rows{a->z, a->ld_z}, bwd ? Rows{a->dy, a->ld_dy} : Rows{nullptr, 0}})
            for (const Rows& out : {bwd ? Rows{a->d_x, a->ld_dx} : Rows{a->y, a->ld_y}, bwd && a->z ? Rows{a->d_z, a->ld_dz} : Rows{nullptr, 0}})
                if (in.p && in.p == out.p && in.ld != out.ld)
                    return fail(c, MAMBA_B200_ERR_ARG, "%s: a result is an input with other strides", what);
    if (bwd && a->z && a->d_z == a->d_x) return fail(c, MAMBA_B200_ERR_ARG, "%s: two results are the same memory", what);
    const long long need = mamba_b200_group_norm_workspace_bytes(a->N, a->S, a->C, a->G, bwd);
    if (need && (!a->workspace || a->workspace_bytes < need))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: a workspace of %lld bytes is needed (%lld given)", what, need, a->workspace ? a->workspace_bytes : 0ll);
    return MAMBA_B200_OK;
}

template <typename T, int VEC>
int configure(Ctx* c) {
    if constexpr (VEC > 1) {
        for (int act = 0; act <= MAMBA_B200_ACT_GELU; ++act)
            for (int gate = 0; gate < 2; ++gate)
                for (const void* f : {rows_fn<T, VEC, 1, true>(act, gate), rows_fn<T, VEC, 2, true>(act, gate)})
                    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, 48 * 1024));
    }
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)slab_kernel<T, VEC, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSlab)));
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)slab_kernel<T, VEC, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSlab)));
    return MAMBA_B200_OK;
}

}  // namespace gn

int group_norm_configure(Ctx* c) {
    int rc = gn::configure<float, 4>(c);
    if (!rc) rc = gn::configure<float, 1>(c);
    if (!rc) rc = gn::configure<__half, 8>(c);
    if (!rc) rc = gn::configure<__half, 1>(c);
    if (!rc) rc = gn::configure<__nv_bfloat16, 8>(c);
    if (!rc) rc = gn::configure<__nv_bfloat16, 1>(c);
    return rc;
}


}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API long long mamba_b200_group_norm_workspace_bytes(int N, int S, int C, int G, int backward) {
    if (N < 1 || S < 1 || C < 1 || G < 1 || C % G || N > kMaxSize || S > gn::kMaxRows || C > kMaxSize) return 0;
    const gn::Room r = gn::room(N, S, C, G, backward);
    return r.part + r.sums;
}

extern "C" MAMBA_B200_API int mamba_b200_group_norm_fwd(void* handle, void* stream, const mamba_b200_group_norm_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gn::check(c, args, false);
    if (rc || args->N == 0 || args->S == 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (args->dtype == MAMBA_B200_F32) return gn::launch_typed<float>(c, *args, false, st);
    if (args->dtype == MAMBA_B200_F16) return gn::launch_typed<__half>(c, *args, false, st);
    return gn::launch_typed<__nv_bfloat16>(c, *args, false, st);
}

extern "C" MAMBA_B200_API int mamba_b200_group_norm_bwd(void* handle, void* stream, const mamba_b200_group_norm_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gn::check(c, args, true);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (args->N == 0 || args->S == 0) {  // no rows: sums of nothing
        if (!args->accumulate) {
            if (args->d_weight) MB200_CUDA_CHECK(c, cudaMemsetAsync(args->d_weight, 0, sizeof(float) * args->C, st));
            if (args->d_bias) MB200_CUDA_CHECK(c, cudaMemsetAsync(args->d_bias, 0, sizeof(float) * args->C, st));
        }
        return MAMBA_B200_OK;
    }
    if (args->dtype == MAMBA_B200_F32) return gn::launch_typed<float>(c, *args, true, st);
    if (args->dtype == MAMBA_B200_F16) return gn::launch_typed<__half>(c, *args, true, st);
    return gn::launch_typed<__nv_bfloat16>(c, *args, true, st);
}
