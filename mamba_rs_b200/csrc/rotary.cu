// Rotation of queries and keys by position.
//
//   (a, b) -> scale (a cos p - b sin p, b cos p + a sin p),   p = position * frequency
//
// One read and one write of every element, so HBM bounds it if instructions do not.  A thread owns one place in the head (16 bytes of
// pairs, or of columns that are handed on) of one token, makes that place's sines and cosines once, and goes through heads of q and k with
// them, four in flight, by pointers that go on by a head.  A block has places of pairs first and places to be handed on behind them, so that
// warps do one or the other.  The angle is reduced to turns in 64 bits: at position 10^6 its 32-bit product is off by 2^-5 of a radian, in
// 64 bits by 2^-34.  8 x 4096 tokens, 2 x 32 heads of 128 columns, bf16, 64 of them turned: 174 us,
// 6.2 TB/s (250 with places of both kinds in a warp and addresses made for every head).
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace rot {

constexpr int kThreads = 256;

struct Params {
    mamba_b200_rotary_args a;
    int units, turned;  // places of a head; of these, places of pairs
    int tokens;         // of a block
    int heads;          // heads of a block
    int copy_q, copy_k; // columns behind the pairs have to be handed on
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
    T v[VEC];
};

// cos and sin of position * frequency, times scale
__device__ __forceinline__ void turn(double position, float freq, float scale, float sign, float* c, float* s) {
    double turns = position * static_cast<double>(freq) * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.0f * static_cast<float>(turns), &sn, &cs);
    *c = cs * scale;
    *s = sn * scale * sign;
}

// VEC: elements of a vector.  A place of pairs is one vector of interleaved pairs or two of halves; with VEC 1 it is the two elements of
// one pair, wherever they lie.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : kThreads) rotary_kernel(const Params p) {
    constexpr bool PACKED = INTERLEAVED && VEC > 1;
    constexpr int NV = PACKED ? 1 : 2, PAIRS = PACKED ? VEC / 2 : VEC, U = 4;
    using V = Vec<T, VEC>;
    const mamba_b200_rotary_args& a = p.a;
    const int item = threadIdx.x, n_pairs = p.tokens * p.turned;
    const bool pairs = item < n_pairs;
    const int per = pairs ? p.turned : p.units - p.turned, i = pairs ? item : item - n_pairs;
    const int own = per > 0 ? i / per : p.tokens, unit = i - own * per;
    const long long token = blockIdx.x * static_cast<long long>(p.tokens) + own;
    if (own >= p.tokens || token >= static_cast<long long>(a.B) * a.T) return;
    const int b = static_cast<int>(token / a.T), t = static_cast<int>(token - static_cast<long long>(b) * a.T);
    const int h0 = blockIdx.y * p.heads, h1 = min(h0 + p.heads, a.Hq + a.Hk);
    const int first = unit * PAIRS;  // pair
    const int col = !pairs ? a.R + unit * VEC : INTERLEAVED ? 2 * first : first;
    const long long other = INTERLEAVED ? 1 : a.R / 2;  // to the second element of a pair
    float cs[PAIRS], sn[PAIRS];
    if (pairs) {
        const double position = static_cast<double>(a.positions[b * a.pos_b + t]);
        const float sign = a.inverse ? -1.0f : 1.0f;
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) turn(position, a.inv_freq[first + k], a.scale, sign, &cs[k], &sn[k]);
    }
    // heads [from, to) of one tensor
    auto heads = [&](const T* in, T* out, long long step_in, long long step_out, int n, bool copy) {
        if (n <= 0 || (!pairs && !copy)) return;
        auto put = [&](V* v, T* dst) {
            if (pairs) {
#pragma unroll
                for (int k = 0; k < PAIRS; ++k) {
                    const float x = to_f(v[0].v[PACKED ? 2 * k : k]), y = to_f(v[NV - 1].v[PACKED ? 2 * k + 1 : k]);
                    // (written out: every variant rounds alike)
                    v[0].v[PACKED ? 2 * k : k] = from_f<T>(fmaf(x, cs[k], -__fmul_rn(y, sn[k])));
                    v[NV - 1].v[PACKED ? 2 * k + 1 : k] = from_f<T>(fmaf(y, cs[k], __fmul_rn(x, sn[k])));
                }
                if (NV == 2) *reinterpret_cast<V*>(dst + other) = v[NV - 1];
            }
            *reinterpret_cast<V*>(dst) = v[0];
        };
        auto get = [&](const T* src, V* v) {
            v[0] = *reinterpret_cast<const V*>(src);
            if (NV == 2 && pairs) v[NV - 1] = *reinterpret_cast<const V*>(src + other);
        };
        for (; n >= U; n -= U) {
            V v[U][NV];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                get(in, v[u]);
                in += step_in;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                put(v[u], out);
                out += step_out;
            }
        }
        for (; n > 0; --n) {
            V v[NV];
            get(in, v);
            put(v, out);
            in += step_in;
            out += step_out;
        }
    };
    const int q0 = min(h0, a.Hq), q1 = min(h1, a.Hq), k0 = max(h0 - a.Hq, 0), k1 = h1 - a.Hq;
    heads(static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + q0 * a.q_h + col, static_cast<T*>(a.q_out) + b * a.qo_b + t * a.qo_t + q0 * a.qo_h + col,
          a.q_h, a.qo_h, q1 - q0, p.copy_q);
    heads(static_cast<const T*>(a.k) + b * a.k_b + t * a.k_t + k0 * a.k_h + col, static_cast<T*>(a.k_out) + b * a.ko_b + t * a.ko_t + k0 * a.ko_h + col,
          a.k_h, a.ko_h, k1 - k0, p.copy_k);
}

template <typename T, int VEC, bool INTERLEAVED>
int launch(Ctx* c, const mamba_b200_rotary_args& a, cudaStream_t st) {
    Params p;
    memset(&p, 0, sizeof(p));
    p.a = a;
    p.copy_q = a.q_out != a.q;
    p.copy_k = a.Hk > 0 && a.k_out != a.k;
    p.turned = INTERLEAVED && VEC > 1 ? a.R / VEC : a.R / 2 / VEC;
    p.units = p.turned + (p.copy_q || p.copy_k ? (a.D - a.R) / VEC : 0);
    if (p.units == 0) return MAMBA_B200_OK;
    // (single elements: up to 1024 places of a head)
    const int threads = p.units <= kThreads ? kThreads : (p.units + 31) / 32 * 32;
    p.tokens = threads / p.units;
    const long long blocks = (static_cast<long long>(a.B) * a.T + p.tokens - 1) / p.tokens;
    if (blocks > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "rotary: too many steps");
    // Heads of a block: all of them where there are enough tokens (a place's sines are made once a block), else as few as four.
    const int heads = a.Hq + a.Hk;
    long long parts = (8ll * c->sm_count + blocks - 1) / blocks;
    if (parts > (heads + 3) / 4) parts = (heads + 3) / 4;
    p.heads = static_cast<int>((heads + parts - 1) / parts);
    p.heads = (p.heads + 3) / 4 * 4;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + p.heads - 1) / p.heads));
    rotary_kernel<T, VEC, INTERLEAVED><<<grid, threads, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

template <typename T>
int launch_typed(Ctx* c, const mamba_b200_rotary_args& a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    // 16-byte vectors where every place of every head starts on 16 bytes
    long long odd = a.interleaved ? a.R : a.R / 2;
    odd |= a.D;
    auto mix = [&](long long sb, long long st_, long long sh, int h) {
        if (a.B > 1) odd |= sb;
        if (a.T > 1) odd |= st_;
        if (h > 1) odd |= sh;
    };
    mix(a.q_b, a.q_t, a.q_h, a.Hq);
    mix(a.qo_b, a.qo_t, a.qo_h, a.Hq);
    if (a.Hk) {
        mix(a.k_b, a.k_t, a.k_h, a.Hk);
        mix(a.ko_b, a.ko_t, a.ko_h, a.Hk);
    }
    const bool wide = odd % W == 0 && aligned_to(16, {a.q, a.q_out, a.Hk ? a.k : nullptr, a.Hk ? a.k_out : nullptr});
    if (a.interleaved) return wide ? launch<T, W, true>(c, a, st) : launch<T, 1, true>(c, a, st);
    return wide ? launch<T, W, false>(c, a, st) : launch<T, 1, false>(c, a, st);
}

}  // namespace rot
}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API int mamba_b200_rotary(void* handle, void* stream, const mamba_b200_rotary_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const mamba_b200_rotary_args& a = *args;
    int cur = -1;
    MB200_CUDA_CHECK(c, cudaGetDevice(&cur));
    if (cur != c->device)
        return fail(c, MAMBA_B200_ERR_DEVICE, "rotary: the handle belongs to device %d but device %d is current", c->device, cur);
    if (!dtype_ok(a.dtype)) return fail(c, MAMBA_B200_ERR_ARG, "rotary: unknown dtype %d", a.dtype);
    if (a.B < 0 || a.T < 0 || a.Hq < 1 || a.Hk < 0 || a.Hq > 65536 || a.Hk > 65536 || a.D < 1 || a.D > 1024)
        return fail(c, MAMBA_B200_ERR_SHAPE, "rotary: B %d T %d heads %d and %d D %d", a.B, a.T, a.Hq, a.Hk, a.D);
    if (a.R < 0 || a.R % 2 || a.R > a.D) return fail(c, MAMBA_B200_ERR_SHAPE, "rotary: %d columns of %d are no pairs", a.R, a.D);
    if (a.B > kMaxSize || a.T > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "rotary: too many steps (%d x %d)", a.B, a.T);
    if (!isfinite(a.scale)) return fail(c, MAMBA_B200_ERR_ARG, "rotary: the scale is not finite");
    if (a.B == 0 || a.T == 0) return MAMBA_B200_OK;
    if (!a.q || !a.q_out || (a.Hk && (!a.k || !a.k_out)) || (a.R && (!a.positions || !a.inv_freq)))
        return fail(c, MAMBA_B200_ERR_ARG, "rotary: null pointer");
    const size_t es = dtype_size(a.dtype);
    if (!aligned_to(es, {a.q, a.q_out, a.k, a.k_out}) || !aligned_to(4, {a.positions, a.inv_freq}))
        return fail(c, MAMBA_B200_ERR_ARG, "rotary: misaligned pointer");
    if (a.q_out == a.q && ((a.B > 1 && a.qo_b != a.q_b) || (a.T > 1 && a.qo_t != a.q_t) || (a.Hq > 1 && a.qo_h != a.q_h)))
        return fail(c, MAMBA_B200_ERR_ARG, "rotary: q_out is q with other strides");
    if (a.Hk && a.k_out == a.k && ((a.B > 1 && a.ko_b != a.k_b) || (a.T > 1 && a.ko_t != a.k_t) || (a.Hk > 1 && a.ko_h != a.k_h)))
        return fail(c, MAMBA_B200_ERR_ARG, "rotary: k_out is k with other strides");
    if (a.Hk && (a.q_out == a.k || a.k_out == a.q || a.q_out == a.k_out))
        return fail(c, MAMBA_B200_ERR_ARG, "rotary: a result of one of q and k is the other's memory");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dtype == MAMBA_B200_F32) return rot::launch_typed<float>(c, a, st);
    if (a.dtype == MAMBA_B200_F16) return rot::launch_typed<__half>(c, a, st);
    return rot::launch_typed<__nv_bfloat16>(c, a, st);
}
