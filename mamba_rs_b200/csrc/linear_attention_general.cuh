// Linear attention on CUDA cores, for any size, type and stride: 128 threads have 32 columns of one pair's state in shared memory and walks chunks of 32 steps,
//   P = mask(X Y^T),  out = P Z + decayed X S,  S <- l^n S + Y^T (weights o Z),
// all in f32 with tiles of registers.  Steps are numbered in the order they are walked, so the roles that run backwards
// differ in what a step's address is alone.  Bound by shared memory, which a load of 16 bytes a lane takes for four cycles: a thread has two
// rows by four columns, so that six loads feed 32 products (one row, five for 16: 3710 us for 3470 at 8 x 4096 x 32 heads of 128 x 64 f32,
// 10640 for 7310 at 4 x 4096 x 16 heads of 256 x 256 f16).  In bf16 the first of them takes 130 on the tensor cores.
// With few pairs the sequence is cut into segments: STATE blocks find what each adds to a state from zero, and the full walk
// starts from the sum of what was before.
#pragma once
#include "linear_attention.cuh"

namespace mb200 {
namespace la {
namespace gen {

constexpr int kCols = 32, kThreads = 128, kRows = 16;  // a thread has rows i and i + kRows of a chunk

// (A: a multiple of four)
inline __host__ __device__ constexpr size_t smem_bytes(int A) { return sizeof(float) * (2 * kSteps * (A + 4) + 2 * kSteps * kCols + kSteps * (kSteps + 4) + A * kCols + 3 * kSteps); }

// Four neighbouring elements, of which n are there (vec: they are one aligned piece).
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int n, bool vec) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (vec && n >= 4) {
        const float2 lo = ld_pair(p), hi = ld_pair(p + 2);
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) v[e] = to_f(p[e]);
    return make_float4(v[0], v[1], v[2], v[3]);
}

// NA: blocks of 32 columns of X and Y (4 or 8).  With 4 a chunk's rows are asked for while the one before is worked on.
// w.tile: 32 columns; sm: smem_bytes(A) bytes; tid: 0 to 127; barrier: one that these threads alone meet at.
template <typename T, int NA, bool STATE>
__device__ __forceinline__ void walk(const Params& p, const Place w, float* sm, const int tid, const int barrier) {
    auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kThreads) : "memory"); };
    const Role& r = p.role[w.role];
    const int A = r.A, Ar = (A + 3) & ~3, LD = Ar + 4, W = r.W;
    const int b = static_cast<int>(w.pair / p.H), h = static_cast<int>(w.pair - static_cast<long long>(b) * p.H);
    const int c0 = w.tile * kCols, nc = min(kCols, W - c0);
    float* X = sm;
    float* Y = X + kSteps * LD;
    float* Z = Y + kSteps * LD;
    float* Zw = Z + kSteps * kCols;
    float* P = Zw + kSteps * kCols;
    float* S = P + kSteps * (kSteps + 4);
    float* pw = S + Ar * kCols;  // l^i, i <= kSteps
    const float ld = p.decay[h], l2 = ld * kLog2e;
    const int t_lo = w.seg * p.seg_len, t_hi = min(p.T, t_lo + p.seg_len);
    const int i4 = tid >> 3, j8 = tid & 7, w4 = j8 * 4;
    // this thread's pieces of a chunk: rows i4 and i4 + kRows, four columns at w4 of every 32
    auto row = [&](int t) { return r.backwards ? p.T - 1 - t : t; };
    const T* xg = static_cast<const T*>(r.x.p) + b * r.x.sb + (h / r.x.group) * r.x.sh + w4;
    const T* yg = static_cast<const T*>(r.y.p) + b * r.y.sb + (h / r.y.group) * r.y.sh + w4;
    const T* zg = static_cast<const T*>(r.z.p) + b * r.z.sb + (h / r.z.group) * r.z.sh + c0 + w4;
    auto whole = [](const T* q, long long st) { return ((reinterpret_cast<uintptr_t>(q) | st * sizeof(T)) & (2 * sizeof(T) - 1)) == 0; };
    const bool vx = whole(xg, r.x.st), vy = whole(yg, r.y.st), vz = whole(zg, r.z.st);
    float4 xr[2][NA], yr[2][NA], zr[2];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = t0 + i4 + kRows * e;
            const bool ok = t < t_hi;
            const long long at = ok ? row(t) : 0;
#pragma unroll
            for (int m = 0; m < NA; ++m) {
                const int n = ok ? A - w4 - 32 * m : 0;
                if (!STATE) xr[e][m] = load4(xg + at * r.x.st + 32 * m, n, vx);
                yr[e][m] = load4(yg + at * r.y.st + 32 * m, n, vy);
            }
            zr[e] = load4(zg + at * r.z.st, ok ? nc - w4 : 0, vz);
        }
    };
    fetch(t_lo);
    if (tid <= kSteps) pw[tid] = decay_at(l2, tid);
    // the state that enters this segment
    const long long slot = static_cast<long long>(A) * W;
    float* slots = r.slots ? r.slots + w.pair * p.segments * slot : nullptr;
    const bool first = w.seg == 0;
    const Pow per_chunk = decay_pow(ld, kSteps);
    bool entered = false;
    if (first ? r.s_in != nullptr : !STATE) entered = true;
    for (int i = tid; i < Ar * kCols; i += kThreads) {
        const int a = i / kCols, c = i % kCols;
        float s = 0.0f;
        if (a < A && c < nc && entered) {
            const long long e = static_cast<long long>(a) * W + c0 + c;
            if (first && (STATE || p.segments == 1)) s = r.s_in[w.pair * slot + static_cast<long long>(a) * r.sa + static_cast<long long>(c0 + c) * r.sw];
            else s = slots[w.seg * slot + e];
            if (STATE && first) slots[e] = s;
        }
        S[i] = s;
    }
    for (int t0 = t_lo; t0 < t_hi; t0 += kSteps) {
        const int n = min(kSteps, t_hi - t0);
        const int late = r.late && first && t0 == t_lo ? 1 : 0;
        if (NA > 4 && t0 > t_lo) fetch(t0);
        meet();  // the last chunk's readers of X, Y, Z, Zw; the state and the powers are whole
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = i4 + kRows * e;
#pragma unroll
            for (int m = 0; m < NA; ++m)
                if (w4 + 32 * m < Ar) {
                    if (!STATE) *reinterpret_cast<float4*>(X + i * LD + w4 + 32 * m) = xr[e][m];
                    *reinterpret_cast<float4*>(Y + i * LD + w4 + 32 * m) = yr[e][m];
                }
            const float f = i < n ? pw[n - 1 - i] * r.alpha_s : 0.0f;
            *reinterpret_cast<float4*>(Z + i * kCols + w4) = zr[e];
            *reinterpret_cast<float4*>(Zw + i * kCols + w4) = make_float4(zr[e].x * f, zr[e].y * f, zr[e].z * f, zr[e].w * f);
        }
        meet();
        if (NA == 4 && t0 + kSteps < t_hi) fetch(t0 + kSteps);
        if (!STATE) {
            // P[i][j8 + 8 m]
            float g[2][4] = {};
            for (int a = 0; a < Ar; a += 4) {
                float4 x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) x[e] = *reinterpret_cast<const float4*>(X + (i4 + kRows * e) * LD + a);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const float4 y = *reinterpret_cast<const float4*>(Y + (j8 + 8 * m) * LD + a);
#pragma unroll
                    for (int e = 0; e < 2; ++e) g[e][m] = fmaf(x[e].x, y.x, fmaf(x[e].y, y.y, fmaf(x[e].z, y.z, fmaf(x[e].w, y.w, g[e][m]))));
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int i = i4 + kRows * e, j = j8 + 8 * m;
                    P[i * (kSteps + 4) + j] = j <= i ? g[e][m] * (pw[max(i - j, 0)] * r.alpha_p) : 0.0f;
                }
            meet();
            float o[2][4] = {};
            auto add = [&](int e, float q, const float4& z) {
                o[e][0] = fmaf(q, z.x, o[e][0]);
                o[e][1] = fmaf(q, z.y, o[e][1]);
                o[e][2] = fmaf(q, z.z, o[e][2]);
                o[e][3] = fmaf(q, z.w, o[e][3]);
            };
            if (entered || t0 > t_lo) {
                for (int a = 0; a < Ar; a += 4) {
                    float xv[2][4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float4 x = *reinterpret_cast<const float4*>(X + (i4 + kRows * e) * LD + a);
                        xv[e][0] = x.x; xv[e][1] = x.y; xv[e][2] = x.z; xv[e][3] = x.w;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float4 s = *reinterpret_cast<const float4*>(S + (a + u) * kCols + w4);
#pragma unroll
                        for (int e = 0; e < 2; ++e) add(e, xv[e][u], s);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = pw[i4 + kRows * e + 1 - late] * r.alpha_x;
#pragma unroll
                    for (int u = 0; u < 4; ++u) o[e][u] *= f;
                }
            }
            // (no row meets a later one's values, which may be infinite)
            for (int j = 0; j <= i4; ++j) {
                const float4 z = *reinterpret_cast<const float4*>(Z + j * kCols + w4);
                add(0, P[i4 * (kSteps + 4) + j], z);
                add(1, P[(i4 + kRows) * (kSteps + 4) + j], z);
            }
            for (int j = i4 + 1; j <= i4 + kRows; ++j)
                add(1, P[(i4 + kRows) * (kSteps + 4) + j], *reinterpret_cast<const float4*>(Z + j * kCols + w4));
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (i4 + kRows * e < n) {
                    const long long at = b * r.ob + row(t0 + i4 + kRows * e) * r.ot + h * r.oh + c0 + w4;
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (w4 + u < nc) {
                            if (r.out_f32) static_cast<float*>(r.out)[at + u] = o[e][u];
                            else static_cast<T*>(r.out)[at + u] = from_f<T>(o[e][u]);
                        }
                }
            meet();  // every reader of S
        }
        // S[a4 .. a4 + 3][w4 .. w4 + 3]
        if (STATE || t0 + n < t_hi || (w.seg + 1 == p.segments && r.s_out)) {
            const Pow f = n - late == kSteps ? per_chunk : decay_pow(ld, n - late);
            for (int a4 = 4 * i4; a4 < Ar; a4 += 4 * (kThreads / 8)) {
                float4 s[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    s[u] = *reinterpret_cast<const float4*>(S + (a4 + u) * kCols + w4);
                    if (entered || t0 > t_lo) s[u] = make_float4(times(f, s[u].x), times(f, s[u].y), times(f, s[u].z), times(f, s[u].w));
                }
                for (int j = 0; j < n; ++j) {
                    const float4 y = *reinterpret_cast<const float4*>(Y + j * LD + a4);
                    const float4 z = *reinterpret_cast<const float4*>(Zw + j * kCols + w4);
                    const float yv[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        s[u].x = fmaf(yv[u], z.x, s[u].x);
                        s[u].y = fmaf(yv[u], z.y, s[u].y);
                        s[u].z = fmaf(yv[u], z.z, s[u].z);
                        s[u].w = fmaf(yv[u], z.w, s[u].w);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) *reinterpret_cast<float4*>(S + (a4 + u) * kCols + w4) = s[u];
            }
        }
    }
    meet();
    float* out = nullptr;
    Pow f{1.0f, 0.0f};
    if (STATE) out = slots + (w.seg + 1) * slot;
    else if (w.seg + 1 == p.segments && r.s_out) {
        out = r.s_out + w.pair * slot;
        if (r.last_decay) f = decay_pow(ld, 1);
    }
    if (out)
        for (int i = tid; i < A * kCols; i += kThreads) {
            const int a = i / kCols, c = i % kCols;
            if (c < nc) out[static_cast<long long>(a) * W + c0 + c] = times(f, S[i]);
        }
}

}  // namespace gen
}  // namespace la
}  // namespace mb200
