// Linear attention with a decay for each head: entry points, decode step, and the kernel for every size, type and stride.
// The formulas and the roles are in linear_attention.cuh; 16-bit rows that TMA can describe go to linear_attention_tc.cu.
#include <math.h>
#include <string.h>

#include "linear_attention.cuh"

namespace mb200 {
namespace la {

// ---------------------------------------------------------------------------------------------------
// One token for each sequence.  S is read and written once (K * V * 8 bytes a head, beside which nothing counts), so a thread has
// four columns of it (one, where V is no multiple of four) and every row of its row group in flight; the groups' parts of o
// are joined through shared memory in their order.  64 sequences x 32 heads of 128 x 64 bf16 take 23.0 us, 90 % of
// the measured copy rate; 32 heads of one sequence 2.8.
// ---------------------------------------------------------------------------------------------------
constexpr int kStepThreads = 256;

template <typename T, int VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const mamba_b200_linear_attention_args a) {
    __shared__ float qs[kMaxDim], ks[kMaxDim];
    __shared__ float part[kStepThreads * VEC];
    const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, tid = threadIdx.x;
    const int K = a.K, V = a.V, lanes = (V + VEC - 1) / VEC, groups = kStepThreads / lanes;
    const T* q = static_cast<const T*>(a.q) + b * a.q_b + (h / (a.H / a.Hq)) * a.q_h;
    const T* k = static_cast<const T*>(a.k) + b * a.k_b + (h / (a.H / a.Hk)) * a.k_h;
    const T* v = static_cast<const T*>(a.v) + b * a.v_b + (h / (a.H / a.Hv)) * a.v_h;
    const long long at = static_cast<long long>(blockIdx.x) * K * V;
    const int g = tid / lanes, c = (tid - g * lanes) * VEC;
    const bool on = g < groups;
    constexpr int U = 8;  // rows in flight
    float s[U][VEC];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[u][e] = 0.0f;
            if (on && r < K && a.state) {
                const float* p = a.state + at + static_cast<long long>(r) * V + c;
                if (VEC == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(p);
                    s[u][0] = f.x; s[u][1 % VEC] = f.y; s[u][2 % VEC] = f.z; s[u][3 % VEC] = f.w;
                } else {
                    s[u][0] = *p;
                }
            }
        }
    };
    fetch(g);  // (before q, k and v: the state is what takes time)
    const float lam = expf(a.decay[h]);
    if (tid < K) {
        qs[tid] = to_f(q[tid]) * a.scale;
        ks[tid] = to_f(k[tid]);
    }
    float vv[VEC], acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        vv[e] = on ? to_f(v[c + e]) : 0.0f;
        acc[e] = 0.0f;
    }
    __syncthreads();
    for (int r0 = g; r0 < K; r0 += U * groups) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
            if (on && r < K) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s[u][e] = a.state ? fmaf(lam, s[u][e], ks[r] * vv[e]) : ks[r] * vv[e];
                    acc[e] = fmaf(qs[r], s[u][e], acc[e]);
                }
                if (a.state_out) {
                    float* p = a.state_out + at + static_cast<long long>(r) * V + c;
                    if (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(s[u][0], s[u][1 % VEC], s[u][2 % VEC], s[u][3 % VEC]);
                    else *p = s[u][0];
                }
            }
        }
        if (r0 + U * groups < K) fetch(r0 + U * groups);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[tid * VEC + e] = acc[e];
    __syncthreads();
    T* o = static_cast<T*>(a.o) + b * a.o_b + h * a.o_h;
    for (int j = tid; j < V; j += kStepThreads) {
        float sum = 0.0f;
        for (int i = 0; i < groups; ++i) sum += part[i * lanes * VEC + j];
        o[j] = from_f<T>(sum);
    }
}

// ---------------------------------------------------------------------------------------------------
// Any size, type and stride: a block has 32 columns of one pair's state in shared memory and walks chunks of 32 steps,
//   P = mask(X Y^T),  out = P Z + decayed X S,  S <- l^n S + Y^T (weights o Z),
// all in f32 with tiles of registers.  Steps are numbered in the order they are walked, so the roles that run backwards
// differ in what a step's address is alone.  Bound by shared memory, which a load of 16 bytes a lane takes for four cycles: a thread has two
// rows by four columns, so that six loads feed 32 products (one row, five for 16: 3710 us for 3470 at 8 x 4096 x 32 heads of 128 x 64 f32,
// 10640 for 7310 at 4 x 4096 x 16 heads of 256 x 256 f16).  In bf16 the first of them takes 130 on the tensor cores.
// With few pairs the sequence is cut into segments: STATE blocks find what each adds to a state from zero, and the full walk
// starts from the sum of what was before.
// ---------------------------------------------------------------------------------------------------
constexpr int kCols = 32, kThreads = 128, kRows = 16;  // a thread has rows i and i + kRows of a chunk

inline size_t gen_smem(int A) { return sizeof(float) * (2 * kSteps * (A + 4) + 2 * kSteps * kCols + kSteps * (kSteps + 4) + A * kCols + 3 * kSteps); }

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
template <typename T, int NA, bool STATE>
__global__ void __launch_bounds__(kThreads, NA == 4 ? 3 : 2) general_kernel(const Params p) {
    extern __shared__ __align__(16) float sm[];
    const Place w = place(p, blockIdx.x, STATE ? p.segments - 1 : p.segments);
    const Role& r = p.role[w.role];
    const int tid = threadIdx.x, A = r.A, Ar = (A + 3) & ~3, LD = Ar + 4, W = r.W;
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
        __syncthreads();  // the last chunk's readers of X, Y, Z, Zw; the state and the powers are whole
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
        __syncthreads();
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
            __syncthreads();
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
            __syncthreads();  // every reader of S
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
    __syncthreads();
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

// A thread has one element of a pair's state (whatever its place in a slot means) and eight segments' in flight; the blocks that
// start from it read one slot then, not all that are before them.
__global__ void __launch_bounds__(256) chain_kernel(const Params p) {
    const Role& r = p.role[blockIdx.y];
    const int size = r.A * r.W, per = (size + 255) / 256;
    const long long pair = blockIdx.x / per;
    const int e = (blockIdx.x - static_cast<int>(pair) * per) * 256 + threadIdx.x;
    if (pair >= static_cast<long long>(p.B) * p.H || e >= size) return;
    float* s = r.slots + pair * p.segments * size + e;
    const Pow f = decay_pow(p.decay[pair % p.H], p.seg_len);
    constexpr int U = 8;
    float run = s[size];
    for (int k = 2; k < p.segments; k += U) {
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = k + u < p.segments ? s[static_cast<long long>(k + u) * size] : 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k + u < p.segments) {
                run = times(f, run) + x[u];
                s[static_cast<long long>(k + u) * size] = run;
            }
    }
}

// Gradients of shared heads: the heads' f32 parts [B, T, H, D], summed in their order.
template <typename T>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* __restrict__ part, T* out, long long ob, long long ot, long long oh,
                                                        long long rows, int T_, int heads, int group, int D) {
    const long long total = rows * heads * D;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int d = static_cast<int>(i % D);
        const long long rh = i / D;
        const int h = static_cast<int>(rh % heads);
        const long long row = rh / heads;
        const float* src = part + (row * heads + h) * group * D + d;
        float s = 0.0f;
        for (int g = 0; g < group; ++g) s += src[static_cast<long long>(g) * D];
        out[(row / T_) * ob + (row % T_) * ot + h * oh + d] = from_f<T>(s);
    }
}

// ---------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------
inline long long up256(long long n) { return (n + 255) / 256 * 256; }

// Segments of a sequence at the most: two blocks an SM, were a pair one block.
inline long long most_segments(long long pairs) {
    const long long n = pairs > 0 ? 2 * 148 / pairs : 1;
    return n < 1 ? 1 : n < kMaxSegments ? n : kMaxSegments;
}

// What a call's scratch holds: the states between segments of each role, and the f32 parts of shared heads' gradients.
struct Room {
    long long slots = 0, parts[3] = {0, 0, 0};
    long long total() const { return slots + parts[0] + parts[1] + parts[2]; }
};
inline Room room(const mamba_b200_linear_attention_args& a, int backward) {
    Room r;
    const long long pairs = static_cast<long long>(a.B) * a.H;
    // (pick_segments() takes no more)
    const long long units = (static_cast<long long>(a.T) + kSteps - 1) / kSteps, most = most_segments(pairs);
    const long long n = units < most ? units : most;
    if (n > 1) r.slots = up256(pairs * n * a.K * a.V * 4) * (backward ? 3 : 1);
    if (backward) {
        const long long rows = static_cast<long long>(a.B) * a.T * a.H * 4;
        if (a.Hq < a.H) r.parts[0] = up256(rows * a.K);
        if (a.Hk < a.H) r.parts[1] = up256(rows * a.K);
        if (a.Hv < a.H) r.parts[2] = up256(rows * a.V);
    }
    return r;
}

int chain_segments(Ctx* c, const Params& p, long long pairs, cudaStream_t st) {
    if (p.segments < 3) return MAMBA_B200_OK;
    int most = 0;
    for (int i = 0; i < p.roles; ++i) most = p.role[i].A * p.role[i].W > most ? p.role[i].A * p.role[i].W : most;
    chain_kernel<<<dim3(static_cast<unsigned>(pairs * ((most + 255) / 256)), p.roles), 256, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

// Segments of a sequence of `units` chunks whose uncut launch has `blocks` blocks, of which `together` run at once: the number that is
// estimated to take least, from the times of a chunk walked in full and for its state alone and what a second kernel costs (us).
int pick_segments(long long together, long long blocks, int units, long long pairs, double full, double state, double second) {
    const long long most = most_segments(pairs);
    int best = 1;
    double best_us = 1e30;
    for (int n = 1; n <= most && n <= units; ++n) {
        const int per = (units + n - 1) / n;
        const double waves = static_cast<double>((blocks * n + together - 1) / together);
        const double us = n == 1 ? waves * per * full : second + waves * per * (full + state);
        if (us < 0.97 * best_us) {
            best = n;
            best_us = us;
        }
    }
    return best;
}

template <typename T>
int launch_general(Ctx* c, Params& p, bool may_cut, long long pairs, cudaStream_t st) {
    int A = 0;
    p.tiles = 0;
    for (int i = 0; i < p.roles; ++i) {
        p.role[i].tiles = (p.role[i].W + kCols - 1) / kCols;
        p.tiles += p.role[i].tiles;
        if (p.role[i].A > A) A = p.role[i].A;
    }
    const long long blocks = pairs * p.tiles;
    // (chunks of 32; two blocks on an SM work at their own speed)
    const int units = (p.T + kSteps - 1) / kSteps;
    const double width = A / 128.0 + 0.4;
    p.segments = may_cut ? pick_segments(2 * c->sm_count, blocks, units, pairs, 4.0 * width, 1.5 * width, 6.0) : 1;
    const int per = (units + p.segments - 1) / p.segments;
    p.segments = (units + per - 1) / per;
    p.seg_len = per * kSteps;
    if (blocks * p.segments > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "linear_attention: too many heads");
    const size_t smem = gen_smem((A + 3) & ~3);
    const unsigned grid = static_cast<unsigned>(blocks * p.segments), before = static_cast<unsigned>(blocks * (p.segments - 1));
    if (before) {
        if (A <= 128) general_kernel<T, 4, true><<<before, kThreads, smem, st>>>(p);
        else general_kernel<T, 8, true><<<before, kThreads, smem, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        const int rc = chain_segments(c, p, pairs, st);
        if (rc) return rc;
    }
    if (A <= 128) general_kernel<T, 4, false><<<grid, kThreads, smem, st>>>(p);
    else general_kernel<T, 8, false><<<grid, kThreads, smem, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

template <typename T>
int launch_step(Ctx* c, const mamba_b200_linear_attention_args& a, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.B) * a.H;
    if (a.V % 4 == 0 && aligned_to(16, {a.state, a.state_out})) step_kernel<T, 4><<<grid, kStepThreads, 0, st>>>(a);
    else step_kernel<T, 1><<<grid, kStepThreads, 0, st>>>(a);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

template <typename T>
int sum_heads(Ctx* c, const float* part, void* out, long long ob, long long ot, long long oh, const mamba_b200_linear_attention_args& a, int heads,
              int D, cudaStream_t st) {
    const long long rows = static_cast<long long>(a.B) * a.T, blocks = (rows * heads * D + 255) / 256;
    const long long most = 32ll * c->sm_count;
    sum_heads_kernel<T><<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, st>>>(part, static_cast<T*>(out), ob, ot, oh, rows, a.T, heads,
                                                                                             a.H / heads, D);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

// Rows of a tensor that a launch of this many steps, heads and sequences may touch, checked against the type's reach.
int check(Ctx* c, const mamba_b200_linear_attention_args* a, bool backward) {
    const char* what = backward ? "linear_attention_bwd" : "linear_attention_fwd";
    int cur = -1;
    MB200_CUDA_CHECK(c, cudaGetDevice(&cur));
    if (cur != c->device)
        return fail(c, MAMBA_B200_ERR_DEVICE, "%s: the handle belongs to device %d but device %d is current", what, c->device, cur);
    if (!dtype_ok(a->dtype)) return fail(c, MAMBA_B200_ERR_ARG, "%s: unknown dtype %d", what, a->dtype);
    if (a->B < 0 || a->T < 0 || a->H < 1 || a->K < 1 || a->V < 1)
        return fail(c, MAMBA_B200_ERR_SHAPE, "%s: B %d T %d H %d K %d V %d", what, a->B, a->T, a->H, a->K, a->V);
    if (a->K > kMaxDim || a->V > kMaxDim) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: K %d and V %d are at most %d", what, a->K, a->V, kMaxDim);
    if (a->T > kMaxSize) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: too many steps (%d)", what, a->T);
    if (static_cast<long long>(a->B) * a->H > 1000000) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: too many sequences x heads (%d x %d)", what, a->B, a->H);
    for (int h : {a->Hq, a->Hk, a->Hv})
        if (h < 1 || a->H % h) return fail(c, MAMBA_B200_ERR_SHAPE, "%s: %d heads are not shared by %d evenly", what, h, a->H);
    if (!isfinite(a->scale)) return fail(c, MAMBA_B200_ERR_ARG, "%s: the scale is not finite", what);
    if (a->B == 0) return MAMBA_B200_OK;
    const bool some = a->T > 0;
    if (!a->decay || (some && (!a->q || !a->k || !a->v))) return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", what);
    if (some && !backward && !a->o) return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", what);
    if (some && backward && (!a->d_o || !a->d_q || !a->d_k || !a->d_v)) return fail(c, MAMBA_B200_ERR_ARG, "%s: null pointer", what);
    if (backward && a->d_state && a->d_state == a->d_state_out)
        return fail(c, MAMBA_B200_ERR_ARG, "%s: d_state and d_state_out are the same memory", what);
    const size_t es = dtype_size(a->dtype);
    if (!aligned_to(es, {a->q, a->k, a->v}) || !aligned_to(es, {backward ? a->d_o : a->o}) ||
        (backward && !aligned_to(es, {a->d_q, a->d_k, a->d_v})) || !aligned_to(4, {a->decay, a->state}) ||
        !aligned_to(4, {backward ? nullptr : a->state_out, backward ? a->d_state : nullptr, backward ? a->d_state_out : nullptr}))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: misaligned pointer", what);
    if (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 256) return fail(c, MAMBA_B200_ERR_ARG, "%s: misaligned workspace", what);
    if (backward && a->d_state && a->d_state == a->state) return fail(c, MAMBA_B200_ERR_ARG, "%s: d_state and state are the same memory", what);
    // (blocks of one head read what others have read: nothing may be written there)
    for (const void* in : {a->q, a->k, a->v, backward ? a->d_o : a->q})
        for (const void* out : {backward ? a->d_q : a->o, backward ? a->d_k : a->o, backward ? a->d_v : a->o})
            if (some && in == out) return fail(c, MAMBA_B200_ERR_ARG, "%s: a result and an input are the same memory", what);
    if (some && backward && (a->d_q == a->d_k || a->d_q == a->d_v || a->d_k == a->d_v))
        return fail(c, MAMBA_B200_ERR_ARG, "%s: two results are the same memory", what);
    return MAMBA_B200_OK;
}

// T = 0: a state goes from `in` to `out`.
int hand_on(Ctx* c, const float* in, float* out, const mamba_b200_linear_attention_args& a, cudaStream_t st) {
    if (!out || in == out) return MAMBA_B200_OK;
    const size_t bytes = sizeof(float) * static_cast<size_t>(a.B) * a.H * a.K * a.V;
    if (in) MB200_CUDA_CHECK(c, cudaMemcpyAsync(out, in, bytes, cudaMemcpyDeviceToDevice, st));
    else MB200_CUDA_CHECK(c, cudaMemsetAsync(out, 0, bytes, st));
    return MAMBA_B200_OK;
}

int dispatch(Ctx* c, const mamba_b200_linear_attention_args& a, Params& p, bool may_cut, cudaStream_t st) {
    const long long pairs = static_cast<long long>(a.B) * a.H;
    bool taken = false;
    const int rc = tc_launch(c, a.dtype, p, may_cut, pairs, st, &taken);
    if (rc || taken) return rc;
    if (a.dtype == MAMBA_B200_F32) return launch_general<float>(c, p, may_cut, pairs, st);
    if (a.dtype == MAMBA_B200_F16) return launch_general<__half>(c, p, may_cut, pairs, st);
    return launch_general<__nv_bfloat16>(c, p, may_cut, pairs, st);
}

}  // namespace la

int linear_attention_configure(Ctx* c) {
    const int most = static_cast<int>(la::gen_smem(la::kMaxDim));
#define MB200_LA(T, NA)                                                                                                                          \
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)la::general_kernel<T, NA, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)); \
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)la::general_kernel<T, NA, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    MB200_LA(float, 4) MB200_LA(float, 8) MB200_LA(__half, 4) MB200_LA(__half, 8) MB200_LA(__nv_bfloat16, 4) MB200_LA(__nv_bfloat16, 8)
#undef MB200_LA
    return MAMBA_B200_OK;
}

}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API long long mamba_b200_linear_attention_workspace_bytes(const mamba_b200_linear_attention_args* a, int backward) {
    if (!a || a->B < 1 || a->T < 1 || a->H < 1 || a->K < 1 || a->V < 1 || a->K > la::kMaxDim || a->V > la::kMaxDim || a->T > kMaxSize ||
        static_cast<long long>(a->B) * a->H > 1000000)
        return 0;
    return la::room(*a, backward).total();
}

extern "C" MAMBA_B200_API int mamba_b200_linear_attention_fwd(void* handle, void* stream, const mamba_b200_linear_attention_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = la::check(c, args, false);
    if (rc || args->B == 0) return rc;
    const mamba_b200_linear_attention_args& a = *args;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.T == 0) return la::hand_on(c, a.state, a.state_out, a, st);
    if (a.T == 1) {
        if (a.dtype == MAMBA_B200_F32) return la::launch_step<float>(c, a, st);
        if (a.dtype == MAMBA_B200_F16) return la::launch_step<__half>(c, a, st);
        return la::launch_step<__nv_bfloat16>(c, a, st);
    }
    la::Params p;
    memset(&p, 0, sizeof(p));
    p.roles = 1;
    p.B = a.B; p.T = a.T; p.H = a.H;
    p.decay = a.decay;
    p.status = c->d_status;
    la::Role& r = p.role[0];
    r.x = {a.q, a.q_b, a.q_t, a.q_h, a.H / a.Hq, a.K};
    r.y = {a.k, a.k_b, a.k_t, a.k_h, a.H / a.Hk, a.K};
    r.z = {a.v, a.v_b, a.v_t, a.v_h, a.H / a.Hv, a.V};
    r.A = a.K; r.W = a.V;
    r.out = a.o; r.ob = a.o_b; r.ot = a.o_t; r.oh = a.o_h;
    r.s_in = a.state; r.sa = a.V; r.sw = 1;
    r.s_out = a.state_out;
    r.alpha_p = r.alpha_x = r.alpha_z = a.scale;
    r.alpha_s = 1.0f;
    const la::Room room = la::room(a, 0);
    const bool may_cut = room.slots > 0 && a.workspace && a.workspace_bytes >= room.slots;
    if (may_cut) r.slots = static_cast<float*>(a.workspace);
    return la::dispatch(c, a, p, may_cut, st);
}

extern "C" MAMBA_B200_API int mamba_b200_linear_attention_bwd(void* handle, void* stream, const mamba_b200_linear_attention_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    int rc = la::check(c, args, true);
    if (rc || args->B == 0) return rc;
    const mamba_b200_linear_attention_args& a = *args;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.T == 0) return la::hand_on(c, a.d_state_out, a.d_state, a, st);
    const la::Room room = la::room(a, 1);
    const long long parts = room.parts[0] + room.parts[1] + room.parts[2];
    if (parts && (!a.workspace || a.workspace_bytes < room.total()))
        return fail(c, MAMBA_B200_ERR_ARG, "linear_attention_bwd: shared heads need a workspace of %lld bytes (%lld given)", room.total(),
                    a.workspace ? a.workspace_bytes : 0ll);
    const bool may_cut = room.slots > 0 && a.workspace && a.workspace_bytes >= room.total();
    char* ws = static_cast<char*>(a.workspace);
    float* part[3] = {nullptr, nullptr, nullptr};
    char* at = ws + room.slots;
    for (int i = 0; i < 3; ++i)
        if (room.parts[i]) {
            part[i] = reinterpret_cast<float*>(at);
            at += room.parts[i];
        }
    la::Params p;
    memset(&p, 0, sizeof(p));
    p.roles = 3;
    p.B = a.B; p.T = a.T; p.H = a.H;
    p.decay = a.decay;
    p.status = c->d_status;
    const la::Operand q = {a.q, a.q_b, a.q_t, a.q_h, a.H / a.Hq, a.K}, k = {a.k, a.k_b, a.k_t, a.k_h, a.H / a.Hk, a.K};
    const la::Operand v = {a.v, a.v_b, a.v_t, a.v_h, a.H / a.Hv, a.V}, d = {a.d_o, a.do_b, a.do_t, a.do_h, 1, a.V};
    void* outs[3] = {a.d_q, a.d_k, a.d_v};
    const long long strides[3][3] = {{a.dq_b, a.dq_t, a.dq_h}, {a.dk_b, a.dk_t, a.dk_h}, {a.dv_b, a.dv_t, a.dv_h}};
    const int heads[3] = {a.Hq, a.Hk, a.Hv};
    for (int i = 0; i < 3; ++i) {
        la::Role& r = p.role[i];
        r.A = i == 2 ? a.K : a.V;
        r.W = i == 2 ? a.V : a.K;
        r.x = i == 0 ? d : i == 1 ? v : k;
        r.y = i == 0 ? v : i == 1 ? d : q;
        r.z = i == 0 ? k : i == 1 ? q : d;
        if (part[i]) {
            r.out = part[i];
            r.out_f32 = 1;
            r.oh = r.W;
            r.ot = static_cast<long long>(a.H) * r.W;
            r.ob = a.T * r.ot;
        } else {
            r.out = outs[i];
            r.ob = strides[i][0]; r.ot = strides[i][1]; r.oh = strides[i][2];
        }
        r.s_in = i == 0 ? a.state : a.d_state_out;
        r.sa = i == 2 ? a.V : 1;
        r.sw = i == 2 ? 1 : a.V;
        r.s_out = i == 2 ? a.d_state : nullptr;
        r.backwards = i > 0;
        r.late = i > 0;
        r.last_decay = i == 2;
        r.alpha_p = a.scale;
        r.alpha_x = i == 0 ? a.scale : 1.0f;
        r.alpha_s = i == 0 ? 1.0f : a.scale;
        r.alpha_z = i == 0 ? a.scale : 1.0f;
        if (may_cut) r.slots = reinterpret_cast<float*>(ws + room.slots / 3 * i);
    }
    rc = la::dispatch(c, a, p, may_cut, st);
    for (int i = 0; i < 3 && !rc; ++i)
        if (part[i]) {
            const int D = i == 2 ? a.V : a.K;
            if (a.dtype == MAMBA_B200_F32) rc = la::sum_heads<float>(c, part[i], outs[i], strides[i][0], strides[i][1], strides[i][2], a, heads[i], D, st);
            else if (a.dtype == MAMBA_B200_F16) rc = la::sum_heads<__half>(c, part[i], outs[i], strides[i][0], strides[i][1], strides[i][2], a, heads[i], D, st);
            else rc = la::sum_heads<__nv_bfloat16>(c, part[i], outs[i], strides[i][0], strides[i][1], strides[i][2], a, heads[i], D, st);
        }
    return rc;
}
