// Linear attention with a decay for each head: entry points, decode step, and the kernel for every size, type and stride.
// The formulas and the roles are in linear_attention.cuh; 16-bit rows that TMA can describe go to linear_attention_tc.cu.
#include <math.h>
#include <string.h>

#include "linear_attention_general.cuh"

namespace mb200 {
namespace la {

// ---------------------------------------------------------------------------------------------------
// One token for each sequence.  S is read and written once (K * V * 8 bytes a head, beside which nothing counts), so a thread has
// four columns of it (one, where V is no multiple of four) and every row of its row group in flight; the groups' parts of o
// are joined through shared memory in their order.  64 sequences x 32 heads of 128 x 64 bf16 take 21.2 to 23.0 us, 90 % of
// the measured copy rate and more (the last states are still in L2 when it ends); 32 heads of one sequence 3.2.
// ---------------------------------------------------------------------------------------------------
constexpr int kStepThreads = 256;

template <typename T, int VEC>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const mamba_b200_linear_attention_args a) {
    __shared__ float qs[kMaxDim], ks[kMaxDim];
    __shared__ float part[kStepThreads * VEC];
    __shared__ Pow factor;  // (two floats: the rounding of one, always the same way, would add up: to 1.4e-4 over 6000 steps at 1 - 2^-12)
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
    if (tid == kStepThreads - 1) factor = decay_pow(a.decay[h], 1);
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
    const Pow lam = factor;
    for (int r0 = g; r0 < K; r0 += U * groups) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
            if (on && r < K) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s[u][e] = a.state ? fmaf(lam.hi, s[u][e], fmaf(lam.lo, s[u][e], ks[r] * vv[e])) : ks[r] * vv[e];
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
// Any size, type and stride (linear_attention_general.cuh).
// ---------------------------------------------------------------------------------------------------
template <typename T, int NA, bool STATE>
__global__ void __launch_bounds__(gen::kThreads, NA == 4 ? 3 : 2) general_kernel(const Params p) {
    extern __shared__ __align__(16) float sm[];
    gen::walk<T, NA, STATE>(p, place(p, blockIdx.x, STATE ? p.segments - 1 : p.segments), sm, threadIdx.x, 0);
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
        p.role[i].tiles = (p.role[i].W + gen::kCols - 1) / gen::kCols;
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
    const size_t smem = gen::smem_bytes((A + 3) & ~3);
    const unsigned grid = static_cast<unsigned>(blocks * p.segments), before = static_cast<unsigned>(blocks * (p.segments - 1));
    if (before) {
        if (A <= 128) general_kernel<T, 4, true><<<before, gen::kThreads, smem, st>>>(p);
        else general_kernel<T, 8, true><<<before, gen::kThreads, smem, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        const int rc = chain_segments(c, p, pairs, st);
        if (rc) return rc;
    }
    if (A <= 128) general_kernel<T, 4, false><<<grid, gen::kThreads, smem, st>>>(p);
    else general_kernel<T, 8, false><<<grid, gen::kThreads, smem, st>>>(p);
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
    const int most = static_cast<int>(la::gen::smem_bytes(la::kMaxDim));
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
