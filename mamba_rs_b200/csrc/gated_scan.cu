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

constexpr int kSave = MAMBA_B200_GATED_SCAN_SAVE;

__device__ __forceinline__ float gate_u(float f) { return 1.0f / (1.0f + ex2(f * kLog2e)); }

template <typename T>
__global__ void __launch_bounds__(128) gated_scan_fwd_kernel(const mamba_b200_gated_scan_args p) {
    const long long i = blockIdx.x * 128ll + threadIdx.x;
    if (i >= static_cast<long long>(p.B) * p.D) return;
    const long long b = i / p.D;
    const int d = static_cast<int>(i - b * p.D);
    const T *x = static_cast<const T*>(p.x), *f = static_cast<const T*>(p.f), *z = static_cast<const T*>(p.z);
    T* y = static_cast<T*>(p.y);
    const int blocks = (p.T + kSave - 1) / kSave;
    float h = p.h0 ? p.h0[i] : 0.0f;
    for (int t = 0; t < p.T; ++t) {
        const long long r = b * p.T + t;
        if (p.chunk_states && t % kSave == 0) p.chunk_states[(b * blocks + t / kSave) * p.D + d] = h;
        const float u = gate_u(to_f(f[r * p.ld_f + d]));
        h = fmaf(u, to_f(x[r * p.ld_x + d]) - h, h);
        y[r * p.ld_y + d] = from_f<T>(z ? h * siluf_fast(to_f(z[r * p.ld_z + d])) : h);
    }
    if (p.h_last) p.h_last[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(128) gated_scan_bwd_kernel(const mamba_b200_gated_scan_args p) {
    const long long i = blockIdx.x * 128ll + threadIdx.x;
    if (i >= static_cast<long long>(p.B) * p.D) return;
    const long long b = i / p.D;
    const int d = static_cast<int>(i - b * p.D);
    const T *x = static_cast<const T*>(p.x), *f = static_cast<const T*>(p.f), *z = static_cast<const T*>(p.z), *dy = static_cast<const T*>(p.dy);
    T *dx = static_cast<T*>(p.d_x), *df = static_cast<T*>(p.d_f), *dz = static_cast<T*>(p.d_z);
    const int blocks = (p.T + kSave - 1) / kSave;
    float g = p.d_last ? p.d_last[i] : 0.0f, hs[kSave];
    for (int k = blocks - 1; k >= 0; --k) {
        const float h_in = p.chunk_states[(b * blocks + k) * p.D + d];
        const int n = min(kSave, p.T - k * kSave);
        float h = h_in;
        for (int j = 0; j < n; ++j) {
            const long long r = b * p.T + k * kSave + j;
            h = fmaf(gate_u(to_f(f[r * p.ld_f + d])), to_f(x[r * p.ld_x + d]) - h, h);
            hs[j] = h;
        }
        for (int j = n - 1; j >= 0; --j) {
            const long long r = b * p.T + k * kSave + j;
            const float u = gate_u(to_f(f[r * p.ld_f + d])), xv = to_f(x[r * p.ld_x + d]);
            float e = to_f(dy[r * p.ld_dy + d]);
            if (z) {
                const float zv = to_f(z[r * p.ld_z + d]), q = sigmoidf_fast(zv);
                dz[r * p.ld_dz + d] = from_f<T>(e * hs[j] * q * (1.0f + zv * (1.0f - q)));
                e *= zv * q;
            }
            g += e;
            dx[r * p.ld_dx + d] = from_f<T>(g * u);
            df[r * p.ld_df + d] = from_f<T>(g * ((j ? hs[j - 1] : h_in) - xv) * u * (1.0f - u));
            g = fmaf(-u, g, g);
        }
    }
    if (p.d_h0) p.d_h0[i] = g;
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

}  // namespace gs
}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API int mamba_b200_gated_scan_fwd(void* handle, void* stream, const mamba_b200_gated_scan_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gs::check(c, args, false);
    if (rc || args->B == 0) return rc;
    const unsigned grid = static_cast<unsigned>((static_cast<long long>(args->B) * args->D + 127) / 128);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (args->dtype == MAMBA_B200_F32) gs::gated_scan_fwd_kernel<float><<<grid, 128, 0, st>>>(*args);
    else if (args->dtype == MAMBA_B200_F16) gs::gated_scan_fwd_kernel<__half><<<grid, 128, 0, st>>>(*args);
    else gs::gated_scan_fwd_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(*args);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

extern "C" MAMBA_B200_API int mamba_b200_gated_scan_bwd(void* handle, void* stream, const mamba_b200_gated_scan_args* args) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c || !args) return MAMBA_B200_ERR_ARG;
    const int rc = gs::check(c, args, true);
    if (rc || args->B == 0) return rc;
    const unsigned grid = static_cast<unsigned>((static_cast<long long>(args->B) * args->D + 127) / 128);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (args->dtype == MAMBA_B200_F32) gs::gated_scan_bwd_kernel<float><<<grid, 128, 0, st>>>(*args);
    else if (args->dtype == MAMBA_B200_F16) gs::gated_scan_bwd_kernel<__half><<<grid, 128, 0, st>>>(*args);
    else gs::gated_scan_bwd_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(*args);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}
