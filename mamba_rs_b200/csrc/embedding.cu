// The token table at a language model's input: lookup with scaling, and the table's gradient.
//   forward   out[r, :] = scale * table[ids[r], :]                    an id outside [0, vocab): a row of zeros
//   backward  d_table[v, :] (+)= scale * sum over r with ids[r] = v of d_out[r, :], r ascending
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace emb {

struct FwdParams {
    const void* table;
    const int* ids;
    void* out;
    long long ld_table, ld_out, rows;
    int dim, vocab;
    float scale;
};

template <typename Tin, typename Tout>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const FwdParams p) {
    const Tin* table = static_cast<const Tin*>(p.table);
    Tout* out = static_cast<Tout*>(p.out);
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const int id = p.ids[r];
        const bool ok = id >= 0 && id < p.vocab;
        for (int c = threadIdx.x; c < p.dim; c += blockDim.x)
            out[r * p.ld_out + c] = from_f<Tout>(ok ? to_f(table[id * p.ld_table + c]) * p.scale : 0.0f);
    }
}

struct BwdParams {
    const void* d_out;
    const int* ids;
    float* d_table;
    long long ld_dout, rows;
    int dim, vocab, accumulate;
    float scale;
};

// A CTA per row of the table: it looks through all ids and adds the rows that are its own.
template <typename Tin>
__global__ void __launch_bounds__(256) embedding_bwd_kernel(const BwdParams p) {
    __shared__ int count[8], list[256];
    const Tin* d_out = static_cast<const Tin*>(p.d_out);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int v = blockIdx.x; v < p.vocab; v += gridDim.x) {
        float* row = p.d_table + static_cast<long long>(v) * p.dim;
        if (!p.accumulate)
            for (int c = tid; c < p.dim; c += 256) row[c] = 0.0f;
        for (long long r0 = 0; r0 < p.rows; r0 += 256) {
            const bool hit = r0 + tid < p.rows && p.ids[r0 + tid] == v;
            const unsigned hits = __ballot_sync(0xffffffffu, hit);
            __syncthreads();
            if (lane == 0) count[warp] = __popc(hits);
            __syncthreads();
            int base = 0, total = 0;
            for (int w = 0; w < 8; ++w) {
                if (w < warp) base += count[w];
                total += count[w];
            }
            if (hit) list[base + __popc(hits & ((1u << lane) - 1))] = tid;
            __syncthreads();
            for (int c = tid; total && c < p.dim; c += 256) {
                float s = 0.0f;
                for (int i = 0; i < total; ++i) s += to_f(d_out[(r0 + list[i]) * p.ld_dout + c]);
                row[c] += s * p.scale;
            }
        }
    }
}

}  // namespace emb
}  // namespace mb200

using namespace mb200;

extern "C" MAMBA_B200_API int mamba_b200_embedding_fwd(void* handle, void* stream, int dtype, const void* table, long long ld_table,
                                                       const int* ids, int out_dtype, void* out, long long ld_out, long long rows,
                                                       int dim, int vocab, float scale) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: bad dtype %d", dtype);
    if (out_dtype != MAMBA_B200_F32 && out_dtype != dtype)
        return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: rows come out as f32 or in the table's dtype, not %d", out_dtype);
    if (rows < 0 || dim <= 0 || vocab <= 0 || ld_table < dim || ld_out < dim) return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: bad dims");
    if (rows == 0) return MAMBA_B200_OK;
    if (!table || !ids || !out) return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: null pointer");
    const emb::FwdParams p{table, ids, out, ld_table, ld_out, rows, dim, vocab, scale};
    const int grid = static_cast<int>(rows < 65536 ? rows : 65536);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) emb::embedding_fwd_kernel<float, float><<<grid, 256, 0, st>>>(p);
    else if (dtype == MAMBA_B200_F16 && out_dtype == dtype) emb::embedding_fwd_kernel<__half, __half><<<grid, 256, 0, st>>>(p);
    else if (dtype == MAMBA_B200_F16) emb::embedding_fwd_kernel<__half, float><<<grid, 256, 0, st>>>(p);
    else if (out_dtype == dtype) emb::embedding_fwd_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else emb::embedding_fwd_kernel<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

extern "C" MAMBA_B200_API long long mamba_b200_embedding_bwd_workspace_bytes(long long rows, int dim, int vocab) {
    (void)rows, (void)dim, (void)vocab;
    return 0;
}

extern "C" MAMBA_B200_API int mamba_b200_embedding_bwd(void* handle, void* stream, int dtype, const void* d_out, long long ld_dout,
                                                       const int* ids, float* d_table, int accumulate, long long rows, int dim,
                                                       int vocab, float scale, void* workspace, long long workspace_bytes) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: bad dtype %d", dtype);
    if (rows < 0 || dim <= 0 || vocab <= 0 || ld_dout < dim) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: bad dims");
    if (rows > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_bwd: too many rows");
    if (!d_table || (rows && (!d_out || !ids))) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: null pointer");
    if (rows == 0 && accumulate) return MAMBA_B200_OK;
    if (workspace_bytes < mamba_b200_embedding_bwd_workspace_bytes(rows, dim, vocab) || (workspace_bytes && !workspace))
        return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: workspace too small");
    const emb::BwdParams p{d_out, ids, d_table, ld_dout, rows, dim, vocab, accumulate, scale};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int grid = vocab < 65536 ? vocab : 65536;
    if (dtype == MAMBA_B200_F32) emb::embedding_bwd_kernel<float><<<grid, 256, 0, st>>>(p);
    else if (dtype == MAMBA_B200_F16) emb::embedding_bwd_kernel<__half><<<grid, 256, 0, st>>>(p);
    else emb::embedding_bwd_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}
