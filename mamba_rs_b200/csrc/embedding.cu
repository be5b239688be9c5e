// The token table at a language model's input: lookup with scaling, and the table's gradient.
//   forward   out[r, :] = scale * table[ids[r], :]                    an id outside [0, vocab): a row of zeros
//   backward  d_table[v, :] (+)= scale * sum over r with ids[r] = v of d_out[r, :], in an order fixed by ids and sizes
#include <string.h>

#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace emb {

// N values at once between memory and f32.
template <typename T, int N> struct __align__(sizeof(T) * N) Vec {
    T v[N];
    __device__ __forceinline__ void widen(float* f) const {
        if constexpr (N % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 p = unpack2<T>(*reinterpret_cast<const uint32_t*>(v + i));
                f[i] = p.x, f[i + 1] = p.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = to_f(v[i]);
        }
    }
    __device__ __forceinline__ void narrow(const float* f) {
        if constexpr (N % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(v + i) = pack2<T>(f[i], f[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = from_f<T>(f[i]);
        }
    }
};

struct FwdParams {
    const void* table;
    const int* ids;
    void* out;
    long long ld_table, ld_out, rows;
    int dim, vocab;
    float scale;
};

// Rows of the output, N elements a thread (16 bytes of the wider type), U pieces in flight: a piece is a row's next kThreads * N
// columns or the next row's.  HBM-bound: a table row read, an f32 row written.
constexpr int kThreads = 256;
template <typename Tin, typename Tout, int N, int U>
__global__ void __launch_bounds__(kThreads) embedding_fwd_kernel(const FwdParams p) {
    const Tin* table = static_cast<const Tin*>(p.table);
    Tout* out = static_cast<Tout*>(p.out);
    const int per_row = (p.dim + N - 1) / N;
    const long long total = p.rows * per_row, i0 = blockIdx.x * static_cast<long long>(kThreads * U) + threadIdx.x;
    Vec<Tin, N> q[U];
    long long r[U];
    int c[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = i0 + u * kThreads;
        r[u] = total <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(per_row) : i / per_row;
        c[u] = static_cast<int>(i - r[u] * per_row) * N;
        ok[u] = false;
        if (i >= total) continue;
        const int id = p.ids[r[u]];
        ok[u] = id >= 0 && id < p.vocab;
        if (ok[u]) q[u] = *reinterpret_cast<const Vec<Tin, N>*>(table + id * p.ld_table + c[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (i0 + u * kThreads >= total) break;
        float f[N];
        q[u].widen(f);
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = ok[u] ? f[k] * p.scale : 0.0f;
        Vec<Tout, N> o;
        o.narrow(f);
        *reinterpret_cast<Vec<Tout, N>*>(out + r[u] * p.ld_out + c[u]) = o;
    }
}

template <typename Tin, typename Tout>
static void launch_fwd(const FwdParams& p, cudaStream_t st) {
    // the widest pieces that sizes, strides and addresses allow: 4 elements are 16 bytes of f32
    auto fits = [&](int n) {
        return p.dim % n == 0 && p.ld_table % n == 0 && p.ld_out % n == 0 && reinterpret_cast<uintptr_t>(p.table) % (n * sizeof(Tin)) == 0 &&
               reinterpret_cast<uintptr_t>(p.out) % (n * sizeof(Tout)) == 0;
    };
    constexpr int U = 4;
    auto blocks = [&](int n) { return static_cast<unsigned>((p.rows * ((p.dim + n - 1) / n) + kThreads * U - 1) / (kThreads * U)); };
    if (fits(4)) embedding_fwd_kernel<Tin, Tout, 4, U><<<blocks(4), kThreads, 0, st>>>(p);
    else embedding_fwd_kernel<Tin, Tout, 1, U><<<blocks(1), kThreads, 0, st>>>(p);
}

// ---------------------------------------------------------------------------------------------------
// The gradient.
//
// Few rows, one kernel: a CTA whose row is the first of its token finds the others among the ids and adds them; further CTAs clear
// the rows of tokens that do not occur.
//
// More rows are sorted by token first.  A CTA of the sort has a range of tokens and reads ALL ids: it counts those below its range
// (where its rows begin in the sorted order) and, for each warp's part of the rows, those of each token of the range.  Prefix sums
// of that table are every row's place, a token's rows in rising order, without exchange between CTAs and without atomics whose
// order shows.  Then a warp adds a run of kRun sorted rows over 32 N columns.  A token whose rows all lie in the run is written at
// once; the sum of one that goes on beyond an end of the run (padding, a frequent token) goes to the workspace, and a third kernel
// adds such a token's sums in the order of the runs.
// ---------------------------------------------------------------------------------------------------
constexpr int kFewRows = 512, kRun = 32, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMaxRange = 1024, kJoinRuns = 8;

struct BwdParams {
    const void* d_out;
    const int* ids;
    float* d_table;
    long long ld_dout;
    int rows, dim, vocab, accumulate, range, slices, runs;
    float scale;
    int2* sorted;            // row, token
    int* counted;            // rows whose token lies in the table
    unsigned char* present;  // [vocab]
    float* part;             // [runs, 2, dim]: a run's sum of the token that came from before, and of the one that goes on
};

template <int N> __device__ __forceinline__ void write_sum(float* to, const float* acc, float scale, bool accumulate) {
    Vec<float, N> o;
    if (accumulate) o = *reinterpret_cast<const Vec<float, N>*>(to);
#pragma unroll
    for (int k = 0; k < N; ++k) o.v[k] = accumulate ? fmaf(acc[k], scale, o.v[k]) : acc[k] * scale;
    *reinterpret_cast<Vec<float, N>*>(to) = o;
}
// Sums of each warp's N columns a lane over the CTA's warps, in their order, in warp 0.
template <int N, int WARPS> __device__ __forceinline__ void add_warps(float* acc, float (*room)[32 * N]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) room[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        acc[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) acc[k] += room[w][k * 32 + lane];
    }
}
// A warp clears rows lo .. hi of the table (where `absent` says so).
template <int N, typename F> __device__ __forceinline__ void clear_rows(float* table, int lo, int hi, int dim, F absent) {
    const int lane = threadIdx.x & 31;
    Vec<float, N> zero;
#pragma unroll
    for (int k = 0; k < N; ++k) zero.v[k] = 0.0f;
    for (int v = lo; v < hi; ++v) {
        if (!absent(v)) continue;
        float* row = table + static_cast<long long>(v) * dim;
        for (int c = lane * N; c < dim; c += 32 * N) *reinterpret_cast<Vec<float, N>*>(row + c) = zero;
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) embedding_bwd_few_kernel(const BwdParams p) {
    constexpr int NF = N == 8 ? 4 : N;
    __shared__ int ids[kFewRows], count[kThreads / 32];
    __shared__ short list[kFewRows];
    __shared__ float room[kThreads / 32][32 * N];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, R = p.rows, tasks = R * p.slices;
    for (int i = tid; i < R; i += kThreads) ids[i] = p.ids[i];
    __syncthreads();
    if (static_cast<int>(blockIdx.x) >= tasks) {  // eight rows of the table, one a warp
        const int v = (static_cast<int>(blockIdx.x) - tasks) * (kThreads / 32) + warp;
        if (v >= p.vocab) return;
        bool any = false;
        for (int i = lane; i < R; i += 32) any |= ids[i] == v;
        any = __any_sync(0xffffffffu, any);
        clear_rows<NF>(p.d_table, v, v + 1, p.dim, [any](int) { return !any; });
        return;
    }
    const int r = static_cast<int>(blockIdx.x) / p.slices, c = (static_cast<int>(blockIdx.x) - r * p.slices) * 32 * N + lane * N, id = ids[r];
    if (id < 0 || id >= p.vocab) return;
    bool earlier = false;
    for (int i = tid; i < r; i += kThreads) earlier |= ids[i] == id;
    if (__syncthreads_or(earlier)) return;
    // the rows of this token in order: each warp has a contiguous part
    const int per = (R + kThreads / 32 - 1) / (kThreads / 32), lo = warp * per, hi = min(R, lo + per);
    int n = 0;
    for (int i = lo; i < hi; i += 32) n += __popc(__ballot_sync(0xffffffffu, i + lane < hi && ids[i + lane] == id));
    if (lane == 0) count[warp] = n;
    __syncthreads();
    int at = 0, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += count[w];
        total += count[w];
    }
    for (int i = lo; i < hi; i += 32) {
        const bool hit = i + lane < hi && ids[i + lane] == id;
        const unsigned hits = __ballot_sync(0xffffffffu, hit);
        if (hit) list[at + __popc(hits & ((1u << lane) - 1))] = static_cast<short>(i + lane);
        at += __popc(hits);
    }
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    const int each = (total + kThreads / 32 - 1) / (kThreads / 32), end = min(total, (warp + 1) * each);
    if (c < p.dim)
        for (int i0 = warp * each; i0 < end; i0 += 8) {
            Vec<T, N> q[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (i0 + u < end) q[u] = *reinterpret_cast<const Vec<T, N>*>(static_cast<const T*>(p.d_out) + list[i0 + u] * p.ld_dout + c);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (i0 + u < end) {
                    float f[N];
                    q[u].widen(f);
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] += f[k];
                }
        }
    if (total > each) add_warps<N, kThreads / 32>(acc, room);  // (one row, most often: it is in warp 0)
    if (warp == 0 && c < p.dim) {
        float* to = p.d_table + static_cast<long long>(id) * p.dim + c;
        write_sum<NF>(to, acc, p.scale, p.accumulate);
        if constexpr (N == 8) write_sum<NF>(to + 4, acc + 4, p.scale, p.accumulate);
    }
}

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const BwdParams p) {
    extern __shared__ int table[];  // [kSortWarps][range]: how many, then the next place
    __shared__ int sums[kSortWarps], base;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, W = p.range, lo = static_cast<int>(blockIdx.x) * W, hi = min(p.vocab, lo + W);
    for (int i = tid; i < kSortWarps * W; i += kSortThreads) table[i] = 0;
    if (tid == 0) base = 0;
    __syncthreads();
    int* mine = table + warp * W;
    const int per = (((p.rows + kSortWarps - 1) / kSortWarps) + 31) / 32 * 32;
    const long long first = static_cast<long long>(warp) * per;
    const int begin = static_cast<int>(first < p.rows ? first : p.rows), end = min(p.rows - begin, per) + begin;
    constexpr int U = 8;
    int below = 0;
    for (int i = begin + lane; i < end; i += 32 * U) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = i + 32 * u < end ? p.ids[i + 32 * u] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            below += id[u] >= 0 && id[u] < lo;
            if (id[u] >= lo && id[u] < hi) atomicAdd(&mine[id[u] - lo], 1);
        }
    }
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0 && below) atomicAdd(&base, below);
    __syncthreads();
    // places: tokens in order, within a token the warps in order
    int total = 0;
    if (tid < W)
        for (int w = 0; w < kSortWarps; ++w) total += table[w * W + tid];
    int sum = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    int before = base;
    for (int w = 0; w < warp; ++w) before += sums[w];
    int at = before + sum - total;
    if (tid < W) {
        for (int w = 0; w < kSortWarps; ++w) {
            const int n = table[w * W + tid];
            table[w * W + tid] = at;
            at += n;
        }
        if (lo + tid < hi) {
            p.present[lo + tid] = total != 0;
            if (lo + tid == p.vocab - 1) *p.counted = at;
        }
    }
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 32 * U) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = i0 + lane + 32 * u < end ? p.ids[i0 + lane + 32 * u] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = id[u] >= lo && id[u] < hi;
            const unsigned any = __ballot_sync(0xffffffffu, in);
            if (any == 0) continue;
            if (in) {
                const unsigned same = __match_any_sync(any, id[u]);
                const int place = mine[id[u] - lo] + __popc(same & ((1u << lane) - 1));
                p.sorted[place] = make_int2(i0 + lane + 32 * u, id[u]);
                __syncwarp(any);
                if ((same >> lane) == 1) mine[id[u] - lo] = place + 1;  // (the last of them)
                __syncwarp(any);
            }
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) embedding_sums_kernel(const BwdParams p, int sum_blocks) {
    constexpr int NF = N == 8 ? 4 : N;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (static_cast<int>(blockIdx.x) >= sum_blocks) {  // 64 rows of the table
        const int lo = ((static_cast<int>(blockIdx.x) - sum_blocks) * (kThreads / 32) + warp) * 8;
        clear_rows<NF>(p.d_table, lo, min(p.vocab, lo + 8), p.dim, [&p](int v) { return !p.present[v]; });
        return;
    }
    const long long task = blockIdx.x * static_cast<long long>(kThreads / 32) + warp;
    const int run = static_cast<int>(task / p.slices), c = (static_cast<int>(task - static_cast<long long>(run) * p.slices) * 32 + lane) * N;
    const int first = run * kRun, total = *p.counted, n = min(kRun, total - first);
    if (n <= 0) return;
    const int2 own = lane < n ? p.sorted[first + lane] : make_int2(0, -1);
    const int before = first > 0 ? p.sorted[first - 1].y : -1, behind = first + kRun < total ? p.sorted[first + kRun].y : -1;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    int start = 0;
    constexpr int U = 8;
    for (int i0 = 0; i0 < n; i0 += U) {
        Vec<T, N> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long row = __shfl_sync(0xffffffffu, own.x, (i0 + u) & 31);
            if (i0 + u < n && c < p.dim) q[u] = *reinterpret_cast<const Vec<T, N>*>(static_cast<const T*>(p.d_out) + row * p.ld_dout + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u, token = __shfl_sync(0xffffffffu, own.y, i & 31), next = __shfl_sync(0xffffffffu, own.y, (i + 1) & 31);
            if (i >= n) break;
            float f[N];
            q[u].widen(f);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += f[k];
            const bool last = i + 1 == n;
            if (!last && next == token) continue;
            const bool begins = start > 0 || before != token, ends = !last || behind != token;
            if (c < p.dim) {
                if (begins && ends) {
                    float* to = p.d_table + static_cast<long long>(token) * p.dim + c;
                    write_sum<NF>(to, acc, p.scale, p.accumulate);
                    if constexpr (N == 8) write_sum<NF>(to + 4, acc + 4, p.scale, p.accumulate);
                } else {
                    float* to = p.part + (2ll * run + (begins ? 1 : 0)) * p.dim + c;
                    write_sum<NF>(to, acc, 1.0f, false);
                    if constexpr (N == 8) write_sum<NF>(to + 4, acc + 4, 1.0f, false);
                }
            }
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] = 0.0f;
            start = i + 1;
        }
    }
}

// Tokens that go on beyond a run, by the CTA of the run that they begin in.
template <int N>
__global__ void __launch_bounds__(kThreads) embedding_join_kernel(const BwdParams p) {
    constexpr int WARPS = kThreads / 32;
    __shared__ float room[WARPS][32 * N];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = (blockIdx.y * 32 + lane) * N;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int total = *p.counted, runs = (total + kRun - 1) / kRun;
    for (int run = blockIdx.x * kJoinRuns; run < min(runs - 1, (static_cast<int>(blockIdx.x) + 1) * kJoinRuns); ++run) {
        const int token = p.sorted[run * kRun + kRun - 1].y;
        if (p.sorted[(run + 1) * kRun].y != token) continue;                      // it ends here
        if (run > 0 && p.sorted[run * kRun - 1].y == token) continue;             // it began before
        int n = 0;  // runs behind this one that it reaches
        for (int i0 = run + 1;; i0 += kThreads) {
            const int here = __syncthreads_count(i0 + tid < runs && p.sorted[(i0 + tid) * kRun].y == token);
            n += here;
            if (here < kThreads) break;
        }
        float acc[N];
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = 0.0f;
        const int each = (n + 1 + WARPS - 1) / WARPS, end = min(n + 1, (warp + 1) * each);
        if (c < p.dim)
            for (int i0 = warp * each; i0 < end; i0 += 8) {
                Vec<float, N> q[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (i0 + u < end) q[u] = *reinterpret_cast<const Vec<float, N>*>(p.part + (2ll * (run + i0 + u) + (i0 + u == 0 ? 1 : 0)) * p.dim + c);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (i0 + u < end)
#pragma unroll
                        for (int k = 0; k < N; ++k) acc[k] += q[u].v[k];
            }
        add_warps<N, WARPS>(acc, room);
        if (warp == 0 && c < p.dim) write_sum<N>(p.d_table + static_cast<long long>(token) * p.dim + c, acc, p.scale, p.accumulate);
    }
}

static int range_of(int vocab) {
    const int w = (vocab + 147) / 148;
    return w < 8 ? 8 : w > kMaxRange ? kMaxRange : w;
}
struct Room {
    long long sorted, counted, present, part, bytes;
};
static Room room_of(long long rows, int dim, int vocab) {
    auto up = [](long long n) { return (n + 255) / 256 * 256; };
    Room r{};
    if (rows <= kFewRows) return r;
    r.counted = up(rows * 8);
    r.present = r.counted + 256;
    r.part = r.present + up(vocab);
    r.bytes = r.part + (rows + kRun - 1) / kRun * 2 * dim * 4;
    return r;
}

template <typename Kernel, typename... Args>
static cudaError_t launch_early(Kernel fn, dim3 grid, int threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute at;
    memset(&at, 0, sizeof(at));
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

template <typename T, int N>
static int launch_bwd(Ctx* c, BwdParams& p, cudaStream_t st) {
    p.slices = (p.dim + 32 * N - 1) / (32 * N);
    if (p.rows <= kFewRows) {
        const long long blocks = static_cast<long long>(p.rows) * p.slices + (p.accumulate ? 0 : (p.vocab + 7) / 8);
        embedding_bwd_few_kernel<T, N><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        return MAMBA_B200_OK;
    }
    p.range = range_of(p.vocab);
    p.runs = (p.rows + kRun - 1) / kRun;
    const long long sums = (static_cast<long long>(p.runs) * p.slices + kThreads / 32 - 1) / (kThreads / 32), clears = p.accumulate ? 0 : (p.vocab + 63) / 64;
    if (sums + clears > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_bwd: too many rows");
    embedding_sort_kernel<<<(p.vocab + p.range - 1) / p.range, kSortThreads, kSortWarps * p.range * sizeof(int), st>>>(p);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    MB200_CUDA_CHECK(c, launch_early(embedding_sums_kernel<T, N>, dim3(static_cast<unsigned>(sums + clears)), kThreads, st, p, static_cast<int>(sums)));
    constexpr int NJ = N == 8 ? 4 : N;
    MB200_CUDA_CHECK(c, launch_early(embedding_join_kernel<NJ>, dim3((p.runs + kJoinRuns - 1) / kJoinRuns, (p.dim + 32 * NJ - 1) / (32 * NJ)), kThreads, st, p));
    return MAMBA_B200_OK;
}
template <typename T>
static int launch_bwd(Ctx* c, BwdParams& p, cudaStream_t st) {
    auto fits = [&](int n) {
        return p.dim % n == 0 && p.ld_dout % n == 0 && reinterpret_cast<uintptr_t>(p.d_out) % (n * sizeof(T)) == 0 &&
               reinterpret_cast<uintptr_t>(p.d_table) % 16 == 0;
    };
    if constexpr (sizeof(T) == 2) {
        if (fits(8)) return launch_bwd<T, 8>(c, p, st);
    }
    return fits(4) ? launch_bwd<T, 4>(c, p, st) : launch_bwd<T, 1>(c, p, st);
}

}  // namespace emb

int embedding_configure(Ctx* c) {
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(emb::embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             emb::kSortWarps * emb::kMaxRange * static_cast<int>(sizeof(int))));
    return MAMBA_B200_OK;
}

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
    if (rows * ((dim + 3) / 4) > 2147483647ll * 256) return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_fwd: too many rows");
    if (!table || !ids || !out) return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: null pointer");
    const emb::FwdParams p{table, ids, out, ld_table, ld_out, rows, dim, vocab, scale};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) emb::launch_fwd<float, float>(p, st);
    else if (dtype == MAMBA_B200_F16 && out_dtype == dtype) emb::launch_fwd<__half, __half>(p, st);
    else if (dtype == MAMBA_B200_F16) emb::launch_fwd<__half, float>(p, st);
    else if (out_dtype == dtype) emb::launch_fwd<__nv_bfloat16, __nv_bfloat16>(p, st);
    else emb::launch_fwd<__nv_bfloat16, float>(p, st);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

extern "C" MAMBA_B200_API long long mamba_b200_embedding_bwd_workspace_bytes(long long rows, int dim, int vocab) {
    return rows > 0 && dim > 0 && vocab > 0 ? emb::room_of(rows, dim, vocab).bytes : 0;
}

extern "C" MAMBA_B200_API int mamba_b200_embedding_bwd(void* handle, void* stream, int dtype, const void* d_out, long long ld_dout,
                                                       const int* ids, float* d_table, int accumulate, long long rows, int dim,
                                                       int vocab, float scale, void* workspace, long long workspace_bytes) {
    Ctx* c = static_cast<Ctx*>(handle);
    if (!c) return MAMBA_B200_ERR_ARG;
    if (!dtype_ok(dtype)) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: bad dtype %d", dtype);
    if (rows < 0 || dim <= 0 || vocab <= 0 || ld_dout < dim) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: bad dims");
    if (rows > 2147483647ll - 1024 || dim > 32 * 65535 || vocab > 2147483647 - 1024)
        return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_bwd: too many rows, columns or tokens");
    if (!d_table || (rows && (!d_out || !ids))) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: null pointer");
    if (rows == 0 && accumulate) return MAMBA_B200_OK;
    const emb::Room r = emb::room_of(rows, dim, vocab);
    if (workspace_bytes < r.bytes || (r.bytes && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)))
        return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: the workspace is %lld bytes, 256-byte aligned", r.bytes);
    emb::BwdParams p{d_out, ids, d_table, ld_dout, static_cast<int>(rows), dim, vocab, accumulate, 0, 0, 0, scale};
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    p.sorted = reinterpret_cast<int2*>(ws + r.sorted);
    p.counted = reinterpret_cast<int*>(ws + r.counted);
    p.present = ws + r.present;
    p.part = reinterpret_cast<float*>(ws + r.part);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) return emb::launch_bwd<float>(c, p, st);
    if (dtype == MAMBA_B200_F16) return emb::launch_bwd<__half>(c, p, st);
    return emb::launch_bwd<__nv_bfloat16>(c, p, st);
}
