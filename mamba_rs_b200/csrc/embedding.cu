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

// A warp has up to 8 pieces a lane of one row, N elements each (4: 16 bytes of f32), their loads in flight together.  HBM-bound: a
// table row is read, an f32 row written.
constexpr int kThreads = 256, kPieces = 8;
template <typename Tin, typename Tout, int N>
__global__ void __launch_bounds__(kThreads) embedding_fwd_kernel(const FwdParams p, int parts) {
    const int lane = threadIdx.x & 31;
    const long long task = blockIdx.x * static_cast<long long>(kThreads / 32) + threadIdx.x / 32, r = parts == 1 ? task : task / parts;
    if (r >= p.rows) return;
    const int id = p.ids[r], c0 = (static_cast<int>(task - r * parts) * kPieces * 32 + lane) * N;
    const bool ok = id >= 0 && id < p.vocab;
    const Tin* from = static_cast<const Tin*>(p.table) + (ok ? id : 0) * p.ld_table + c0;
    Tout* to = static_cast<Tout*>(p.out) + r * p.ld_out + c0;
    Vec<Tin, N> q[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
        if (c0 + u * 32 * N < p.dim) q[u] = *reinterpret_cast<const Vec<Tin, N>*>(from + u * 32 * N);
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
        if (c0 + u * 32 * N >= p.dim) break;
        float f[N];
        q[u].widen(f);
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = ok ? f[k] * p.scale : 0.0f;
        Vec<Tout, N> o;
        o.narrow(f);
        *reinterpret_cast<Vec<Tout, N>*>(to + u * 32 * N) = o;
    }
}

template <typename Tin, typename Tout>
static void launch_fwd(const FwdParams& p, cudaStream_t st) {
    // the widest pieces that sizes, strides and addresses allow: 4 elements are 16 bytes of f32
    auto fits = [&](int n) {
        return p.dim % n == 0 && p.ld_table % n == 0 && p.ld_out % n == 0 && reinterpret_cast<uintptr_t>(p.table) % (n * sizeof(Tin)) == 0 &&
               reinterpret_cast<uintptr_t>(p.out) % (n * sizeof(Tout)) == 0;
    };
    auto run = [&](auto kernel, int n) {
        const int parts = (p.dim + 32 * n * kPieces - 1) / (32 * n * kPieces);
        kernel<<<static_cast<unsigned>((p.rows * parts + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(p, parts);
    };
    if (fits(4)) run(embedding_fwd_kernel<Tin, Tout, 4>, 4);
    else run(embedding_fwd_kernel<Tin, Tout, 1>, 1);
}

// ---------------------------------------------------------------------------------------------------
// The gradient.
//
// Few rows, one kernel: a CTA whose row is the first of its token finds the others among the ids and adds them; further CTAs clear
// the rows of tokens that do not occur.
//
// More rows are sorted by token first, by one cluster of 16 CTAs: 8 bits of the token at a time, rows of equal bits in rising
// order, counts of each warp's contiguous rows in shared memory, the CTAs' counts joined through distributed shared memory.  The
// other SMs clear rows of the table meanwhile.  (A sort by 148 CTAs with a range of tokens each, without exchange, read all ids
// 148 times: 23 us for 32768 rows.)  Then a warp adds a run of up to 32 sorted rows over 32 N columns.  A token whose rows all lie
// in the run is written at once; the sum of one that goes on beyond an end of the run (padding, a frequent token) goes to the
// workspace, and a third kernel adds such a token's sums in the order of the runs.
// ---------------------------------------------------------------------------------------------------
constexpr int kFewRows = 512, kMaxRun = 32, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSorters = 16, kDigits = 256;

struct BwdParams {
    const void* d_out;
    const int* ids;
    float* d_table;
    long long ld_dout;
    int rows, dim, vocab, accumulate, slices, run, runs;
    int cleared;             // rows from here on are cleared beside the sort, whether their token occurs or not
    int passes;              // of the sort
    float scale;
    int2* sorted;            // [(runs + 1) * run] row, token; behind the last one token -1
    int2* other;             // of the sort's passes before the last
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
// A warp clears a row of the table.
template <int N> __device__ __forceinline__ void clear_row(float* row, int dim) {
    Vec<float, N> zero;
#pragma unroll
    for (int k = 0; k < N; ++k) zero.v[k] = 0.0f;
#pragma unroll 4
    for (int c = (threadIdx.x & 31) * N; c < dim; c += 32 * N) *reinterpret_cast<Vec<float, N>*>(row + c) = zero;
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
        if (!any) clear_row<NF>(p.d_table + static_cast<long long>(v) * p.dim, p.dim);
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

// Clears the rows from p.cleared on.  The sort starts while this runs, and ends after it.
template <int N>
__global__ void __launch_bounds__(kThreads) embedding_clear_kernel(const BwdParams p) {
    asm volatile("griddepcontrol.launch_dependents;");
    for (int v = p.cleared + static_cast<int>(blockIdx.x) * (kThreads / 32) + static_cast<int>(threadIdx.x) / 32; v < p.vocab; v += gridDim.x * (kThreads / 32))
        clear_row<N>(p.d_table + static_cast<long long>(v) * p.dim, p.dim);
}

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const BwdParams p) {
    __shared__ int table[kSortWarps][kDigits], digit[kDigits], sums[kSortWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x;
    for (int v = rank * kSortThreads + tid; v < p.vocab; v += kSorters * kSortThreads) p.present[v] = 0;
    int n = p.rows;
    constexpr int U = 4;
    for (int pass = 0; pass < p.passes; ++pass) {
        const bool first = pass == 0, last = pass + 1 == p.passes;
        const int2* from = (p.passes - pass) % 2 ? p.other : p.sorted;
        int2* to = (p.passes - pass) % 2 ? p.sorted : p.other;
        // this warp's elements
        const int per = ((n + kSorters * kSortWarps - 1) / (kSorters * kSortWarps) + 31) / 32 * 32;
        const long long lo = static_cast<long long>(rank * kSortWarps + warp) * per;
        const int begin = static_cast<int>(lo < n ? lo : n), end = min(n - begin, per) + begin, shift = 8 * pass;
        auto element = [&](int i) -> int2 {
            if (i >= end) return make_int2(0, -1);
            if (!first) return from[i];
            const int id = p.ids[i];
            return make_int2(i, id < p.vocab ? id : -1);
        };
        int2 e[U];  // (all that a warp has, most often: it is fetched once)
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = element(begin + 32 * u + lane);
        for (int i = tid; i < kSortWarps * kDigits; i += kSortThreads) (&table[0][0])[i] = 0;
        __syncthreads();
        for (int i0 = begin; i0 < end; i0 += 32 * U) {
            if (i0 > begin) {
#pragma unroll
                for (int u = 0; u < U; ++u) e[u] = element(i0 + 32 * u + lane);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int d = e[u].y < 0 ? kDigits : (e[u].y >> shift) & (kDigits - 1);
                const unsigned same = __match_any_sync(0xffffffffu, d);
                if (d < kDigits && (same & ((1u << lane) - 1)) == 0) atomicAdd(&table[warp][d], __popc(same));
            }
        }
        __syncthreads();
        int mine = 0;
        if (tid < kDigits) {
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) mine += table[w][tid];
            digit[tid] = mine;
        }
        cluster_sync();
        int before = 0, all = 0;
        if (tid < kDigits) {
            int of[kSorters];
#pragma unroll
            for (int k = 0; k < kSorters; ++k) of[k] = __float_as_int(ld_cluster1(cluster_addr(smem_u32(digit + tid), k)));
#pragma unroll
            for (int k = 0; k < kSorters; ++k) {
                if (k < rank) before += of[k];
                all += of[k];
            }
            int sum = all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            if (lane == 31) sums[warp] = sum;
            before += sum - all;
        }
        __syncthreads();
        if (tid < kDigits) {
            for (int w = 0; w < warp; ++w) before += sums[w];
#pragma unroll
            for (int w0 = 0; w0 < kSortWarps; w0 += 8) {
                int c[8];
#pragma unroll
                for (int w = 0; w < 8; ++w) c[w] = table[w0 + w][tid];
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    table[w0 + w][tid] = before;
                    before += c[w];
                }
            }
        }
        __syncthreads();
        n = 0;
        for (int w = 0; w < kDigits / 32; ++w) n += sums[w];
        for (int i0 = begin; i0 < end; i0 += 32 * U) {
            if (end - begin > 32 * U) {
#pragma unroll
                for (int u = 0; u < U; ++u) e[u] = element(i0 + 32 * u + lane);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int d = e[u].y < 0 ? kDigits : (e[u].y >> shift) & (kDigits - 1);
                const unsigned same = __match_any_sync(0xffffffffu, d);
                const int place = d < kDigits ? table[warp][d] + __popc(same & ((1u << lane) - 1)) : 0;
                __syncwarp();
                if (d < kDigits) {
                    to[place] = e[u];
                    if (last) p.present[e[u].y] = 1;
                    if ((same >> lane) == 1) table[warp][d] = place + 1;  // (the last of them)
                }
                __syncwarp();
            }
        }
        cluster_sync();  // the elements are there, and nobody reads this CTA's counts any more
    }
    for (int i = n + rank * kSortThreads + tid; i < (p.runs + 1) * p.run; i += kSorters * kSortThreads) p.sorted[i] = make_int2(0, -1);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (what comes next relies on the cleared rows too)
}

// What a warp of the sums has: a run of sorted rows and a part of the columns, or rows of the table to clear (kClear of them).  Those
// that clear lie evenly between those that add: the ones write, the others read.
constexpr int kClear = 32;
struct Task {
    int run, slice;  // run < 0: done
    int2 own;        // lane l: the run's l-th row and its token
    int n;
    unsigned ends;   // last rows of a token in this run
    bool from_before, goes_on;
};
template <int NF>
__device__ __forceinline__ Task next_task(const BwdParams& p, long long index, long long sums, long long clears) {
    const int lane = threadIdx.x & 31;
    Task t;
    t.run = -1;
    const long long total = sums + clears, cleared = index * clears / total;
    if (index >= total) return t;
    if ((index + 1) * clears / total != cleared) {
        const int v0 = static_cast<int>(cleared) * kClear;
        const unsigned absent = __ballot_sync(0xffffffffu, v0 + lane < p.cleared && !p.present[v0 + lane]);
        for (unsigned m = absent; m; m &= m - 1) clear_row<NF>(p.d_table + static_cast<long long>(v0 + __ffs(m) - 1) * p.dim, p.dim);
        return t;
    }
    const long long task = index - cleared;
    const int run = static_cast<int>(task / p.slices), first = run * p.run;
    t.slice = static_cast<int>(task - static_cast<long long>(run) * p.slices);
    t.own = lane < p.run ? p.sorted[first + lane] : make_int2(0, -1);
    const int before = first > 0 ? p.sorted[first - 1].y : -1, behind = p.sorted[first + p.run].y;
    t.n = __popc(__ballot_sync(0xffffffffu, t.own.y >= 0));
    if (t.n == 0) return t;
    const int next = __shfl_down_sync(0xffffffffu, t.own.y, 1);
    t.ends = __ballot_sync(0xffffffffu, lane + 1 < t.n && next != t.own.y) | 1u << (t.n - 1);
    t.from_before = before == __shfl_sync(0xffffffffu, t.own.y, 0);
    t.goes_on = behind == __shfl_sync(0xffffffffu, t.own.y, t.n - 1);
    t.run = run;
    return t;
}
// Where the sum of the token that ends with row i of the run goes: the token's row, or the run's part of a token that goes on.
__device__ __forceinline__ float* sum_place(const BwdParams& p, const Task& t, int i, int c, bool& whole) {
    whole = !t.from_before && !(t.goes_on && i + 1 == t.n);
    return whole ? p.d_table + static_cast<long long>(__shfl_sync(0xffffffffu, t.own.y, i)) * p.dim + c
                 : p.part + (2ll * t.run + (t.from_before ? 0 : 1)) * p.dim + c;
}

// Rows whose parts are 16-byte aligned come to shared memory by bulk copies, a lane asking for one row's part: a run's 16 or 32 KB are
// in flight at once.  Parts of 512 bytes in f32, 1 KB in 16 bits: 32768 x 768 f32 takes 71 us (with 1 KB 2 more), 16384 x 2560 bf16 123
// (with 512 bytes 5 more).  Some 30 us of the first are this kernel, whose 155 MB (rows read, rows of tokens written, what is left to
// clear) are 24.
template <typename T> constexpr int kPartBytes = sizeof(T) == 2 ? 1024 : 512;
template <typename T>
__global__ void __launch_bounds__(32) embedding_sums_kernel(const BwdParams p, long long sums, long long clears, int* status) {
    constexpr int N = 16 / sizeof(T), NF = 4, kPart = kPartBytes<T>, M = kPart / 512;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + (128 - (smem_u32(raw) & 127)) % 128;
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + p.run * kPart);
    const int lane = threadIdx.x;
    if (lane == 0) {
        mbar_init(bar, 1);
        fence_barrier_init();
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Task t = next_task<NF>(p, blockIdx.x, sums, clears);
    if (t.run < 0) return;
    const int c0 = t.slice * (kPart / static_cast<int>(sizeof(T))), c = c0 + lane * N;
    const uint32_t bytes = static_cast<uint32_t>(min(kPart, (p.dim - c0) * static_cast<int>(sizeof(T))));
    if (lane == 0) mbar_expect_tx(bar, bytes * t.n);
    __syncwarp();
    if (lane < t.n) bulk_load(sm + lane * kPart, static_cast<const T*>(p.d_out) + t.own.x * p.ld_dout + c0, bytes, bar);
    bool in[M];
    float acc[M][N];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        in[m] = c + m * 32 * N < p.dim;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[m][k] = 0.0f;
    }
    if (!mbar_wait(bar, 0, status)) return;
#pragma unroll 4
    for (int i = 0; i < t.n; ++i) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
            float f[N];
            reinterpret_cast<const Vec<T, N>*>(sm + i * kPart + m * 512 + lane * 16)->widen(f);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[m][k] += f[k];
        }
        if (!(t.ends >> i & 1)) continue;
        bool whole;
        float* to = sum_place(p, t, i, c, whole);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if (in[m])
#pragma unroll
                for (int k = 0; k < N; k += NF)
                    write_sum<NF>(to + m * 32 * N + k, acc[m] + k, whole ? p.scale : 1.0f, whole && p.accumulate);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[m][k] = 0.0f;
        }
        t.from_before = false;
    }
}

// Other rows: M columns a lane, 32 apart.  (Two rows' loads at once took 98 us for 32768 x 769, one row's 84: the warps of an SM suffice.)
template <typename T>
__global__ void __launch_bounds__(kThreads) embedding_sums_plain_kernel(const BwdParams p, long long sums, long long clears) {
    constexpr int M = 4;
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Task t = next_task<1>(p, blockIdx.x * static_cast<long long>(kThreads / 32) + threadIdx.x / 32, sums, clears);
    if (t.run < 0) return;
    const int c = t.slice * 32 * M + lane;
    const T* columns = static_cast<const T*>(p.d_out) + c;
    float acc[M];
#pragma unroll
    for (int m = 0; m < M; ++m) acc[m] = 0.0f;
    for (int i = 0; i < t.n; ++i) {
        const T* row = columns + __shfl_sync(0xffffffffu, t.own.x, i) * p.ld_dout;
        T q[M];
#pragma unroll
        for (int m = 0; m < M; ++m) q[m] = c + 32 * m < p.dim ? row[32 * m] : from_f<T>(0.0f);
#pragma unroll
        for (int m = 0; m < M; ++m) acc[m] += to_f(q[m]);
        if (!(t.ends >> i & 1)) continue;
        bool whole;
        float* to = sum_place(p, t, i, c, whole);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if (c + 32 * m < p.dim) write_sum<1>(to + 32 * m, acc + m, whole ? p.scale : 1.0f, whole && p.accumulate);
            acc[m] = 0.0f;
        }
        t.from_before = false;
    }
}

// Tokens that go on beyond a run.  A warp looks after the one that begins in its run and adds its runs' sums, if they are few; the
// CTAs of a cluster share one that reaches 32 runs or more.  What counts for the many short ones is how many CTAs an SM has: with 8
// loads in flight a warp and four CTAs 8192 x 768 f32 took 47.4 us, with 16 and two 53, with 4 and six 46.6.
constexpr int kJoinThreads = 256, kJoinCtas = 4;
template <int N>
__global__ void __launch_bounds__(kJoinThreads, 6) embedding_join_kernel(const BwdParams p) {
    constexpr int WARPS = kJoinThreads / 32, RUNS = kJoinCtas * WARPS, kCount = 8;
    static_assert(RUNS % 32 == 0 && RUNS <= kJoinThreads, "a thread for each of the cluster's runs");
    __shared__ float room[WARPS][32 * N], joined[32 * N];
    __shared__ unsigned far[RUNS / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = (blockIdx.y * 32 + lane) * N, rank = blockIdx.x % kJoinCtas;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int runs = p.runs, first = (static_cast<int>(blockIdx.x) - rank) * WARPS;
    auto starts_with = [&](int run) { return p.sorted[run * p.run].y; };
    auto ends_with = [&](int run) { return p.sorted[run * p.run + p.run - 1].y; };
    if (warp < RUNS / 32) {  // the same in all CTAs of the cluster
        const int run = first + tid;
        const int token = run + 32 < runs ? ends_with(run) : -1;
        const unsigned mask = __ballot_sync(0xffffffffu, token >= 0 && starts_with(run + 32) == token && (run == 0 || ends_with(run - 1) != token));
        if (lane == 0) far[warp] = mask;
    }
    auto add = [&](float* acc, int run, int begin, int end) {  // sums begin .. end of the token that begins in the run
        if (c >= p.dim) return;
        constexpr int U = 4;
        for (int i0 = begin; i0 < end; i0 += U) {
            Vec<float, N> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u < end) q[u] = *reinterpret_cast<const Vec<float, N>*>(p.part + (2ll * (run + i0 + u) + (i0 + u == 0 ? 1 : 0)) * p.dim + c);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u < end)
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] += q[u].v[k];
        }
    };
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    const int run = first + rank * WARPS + warp;
    // lane l: the token at the start of run run + 1 + l; and those before this run and at its end
    const int ahead = run + 1 + lane < runs ? starts_with(run + 1 + lane) : -1;
    const int before = run > 0 && run < runs ? ends_with(run - 1) : -1, end = run + 1 < runs ? ends_with(run) : -1;
    const int token = end >= 0 ? end : -2;  // (-2: none goes on from here)
    const unsigned same = __ballot_sync(0xffffffffu, ahead == token);
    if ((same & 1) && before != token && same != 0xffffffffu) {
        add(acc, run, 0, __ffs(~same));
        if (c < p.dim) write_sum<N>(p.d_table + static_cast<long long>(token) * p.dim + c, acc, p.scale, p.accumulate);
    }
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < RUNS / 32; ++w)
#pragma unroll 1
        for (unsigned m = far[w]; m; m &= m - 1) {
            const int from = first + 32 * w + __ffs(m) - 1, its = ends_with(from);
            int n = 0, here = 1;  // runs behind this one that it reaches
            for (int i0 = from + 1 + tid; here; i0 += kCount * kJoinThreads) {
                int starts[kCount];
#pragma unroll
                for (int u = 0; u < kCount; ++u) starts[u] = i0 + u * kJoinThreads < runs ? starts_with(i0 + u * kJoinThreads) : -1;
                here = 0;
#pragma unroll
                for (int u = 0; u < kCount; ++u) here += __syncthreads_count(starts[u] == its);
                n += here;
            }
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] = 0.0f;
            const int each = (n + 1 + RUNS - 1) / RUNS, at = (rank * WARPS + warp) * each;
            add(acc, from, at, min(n + 1, at + each));
            add_warps<N, WARPS>(acc, room);
            if (warp == 0) {
#pragma unroll
                for (int k = 0; k < N; ++k) joined[k * 32 + lane] = acc[k];
            }
            __syncwarp();
            cluster_sync();
            if (rank == 0 && warp == 0) {
#pragma unroll
                for (int i = 1; i < kJoinCtas; ++i)
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] += ld_cluster1(cluster_addr(smem_u32(joined + k * 32 + lane), i));
                if (c < p.dim) write_sum<N>(p.d_table + static_cast<long long>(its) * p.dim + c, acc, p.scale, p.accumulate);
            }
            __syncwarp();
            cluster_sync();
        }
}

constexpr long long kClearBeside = 128 << 20;
// Rows of a run: fewer where that gives more warps something to do.
static int run_of(long long rows, int dim) {
    int run = kMaxRun;
    while (run > 8 && rows / run * ((dim + 255) / 256) < 148 * 12) run /= 2;
    return run;
}
struct Room {
    long long sorted, other, present, part, bytes;
};
static Room room_of(long long rows, int dim, int vocab) {
    auto up = [](long long n) { return (n + 255) / 256 * 256; };
    Room r{};
    if (rows <= kFewRows) return r;
    const int run = run_of(rows, dim);
    r.other = up(((rows + run - 1) / run + 1) * run * 8);
    r.present = r.other + up(rows * 8);
    r.part = r.present + up(vocab);
    r.bytes = r.part + (rows + run - 1) / run * 2 * dim * 4;
    return r;
}

// With `early` the kernel may start before the one ahead of it in the stream has ended, and waits for it itself.
template <typename Kernel, typename... Args>
static cudaError_t launch_early(Kernel fn, dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, bool early, Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    memset(at, 0, sizeof(at));
    if (early) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = cluster;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = at;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

template <typename T, int N>
static int launch_bwd(Ctx* c, BwdParams& p, cudaStream_t st) {
    if (p.rows <= kFewRows) {
        p.slices = (p.dim + 32 * N - 1) / (32 * N);
        const long long blocks = static_cast<long long>(p.rows) * p.slices + (p.accumulate ? 0 : (p.vocab + 7) / 8);
        embedding_bwd_few_kernel<T, N><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        return MAMBA_B200_OK;
    }
    constexpr int NF = N == 1 ? 1 : 4, kJoinRuns = kJoinCtas * (kJoinThreads / 32), kColumns = N == 1 ? 128 : kPartBytes<T> / static_cast<int>(sizeof(T));
    p.slices = (p.dim + kColumns - 1) / kColumns;
    p.run = run_of(p.rows, p.dim);
    p.runs = (p.rows + p.run - 1) / p.run;
    for (p.passes = 1; p.passes < 4 && (p.vocab - 1) >> (8 * p.passes); ++p.passes) {}
    // what HBM can clear while the sort runs (some 20 us), of the last tokens: the rare ones where tokens are in order of frequency
    const long long beside = p.accumulate ? 0 : kClearBeside / (4ll * p.dim);
    p.cleared = p.vocab - static_cast<int>(beside < p.vocab ? beside : p.vocab);
    const long long sums = static_cast<long long>(p.runs) * p.slices, clears = p.accumulate ? 0 : (p.cleared + kClear - 1) / kClear;
    if (sums + clears > 2147483647ll) return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_bwd: too many rows");
    const bool beside_sort = p.cleared < p.vocab;
    if (beside_sort) {
        embedding_clear_kernel<NF><<<2 * c->sm_count, kThreads, 0, st>>>(p);
        MB200_CUDA_CHECK(c, cudaGetLastError());
    }
    MB200_CUDA_CHECK(c, launch_early(embedding_sort_kernel, dim3(kSorters), kSortThreads, 0, st, kSorters, beside_sort, p));
    const unsigned tasks = static_cast<unsigned>(sums + clears);
    if constexpr (N == 1)
        MB200_CUDA_CHECK(c, launch_early(embedding_sums_plain_kernel<T>, dim3((tasks + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st, 1, true, p, sums, clears));
    else
        MB200_CUDA_CHECK(c, launch_early(embedding_sums_kernel<T>, dim3(tasks), 32, p.run * kPartBytes<T> + 16 + 128, st, 1, true, p, sums, clears, c->d_status));
    MB200_CUDA_CHECK(c, launch_early(embedding_join_kernel<NF>, dim3((p.runs + kJoinRuns - 1) / kJoinRuns * kJoinCtas, (p.dim + 32 * NF - 1) / (32 * NF)),
                                     kJoinThreads, 0, st, kJoinCtas, true, p));
    return MAMBA_B200_OK;
}
template <typename T>
static int launch_bwd(Ctx* c, BwdParams& p, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = p.dim % N == 0 && p.ld_dout % N == 0 && reinterpret_cast<uintptr_t>(p.d_out) % 16 == 0 && reinterpret_cast<uintptr_t>(p.d_table) % 16 == 0;
    return wide ? launch_bwd<T, N>(c, p, st) : launch_bwd<T, 1>(c, p, st);
}

}  // namespace emb

int embedding_configure(Ctx* c) {
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute(emb::embedding_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
    if (dim > kMaxSize || rows > 2147483647ll * 8 / ((dim + 255) / 256)) return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_fwd: too many rows or columns");
    if (!aligned_to(dtype_size(dtype), {table}) || !aligned_to(dtype_size(out_dtype), {out}) || !aligned_to(4, {ids}))
        return fail(c, MAMBA_B200_ERR_ARG, "embedding_fwd: misaligned pointer");
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
    if (rows > kMaxSize || dim > 32 * 65535 || vocab > kMaxSize)
        return fail(c, MAMBA_B200_ERR_SHAPE, "embedding_bwd: too many rows, columns or tokens");
    if (!aligned_to(dtype_size(dtype), {d_out}) || !aligned_to(4, {ids, d_table})) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: misaligned pointer");
    if (!d_table || (rows && (!d_out || !ids))) return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: null pointer");
    if (rows == 0 && accumulate) return MAMBA_B200_OK;
    const emb::Room r = emb::room_of(rows, dim, vocab);
    if (workspace_bytes < r.bytes || (r.bytes && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)))
        return fail(c, MAMBA_B200_ERR_ARG, "embedding_bwd: the workspace is %lld bytes, 256-byte aligned", r.bytes);
    emb::BwdParams p{d_out, ids, d_table, ld_dout, static_cast<int>(rows), dim, vocab, accumulate};
    p.scale = scale;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    p.sorted = reinterpret_cast<int2*>(ws + r.sorted);
    p.other = reinterpret_cast<int2*>(ws + r.other);
    p.present = ws + r.present;
    p.part = reinterpret_cast<float*>(ws + r.part);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MAMBA_B200_F32) return emb::launch_bwd<float>(c, p, st);
    if (dtype == MAMBA_B200_F16) return emb::launch_bwd<__half>(c, p, st);
    return emb::launch_bwd<__nv_bfloat16>(c, p, st);
}
