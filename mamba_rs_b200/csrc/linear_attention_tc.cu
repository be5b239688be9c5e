// Linear attention with a decay for each head on the tensor cores: 16-bit rows that TMA can describe, K and V up to 128.
//
// A block has 64 columns of one pair's (sequence, head) state and walks chunks of 128 steps (roles and names: linear_attention.cuh):
//   G = X Y^T,  P = G o l^{distance},  out = P Z + l^{row} o (X S),  S <- l^n S + Y^T (w o Z)
// Beside HBM, which a chunk of 128 x 64 heads of 128 x 64 keeps busy for 4100 cycles an SM, its products take some 2000 cycles of the
// tensor pipe, so one block on an SM reaches HBM's rate if nothing waits for anything else: every part has warps of its own, and the
// state, the only thing that is carried from chunk to chunk, stays in tensor memory,
//   warp 0      asks for the tiles (X and Y, Z), as many chunks ahead as there are stages
//   warp 1      issues X Y^T, up to two chunks ahead
//   warp 2      issues Y^T (w o Z), the chain from chunk to chunk
//   warp 3      issues X S and P Z
//   warps 4-7   make P from G, of every other chunk; it goes back to tensor memory and is read there as an operand
//   warps 8-11  leave a 16-bit copy of S for X S, and in its place what is left of it after the chunk
//   warps 12-15 join P Z and X S and write rows, by TMA from Z's place (a thread's own row in pieces of 32 bytes took 2100 cycles)
//   warps 16-19 weigh Z
//   warps 20-23 make P of the other chunks
// and they meet on mbarriers alone; every wait gives up after a limit and takes the block to its end.
//
// Slow decays (`fold`, bf16): w_j = l^{n-1-j} stands in for l^{i-j} = l^{i-(n-1)} w_j too.  w o Z takes Z's place, P is G with its future cut
// off, and l^{i-(n-1)} is one factor a row of the result, in 32 bits.  Fast ones, whose l^127 takes the first rows' products far
// below their size (kSlow), and f16 weigh P instead.
//
// Roundings to 16 bits: the scores (made in f32), the weighted values beside them where they are folded, and the copy of S that is read,
// each once, as the result is.  The state itself is f32: w o Z, which it is made of, is kept to f32 accuracy where a state is handed on:
// three bf16 terms of 8 bits each; where only out is wanted one term is enough.  In f16 a second term of 2^-11 of the first gives 22 bits (down
// to 2^-26 of a tile's largest value, fewer below), P is scaled by a power of two a row, S and w o Z by one a tile, so that neither their size
// nor their smallness leaves the type.
//
// Device time of 8 x 4096 x 32 heads of 128 x 64, bf16: 127 to 134 us, 92 to 97 % of the measured copy rate (a block alone needs 2600 cycles a
// chunk; with 148 of them HBM has them wait); its backward 458 to 482, 47 to 49 % (2200 cycles a chunk and 64 columns, of which the products
// and the rows' warps are busy for most).  Calls one after another, each on inputs of its own, take 142 to 152 and 532 to 563.  f16: 265 to 275, its
// backward 1125 to 1165 (weights, scores and states are looked over once more for their magnitudes, and nothing is folded).
// What the steps gave is told where it matters.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "linear_attention_general.cuh"
#include "m3_tc.cuh"

namespace mb200 {
namespace la {
namespace tcl {

using namespace mb200::tc;

constexpr int kThreads = 768, kTile = 64;
constexpr uint32_t kSub = kSwSub;  // a [128 x 64] sub-tile
// Tensor memory: two buffers of G, whose left half P takes and whose right half P Z (not folded); two of X S (f16: one) and, folded, P Z in
// one sum; S, and where it has one a chunk's sum; in f16 the sum of the second terms.
constexpr uint32_t cG = 0, cY1 = 64, cY2 = 256, cDf = 320, cS = 384, cSlo = 448, kCols = 512;

struct TcParams {
    CUtensorMap x[3], y[3], z[3], out[3];
    Params p;
    int na, stages, z_tiles;  // sub-tiles of X (and of Y) in a stage; stages of X and Y; tiles for stages of Z and terms of w o Z
    int out_map[3];  // 1: out can be described too, and rows leave in tiles of 32
};

// Tiles beside the stages of X and Y: copies of S, and those for Z and w o Z.
template <int TERMS>
constexpr int kCopies = TERMS == 1 ? 2 : 1;
constexpr int kTiles = 6;  // beside two stages of X and Y of two sub-tiles, or four of one
// A chunk's smallest weight is above e^-kSlow = 2^-8 where w o Z stands in for Z: the first rows' products are that much smaller than the
// formula's, and one of 2^-126 still has 15 bits (a limit of e^-40 lost those below 3e-21.  Decays from 1 / 1.4 to 1 / 256 a step, of which this
// limit weighs half and that one a sixth, 8 x 4096 x 32 heads of 128 x 64: 187 us for 180, backward 640 for 580).
constexpr float kSlow = 5.545f;

// behind the stages, the terms of w o Z and the copies of S
struct Small {
    float col[32];         // l^{31 - u} (back: l^u)
    float diag[64];        // alpha_p l^{d} at 31 + d
    float row_scale[2][128];
    float tile_scale[4];  // (a copy's is read until its rows are out, which is known of the chunk three before)
    float warp_max[2][4];
    float z_max[2][4], z_scale[2];  // f16: magnitudes of w o Z, and what its tile's products are multiplied by
    uint64_t full[4], empty[4], z_full[8], z_empty[8], g_full[2], p_full[2], y_full[2], y_empty[2], s_full[2], s_empty[2], w_full[8], z_read[8], d_full, d_read, max_full, z_max_full, drain[3];
    // Values that are not finite may change no row before their own, as 0 times them in a product would: w o Z has 0 in their place, and
    // of their column the rows from the first of them on, counted as they are walked, are NaN (as is the state that leaves).
    int bad[kTile], any_bad;
    uint32_t tmem;
    int dead;
};
constexpr int kNever = 0x7fffffff;
static_assert(14 * kSub + sizeof(Small) <= 227 * 1024, "a block's shared memory");

template <int TERMS>
uint32_t smem_bytes(int na, int stages, int z_tiles) {
    return (stages * 2 * na + z_tiles + kCopies<TERMS>) * kSub + sizeof(Small);
}

__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* w) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11]),
        "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A bounded wait that also ends when another role has given up.
__device__ __forceinline__ bool look(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool free_now(uint64_t* bar, uint32_t parity) {  // (look() may sleep for a while)
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, Small* sm, int* status) {
    for (int it = 0; it < kMbarMaxPolls; ++it) {
        if (look(bar, parity)) return true;
        if ((it & 15) == 15 && *reinterpret_cast<volatile int*>(&sm->dead)) return false;
    }
    *reinterpret_cast<volatile int*>(&sm->dead) = 1;
    atomicCAS(status, kStatusOk, kStatusBarrierTimeout);
    return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Small* sm, int* status) {
    return look(bar, parity) || wait_on(bar, parity, sm, status);
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Small* sm, int* status) {
    return __all_sync(0xffffffffu, wait(bar, parity, sm, status));
}

// One lane of a converged warp.  The products' warp goes through its loop as a whole and this lane issues them: descriptors then stay
// in uniform registers (a branch on the lane's number had them moved there one by one, 130 cycles a product).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// 2^e that brings a magnitude to [2^13, 2^14), and back (0, infinities and NaN: as it is)
__device__ __forceinline__ float scale_to(float m, float* back) {
    const int e = static_cast<int>((__float_as_uint(m) >> 23) & 255);
    if (e == 255 || m == 0.0f) {
        *back = 1.0f;
        return 1.0f;
    }
    const int d = max(e - 127 - 13, -126);
    *back = __uint_as_float(static_cast<uint32_t>(127 + d) << 23);
    return __uint_as_float(static_cast<uint32_t>(127 - d) << 23);
}

// The largest finite magnitude of a row of an f16 tile that also holds others.
__device__ __noinline__ float finite_max(const unsigned char* z, int row) {
    float m = 0.0f;
    for (int c = 0; c < kTile; ++c) {
        const float v = fabsf(__half2float(*reinterpret_cast<const __half*>(z + sw_chunk(row, c >> 3) + 2 * (c & 7))));
        if (v < INFINITY) m = fmaxf(m, v);
    }
    return m;
}
// A row of w o Z (its terms' tiles lie together) and of Z (which may be w o Z's first term), some of whose values are not finite.
template <typename Th>
__device__ __noinline__ void set_aside(unsigned char* w0, unsigned char* w1, int more, unsigned char* z, int row, int pos, Small* sm) {
    constexpr unsigned inf = std::is_same<Th, __half>::value ? 0x7c00u : 0x7f80u;
    for (int c = 0; c < kTile; ++c) {
        const uint32_t at = sw_chunk(row, c >> 3) + 2 * (c & 7);
        if ((*reinterpret_cast<uint16_t*>(z + at) & inf) != inf) continue;
        *reinterpret_cast<uint16_t*>(w0 + at) = 0;
        *reinterpret_cast<uint16_t*>(z + at) = 0;
        for (int t = 0; t < more; ++t) *reinterpret_cast<uint16_t*>(w1 + t * kSub + at) = 0;
        atomicMin(&sm->bad[c], pos);
    }
    *reinterpret_cast<volatile int*>(&sm->any_bad) = 1;
}
// ... and the rows behind them: columns c < left of a row at out, `step` elements apart, or of row `row` of a swizzled tile.
template <typename To>
__device__ __noinline__ void spoil(To* out, int step, int left, int pos, const Small* sm) {
    for (int c = 0; c < left; ++c)
        if (sm->bad[c] <= pos) out[c * step] = from_f<To>(__int_as_float(0x7fffffff));
}
template <typename To>
__device__ __noinline__ void spoil_tile(unsigned char* tile, int row, int pos, const Small* sm) {
    for (int c = 0; c < kTile; ++c)
        if (sm->bad[c] <= pos) *reinterpret_cast<To*>(tile + sw_chunk(row, c >> 3) + 2 * (c & 7)) = from_f<To>(__int_as_float(0x7fffffff));
}

// (`fold` is known to the compiler: code that is not taken lies elsewhere, and what is fits the instruction cache: 137 -> 126 us, the
// backward 559 -> 449.  `back` is not: blocks of both directions share a cache, and two more variants took 634)
template <typename Th, int TERMS, bool STATE, bool fold>
__device__ __forceinline__ void walk(const TcParams& tp, unsigned char* smem, const Place& w, const float ld) {
    constexpr bool F16 = std::is_same<Th, __half>::value;
    constexpr int SB = kCopies<TERMS>;
    // A product adds to its accumulator by cutting off, always towards zero: with a chunk's 24 of them on top of S, a state that decays slowly
    // lost 2^-25 of itself each time, 10^-5 over 40 chunks.  Where a state has to keep its digits a chunk's sum has an accumulator of its
    // own, and joins S in a rounded f32 sum.  (Where only 16-bit rows are wanted, S itself: 464 us for 500 of a backward.)
    constexpr bool FRESH = TERMS > 1;
    constexpr uint32_t cD = !FRESH ? cS : F16 ? cDf : cSlo;
    constexpr uint32_t fmt = F16 ? 0u : 1u;
    const Params& p = tp.p;
    const Role& r = p.role[w.role];
    const int A = r.A, W = r.W, na = (A + 63) >> 6, c0 = w.tile * kTile, stages = tp.stages;
    const uint32_t stage = 2 * tp.na * kSub, oY = tp.na * kSub, kZ = stages * stage, kS = kZ + tp.z_tiles * kSub;
    Small* sm = reinterpret_cast<Small*>(smem + kS + SB * kSub);
    const uint32_t sbase = smem_u32(smem);
    const int b = static_cast<int>(w.pair / p.H), h = static_cast<int>(w.pair - static_cast<long long>(b) * p.H);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, role = warp >> 2, row = threadIdx.x & 127;
    const bool back = r.backwards;
    const float l2 = ld * kLog2e;
    const int zs = tp.z_tiles - TERMS + (fold ? 1 : 0);  // stages of Z
    const uint32_t kW = kZ + zs * kSub;
    // chunks of this segment, numbered as they are walked
    const int all = (p.T + kChunk - 1) / kChunk, per = p.seg_len / kChunk;
    const int first = w.seg * per, n = min(all - first, per);
    auto start = [&](int i) { return (back ? all - 1 - (first + i) : first + i) * kChunk; };
    const bool enters = w.seg > 0 ? !STATE : r.s_in != nullptr;
    const bool leaves = STATE || (w.seg + 1 == p.segments && r.s_out != nullptr);
    const int late0 = r.late && w.seg == 0 ? 1 : 0;  // of chunk 0

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sm->full[i], 1);
            mbar_init(&sm->empty[i], STATE ? 1 : 3);
        }
        for (int i = 0; i < 8; ++i) {
            mbar_init(&sm->z_full[i], 1);
            mbar_init(&sm->z_empty[i], STATE ? 1 : 4);
            mbar_init(&sm->w_full[i], 128);
            mbar_init(&sm->z_read[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm->g_full[i], 1);
            mbar_init(&sm->p_full[i], 128);
            mbar_init(&sm->s_full[i], 128);
            mbar_init(&sm->s_empty[i], 1);
            mbar_init(&sm->y_full[i], 1);
            mbar_init(&sm->y_empty[i], 128);
        }
        for (int i = 0; i < 3; ++i) mbar_init(&sm->drain[i], 1);
        mbar_init(&sm->d_full, 1);
        mbar_init(&sm->max_full, 128);
        mbar_init(&sm->z_max_full, 4);
        mbar_init(&sm->d_read, 128);
        sm->dead = 0;
        sm->any_bad = 0;
        fence_barrier_init();
    }
    if (threadIdx.x >= 64 && threadIdx.x < 64 + kTile) sm->bad[threadIdx.x - 64] = kNever;
    if (threadIdx.x >= 32 && threadIdx.x < 64) {
        sm->col[lane] = decay_at(l2, back ? lane : 31 - lane);
        sm->diag[lane] = 0.0f;  // (31 is written below)
        __syncwarp();
        sm->diag[31 + lane] = decay_at(l2, lane) * r.alpha_p;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm->tmem)), "r"(kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sm->tmem;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);  // this warp's 32 rows

    const uint32_t per_stage = stage >> 4;  // in descriptors
    constexpr uint32_t kStep = 32 >> 4, mStep = 2048 >> 4, sub = kSub >> 4;

    if (warp == 0) {
        if (lane == 0) {
            // X and Y are free when the products of S are, Z only with the rows: neither waits for the other's turn
            const int hx = h / r.x.group, hy = h / r.y.group, hz = h / r.z.group;
            int i = 0, st = 0, turn = 0, iz = 0, sz = 0, turn_z = 0, polls = 0;
            while (i < n || iz < n) {
                bool did = false;
                if (i < n && (turn == 0 || free_now(&sm->empty[st], (turn - 1) & 1))) {
                    const int t0 = start(i);
                    unsigned char* at = smem + st * stage;
                    mbar_expect_tx(&sm->full[st], (STATE ? 1 : 2) * na * kSub);
                    for (int s = 0; s < na; ++s) {
                        if (!STATE) tma_load_4d(at + s * kSub, &tp.x[w.role], &sm->full[st], 64 * s, hx, t0, b);
                        tma_load_4d(at + oY + s * kSub, &tp.y[w.role], &sm->full[st], 64 * s, hy, t0, b);
                    }
                    ++i;
                    if (++st == stages) {
                        st = 0;
                        ++turn;
                    }
                    did = true;
                }
                if (iz < n && (turn_z == 0 || free_now(&sm->z_empty[sz], (turn_z - 1) & 1))) {
                    mbar_expect_tx(&sm->z_full[sz], kSub);
                    tma_load_4d(smem + kZ + sz * kSub, &tp.z[w.role], &sm->z_full[sz], c0, hz, start(iz), b);
                    ++iz;
                    if (++sz == zs) {
                        sz = 0;
                        ++turn_z;
                    }
                    did = true;
                }
                polls = did ? 0 : polls + 1;
                if (!did) {
                    if (polls > kMbarMaxPolls || ((polls & 15) == 15 && *reinterpret_cast<volatile int*>(&sm->dead))) {
                        *reinterpret_cast<volatile int*>(&sm->dead) = 1;
                        atomicCAS(p.status, kStatusOk, kStatusBarrierTimeout);
                        break;
                    }
                    __nanosleep(32);
                }
            }
            // nothing may be in flight when the block ends (where all went well, it has long landed)
            for (int k = max(0, i - stages); k < i; ++k) mbar_wait(&sm->full[k % stages], (k / stages) & 1, p.status);
            for (int k = max(0, iz - zs); k < iz; ++k) mbar_wait(&sm->z_full[k % zs], (k / zs) & 1, p.status);
        }
    } else if (warp == 1) {
        // ---- X Y^T ----
        if (!STATE) {
            const uint32_t idG = instr_desc(fmt, 0, 0, 128);
            // descriptors of stage 0; a step along K is a constant more (m3_tc.cuh), a stage `per_stage`
            const uint64_t xk = desc_sw_k(sbase, 0), yk = desc_sw_k(sbase + oY, 0);
            bool ok = true;
            for (int i = 0, st = 0, turn = 0; i < n; ++i) {
                const uint32_t at = st * per_stage;
                // the buffer's P has been read (not folded: and P Z, beside it, by the rows)
                if (i > 1) ok = wait_warp(fold ? &sm->y_full[i & 1] : &sm->y_empty[i & 1], ((i >> 1) - 1) & 1, sm, p.status);
                if (ok) ok = wait_warp(&sm->full[st], turn & 1, sm, p.status);
                if (!ok) break;
                fence_after();
                const uint32_t d = tmem + cG + (i & 1) * 128;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma(d, xk + at + k * kStep, yk + at + k * kStep, idG, k > 0);
                    if (na == 2) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma(d, xk + at + sub + k * kStep, yk + at + sub + k * kStep, idG, true);
                    }
                    commit(&sm->g_full[i & 1]);
                    commit(&sm->empty[st]);
                }
                __syncwarp();
                if (++st == stages) {
                    st = 0;
                    ++turn;
                }
            }
            if (!ok) {  // what was issued has to end before tensor memory is given back
                if (elect_one()) commit(&sm->drain[0]);
                __syncwarp();
                mbar_wait(&sm->drain[0], 0, p.status);
            }
        }
    } else if (warp == 2) {
        // ---- Y^T (w o Z) ----
        const uint32_t idD = instr_desc(fmt, 1, 1, 64);
        const uint64_t ym = desc_sw_mn(sbase + oY, 0), zm = desc_sw_mn(sbase + kZ, 0), wm = desc_sw_mn(sbase + kW, 0);
        bool ok = true;
        int st = 0, turn = 0, sz = 0, turn_z = 0;
        for (int i = 0; i < n; ++i) {
            const uint32_t at = st * per_stage;
            const bool reads = i > 0 || enters, adds = leaves || i + 1 < n;
            const int u = enters ? i : i - 1;  // number of the copy of S
            // (without a product too: what this warp commits counts for the tiles of this chunk, which have to be there)
            ok = wait_warp(&sm->full[st], turn & 1, sm, p.status);
            if (ok) ok = wait_warp(&sm->w_full[sz], turn_z & 1, sm, p.status);
            // the sum of the last chunk has been read; or, where it is S itself, what is left of S is in its place (with the copy of S)
            if (FRESH && ok && adds && i > 0) ok = wait_warp(&sm->d_read, (i - 1) & 1, sm, p.status);
            if (!FRESH && ok && adds && reads) ok = wait_warp(&sm->s_full[STATE ? 0 : u % SB], (STATE ? u : u / SB) & 1, sm, p.status);
            if (!ok) break;
            fence_after();
            // first term; the others
            const uint64_t w0 = fold ? zm + sz * sub : wm, w1 = fold ? wm - sub : wm;
            if (elect_one()) {
                if (adds) {
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const bool own = F16 && t == 1;  // (the second f16 term is summed apart)
#pragma unroll
                        for (int k = 0; k < kChunk / 16; ++k)
                            mma(tmem + (own ? cSlo : cD), ym + at + k * mStep, (t == 0 ? w0 : w1 + t * sub) + k * mStep, idD,
                                own ? k > 0 : (!FRESH && reads) || k > 0 || t > 0);
                    }
                    commit(&sm->d_full);
                }
                commit(&sm->empty[st]);
                commit(STATE ? &sm->z_empty[sz] : &sm->z_read[sz]);
            }
            __syncwarp();
            if (++st == stages) {
                st = 0;
                ++turn;
            }
            if (++sz == zs) {
                sz = 0;
                ++turn_z;
            }
        }
        if (!ok) {
            if (elect_one()) commit(&sm->drain[1]);
            __syncwarp();
            mbar_wait(&sm->drain[1], 0, p.status);
        }
    } else if (warp == 3) {
        // ---- X S and P Z ----
        if (!STATE) {
            const uint32_t idY = instr_desc(fmt, 0, 1, 64);
            const uint64_t xk = desc_sw_k(sbase, 0), sc = desc_sw_mn(sbase + kS, 0), zm = desc_sw_mn(sbase + kZ, 0);
            bool ok = true;
            int st = 0, turn = 0, sz = 0, turn_z = 0;
            for (int i = 0; i < n; ++i) {
                const uint32_t at = st * per_stage, d = tmem + cY2 + (F16 ? 0 : (i & 1) * 64);
                const bool reads = i > 0 || enters;
                const int u = enters ? i : i - 1;  // number of the copy of S
                const int j = F16 ? i - 1 : i - 2;  // the chunk that had this buffer before
                if (j >= 0) ok = wait_warp(&sm->y_empty[j & 1], (j >> 1) & 1, sm, p.status);
                if (ok) ok = wait_warp(&sm->full[st], turn & 1, sm, p.status);
                if (ok && reads) ok = wait_warp(&sm->s_full[u % SB], (u / SB) & 1, sm, p.status);
                if (!ok) break;
                fence_after();
                if (elect_one()) {
                    if (reads) {
                        const uint32_t copy = (u % SB) * sub;
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma(d, xk + at + k * kStep, sc + copy + k * mStep, idY, k > 0);
                        if (na == 2) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) mma(d, xk + at + sub + k * kStep, sc + copy + (4 + k) * mStep, idY, true);
                        }
                        commit(&sm->s_empty[u % SB]);
                    }
                    commit(&sm->empty[st]);
                }
                __syncwarp();
                ok = wait_warp(&sm->w_full[sz], turn_z & 1, sm, p.status);
                if (ok) ok = wait_warp(&sm->p_full[i & 1], (i >> 1) & 1, sm, p.status);
                if (!ok) break;
                fence_after();
                const uint32_t g = tmem + cG + (i & 1) * 128, z = sz * sub, y = fold ? d : g + cY1;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kChunk / 16; ++k) mma_ta(y, g + k * 8, zm + z + k * mStep, idY, k > 0 || (fold && reads));
                    commit(&sm->y_full[i & 1]);
                }
                __syncwarp();
                if (++st == stages) {
                    st = 0;
                    ++turn;
                }
                if (++sz == zs) {
                    sz = 0;
                    ++turn_z;
                }
            }
            if (!ok) {
                if (elect_one()) commit(&sm->drain[2]);
                __syncwarp();
                mbar_wait(&sm->drain[2], 0, p.status);
            }
        }
    } else if (role == 1 || role == 5) {
        // ---- P ----
        if (!STATE) {
            const int q = warp & 3;  // the 32 columns that hold this warp's diagonal
            // other blocks: l^{row - column} in two factors, col[u] = l^{31 - u} (back: l^u) and what is left, here of the blocks one, two and
            // three away
            float rf[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) rf[k] = decay_at(l2, back ? 32 * (k + 1) - lane : lane + 32 * (k + 1) - 31) * r.alpha_p;
            const float bound = fabsf(r.alpha_p) * fmaxf(1.0f, decay_at(l2, kChunk - 1));  // (a decay above 0 makes them grow)
            const float* diag = sm->diag + 31 + (back ? -lane : lane);
            for (int i = role == 1 ? 0 : 1; i < n; i += 2) {
                if (!wait_warp(&sm->g_full[i & 1], (i >> 1) & 1, sm, p.status)) break;
                fence_after();
                const uint32_t g0 = lanes + cG + (i & 1) * 128;
                if (fold) {
                    // (P takes the place of G's columns that have been read: from the left.  One block a turn: code unrolled over a chunk waits for
                    // instructions, 8000 cycles a chunk)
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        uint32_t o[16];
                        if (back ? k >= q : k <= q) {
                            float g[32];
                            tmem_ld32(g0 + 32 * k, g);
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = pack2<Th>(g[2 * u], g[2 * u + 1]);
                            if (k == q) {
                                // (cut off, not multiplied by 0: what lies behind the edge may be infinite)
#pragma unroll
                                for (int u = 0; u < 16; ++u) {
                                    const bool lo = back ? 2 * u >= lane : 2 * u <= lane, hi = back ? 2 * u + 1 >= lane : 2 * u + 1 <= lane;
                                    o[u] &= (lo ? 0xffffu : 0u) | (hi ? 0xffff0000u : 0u);
                                }
                            }
                        } else {
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = 0;
                        }
                        tmem_st16(g0 + 16 * k, o);
                    }
                    tmem_st_wait();
                    fence_before();
                    mbar_arrive(&sm->p_full[i & 1]);
                    continue;
                }
                // weighted scores of block k
                auto weigh = [&](int k, float* g) {
                    tmem_ld32(g0 + 32 * k, g);
                    if (k == q) {
#pragma unroll
                        for (int u = 0; u < 32; ++u) {
                            // (a choice, not a product with 0: what lies behind the edge may be infinite)
                            const bool in = back ? u >= lane : u <= lane;
                            g[u] = in ? g[u] * diag[back ? u : -u] : 0.0f;
                        }
                    } else {
                        const int away = back ? k - q : q - k;
                        const float2 f = splat2(away == 1 ? rf[0] : away == 2 ? rf[1] : rf[2]);
#pragma unroll
                        for (int u = 0; u < 32; u += 4) {
                            const float4 c = *reinterpret_cast<const float4*>(sm->col + u);
                            const float2 a = mul2(mul2(make_float2(g[u], g[u + 1]), make_float2(c.x, c.y)), f);
                            const float2 e = mul2(mul2(make_float2(g[u + 2], g[u + 3]), make_float2(c.z, c.w)), f);
                            g[u] = a.x; g[u + 1] = a.y; g[u + 2] = e.x; g[u + 3] = e.y;
                        }
                    }
                };
                float scale = 1.0f;
                if (F16) {
                    // the scores themselves bound their weighted values (up to the diagonal's alpha_p), and below 2^-28 of the bound an f16 still
                    // has all its digits
                    float m = 0.0f;
#pragma unroll 1
                    for (int k = back ? q : 0; k <= (back ? 3 : q); ++k) {
                        float g[32];
                        tmem_ld32(g0 + 32 * k, g);
                        if (k == q) {
#pragma unroll
                            for (int u = 0; u < 32; ++u) g[u] = (back ? u >= lane : u <= lane) ? g[u] : 0.0f;
                        }
#pragma unroll
                        for (int u = 0; u < 32; u += 2) m = fmaxf(m, fmaxf(fabsf(g[u]), fabsf(g[u + 1])));
                    }
                    float undo;
                    scale = scale_to(m * bound, &undo);
                    sm->row_scale[i & 1][row] = undo;
                }
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    uint32_t o[16];
                    if (back ? k >= q : k <= q) {
                        float g[32];
                        weigh(k, g);
#pragma unroll
                        for (int u = 0; u < 16; ++u) o[u] = F16 ? pack2<Th>(g[2 * u] * scale, g[2 * u + 1] * scale) : pack2<Th>(g[2 * u], g[2 * u + 1]);
                    } else {
#pragma unroll
                        for (int u = 0; u < 16; ++u) o[u] = 0;
                    }
                    tmem_st16(g0 + 16 * k, o);
                }
                tmem_st_wait();
                fence_before();
                mbar_arrive(&sm->p_full[i & 1]);
            }
        }
    } else if (role == 2) {
        // ---- S ----
        const long long slot = static_cast<long long>(A) * W;
        float* slots = r.slots ? r.slots + w.pair * p.segments * slot : nullptr;
        const bool mine = row < A;
        const int nc = min(kTile, W - c0);
        // (states between segments lie column by column here: a warp's rows are neighbours)
        if (enters) {
            const bool given = w.seg == 0 && (STATE || p.segments == 1);
            const int at = mine ? row : 0;  // (rows that are none read the first one, and drop it: loads without a branch are in flight together)
            const float* in = r.s_in + w.pair * slot + static_cast<long long>(at) * r.sa + static_cast<long long>(c0) * r.sw;
            const bool quads = given && r.sw == 1 && nc == kTile && (reinterpret_cast<uintptr_t>(r.s_in) | (r.sa * sizeof(float))) % 16 == 0;
            const float* between = slots + w.seg * slot + static_cast<long long>(c0) * A + at;
#pragma unroll 1
            for (int s = 0; s < 2; ++s) {
                float v[32];
                const int last = max(nc - 32 * s, 1) - 1;  // columns behind the last one read that, and drop it
                if (quads) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(in + 32 * s + c);
                        v[c] = x.x; v[c + 1] = x.y; v[c + 2] = x.z; v[c + 3] = x.w;
                    }
                } else if (nc > 32 * s) {
                    const float* q = given ? in + static_cast<long long>(32 * s) * r.sw : between + static_cast<long long>(32 * s) * A;
                    const int step = given ? r.sw : A;
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] = q[min(c, last) * step];
                }
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (!mine || 32 * s + c >= nc) v[c] = 0.0f;
                if (STATE && mine) {
                    float* q = slots + static_cast<long long>(c0 + 32 * s) * A + row;
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (32 * s + c < nc) q[c * A] = v[c];
                }
                tmem_st32(lanes + cS + 32 * s, v);
            }
        }
        if (FRESH && !enters) {
            const float none[32] = {};
            tmem_st32(lanes + cS, none);
            tmem_st32(lanes + cS + 32, none);
        }
        const Pow whole = decay_pow(ld, kChunk);
        float undo = 1.0f;  // of the last chunk's w o Z (f16)
        auto sum_scale = [&](int i) {
            if (!F16) return true;
            if (!wait_warp(&sm->w_full[i % zs], (i / zs) & 1, sm, p.status)) return false;  // (long over: the products have read what it says)
            undo = sm->z_scale[i & 1];
            return true;
        };
        // 32 columns of S with the last chunk's sum
        auto read = [&](int s, float* v) {
            if (!FRESH) {
                tmem_ld32(lanes + cS + 32 * s, v);
                return;
            }
            float d[32];
            if (F16) {
                tmem_ld32x2(lanes + cD + 32 * s, v, lanes + cSlo + 32 * s, d);
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = fmaf(d[c], 1.0f / 2048, v[c]);
                tmem_ld32(lanes + cS + 32 * s, d);
            } else {
                tmem_ld32x2(lanes + cS + 32 * s, v, lanes + cD + 32 * s, d);
            }
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = F16 ? fmaf(v[c], undo, d[c]) : v[c] + d[c];
        };
        auto has_read = [&]() {
            fence_before();
            mbar_arrive(&sm->d_read);
        };
        int u = 0;  // copies of S
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int rows = min(kChunk, p.T - start(i));
            const bool adds = leaves || i + 1 < n;
            if (i > 0) {
                ok = wait_warp(&sm->d_full, (i - 1) & 1, sm, p.status);
                if (ok) ok = sum_scale(i - 1);
                if (!ok) break;
                fence_after();
            }
            if (i > 0 || enters) {
                // S enters chunk i: a copy for X S, and what is left of it when the chunk is over
                float scale = 1.0f;
                if (!STATE) {
                    if (F16) {
                        float m = 0.0f;
#pragma unroll 1
                        for (int s = 0; s < 2; ++s) {
                            float v[32];
                            if (i > 0) {
                                read(s, v);
                                tmem_st32(lanes + cS + 32 * s, v);
                            } else {
                                tmem_ld32(lanes + cS + 32 * s, v);
                            }
                            if (mine) {
#pragma unroll
                                for (int c = 0; c < 32; c += 2) m = fmaxf(m, fmaxf(fabsf(v[c]), fabsf(v[c + 1])));
                            }
                        }
                        if (i > 0) has_read();
                        // (NaN are passed over, and an infinity, which only a given state brings, is: other columns keep their digits)
                        if (__any_sync(0xffffffffu, m == INFINITY)) {
                            tmem_st_wait();
                            m = 0.0f;
#pragma unroll 1
                            for (int s = 0; s < 2; ++s) {
                                float v[32];
                                tmem_ld32(lanes + cS + 32 * s, v);
                                if (mine)
                                    for (int c = 0; c < 32; ++c) m = fmaxf(m, fabsf(v[c]) < INFINITY ? fabsf(v[c]) : 0.0f);
                            }
                        }
                        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
                        if (lane == 0) sm->warp_max[u & 1][warp & 3] = m;
                        mbar_arrive(&sm->max_full);
                        ok = wait_warp(&sm->max_full, u & 1, sm, p.status);
                        if (!ok) break;
                        const float* wm = sm->warp_max[u & 1];
                        float undo;
                        scale = scale_to(fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3])), &undo);
                        if (row == 0) sm->tile_scale[u & 3] = undo;
                    }
                    if (u >= SB) ok = wait_warp(&sm->s_empty[u % SB], (u / SB - 1) & 1, sm, p.status);
                    if (!ok) break;
                }
                const bool odd = rows != kChunk || (i == 0 && late0);
                const Pow f = odd ? decay_pow(ld, rows - (i == 0 ? late0 : 0)) : whole;
                unsigned char* copy = smem + kS + (u % SB) * kSub;
#pragma unroll 1
                for (int s = 0; s < 2; ++s) {
                    float v[32];
                    if (i > 0 && (!F16 || STATE)) {
                        read(s, v);
                        if (FRESH && s == 1) has_read();
                    } else {
                        tmem_ld32(lanes + cS + 32 * s, v);  // (joined above, or nothing to join)
                    }
                    // (folded: rows take the factor that w o Z lacks, and with it X S is wanted of what is left of S)
                    auto decay = [&]() {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float2 x = make_float2(v[c], v[c + 1]);
                            x = TERMS == 1 ? mul2(x, splat2(f.hi)) : fma2(x, splat2(f.hi), mul2(x, splat2(f.lo)));
                            v[c] = x.x;
                            v[c + 1] = x.y;
                        }
                    };
                    if (fold) decay();
                    if (!STATE) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int c = 8 * j + 2 * e;
                                o[e] = F16 ? pack2<Th>(v[c] * scale, v[c + 1] * scale) : pack2<Th>(v[c], v[c + 1]);
                            }
                            *reinterpret_cast<uint4*>(copy + sw_chunk(row, 4 * s + j)) = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                    if (!fold) decay();
                    if (adds) tmem_st32(lanes + cS + 32 * s, v);
                }
                if (!STATE) fence_proxy_async();
                fence_before();
                if (!STATE || !FRESH) mbar_arrive(&sm->s_full[STATE ? 0 : u % SB]);
                ++u;
            }
        }
        if (ok && leaves && n > 0) {
            ok = wait_warp(&sm->d_full, (n - 1) & 1, sm, p.status);
            if (ok) ok = wait_warp(&sm->w_full[(n - 1) % zs], ((n - 1) / zs) & 1, sm, p.status);
            if (ok) ok = sum_scale(n - 1);
            if (ok) {
                fence_after();
                const Pow f = !STATE && r.last_decay ? decay_pow(ld, 1) : Pow{1.0f, 0.0f};
                float* out = STATE ? slots + (w.seg + 1) * slot + static_cast<long long>(c0) * A + row
                                   : r.s_out + w.pair * slot + static_cast<long long>(row) * W + c0;
                const bool quads = !STATE && nc == kTile && (reinterpret_cast<uintptr_t>(out) | (W * sizeof(float))) % 16 == 0;
#pragma unroll 1
                for (int s = 0; s < 2; ++s) {
                    float v[32];
                    read(s, v);
                    const int left = mine ? nc - 32 * s : 0;
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] = times(f, v[c]);
                    if (quads) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            if (mine) *reinterpret_cast<float4*>(out + 32 * s + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (c < left) out[(32 * s + c) * (STATE ? A : 1)] = v[c];
                    }
                }
                if (*reinterpret_cast<volatile int*>(&sm->any_bad) && mine) spoil(out, STATE ? A : 1, nc, kNever - 1, sm);
            }
        }
    } else if (role == 3 && !STATE) {
        // ---- out ----
        const float x_whole = decay_at(l2, back ? kChunk - row : row + 1) * r.alpha_x;
        const float y_whole = fold ? decay_at(-l2, back ? row : kChunk - 1 - row) * r.alpha_z : 1.0f;
        const int nc = min(kTile, W - c0);
        const bool tiles = tp.out_map[w.role];
        for (int i = 0, sz = 0, turn_z = 0; i < n; ++i) {
            // (Z's place, where the rows go, is read by the products of S too)
            if (!wait_warp(&sm->z_read[sz], turn_z & 1, sm, p.status)) break;
            if (!wait_warp(&sm->y_full[i & 1], (i >> 1) & 1, sm, p.status)) break;
            if (!wait_warp(&sm->w_full[sz], turn_z & 1, sm, p.status)) break;  // (long over; what it says of bad values is read here)
            fence_after();
            const bool bad = *reinterpret_cast<volatile int*>(&sm->any_bad);
            const int pos = i * kChunk + (back ? kChunk - 1 - row : row);
            const int t0 = start(i), rows = min(kChunk, p.T - t0);
            const bool reads = i > 0 || enters;
            const int late = i == 0 ? late0 : 0;
            float f = x_whole, f1 = y_whole;
            if (fold && !back && rows != kChunk) f1 = decay_at(-l2, max(rows - 1 - row, 0)) * r.alpha_z;
            if (!fold && (late || (back && rows != kChunk))) f = decay_at(l2, back ? rows - row - late : row + 1 - late) * r.alpha_x;
            if (F16) {
                f1 = sm->row_scale[i & 1][row];
                if (reads) f *= sm->tile_scale[(enters ? i : i - 1) & 3];
            }
            const uint32_t y2 = lanes + cY2 + (F16 ? 0 : (i & 1) * 64), y1 = fold ? y2 : lanes + cG + (i & 1) * 128 + cY1;
            // 32 columns of out
            auto read = [&](int s, float* y) {
                if (!fold && reads) {
                    float x[32];
                    tmem_ld32x2(y1 + 32 * s, y, y2 + 32 * s, x);
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float2 o = mul2(make_float2(y[c], y[c + 1]), splat2(f1));
                        o = fma2(make_float2(x[c], x[c + 1]), splat2(f), o);
                        y[c] = o.x;
                        y[c + 1] = o.y;
                    }
                } else {
                    tmem_ld32(y1 + 32 * s, y);
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float2 o = mul2(make_float2(y[c], y[c + 1]), splat2(f1));
                        y[c] = o.x;
                        y[c + 1] = o.y;
                    }
                }
            };
            if (tiles) {
                // Rows go to Z's place, which the products have read, and leave from there in whole lines (a thread's own row in pieces of 32
                // bytes took 2100 cycles a chunk).
                unsigned char* at = smem + kZ + sz * kSub;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    float y[32];
                    read(s, y);
                    if (s == 1) {
                        fence_before();
                        mbar_arrive(&sm->y_empty[i & 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<uint4*>(at + sw_chunk(row, 4 * s + j)) =
                            make_uint4(pack2<Th>(y[8 * j], y[8 * j + 1]), pack2<Th>(y[8 * j + 2], y[8 * j + 3]),
                                       pack2<Th>(y[8 * j + 4], y[8 * j + 5]), pack2<Th>(y[8 * j + 6], y[8 * j + 7]));
                }
                if (bad) spoil_tile<Th>(at, row, pos, sm);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (t0 + (row & ~31) < p.T) tma_store_4d(&tp.out[w.role], at + (row & ~31) * 128, c0, h, t0 + (row & ~31), b);
                    tma_commit();
                    // (the last chunk's rows have been read from their place meanwhile: nobody waits for this chunk's)
                    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    if (i > 0) mbar_arrive(&sm->z_empty[sz == 0 ? zs - 1 : sz - 1]);
                }
            } else {
                const long long at = b * r.ob + static_cast<long long>(t0 + row) * r.ot + h * r.oh + c0;
                const int left = row < rows ? nc : 0;
#pragma unroll 1
                for (int s = 0; s < 2; ++s) {
                    float y[32];
                    read(s, y);
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (32 * s + c < left) {
                            if (r.out_f32) static_cast<float*>(r.out)[at + 32 * s + c] = y[c];
                            else static_cast<Th*>(r.out)[at + 32 * s + c] = from_f<Th>(y[c]);
                        }
                }
                if (bad) {
                    if (r.out_f32) spoil(static_cast<float*>(r.out) + at, 1, left, pos, sm);
                    else spoil(static_cast<Th*>(r.out) + at, 1, left, pos, sm);
                }
                fence_before();
                mbar_arrive(&sm->y_empty[i & 1]);
            }
            if (!tiles && lane == 0) mbar_arrive(&sm->z_empty[sz]);
            if (++sz == zs) {
                sz = 0;
                ++turn_z;
            }
        }
        if (tiles && lane == 0) tma_wait_read0();
    } else if (role == 4) {
        // ---- w o Z ----
        const float w_whole = decay_at(l2, back ? row : kChunk - 1 - row) * r.alpha_s;
        // The terms' own tiles are the last chunk's products' until they are done.  Folded, two tiles' worth is made meanwhile and kept in
        // registers, so that the stores alone stand between one chunk's products and the next one's: 1021 steps of 32 heads of 64 x 64 with their
        // states 23.4 -> 21.5 us.  (f16's two, in code that is twice as long, took a long text from 140 to 170.)
        constexpr bool ahead = fold && TERMS == 3;
        for (int i = 0, st = 0, turn = 0; i < n; ++i) {
            const int rows = min(kChunk, p.T - start(i));
            if (!wait_warp(&sm->z_full[st], turn & 1, sm, p.status)) break;
            float f = rows == kChunk ? w_whole : row < rows ? decay_at(l2, back ? row : rows - 1 - row) * r.alpha_s : 0.0f;
            unsigned char* z = smem + kZ + st * kSub;
            float undo = 1.0f;
            bool bad = false;
            if (F16) {
                // a power of two takes the tile's largest magnitude to 2^13: neither small values and weights nor those that grow leave the type
                __half2 top = __float2half2_rn(0.0f);
#pragma unroll 2
                for (int j = 0; j < 8; ++j) {
                    const uint4 v = *reinterpret_cast<const uint4*>(z + sw_chunk(row, j));
                    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(in + e)));
                }
                float m = __low2float(__hmax2_nan(top, __lowhigh2highlow(top)));
                bad = !(m < INFINITY);
                if (bad) m = finite_max(z, row);
                m = m > 0.0f ? m * fabsf(f) : 0.0f;
                m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
                if (lane == 0) {
                    sm->z_max[i & 1][warp & 3] = m;
                    mbar_arrive(&sm->z_max_full);
                }
                __syncwarp();
                if (!wait_warp(&sm->z_max_full, i & 1, sm, p.status)) break;
                const float* zm = sm->z_max[i & 1];
                f *= scale_to(fmaxf(fmaxf(zm[0], zm[1]), fmaxf(zm[2], zm[3])), &undo);
            }
            if (!ahead && (TERMS > 1 || !fold) && i > 0 && !wait_warp(&sm->d_full, (i - 1) & 1, sm, p.status)) break;
            if (F16 && row == 0) sm->z_scale[i & 1] = undo;  // (the sum of the chunk that had this place has been read: d_full of the one between)
            unsigned char* w0 = fold ? z : smem + kW;
            unsigned char* w1 = fold ? smem + kW - kSub : smem + kW;
            float2 zero = make_float2(0.0f, 0.0f);  // NaN, if a value is not finite
            uint4 kept[ahead ? 2 : 1][ahead ? 8 : 1];
#pragma unroll(ahead ? 8 : 2)
            for (int j = 0; j < 8; ++j) {
                const uint4 v = *reinterpret_cast<const uint4*>(z + sw_chunk(row, j));
                const uint32_t in[4] = {v.x, v.y, v.z, v.w};
                uint32_t o[TERMS][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float2 x = mul2(unpack2<Th>(in[e]), splat2(f));
                    if (!F16) zero = fma2(x, splat2(0.0f), zero);
                    o[0][e] = pack2<Th>(x.x, x.y);
#pragma unroll
                    for (int t = 1; t < TERMS; ++t) {
                        const float2 hi = unpack2<Th>(o[t - 1][e]);
                        x = make_float2(x.x - hi.x, x.y - hi.y);
                        if (F16) x = make_float2(x.x * 2048.0f, x.y * 2048.0f);
                        o[t][e] = pack2<Th>(x.x, x.y);
                    }
                }
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    const uint4 w = make_uint4(o[t][0], o[t][1], o[t][2], o[t][3]);
                    if (ahead && t > 0) kept[ahead ? t - 1 : 0][ahead ? j : 0] = w;
                    else *reinterpret_cast<uint4*>((t == 0 ? w0 : w1 + t * kSub) + sw_chunk(row, j)) = w;
                }
            }
            if (ahead) {
                if (i > 0 && !wait_warp(&sm->d_full, (i - 1) & 1, sm, p.status)) break;
#pragma unroll
                for (int t = 1; t < TERMS; ++t)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        *reinterpret_cast<uint4*>(w1 + t * kSub + sw_chunk(row, j)) = kept[ahead ? t - 1 : 0][ahead ? j : 0];
            }
            if (F16 ? bad : !(zero.x + zero.y == 0.0f)) set_aside<Th>(w0, w1 + kSub, TERMS - 1, z, row, i * kChunk + (back ? kChunk - 1 - row : row), sm);
            fence_proxy_async();
            mbar_arrive(&sm->w_full[st]);
            if (++st == zs) {
                st = 0;
                ++turn;
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    __syncwarp();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

// Heads whose state grows by more than kGrows over a chunk: the first 256 threads take the block's columns in 32 bits (a f16 tile whose weights
// lie further apart has no digits for the small ones, and they are all there is where the first keys are zeros).
constexpr float kGrows = 5.545f;  // 2^8
template <typename Th, bool STATE>
__device__ __noinline__ void grown(const TcParams& tp, unsigned char* smem, Place w) {
    const int half = threadIdx.x / gen::kThreads;
    w.tile = 2 * w.tile + half;
    static_assert(kTile == 2 * gen::kCols && 2 * gen::smem_bytes(128) <= 14 * kSub, "two parts of a block");
    if (half > 1 || w.tile * gen::kCols >= tp.p.role[w.role].W) return;
    gen::walk<Th, 4, STATE>(tp.p, w, reinterpret_cast<float*>(smem + half * gen::smem_bytes(128)), threadIdx.x % gen::kThreads, 1 + half);
}

template <typename Th, int TERMS, bool STATE>
__global__ void __launch_bounds__(kThreads, 1) walk_kernel(const __grid_constant__ TcParams tp) {
    extern __shared__ __align__(1024) unsigned char smem[];
    const Place w = place(tp.p, blockIdx.x, STATE ? tp.p.segments - 1 : tp.p.segments);
    const float ld = tp.p.decay[w.pair % tp.p.H];
    // `fold`: w o Z takes Z's place and P is G with its future cut off; what is missing, l^{row} up to a constant, is one factor a row of the
    // result.  Not where l^127 is small (kSlow), nor in f16.
    if constexpr (!std::is_same<Th, __half>::value) {
        if (ld <= 0.0f && ld * (kChunk - 1) >= -kSlow) {
            walk<Th, TERMS, STATE, true>(tp, smem, w, ld);
            return;
        }
    } else if (ld * (kChunk - 1) > kGrows) {
        grown<Th, STATE>(tp, smem, w);
        return;
    }
    walk<Th, TERMS, STATE, false>(tp, smem, w, ld);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [rows x 64 columns] of one head, 128-byte swizzled; rows behind the last step and columns behind the last one are zeros.
static bool make_map(Ctx* c, CUtensorMap* map, int dtype, const Operand& o, int H, int T, int B, int rows) {
    const int heads = H / o.group;
    if (!c->encode_tiled || reinterpret_cast<uintptr_t>(o.p) % 16) return false;
    const long long st = T > 1 ? o.st : (o.cols + 7) & ~7, sh = heads > 1 ? o.sh : 8, sb = B > 1 ? o.sb : 8;
    for (long long s : {st, sh, sb})
        if (s <= 0 || s % 8 || s >= (1ll << 38)) return false;
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(o.cols), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(T), static_cast<cuuint64_t>(B)};
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(st) * 2, static_cast<cuuint64_t>(sb) * 2};
    cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(rows), 1}, each[4] = {1, 1, 1, 1};
    return reinterpret_cast<EncodeTiledFn>(c->encode_tiled)(
               map, dtype == MAMBA_B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(o.p), dims,
               strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Th, int TERMS>
int launch(Ctx* c, TcParams& tp, long long pairs, cudaStream_t st) {
    tp.na = 1;
    tp.p.tiles = 0;
    for (int i = 0; i < tp.p.roles; ++i) {
        tp.p.tiles += tp.p.role[i].tiles;
        if (tp.p.role[i].A > 64) tp.na = 2;
    }
    const long long blocks = pairs * tp.p.tiles;
    tp.stages = tp.na == 2 ? 2 : 4;
    tp.z_tiles = kTiles - kCopies<TERMS>;
    const uint32_t smem = smem_bytes<TERMS>(tp.na, tp.stages, tp.z_tiles);
    if (tp.p.segments > 1) {
        walk_kernel<Th, TERMS, true><<<static_cast<unsigned>(blocks * (tp.p.segments - 1)), kThreads, smem, st>>>(tp);
        MB200_CUDA_CHECK(c, cudaGetLastError());
        const int rc = chain_segments(c, tp.p, pairs, st);
        if (rc) return rc;
    }
    walk_kernel<Th, TERMS, false><<<static_cast<unsigned>(blocks * tp.p.segments), kThreads, smem, st>>>(tp);
    MB200_CUDA_CHECK(c, cudaGetLastError());
    return MAMBA_B200_OK;
}

}  // namespace tcl

// Takes the call where the tensor cores' kernel can: 16-bit types, both widths up to 128, tensors that TMA can describe.  A tile has 128 rows
// whatever T is, and still a few steps take less than in the general kernel's chunks of 32: 2 of 32 heads of 128 x 64 5.8 us (8.0 there), with
// states 8.8 (14.3), 64 sequences of 32 steps with states 123 (372).
int tc_launch(Ctx* c, int dtype, Params& p, bool may_cut, long long pairs, cudaStream_t st, bool* taken) {
    using namespace tcl;
    *taken = false;
    if (dtype == MAMBA_B200_F32) return MAMBA_B200_OK;
    for (int i = 0; i < p.roles; ++i)
        if (p.role[i].A > 128 || p.role[i].W > 128) return MAMBA_B200_OK;
    // Roles that leave a state are kept in more terms, and those of narrow X and Y have room for more stages: up to four launches.
    TcParams tp[4];
    memset(tp, 0, sizeof(tp));
    auto kind = [](const Role& r) { return (r.s_out ? 2 : 0) + (r.A > 64 ? 1 : 0); };
    long long blocks = 0;
    int roles[4] = {0, 0, 0, 0};
    for (int i = 0; i < p.roles; ++i) {
        Role& r = p.role[i];
        TcParams& to = tp[kind(r)];
        int& k = roles[kind(r)];
        if (!make_map(c, &to.x[k], dtype, r.x, p.H, p.T, p.B, kChunk) || !make_map(c, &to.y[k], dtype, r.y, p.H, p.T, p.B, kChunk) ||
            !make_map(c, &to.z[k], dtype, r.z, p.H, p.T, p.B, kChunk))
            return MAMBA_B200_OK;
        const Operand out = {r.out, r.ob, r.ot, r.oh, 1, r.W};
        to.out_map[k] = !r.out_f32 && make_map(c, &to.out[k], dtype, out, p.H, p.T, p.B, 32);
        r.tiles = (r.W + kTile - 1) / kTile;
        blocks += pairs * r.tiles;
        ++k;
    }
    if (blocks > 1000000000ll / kMaxSegments) return MAMBA_B200_OK;
    const int chunks = (p.T + kChunk - 1) / kChunk;
    p.segments = may_cut ? pick_segments(c->sm_count, blocks, chunks, pairs, 1.9, 1.3, 14.0) : 1;
    const int per = (chunks + p.segments - 1) / p.segments;
    p.segments = (chunks + per - 1) / per;
    p.seg_len = per * kChunk;
    *taken = true;
    for (int q = 0; q < 4; ++q) {
        if (!roles[q]) continue;
        tp[q].p = p;
        tp[q].p.roles = 0;
        for (int i = 0; i < p.roles; ++i)
            if (kind(p.role[i]) == q) tp[q].p.role[tp[q].p.roles++] = p.role[i];
        const int rc = dtype == MAMBA_B200_F16 ? launch<__half, 2>(c, tp[q], pairs, st)
                       : q >= 2                ? launch<__nv_bfloat16, 3>(c, tp[q], pairs, st)
                                               : launch<__nv_bfloat16, 1>(c, tp[q], pairs, st);
        if (rc) return rc;
    }
    return MAMBA_B200_OK;
}

}  // namespace la

int linear_attention_tc_configure(Ctx* c) {
    using namespace la::tcl;
#define MB200_LA(Th, TERMS)                                                                                                              \
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)walk_kernel<Th, TERMS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,     \
                                             static_cast<int>(smem_bytes<TERMS>(2, 2, kTiles - kCopies<TERMS>))));                                                \
    MB200_CUDA_CHECK(c, cudaFuncSetAttribute((const void*)walk_kernel<Th, TERMS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,      \
                                             static_cast<int>(smem_bytes<TERMS>(2, 2, kTiles - kCopies<TERMS>))));
    MB200_LA(__half, 2)
    MB200_LA(__nv_bfloat16, 1)
    MB200_LA(__nv_bfloat16, 3)
#undef MB200_LA
    return MAMBA_B200_OK;
}

}  // namespace mb200
