// Linear attention with a decay for each head: what its two kernels share.
//
// Forward and every gradient are one operation on other operands,
//   out_t = alpha_p * sum_{s <= t} l^{t-s} (x_t . y_s) z_s + alpha_x * (decayed entering state)^T x_t,   l = exp(decay[h]),
//   state: S <- l S + alpha_s y z^T  (rows: y's columns, columns: z's),
// with time running from the start or from the end ("role"):
//   o   : x = q,  y = k,  z = v,  forwards,  state S                  alpha_p = alpha_x = scale, alpha_s = 1
//   d_q : x = do, y = v,  z = k,  forwards,  state S^T                alpha_p = alpha_x = scale, alpha_s = 1
//   d_k : x = v,  y = do, z = q,  backwards, gradient of S^T          alpha_p = alpha_s = scale, alpha_x = 1
//   d_v : x = k,  y = q,  z = do, backwards, gradient of S            alpha_p = alpha_s = scale, alpha_x = 1
// so the backward makes the states again on the way and reads nothing that the forward would have to save.  The gradient of the
// state that left belongs to the last step itself (`late`: it decays one step less than an entering state), and the gradient
// of the state that entered has one decay more (`last_decay`).
#pragma once
#include "common.cuh"
#include "internal.h"

namespace mb200 {
namespace la {

constexpr int kChunk = 128;     // steps of a tensor-core tile
constexpr int kSteps = 32;      // steps of a chunk of the general kernel (segments are whole chunks)
constexpr int kMaxSegments = 64;
constexpr int kMaxDim = 256;    // of K and V

struct Operand {
    const void* p;
    long long sb, st, sh;  // strides of batch, step, head (elements)
    int group;             // heads that read one of its heads
    int cols;
};

struct Role {
    Operand x, y, z;
    int A, W;  // columns of x and y, columns of z and out
    void* out;
    long long ob, ot, oh;
    int out_f32;          // partial sums of shared heads
    const float* s_in;    // entering state: element (a, w) of a head at a * sa + w * sw (null: zeros)
    int sa, sw;
    float* s_out;         // leaving state [A, W] (null: not wanted)
    int backwards, late, last_decay;
    float alpha_p, alpha_x, alpha_s;
    float alpha_z;        // alpha_p / alpha_s
    int tiles;            // column tiles of W
    float* slots;         // [B * H][segments][A * W]: slot 0 the entering state, slot r what segment r - 1 leaves of it or adds to a state,
                          // and after chain_segments() the state that enters segment r
};

struct Params {
    Role role[3];
    int roles, tiles, B, T, H;  // tiles: of all roles
    int segments, seg_len;  // seg_len: steps of a segment, whole chunks
    const float* decay;
    int* status;
};

// The role and place of a block: pair = b * H + h.  The roles and column tiles of a pair's segment are neighbours: they read the same
// rows at about the same time, which the later ones find in L2.
struct Place {
    int role, tile, seg;
    long long pair;
};
__device__ __forceinline__ Place place(const Params& p, long long block, int segments) {
    Place w;
    const long long i = block / p.tiles;
    w.tile = static_cast<int>(block - i * p.tiles);
    w.role = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r)
        if (r + 1 < p.roles && w.role == r && w.tile >= p.role[r].tiles) {
            w.tile -= p.role[r].tiles;
            w.role = r + 1;
        }
    w.seg = static_cast<int>(i % segments);
    w.pair = i / segments;
    return w;
}

// l^n for n steps as a sum of two floats: a state that is carried over many chunks is multiplied by it again and again, and
// the rounding of one float (2^-25, always the same way) would add up.
struct Pow {
    float hi, lo;
};
__device__ __forceinline__ Pow decay_pow(float log_decay, int n) {
    Pow r{1.0f, 0.0f};
    if (n > 0) {
        const double e = exp(static_cast<double>(log_decay) * n);
        r.hi = static_cast<float>(e);
        r.lo = isinf(r.hi) ? 0.0f : static_cast<float>(e - static_cast<double>(r.hi));
    }
    return r;
}
__device__ __forceinline__ float times(const Pow& f, float s) { return fmaf(f.hi, s, f.lo * s); }
// l^n, n >= 0, in 32 bits (n = 0: 1 for every decay, minus infinity among them)
__device__ __forceinline__ float decay_at(float log2_decay, int n) { return n > 0 ? exp2f(log2_decay * n) : 1.0f; }

// Turns what each segment adds to a state (slots 1 ...) into what enters the next one, in place.
int chain_segments(Ctx* c, const Params& p, long long pairs, cudaStream_t st);
int pick_segments(long long together, long long blocks, int units, long long pairs, double full, double state, double second);
// linear_attention_tc.cu: launches, if it takes such a call (`taken`).
int tc_launch(Ctx* c, int dtype, Params& p, bool may_cut, long long pairs, cudaStream_t st, bool* taken);

}  // namespace la
}  // namespace mb200
