// Gated delta rule: sizes, buffers and launchers shared by its translation units.
//
// Per value head, with a_t = exp(g_t), state S (dk, dv) and e_t = beta_t (v_t - a_t S_{t-1}^T k_t):
//     S_t = a_t S_{t-1} + k_t e_t^T,     o_t = scale S_t^T q_t.
// Over a chunk of C = 64 steps with entry state S, G_i = g_1 + ... + g_i, the e_i are the rows of the V' that solves
//     (I + A) V' = beta (V - e^G K S),   A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i),
// so with T = (I + A)^-1, W = T beta e^G K, P_ij = scale e^(G_i - G_j) q_i.k_j (j <= i), Qt = scale e^G Q and
// Kt = e^(G_C - G) K:
//     V' = T beta V - W S,     O = Qt S + P V',     S <- e^(G_C) S + Kt^T V'.
// Backward, from the gradient dS of the chunk's exit state and dO:
//     dV' = P^T dO + Kt dS,   X = T^T dV',   dV = beta X,   dS <- e^(G_C) dS + Qt^T dO - W^T dV',
//     dP = tril(dO V'^T),  dA = -stril(X V'^T),  dQt = dO S^T,  Z = X S^T,  dKt = V' dS^T,
// and from these the gradients of q, k, beta and g.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/aussm_b200.h"

namespace aussm {

constexpr int kDeltaChunk = 64;
inline int delta_chunks(int steps) { return steps / kDeltaChunk + (steps % kDeltaChunk != 0); }      // L + 63 need not fit

// ---- operand tiles -----------------------------------------------------------------------------------------------
// Products run on FP16 parts: with S the power of two that brings a tile's largest magnitude to 2^13..2^14,
// hi = fp16(S a), lo = fp16(S a - hi): 22 significant bits down to 2^-17 of the largest element and an absolute error of
// 2^-39 of it below; a product is hi hi + hi lo + lo hi.  A tile of 64 rows is stored the way the tensor core reads it
// from shared memory: panels of 64 columns (64 rows of 128 bytes, 16-byte pieces swizzled by the row), the hi panels
// and then the lo panels.  Rows of 128 bytes serve as K-major and as MN-major operands alike.
//
// Queries differ in size, and no output has a share in another's query: rows of Q are brought to one size by a power of two
// of their own, r_i, before anything else (Q / r in P and Qt).  O's rows are multiplied with r_i when they leave, dO's rows
// with r_i when they come in as the operand of P and Qt.
// Keys above 1 would have their share of a tile's scale even where beta is zero (a padded step: unwritten memory may lie
// there).  Their rows are divided by a power of two kappa_i >= 1 that brings them into 1..2 (unit keys: 1): with k^ = k /
// kappa, beta^ = beta kappa^2 and v^ = v / kappa the rule is the same, S and O are the same and V'^ = kappa V', X^ = X / kappa.
// K, beta and V' stand for these in all tiles and kernels; beta^ v^ = (beta kappa) v, dv = (beta kappa) X^, dk = dk^ / kappa,
// dbeta = kappa^2 dbeta^.
//
// Per chunk and value head one record of such tiles (`key` = DK rounded up to 64 or 128):
struct DeltaRecord {
    int key;                                            // columns of W, Kt, Q
    static constexpr int kHead = 1536;                  // bytes of the header
    static constexpr int kSquare = 16384;               // bytes of a 64 x 64 tile, hi and lo
    __host__ __device__ int tile() const { return key * 256; }
    __host__ __device__ int w() const { return kHead; }                             // W = T beta e^G K
    __host__ __device__ int kt() const { return kHead + tile(); }                   // Kt = e^(G_C - G) K
    __host__ __device__ int q() const { return kHead + 2 * tile(); }                // Qt = scale e^G Q / r
    __host__ __device__ int t() const { return kHead + 3 * tile(); }                // T = (I + A)^-1
    __host__ __device__ int p() const { return kHead + 3 * tile() + kSquare; }      // P / r
    __host__ __device__ int bytes() const { return kHead + 3 * tile() + 2 * kSquare; }
};
// header, in floats: what a stored part is to be multiplied with (1 / S) ...
enum : int { kUnW = 0, kUnKt = 1, kUnQ = 2, kUnT = 3, kUnP = 4, kGamma = 5 /* e^(G_C) */,
             kBeta = 16 /* beta kappa, 64 */, kGHi = 80, kGLo = 144 /* G_i = hi + lo, 64 each */, kRow = 208 /* r, 64 */,
             kKey = 272 /* kappa, 64 */,
             kIdle = 6 /* 2 words: bit i of the first is set when beta of step 2 i is zero, of the second 2 i + 1 */ };

// byte offset of element (row, col) in the hi panels of a tile
__host__ __device__ __forceinline__ int panel_at(int row, int col) {
    return (col >> 6) * 8192 + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

__host__ __device__ __forceinline__ float pow2_float(int k) {
#ifdef __CUDA_ARCH__
    return __uint_as_float((unsigned)(127 + k) << 23);
#else
    return 0.f;
#endif
}
// 1 / x for a power of two x from 2^-126 to 2^126
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
// exponent k of the scale 2^k for a tile whose largest magnitude is m
__device__ __forceinline__ int part_exponent(float m) {
    const int e = (int)((__float_as_uint(m) >> 23) & 0xffu) - 127;
    return max(-115, min(115, 13 - e));                  // the whole range of float32
}
// The same from the largest of the values' ranks: unsigned numbers in the order of the magnitudes, with what is not finite
// below zero.  An infinity would set a scale that turns every finite element of its tile into zero; so it sets none, and
// stays an infinity (and its lo part a NaN) in the conversion.
__device__ __forceinline__ uint32_t rank_of(float x) { return (__float_as_uint(x) << 1) + 0x01000000u; }
__device__ __forceinline__ int rank_exponent(uint32_t r) { return max(-115, min(115, 13 + 128 - (int)(r >> 24))); }
// exponent of kappa for a row of keys, and the rank of what is left of x behind the division
__device__ __forceinline__ int key_exponent(uint32_t r) { return max(0, min(126, (int)(r >> 24) - 128)); }
__device__ __forceinline__ int key_exponent_of(float kappa) { return (int)(__float_as_uint(kappa) >> 23) - 127; }
__device__ __forceinline__ uint32_t rank_less(uint32_t r, int c) { return r - min(r, (uint32_t)c << 24); }
// hi and lo parts of two values that are scaled already, packed
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

struct DeltaInputs {
    const void *q, *k, *v;
    const float *g, *beta;
};

// Keys and values of a step with beta = 0 (padding: unwritten memory may lie there) count as zero where they are not finite:
// they are multiplied with zeros only, which would make NaN of them.
__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.f; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// exp(-200) is zero in float32: g of -inf (forget everything) would make differences of its sums NaN
__device__ __forceinline__ float clamp_log_decay(float g) { return g < -200.f ? -200.f : g; }

// What the recurrences leave for the gradients, per chunk, value head and slice of 128 value columns, as it lies in tensor
// memory: 16 bytes of a lane (value column) after the other, [words / 4][128 lanes].  A state: `key` words a lane (8 keys in
// 4 words of hi parts, then the lo parts), V': 64 words (8 steps in 4 words), and behind them the lanes' float32 factors.
// X: 64 float32 words a lane.
//
// Sizes and buffers of a problem.  keep: [records][transitions][ends][V'][entry states] (the first three are the workspace
// of a forward call without a backward one), backward workspace: [X][gradients of exit states][ends].
//
// Few heads leave most of the GPU idle: the chunks are then cut into `segs` segments of `span` that run side by side.  A pass
// gives what a segment makes of a zero state and one what it does to a state (its transition, DK x DK; the backward pass
// uses the transposed ones of the forward pass), a chain over the segments the states at their boundaries, and the pass
// with all outputs starts every segment from its own.
struct DeltaPlan {
    int n;                 // chunks of a sequence
    int slices;            // of 128 value columns
    int segs, span;        // segments of the recurrences, chunks of one
    __host__ __device__ static size_t state_bytes(int key) { return (size_t)key * 512 + 512; }
    __host__ __device__ static size_t news_bytes() { return 64 * 512 + 512; }
    __host__ __device__ static size_t x_bytes() { return 64 * 512; }
    size_t heads;          // chunk heads: (b * HV + h) * n + chunk
    DeltaRecord rec;
    size_t keep_bytes, fwd_bytes, bwd_bytes;
    size_t transitions, ends, news, states;   // byte offsets in keep
    size_t dstates, bwd_ends;                 // byte offsets in the backward workspace
};
DeltaPlan delta_plan(const aussm_b200_delta_t& p);

cudaError_t launch_delta_prepare(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaInputs& in, void* records,
                                 cudaStream_t stream);
// the recurrence over chunks, forward or (V -> dO, O -> dV, V' -> X, states -> gradients) backward
struct DeltaScan {
    const void* records;
    const void* v;
    const float* s0;
    float* s1;
    void* out;
    void *rows, *states;       // V' / X and entry states / gradients of exit states; forward: NULL = not kept
    void *transitions, *ends;  // of the segments (forward writes the transitions, backward reads them)
};
cudaError_t launch_delta_scan(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaScan& io, bool backward,
                              cudaStream_t stream);
struct DeltaGrads {
    const void *records, *go;
    const void *news, *x, *states, *dstates;
    void *dq, *dk;
    float *dg, *dbeta;
};
cudaError_t launch_delta_grads(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaInputs& in, const DeltaGrads& io,
                               cudaStream_t stream);
cudaError_t launch_delta_fwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* s0, void* o, float* s1,
                             void* keep, bool train, cudaStream_t stream);
cudaError_t launch_delta_bwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const void* go, const float* gs1,
                             const void* keep, void* dq, void* dk, void* dv, float* dg, float* dbeta, float* ds0,
                             void* workspace, cudaStream_t stream);
cudaError_t launch_delta_step(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* state, float* new_state,
                              void* o, cudaStream_t stream);

}  // namespace aussm
