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

struct DeltaInputs {
    const void *q, *k, *v;
    const float *g, *beta;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// exp(-200) is zero in float32: g of -inf (forget everything) would make differences of its sums NaN
__device__ __forceinline__ float clamp_log_decay(float g) { return g < -200.f ? -200.f : g; }

cudaError_t launch_delta_fwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* s0, void* o, float* s1,
                             void* keep, cudaStream_t stream);
cudaError_t launch_delta_bwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const void* go, const float* gs1,
                             const void* keep, void* dq, void* dk, void* dv, float* dg, float* dbeta, float* ds0,
                             void* workspace, cudaStream_t stream);
cudaError_t launch_delta_step(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* state, float* new_state,
                              void* o, cudaStream_t stream);
size_t delta_keep_bytes(const aussm_b200_delta_t& p);
size_t delta_bwd_bytes(const aussm_b200_delta_t& p);

}  // namespace aussm
