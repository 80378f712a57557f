// Gated delta rule, the recurrence itself: for one or a few new steps of each sequence.
//
// Bound: every state is read once and written once (2 DK DV 4 bytes a value head; everything else is small).  A block
// holds 32 or 128 value columns of one state in registers: 8 or 32 lanes of 4 columns make a piece of a row, all of up to
// 128 rows are in flight at once.  Since
//     S' = a S + k e^T  with  e = beta (v - a S^T k),     S'^T q = a S^T q + (k.q) e,
// one pass over the state gives both S^T k and S^T q: one reduction over the block and the state is written back, past the
// L2 (streaming accesses: 104 -> 91 us).  4096 states of 128 x 128: 91 us, 5.9 TB/s, with whole rows a block, 129 us with 32
// columns (before streaming).  One sequence of 8 heads fills 32 SMs with 32 columns a block, 8 with whole rows, and takes
// 2.8 us: hence whole rows only from 4 states an SM on.
#include "delta.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int NT = 256, WARPS = NT / 32;

struct StepParams {
    aussm_b200_delta_t p;
    DeltaInputs in;
    const float* state;
    float* new_state;
    void* o;
};

// VEC 4: 8 lanes a row, VEC 1 (DV no multiple of 4, or unaligned states): 32 lanes a row
template <typename T, int VEC, int COLS>
__global__ void __launch_bounds__(NT) delta_step_kernel(const StepParams a) {
    constexpr int LANES = COLS / VEC, ROWS = NT / LANES, RPT = AUSSM_MAX_DELTA_KEY / ROWS;
    __shared__ float ks[2][AUSSM_MAX_DELTA_KEY], qs[2][AUSSM_MAX_DELTA_KEY];
    __shared__ float rk[2][WARPS][COLS], rq[2][WARPS][COLS], rkq[2][WARPS];
    const aussm_b200_delta_t& p = a.p;
    const int slices = (p.DV + COLS - 1) / COLS;
    const int slice = blockIdx.x % slices, bh = blockIdx.x / slices, b = bh / p.HV, h = bh % p.HV, hk = h / (p.HV / p.HK);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = threadIdx.x / LANES, lcol = lane % LANES * VEC, col = slice * COLS + lcol;
    const bool mine = col < p.DV;
    const size_t base = (size_t)bh * p.DK * p.DV + col;
    float S[RPT][VEC];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = row0 + i * ROWS;
        const float* src = a.state + base + (size_t)row * p.DV;
#pragma unroll
        for (int c = 0; c < VEC; ++c) S[i][c] = 0.f;
        if (mine && row < p.DK) {
            if (VEC == 4) {
                const float4 x = __ldcs(reinterpret_cast<const float4*>(src));     // read once: first to leave the L2
                S[i][0] = x.x; S[i][1 % VEC] = x.y; S[i][2 % VEC] = x.z; S[i][3 % VEC] = x.w;
            } else {
                S[i][0] = *src;
            }
        }
    }
    const T* q = static_cast<const T*>(a.in.q) + b * p.q_stride[0] + hk * p.q_stride[2];
    const T* k = static_cast<const T*>(a.in.k) + b * p.k_stride[0] + hk * p.k_stride[2];
    const T* v = static_cast<const T*>(a.in.v) + b * p.v_stride[0] + h * p.v_stride[2];
    for (int t = 0; t < p.L; ++t) {
        const int buf = t & 1;
        const long long gh = ((long long)b * p.L + t) * p.HV + h;
        const float decay = expf(a.in.g[gh]), beta = a.in.beta[gh];
        auto taken = [&](float x) { return beta == 0.f ? finite_or_zero(x) : x; };         // a key or value
        if (threadIdx.x < AUSSM_MAX_DELTA_KEY)
            ks[buf][threadIdx.x] = threadIdx.x < p.DK ? taken(to_f32(k[t * p.k_stride[1] + threadIdx.x])) : 0.f;
        else if (threadIdx.x < 2 * AUSSM_MAX_DELTA_KEY) {
            const int x = threadIdx.x - AUSSM_MAX_DELTA_KEY;
            qs[buf][x] = x < p.DK ? to_f32(q[t * p.q_stride[1] + x]) : 0.f;
        }
        float val[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) val[c] = mine ? taken(to_f32(v[t * p.v_stride[1] + col + c])) : 0.f;
        __syncthreads();
        float pk[VEC] = {}, pq[VEC] = {}, kq = 0.f;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float kr = ks[buf][row0 + i * ROWS], qr = qs[buf][row0 + i * ROWS];
            kq += kr * qr;
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                S[i][c] *= decay;
                pk[c] += kr * S[i][c];
                pq[c] += qr * S[i][c];
            }
        }
#pragma unroll
        for (int m = LANES; m < 32; m *= 2) {
            kq += __shfl_xor_sync(0xffffffffu, kq, m);
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                pk[c] += __shfl_xor_sync(0xffffffffu, pk[c], m);
                pq[c] += __shfl_xor_sync(0xffffffffu, pq[c], m);
            }
        }
        if (lane < LANES) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                rk[buf][warp][lcol + c] = pk[c];
                rq[buf][warp][lcol + c] = pq[c];
            }
            if (lane == 0) rkq[buf][warp] = kq;
        }
        __syncthreads();
        float e[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) s += rk[buf][w][lcol + c];
            e[c] = beta * (val[c] - s);
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int c = 0; c < VEC; ++c) S[i][c] = fmaf(ks[buf][row0 + i * ROWS], e[c], S[i][c]);
        if (threadIdx.x < LANES && mine) {
            float kqs = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) kqs += rkq[buf][w];
            T* o = static_cast<T*>(a.o) + gh * p.DV + col;
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) s += rq[buf][w][lcol + c];
                o[c] = from_f32<T>(p.scale * fmaf(kqs, e[c], s));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int row = row0 + i * ROWS;
        float* dst = a.new_state + base + (size_t)row * p.DV;
        if (mine && row < p.DK) {
            if (VEC == 4) __stcs(reinterpret_cast<float4*>(dst), make_float4(S[i][0], S[i][1 % VEC], S[i][2 % VEC], S[i][3 % VEC]));
            else *dst = S[i][0];
        }
    }
}

template <typename T>
void step(const StepParams& a, cudaStream_t st) {
    const long long heads = (long long)a.p.B * a.p.HV;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.new_state);
    const bool vec = a.p.DV % 4 == 0 && bits % 16 == 0;
    if (vec && heads >= 148 * 4 && a.p.DV > 64) delta_step_kernel<T, 4, 128><<<(unsigned)(heads * ((a.p.DV + 127) / 128)), NT, 0, st>>>(a);
    else if (vec) delta_step_kernel<T, 4, 32><<<(unsigned)(heads * ((a.p.DV + 31) / 32)), NT, 0, st>>>(a);
    else delta_step_kernel<T, 1, 32><<<(unsigned)(heads * ((a.p.DV + 31) / 32)), NT, 0, st>>>(a);
    count_launch();
}

}  // namespace

cudaError_t launch_delta_step(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* state, float* new_state,
                              void* o, cudaStream_t st) {
    const StepParams a = {p, in, state, new_state, o};
    if (p.dtype == AUSSM_FLOAT32) step<float>(a, st);
    else if (p.dtype == AUSSM_BFLOAT16) step<__nv_bfloat16>(a, st);
    else step<__half>(a, st);
    return cudaGetLastError();
}

}  // namespace aussm
