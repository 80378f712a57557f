// Gated delta rule: shared pieces of the kernels that build operand tiles in shared memory and multiply them with
// mma.sync (fragments of 16 x 16 and 16 x 8 blocks of the swizzled panels of delta.cuh).
#pragma once

#include "common.cuh"
#include "delta.cuh"

namespace aussm {

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Addresses of the four 8 x 8 blocks that a lane names to ldmatrix (tile: rows x columns as stored):
// A block of 16 rows x 16 contraction columns at (row, col)
__device__ __forceinline__ int frag_a(int row, int col) {
    const int lane = threadIdx.x & 31;
    return panel_at(row + (lane & 15), col + (lane >> 4) * 8);
}
// the same block of A^T: contraction along the rows as stored (for ldmatrix4_trans)
__device__ __forceinline__ int frag_at(int krow, int mcol) {
    const int lane = threadIdx.x & 31;
    return panel_at(krow + (lane & 7) + (lane >> 4) * 8, mcol + ((lane >> 3) & 1) * 8);
}
// B: 16 columns n stored as rows, contraction along the columns
__device__ __forceinline__ int frag_b(int nrow, int kcol) {
    const int lane = threadIdx.x & 31;
    return panel_at(nrow + (lane & 7) + ((lane >> 4) << 3), kcol + ((lane >> 3) & 1) * 8);
}
// B: contraction along the rows as stored, 16 columns n (for ldmatrix4_trans)
__device__ __forceinline__ int frag_bt(int krow, int ncol) {
    const int lane = threadIdx.x & 31;
    return panel_at(krow + (lane & 15), ncol + (lane >> 4) * 8);
}

// whether beta of a step is zero for all `heads` value heads that share a key head
__device__ __forceinline__ bool all_idle(const float* beta, int heads) {
    bool idle = true;
    for (int h = 0; h < heads; ++h) idle = idle && beta[h] == 0.f;
    return idle;
}
__device__ __forceinline__ bool finite8(const float (&f)[8]) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = all && rank_of(f[i]) >= 0x01000000u;
    return all;
}
__device__ __forceinline__ void keep_finite8(float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = finite_or_zero(f[i]);
}

// eight consecutive elements of a row, zeros from `cols` on
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int cols, bool vec, float (&f)[8]) {
    if (vec) {
        if (c < cols) {
            constexpr int N = 16 / sizeof(T);
            struct alignas(16) Raw { T v[N]; };
#pragma unroll
            for (int k = 0; k < 8 / N; ++k) {
                const Raw r = *reinterpret_cast<const Raw*>(row + c + k * N);
#pragma unroll
                for (int i = 0; i < N; ++i) f[k * N + i] = to_f32(r.v[i]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = c + i < cols ? to_f32(row[c + i]) : 0.f;
    }
}
__device__ __forceinline__ void zero8(float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
}
__device__ __forceinline__ uint32_t max8(const float (&f)[8], uint32_t m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, rank_of(f[i]));
    return m;
}
__device__ __forceinline__ void split8(const float (&f)[8], float s, uint4& hi, uint4& lo) {
    split2(f[0] * s, f[1] * s, hi.x, lo.x);
    split2(f[2] * s, f[3] * s, hi.y, lo.y);
    split2(f[4] * s, f[5] * s, hi.z, lo.z);
    split2(f[6] * s, f[7] * s, hi.w, lo.w);
}
// the parts of eight values to a tile
__device__ __forceinline__ void put8(uint8_t* at, int lo_off, const float (&f)[8], float s) {
    uint4 hi, lo;
    split8(f, s, hi, lo);
    *reinterpret_cast<uint4*>(at) = hi;
    *reinterpret_cast<uint4*>(at + lo_off) = lo;
}
// what eight stored hi and lo parts stand for, times f
__device__ __forceinline__ void join8(const uint8_t* hi, const uint8_t* lo, float f, float (&v)[8]) {
    const uint4 h4 = *reinterpret_cast<const uint4*>(hi), l4 = *reinterpret_cast<const uint4*>(lo);
    const __half2 *hp = reinterpret_cast<const __half2*>(&h4), *lp = reinterpret_cast<const __half2*>(&l4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(hp[i]), b = __half22float2(lp[i]);
        v[2 * i] = (a.x + b.x) * f;
        v[2 * i + 1] = (a.y + b.y) * f;
    }
}

// maximum over LANES neighbouring lanes
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
#pragma unroll
    for (int m = 1; m < LANES; m *= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// maxima of N ranks over the block of WARPS warps; `buf` has N * WARPS words and is free again after the next barrier
template <int WARPS, int N>
__device__ __forceinline__ void block_max(uint32_t (&v)[N], uint32_t* buf) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __reduce_max_sync(0xffffffffu, v[i]);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) buf[i * WARPS + (threadIdx.x >> 5)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v[i] = max(v[i], buf[i * WARPS + w]);
    }
}

}  // namespace aussm
