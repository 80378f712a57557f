// Queries and keys: norm over each head and rotation by position in one pass, forward and backward.
//
//     y = R(position) (x r w),   r = rsqrt(mean(x^2) + eps)  (rms)  or  rsqrt(sum(x^2) + eps)  (l2)  or  1,
// R turns pair p by position * frequency_p and scales it by `magnitude`; elements behind the rotated part pass.
// Backward, with h = R^T dy and the mean / sum over the head:  dw = sum h x r,  dx = r (h w - x r^2 mean(h w x)).
//
// Bound: memory, every element read once and written once.  A group of 8, 16 or 32 lanes holds a head, both elements
// of a pair in the same lane: the norm is a few shuffles, the rotation none.  The lane's angles and weights serve the
// heads of a token that the group walks: all of them where the tokens fill the GPU, fewer otherwise.  Angles are reduced in 64 bits: position *
// (frequency / 2 pi), less its nearest integer, so a position of 2^22 is turned as exactly as position 1.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/aussm_b200.h"
#include "delta.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int NT = 256;
constexpr int IN_FLIGHT = 4;             // heads of a group whose loads are in flight together
constexpr int MAX_BLOCKS = 148 * 8;      // of the backward kernel: each leaves one partial sum of the weights' gradients

struct RotateParams {
    aussm_b200_rotate_t p;
    const void *x[2], *dy[2];
    void* out[2];                        // y, or dx
    const float* w[2];
    const double* frequencies;
    const long long* positions;
    float* part;                         // (blocks, 2, d) partial sums of dw, or NULL
    int split;                           // groups a token: group k walks heads k, k + split, ..
    int units, rot_units;
    unsigned groups;
};

// VEC consecutive elements as one access (VEC 4: the row is aligned to 4 elements)
template <int VEC, typename T>
__device__ __forceinline__ void load(const T* p, float (&f)[VEC]) {
    if (VEC == 1) f[0] = to_f32(*p);
    else {
        struct alignas(sizeof(T) * VEC) Raw { T v[VEC]; };
        const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = to_f32(r.v[i]);
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    if (VEC == 1) *p = from_f32<T>(f[0]);
    else {
        struct alignas(sizeof(T) * VEC) Raw { T v[VEC]; } r;
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = from_f32<T>(f[i]);
        *reinterpret_cast<Raw*>(p) = r;
    }
}

// A unit: VEC elements at e0 and VEC at e1.  Rotated units come first: in the half layout e1 = e0 + n and pair i is
// (e0 + i, e1 + i); in the interleaved one the 2 VEC elements are consecutive and hold VEC pairs.  Units behind them
// hold 2 VEC consecutive elements that are not rotated; `second`: whether the row has the last VEC of them.
template <int VEC>
struct Unit {
    int e0, e1;
    bool any, second, turns;
    __device__ Unit(const RotateParams& a, int u) {
        const int n = a.p.rot / 2;
        any = u < a.units;
        turns = u < a.rot_units;
        if (turns && !a.p.interleaved) { e0 = u * VEC; e1 = e0 + n; second = true; }
        else if (turns) { e0 = 2 * u * VEC; e1 = e0 + VEC; second = true; }
        else { e0 = a.p.rot + 2 * (u - a.rot_units) * VEC; e1 = e0 + VEC; second = any && e1 < a.p.d; }
    }
};

template <int VEC>
struct Angles {
    float c[VEC], s[VEC];
    // pairs VEC * u ... of the rotated part
    __device__ void set(const RotateParams& a, int u, bool turns, long long pos) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) { c[i] = 1.f; s[i] = 0.f; }
        if (turns) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const double turn = (double)pos * (a.frequencies[u * VEC + i] * 0.15915494309189535);    // 1 / (2 pi)
                sincospif(2.f * (float)(turn - rint(turn)), &s[i], &c[i]);
                s[i] *= a.p.magnitude;
                c[i] *= a.p.magnitude;
            }
        }
    }
    // (x, y) -> the turned pairs; sign -1 turns back
    __device__ __forceinline__ void turn(bool interleaved, float (&x)[VEC], float (&y)[VEC], float sign) const {
        if (interleaved) {
            float z[2 * VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) { z[i] = x[i]; z[VEC + i] = y[i]; }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float u = z[2 * i], v = z[2 * i + 1], t = sign * s[i];
                z[2 * i] = u * c[i] - v * t;
                z[2 * i + 1] = v * c[i] + u * t;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) { x[i] = z[i]; y[i] = z[VEC + i]; }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float u = x[i], v = y[i], t = sign * s[i];
                x[i] = u * c[i] - v * t;
                y[i] = v * c[i] + u * t;
            }
        }
    }
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int m = 1; m < G; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// The heads of one token and tensor that this group walks.  FLY of them are in flight together.
template <typename T, int VEC, int G, int UPL, bool BWD>
struct Walk {
    static constexpr int FLY = UPL > 1 ? 1 : BWD ? IN_FLIGHT / 2 : IN_FLIGHT;
    float w[UPL][2][VEC];                // weights of the lane's elements
    float dw[BWD ? UPL : 1][2][VEC];     // their gradients

    __device__ void start(const RotateParams& a, int which, int lane) {
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
            const Unit<VEC> at(a, lane + u * G);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                w[u][0][i] = w[u][1][i] = 1.f;
                if (BWD) dw[u][0][i] = dw[u][1][i] = 0.f;
            }
            if (a.w[which] && at.any) load<VEC>(a.w[which] + at.e0, w[u][0]);
            if (a.w[which] && at.second) load<VEC>(a.w[which] + at.e1, w[u][1]);
        }
    }
    // x, g, out: the token's first head; `heads` of them, the strides between them
    __device__ void run(const RotateParams& a, const Angles<VEC> (&ang)[UPL], int lane, const T* x, long long xs, const T* g,
                        long long gs, T* out, int part, int heads, bool live) {
        const bool norm = a.p.norm != AUSSM_NORM_NONE, need = !BWD || norm || a.part;
        const float inv_d = a.p.norm == AUSSM_NORM_RMS ? 1.f / (float)a.p.d : 1.f;
        for (int base = 0; base < heads; base += FLY * a.split) {          // as often for all groups of a warp: shuffles
            const int h = base + part;
            float v[FLY][UPL][2][VEC], y[BWD ? FLY : 1][UPL][2][VEC];
#pragma unroll
            for (int f = 0; f < FLY; ++f) {
                const int hh = h + f * a.split;
#pragma unroll
                for (int u = 0; u < UPL; ++u) {
                    const Unit<VEC> at(a, lane + u * G);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        v[f][u][0][i] = v[f][u][1][i] = 0.f;
                        if (BWD) y[f % (BWD ? FLY : 1)][u][0][i] = y[f % (BWD ? FLY : 1)][u][1][i] = 0.f;
                    }
                    if (hh >= heads) continue;
                    if (need && at.any) load<VEC>(x + hh * xs + at.e0, v[f][u][0]);
                    if (need && at.second) load<VEC>(x + hh * xs + at.e1, v[f][u][1]);
                    if (BWD && at.any) load<VEC>(g + hh * gs + at.e0, y[f % (BWD ? FLY : 1)][u][0]);
                    if (BWD && at.second) load<VEC>(g + hh * gs + at.e1, y[f % (BWD ? FLY : 1)][u][1]);
                }
            }
#pragma unroll
            for (int f = 0; f < FLY; ++f) {
                const int hh = h + f * a.split;
                const bool keep = live && hh < heads;
                float rstd = 1.f, dot = 0.f;
                if (norm) {
                    float sq = 0.f;
#pragma unroll
                    for (int u = 0; u < UPL; ++u)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) sq += v[f][u][0][i] * v[f][u][0][i] + v[f][u][1][i] * v[f][u][1][i];
                    rstd = rsqrtf(group_sum<G>(sq) * inv_d + a.p.eps);
                }
                T* dst = out + (long long)hh * a.p.d;
#pragma unroll
                for (int u = 0; u < UPL; ++u) {
                    const Unit<VEC> at(a, lane + u * G);
                    float (&v0)[VEC] = v[f][u][0], (&v1)[VEC] = v[f][u][1];
                    if (!BWD) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            v0[i] *= rstd * w[u][0][i];
                            v1[i] *= rstd * w[u][1][i];
                        }
                        if (at.turns) ang[u].turn(a.p.interleaved, v0, v1, 1.f);
                        if (keep && at.any) store<VEC>(dst + at.e0, v0);
                        if (keep && at.second) store<VEC>(dst + at.e1, v1);
                    } else {
                        float (&g0)[VEC] = y[f % (BWD ? FLY : 1)][u][0], (&g1)[VEC] = y[f % (BWD ? FLY : 1)][u][1];
                        if (at.turns) ang[u].turn(a.p.interleaved, g0, g1, -1.f);
                        const float r = keep ? rstd : 0.f;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            if (a.part && keep) {
                                dw[u][0][i] = fmaf(g0[i], v0[i] * r, dw[u][0][i]);
                                dw[u][1][i] = fmaf(g1[i], v1[i] * r, dw[u][1][i]);
                            }
                            g0[i] *= w[u][0][i];
                            g1[i] *= w[u][1][i];
                            dot += g0[i] * v0[i] + g1[i] * v1[i];
                        }
                    }
                }
                if (BWD) {
                    const float back = norm ? group_sum<G>(dot) * inv_d * rstd * rstd : 0.f;
#pragma unroll
                    for (int u = 0; u < UPL; ++u) {
                        const Unit<VEC> at(a, lane + u * G);
                        float (&g0)[VEC] = y[f % (BWD ? FLY : 1)][u][0], (&g1)[VEC] = y[f % (BWD ? FLY : 1)][u][1];
                        if (norm) {
#pragma unroll
                            for (int i = 0; i < VEC; ++i) {
                                g0[i] = rstd * (g0[i] - back * v[f][u][0][i]);
                                g1[i] = rstd * (g1[i] - back * v[f][u][1][i]);
                            }
                        }
                        if (keep && at.any) store<VEC>(dst + at.e0, g0);
                        if (keep && at.second) store<VEC>(dst + at.e1, g1);
                    }
                }
            }
        }
    }
};

// G lanes a head, UPL units a lane (UPL > 1 only for VEC 1)
template <typename T, int VEC, int G, int UPL, bool BWD>
__global__ void __launch_bounds__(NT) rotate_kernel(const RotateParams a) {
    const int lane = threadIdx.x % G;
    const unsigned first = (blockIdx.x * NT + threadIdx.x) / G, stride = gridDim.x * (NT / G);
    Walk<T, VEC, G, UPL, BWD> q, k;
    q.start(a, 0, lane);
    k.start(a, 1, lane);
    // all lanes of a warp stay together for the shuffles: a group behind the last one repeats it without storing
    const unsigned rounds = (a.groups + stride - 1) / stride;
    for (unsigned it = 0; it < rounds; ++it) {
        unsigned gr = first + it * stride;
        const bool live = gr < a.groups;
        if (!live) gr = a.groups - 1;
        const unsigned token = a.split == 1 ? gr : gr / a.split, part = gr - token * a.split;
        const unsigned b = token / (unsigned)a.p.L, t = token - b * a.p.L;
        const long long pos = a.positions ? a.positions[b * a.p.position_stride + t] : t;
        Angles<VEC> ang[UPL];
#pragma unroll
        for (int u = 0; u < UPL; ++u) ang[u].set(a, lane + u * G, lane + u * G < a.rot_units, pos);
        const long long *xs = a.p.q_stride, *gs = a.p.gq_stride, *ks = a.p.k_stride, *hs = a.p.gk_stride;
        q.run(a, ang, lane, static_cast<const T*>(a.x[0]) + b * xs[0] + t * xs[1], xs[2],
              BWD ? static_cast<const T*>(a.dy[0]) + b * gs[0] + t * gs[1] : nullptr, gs[2],
              static_cast<T*>(a.out[0]) + (long long)token * a.p.HQ * a.p.d, part, a.p.HQ, live);
        k.run(a, ang, lane, static_cast<const T*>(a.x[1]) + b * ks[0] + t * ks[1], ks[2],
              BWD ? static_cast<const T*>(a.dy[1]) + b * hs[0] + t * hs[1] : nullptr, hs[2],
              static_cast<T*>(a.out[1]) + (long long)token * a.p.HK * a.p.d, part, a.p.HK, live);
    }
    if constexpr (BWD) {
        if (!a.part) return;             // the block's groups add up in a fixed order, each element one thread
        __shared__ float sum[NT / G][G * UPL * 2 * VEC];
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < UPL; ++u)
#pragma unroll
                for (int i = 0; i < 2 * VEC; ++i)
                    sum[threadIdx.x / G][((lane + u * G) * 2 + i / VEC) * VEC + i % VEC] = (which ? k : q).dw[u][i / VEC][i % VEC];
            __syncthreads();
            for (int e = threadIdx.x; e < G * UPL * 2 * VEC; e += NT) {
                const int u = e / (2 * VEC), i = e % (2 * VEC);
                const Unit<VEC> at(a, u);
                const bool there = i < VEC ? at.any : at.second;
                if (!there) continue;
                float s = 0.f;
                for (int gq = 0; gq < NT / G; ++gq) s += sum[gq][e];
                a.part[((long long)blockIdx.x * 2 + which) * a.p.d + (i < VEC ? at.e0 + i : at.e1 + i - VEC)] = s;
            }
        }
    }
}

// dw = sum of the blocks' partial sums: a block per element, in a fixed order
__global__ void __launch_bounds__(128) rotate_weights_kernel(const float* part, int blocks, int d, float* dwq, float* dwk) {
    __shared__ float s[4];
    const int which = blockIdx.x / d, e = blockIdx.x % d;
    float v = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 128) v += part[((long long)b * 2 + which) * d + e];
    v = group_sum<32>(v);
    if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
    __syncthreads();
    float* out = which ? dwk : dwq;
    if (threadIdx.x == 0 && out) out[e] = s[0] + s[1] + s[2] + s[3];
}

// Whether rows can be taken four elements at a time: every piece of a row starts on a multiple of 4 elements.
bool quads(const aussm_b200_rotate_t& p, const RotateParams& a, size_t size, bool bwd) {
    const int rest = p.d - p.rot;
    bool ok = p.rot % 8 == 0 && rest % 4 == 0;
    auto row = [&](const void* base, const long long* s) {
        if (!base) return true;
        return reinterpret_cast<uintptr_t>(base) % (4 * size) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
    };
    ok = ok && row(a.x[0], p.q_stride) && row(a.x[1], p.k_stride);
    if (bwd) ok = ok && row(a.dy[0], p.gq_stride) && row(a.dy[1], p.gk_stride);
    for (int i = 0; i < 2; ++i) {
        ok = ok && reinterpret_cast<uintptr_t>(a.out[i]) % (4 * size) == 0;
        ok = ok && reinterpret_cast<uintptr_t>(a.w[i]) % 16 == 0;
    }
    return ok;
}

template <typename T, bool BWD>
void launch(RotateParams& a, int blocks_max, int* blocks_out, cudaStream_t st) {
    const bool vec = quads(a.p, a, sizeof(T), BWD);
    const int vw = vec ? 4 : 1, rest = a.p.d - a.p.rot;
    a.rot_units = a.p.rot / 2 / vw;
    a.units = a.rot_units + (rest + 2 * vw - 1) / (2 * vw);
    const long long tokens = (long long)a.p.B * a.p.L;
    // as many groups a token as give 16 groups an SM, at most one for each head of the longer of q and k
    const int heads = a.p.HQ > a.p.HK ? a.p.HQ : a.p.HK;
    const long long split = (148 * 16 + tokens - 1) / tokens;
    a.split = (int)(split < heads ? split : heads);
    a.groups = (unsigned)(tokens * a.split);
    const int g = a.units <= 8 ? 8 : a.units <= 16 ? 16 : 32;
    const unsigned want = (a.groups + NT / g - 1) / (NT / g);
    const unsigned grid = want < (unsigned)blocks_max ? want : (unsigned)blocks_max;
    if (vec) {
        if (g == 8) rotate_kernel<T, 4, 8, 1, BWD><<<grid, NT, 0, st>>>(a);
        else if (g == 16) rotate_kernel<T, 4, 16, 1, BWD><<<grid, NT, 0, st>>>(a);
        else rotate_kernel<T, 4, 32, 1, BWD><<<grid, NT, 0, st>>>(a);
    } else if (g == 8) rotate_kernel<T, 1, 8, 1, BWD><<<grid, NT, 0, st>>>(a);
    else if (g == 16) rotate_kernel<T, 1, 16, 1, BWD><<<grid, NT, 0, st>>>(a);
    else rotate_kernel<T, 1, 32, 4, BWD><<<grid, NT, 0, st>>>(a);
    count_launch();
    *blocks_out = (int)grid;
}

template <bool BWD>
void launch_typed(RotateParams& a, int blocks_max, int* blocks, cudaStream_t st) {
    if (a.p.dtype == AUSSM_FLOAT32) launch<float, BWD>(a, blocks_max, blocks, st);
    else if (a.p.dtype == AUSSM_BFLOAT16) launch<__nv_bfloat16, BWD>(a, blocks_max, blocks, st);
    else launch<__half, BWD>(a, blocks_max, blocks, st);
}

int rotate_check(const char* who, const aussm_b200_rotate_t* p) {
    if (!p) {
        set_error("%s: null problem", who);
        return AUSSM_EINVAL;
    }
    if (p->B <= 0 || p->L <= 0 || p->HQ <= 0 || p->HK <= 0 || p->d <= 0 || p->d > AUSSM_MAX_ROTATE_HEAD) {
        set_error("%s: bad sizes (B=%d L=%d HQ=%d HK=%d d=%d, d at most %d)", who, p->B, p->L, p->HQ, p->HK, p->d,
                  AUSSM_MAX_ROTATE_HEAD);
        return AUSSM_EINVAL;
    }
    if ((long long)p->B * p->L > 0x0fffffffLL) {
        set_error("%s: B*L=%lld tokens, at most 2^28 are supported", who, (long long)p->B * p->L);
        return AUSSM_EINVAL;
    }
    if (p->rot < 0 || p->rot % 2 || p->rot > p->d) {
        set_error("%s: the rotated part of %d elements must be even and at most the head's %d", who, p->rot, p->d);
        return AUSSM_EINVAL;
    }
    if (p->dtype < AUSSM_FLOAT32 || p->dtype > AUSSM_FLOAT16 || p->norm < AUSSM_NORM_NONE || p->norm > AUSSM_NORM_L2) {
        set_error("%s: unknown type %d or norm %d", who, p->dtype, p->norm);
        return AUSSM_EINVAL;
    }
    return AUSSM_OK;
}

int finished(const char* who) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return AUSSM_OK;
    set_error("%s launch: %s", who, cudaGetErrorString(e));
    return AUSSM_ECUDA;
}

}  // namespace
}  // namespace aussm

using namespace aussm;

extern "C" {

int aussm_b200_rotate_fwd(const aussm_b200_rotate_t* p, const void* q, const void* k, const double* frequencies,
                          const long long* positions, const float* q_weight, const float* k_weight, void* yq, void* yk,
                          aussm_stream_t stream) {
    if (int rc = rotate_check("rotate_fwd", p)) return rc;
    if (!q || !k || !yq || !yk || (p->rot && !frequencies)) {
        set_error("rotate_fwd: null input or output pointer");
        return AUSSM_EINVAL;
    }
    RotateParams a = {};
    a.p = *p;
    a.x[0] = q; a.x[1] = k; a.out[0] = yq; a.out[1] = yk; a.w[0] = q_weight; a.w[1] = k_weight;
    a.frequencies = frequencies; a.positions = positions;
    int blocks;
    launch_typed<false>(a, 0x7fffffff, &blocks, (cudaStream_t)stream);
    return finished("rotate_fwd");
}

size_t aussm_b200_rotate_bwd_workspace_bytes(const aussm_b200_rotate_t* p) {
    return rotate_check("rotate_bwd_workspace_bytes", p) ? 0 : ((size_t)MAX_BLOCKS * 2 * p->d * sizeof(float) + 255) / 256 * 256;
}

int aussm_b200_rotate_bwd(const aussm_b200_rotate_t* p, const void* gq, const void* gk, const void* q, const void* k,
                          const double* frequencies, const long long* positions, const float* q_weight,
                          const float* k_weight, void* dq, void* dk, float* dq_weight, float* dk_weight, void* workspace,
                          size_t workspace_bytes, aussm_stream_t stream) {
    if (int rc = rotate_check("rotate_bwd", p)) return rc;
    if (!gq || !gk || !q || !k || !dq || !dk || (p->rot && !frequencies)) {
        set_error("rotate_bwd: null input or output pointer");
        return AUSSM_EINVAL;
    }
    RotateParams a = {};
    a.p = *p;
    a.x[0] = q; a.x[1] = k; a.dy[0] = gq; a.dy[1] = gk; a.out[0] = dq; a.out[1] = dk; a.w[0] = q_weight; a.w[1] = k_weight;
    a.frequencies = frequencies; a.positions = positions;
    if (dq_weight || dk_weight) {
        if (!workspace || workspace_bytes < aussm_b200_rotate_bwd_workspace_bytes(p)) {
            set_error("rotate_bwd: workspace of %zu bytes required, got %zu", aussm_b200_rotate_bwd_workspace_bytes(p), workspace_bytes);
            return AUSSM_EWORKSPACE;
        }
        a.part = static_cast<float*>(workspace);
    }
    int blocks;
    launch_typed<true>(a, MAX_BLOCKS, &blocks, (cudaStream_t)stream);
    if (a.part) {
        rotate_weights_kernel<<<2 * p->d, 128, 0, (cudaStream_t)stream>>>(a.part, blocks, p->d, dq_weight, dk_weight);
        count_launch();
    }
    return finished("rotate_bwd");
}

}  // extern "C"
