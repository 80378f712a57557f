// Queries and keys: norm over each head and rotation by position in one pass, forward and backward.
//
//     y = R(position) (x r w),   r = rsqrt(mean(x^2) + eps)  (rms)  or  rsqrt(sum(x^2) + eps)  (l2)  or  1,
// R turns pair p by position * frequency_p and scales it by `magnitude`; elements behind the rotated part pass.
// Backward, with h = R^T dy and the mean / sum over the head:  dw = sum h x r,  dx = r (h w - x r^2 mean(h w x)).
//
// Bound: memory, every element read once and written once.  4 x 4096 steps, 16 heads of 128 in float32: forward 44 us
// (6.1 TB/s), backward 83 us (4.9 TB/s, three streams and the weights' sums); 2 x 65536 steps, 12 heads of 128 in bfloat16,
// forward 211 us (3.8 TB/s: half as many bytes for the same scalar float32 arithmetic, 71 % of the issue slots).  A group of 8, 16 or 32 lanes holds a head, both
// elements of a pair in the same lane: the norm is a few shuffles, the rotation none.  The lane's angles and weights serve
// the heads of a token that the group walks: all of them where the tokens fill the GPU, fewer otherwise.  Angles are reduced
// in 64 bits: position * (frequency / 2 pi), less its nearest integer, so a position of 2^22 is turned as exactly as 1.
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

// VEC consecutive elements as one access (VEC > 1: the row is aligned to it), kept as the words they are
template <typename T, int VEC>
struct Piece {
    static constexpr int BYTES = VEC * (int)sizeof(T), N = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[N];
};
template <int VEC, typename T>
__device__ __forceinline__ Piece<T, VEC> fetch(const T* p) {
    using P = Piece<T, VEC>;
    P r;
    if constexpr (P::BYTES == 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (P::BYTES == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    } else if constexpr (P::BYTES == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        r.w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
    return r;
}
__device__ __forceinline__ float2 two(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 two(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Piece<T, VEC>& r, float (&f)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 v = two(r.w[i / 2], T());
            f[i] = v.x;
            if (i + 1 < VEC) f[i + 1] = v.y;
        }
    }
}
template <int VEC, typename T>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    using P = Piece<T, VEC>;
    if constexpr (VEC == 1) *p = from_f32<T>(f[0]);
    else {
        P r;
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
            if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(f[i]);
            else if constexpr (sizeof(T) == 2) {
                const T lo = from_f32<T>(f[2 * i]), hi = from_f32<T>(f[2 * i + 1]);
                r.w[i] = (uint32_t)*reinterpret_cast<const unsigned short*>(&lo) | (uint32_t)*reinterpret_cast<const unsigned short*>(&hi) << 16;
            }
        }
        if constexpr (P::BYTES == 16) *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
        else *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
    }
}
// weights are float32 whatever the elements are: pieces of 16 bytes
template <int VEC>
__device__ __forceinline__ void load_weights(const float* p, float (&f)[VEC]) {
    constexpr int P = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int k = 0; k < VEC; k += P) {
        const Piece<float, P> r = fetch<P>(p + k);
#pragma unroll
        for (int i = 0; i < P; ++i) f[k + i] = __uint_as_float(r.w[i]);
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

// The heads of one token and tensor that this group walks, FLY of them in flight together: `start` asks for the first ones
// (before the angles are worked out), `run` does them all.
template <typename T, int VEC, int G, int UPL, bool BWD>
struct Walk {
    static constexpr int FLY = UPL > 1 ? 1 : BWD ? IN_FLIGHT / 2 : IN_FLIGHT;
    float dw[BWD ? UPL : 1][2][VEC];     // gradients of the weights of the lane's elements
    const T *x, *g;                      // the token's first head
    long long xs, gs;                    // strides between heads
    T* out;
    int heads, part;
    Piece<T, VEC> px[FLY][UPL][2], pg[BWD ? FLY : 1][UPL][2];

    __device__ __forceinline__ void ask(const RotateParams& a, int lane, int h) {
        const bool need = !BWD || a.p.norm != AUSSM_NORM_NONE || a.part;
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            const int hh = h + f * a.split;
#pragma unroll
            for (int u = 0; u < UPL; ++u) {
                const Unit<VEC> at(a, lane + u * G);
#pragma unroll
                for (int i = 0; i < Piece<T, VEC>::N; ++i) {
                    px[f][u][0].w[i] = px[f][u][1].w[i] = 0;
                    if (BWD) pg[BWD ? f : 0][u][0].w[i] = pg[BWD ? f : 0][u][1].w[i] = 0;
                }
                if (hh >= heads) continue;
                if (need && at.any) px[f][u][0] = fetch<VEC>(x + hh * xs + at.e0);
                if (need && at.second) px[f][u][1] = fetch<VEC>(x + hh * xs + at.e1);
                if (BWD && at.any) pg[BWD ? f : 0][u][0] = fetch<VEC>(g + hh * gs + at.e0);
                if (BWD && at.second) pg[BWD ? f : 0][u][1] = fetch<VEC>(g + hh * gs + at.e1);
            }
        }
    }
    __device__ __forceinline__ void run(const RotateParams& a, const Angles<VEC> (&ang)[UPL], int which, int lane, bool live) {
        const bool norm = a.p.norm != AUSSM_NORM_NONE;
        const float inv_d = a.p.norm == AUSSM_NORM_RMS ? 1.f / (float)a.p.d : 1.f;
        float w[UPL][2][VEC];
#pragma unroll
        for (int u = 0; u < UPL; ++u) {
            const Unit<VEC> at(a, lane + u * G);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[u][0][i] = w[u][1][i] = 1.f;
            if (a.w[which] && at.any) load_weights<VEC>(a.w[which] + at.e0, w[u][0]);
            if (a.w[which] && at.second) load_weights<VEC>(a.w[which] + at.e1, w[u][1]);
        }
        for (int base = 0; base < heads; base += FLY * a.split) {          // as often for all groups of a warp: shuffles
            if (base) ask(a, lane, base + part);
#pragma unroll
            for (int f = 0; f < FLY; ++f) {
                const int hh = base + part + f * a.split;
                const bool keep = live && hh < heads;
                float v[UPL][2][VEC], rstd = 1.f, dot = 0.f, sq = 0.f;
#pragma unroll
                for (int u = 0; u < UPL; ++u) {
                    unpack(px[f][u][0], v[u][0]);
                    unpack(px[f][u][1], v[u][1]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) sq += v[u][0][i] * v[u][0][i] + v[u][1][i] * v[u][1][i];
                }
                if (norm) rstd = rsqrtf(group_sum<G>(sq) * inv_d + a.p.eps);
                T* dst = out + (long long)hh * a.p.d;
                if (!BWD) {
#pragma unroll
                    for (int u = 0; u < UPL; ++u) {
                        const Unit<VEC> at(a, lane + u * G);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            v[u][0][i] *= rstd * w[u][0][i];
                            v[u][1][i] *= rstd * w[u][1][i];
                        }
                        if (at.turns) ang[u].turn(a.p.interleaved, v[u][0], v[u][1], 1.f);
                        if (keep && at.any) store<VEC>(dst + at.e0, v[u][0]);
                        if (keep && at.second) store<VEC>(dst + at.e1, v[u][1]);
                    }
                } else {
                    float y[UPL][2][VEC];
#pragma unroll
                    for (int u = 0; u < UPL; ++u) {
                        const Unit<VEC> at(a, lane + u * G);
                        unpack(pg[BWD ? f : 0][u][0], y[u][0]);
                        unpack(pg[BWD ? f : 0][u][1], y[u][1]);
                        if (at.turns) ang[u].turn(a.p.interleaved, y[u][0], y[u][1], -1.f);
#pragma unroll
                        for (int z = 0; z < 2; ++z)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) {
                                if (a.part && keep) dw[BWD ? u : 0][z][i] = fmaf(y[u][z][i], v[u][z][i] * rstd, dw[BWD ? u : 0][z][i]);
                                y[u][z][i] *= w[u][z][i];
                                dot += y[u][z][i] * v[u][z][i];
                            }
                    }
                    const float back = norm ? group_sum<G>(dot) * inv_d * rstd * rstd : 0.f;
#pragma unroll
                    for (int u = 0; u < UPL; ++u) {
                        const Unit<VEC> at(a, lane + u * G);
                        if (norm) {
#pragma unroll
                            for (int z = 0; z < 2; ++z)
#pragma unroll
                                for (int i = 0; i < VEC; ++i) y[u][z][i] = rstd * (y[u][z][i] - back * v[u][z][i]);
                        }
                        if (keep && at.any) store<VEC>(dst + at.e0, y[u][0]);
                        if (keep && at.second) store<VEC>(dst + at.e1, y[u][1]);
                    }
                }
            }
        }
    }
};

// G lanes a head, UPL units a lane (UPL > 1 only for VEC 1)
template <typename T, int VEC, int G, int UPL, bool BWD>
__global__ void __launch_bounds__(NT, BWD ? 2 : 3) rotate_kernel(const RotateParams a) {
    const int lane = threadIdx.x % G;
    const unsigned first = blockIdx.x * (NT / G) + threadIdx.x / G, stride = gridDim.x * (NT / G);
    Walk<T, VEC, G, UPL, BWD> q, k;
    if (BWD) {
#pragma unroll
        for (int u = 0; u < (BWD ? UPL : 1); ++u)
#pragma unroll
            for (int i = 0; i < 2 * VEC; ++i) q.dw[u][i / VEC][i % VEC] = k.dw[u][i / VEC][i % VEC] = 0.f;
    }
    // all lanes of a warp stay together for the shuffles: a group behind the last one repeats it without storing
    const unsigned rounds = (a.groups + stride - 1) / stride;
    for (unsigned it = 0; it < rounds; ++it) {
        unsigned gr = first + it * stride;
        const bool live = gr < a.groups;
        if (!live) gr = a.groups - 1;
        const unsigned token = a.split == 1 ? gr : gr / a.split, part = gr - token * a.split;
        const unsigned b = token / (unsigned)a.p.L, t = token - b * a.p.L;
        const long long pos = a.positions ? a.positions[b * a.p.position_stride + t] : t;
        auto place = [&](Walk<T, VEC, G, UPL, BWD>& w, int which, const long long* xs, const long long* gs, int heads) {
            w.x = static_cast<const T*>(a.x[which]) + b * xs[0] + t * xs[1];
            w.g = BWD ? static_cast<const T*>(a.dy[which]) + b * gs[0] + t * gs[1] : nullptr;
            w.xs = xs[2];
            w.gs = gs[2];
            w.out = static_cast<T*>(a.out[which]) + (long long)token * heads * a.p.d;
            w.heads = heads;
            w.part = part;
        };
        place(q, 0, a.p.q_stride, a.p.gq_stride, a.p.HQ);
        q.ask(a, lane, part);
        Angles<VEC> ang[UPL];
#pragma unroll
        for (int u = 0; u < UPL; ++u) ang[u].set(a, lane + u * G, lane + u * G < a.rot_units, pos);
        q.run(a, ang, 0, lane, live);
        place(k, 1, a.p.k_stride, a.p.gk_stride, a.p.HK);
        k.ask(a, lane, part);
        k.run(a, ang, 1, lane, live);
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

// Whether rows can be taken n elements at a time: every piece of a row starts on a multiple of n elements.
bool pieces(const aussm_b200_rotate_t& p, const RotateParams& a, int n, size_t size, bool bwd) {
    auto row = [&](const void* base, const long long* s) {
        return reinterpret_cast<uintptr_t>(base) % (n * size) == 0 && s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0;
    };
    bool ok = p.rot % (2 * n) == 0 && (p.d - p.rot) % n == 0 && row(a.x[0], p.q_stride) && row(a.x[1], p.k_stride);
    if (bwd) ok = ok && row(a.dy[0], p.gq_stride) && row(a.dy[1], p.gk_stride);
    for (int i = 0; i < 2; ++i)
        ok = ok && reinterpret_cast<uintptr_t>(a.out[i]) % (n * size) == 0 && reinterpret_cast<uintptr_t>(a.w[i]) % 16 == 0;
    return ok;
}

// VEC elements an access: 4 where rows allow it, single ones otherwise.  (8 of a 16-bit type, 16 bytes a lane, need more
// registers than three blocks an SM have: 231 us against 213 us, forward, 2 x 65536 steps of 12 heads of 128.)
template <typename T, int VEC, bool BWD>
int launch_vec(RotateParams& a, int blocks_max, cudaStream_t st) {
    const int rest = a.p.d - a.p.rot;
    a.rot_units = a.p.rot / 2 / VEC;
    a.units = a.rot_units + (rest + 2 * VEC - 1) / (2 * VEC);
    const long long tokens = (long long)a.p.B * a.p.L;
    // as many groups a token as give 16 groups an SM, at most one for each head of the longer of q and k
    const int heads = a.p.HQ > a.p.HK ? a.p.HQ : a.p.HK;
    const long long split = (148 * 16 + tokens - 1) / tokens;
    a.split = (int)(split < heads ? split : heads);
    a.groups = (unsigned)(tokens * a.split);
    const int g = a.units <= 8 ? 8 : a.units <= 16 ? 16 : 32;
    const unsigned want = (a.groups + NT / g - 1) / (NT / g);
    const unsigned grid = want < (unsigned)blocks_max ? want : (unsigned)blocks_max;
    constexpr int MOST = AUSSM_MAX_ROTATE_HEAD / 2 / VEC;         // units of the widest head
    if (g == 8) rotate_kernel<T, VEC, 8, 1, BWD><<<grid, NT, 0, st>>>(a);
    else if (g == 16) rotate_kernel<T, VEC, 16, 1, BWD><<<grid, NT, 0, st>>>(a);
    else if constexpr (MOST > 16) rotate_kernel<T, VEC, 32, (MOST + 31) / 32, BWD><<<grid, NT, 0, st>>>(a);
    count_launch();
    return (int)grid;
}
template <typename T, bool BWD>
void launch(RotateParams& a, int blocks_max, int* blocks_out, cudaStream_t st) {
    *blocks_out = pieces(a.p, a, 4, sizeof(T), BWD) ? launch_vec<T, 4, BWD>(a, blocks_max, st) : launch_vec<T, 1, BWD>(a, blocks_max, st);
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
