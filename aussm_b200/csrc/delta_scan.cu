// Gated delta rule, the recurrences over chunks on the tensor cores (formulas in delta.cuh).
//
// A block walks one sequence and value head for up to 128 value columns.  The state is kept transposed: TMEM lane =
// value column, so a thread owns one row S^T[v][:] in float32 registers and the products of a chunk are
//     forward:   V'^T = (beta V)^T T^T - S^T W^T       S^T <- e^(G_C) S^T + V'^T Kt      O^T = S^T Qt^T + V'^T P^T
//     backward:  dV'^T = dO^T P + dS^T Kt^T            dS^T <- e^(G_C) dS^T + dO^T Qt - dV'^T W      X^T = dV'^T T
// all with A (128 value columns) from tensor memory and B (the record's tiles) from shared memory: what comes out of one
// product is converted by the thread that owns the row and goes back as the next product's A without leaving the lane.
// A row's FP16 parts are scaled by a power of two of the row's own: no reduction between threads.
//
// Warps 0-3 own the state (the chain: convert S, product, convert V', product, add), warps 4-7 bring V (dO) in and
// O (X) out, warp 8 copies the records' tiles (bulk copies), warp 9 issues the MMAs
// (10 and 11 fill their warpgroup, which hands its registers to the other two).  Tensor memory, 512 columns:
// [X | Y] take turns as the parts of S and as the product that updates it, two accumulators of 64 columns, the parts of
// V' and of V.  Every wait is bounded: one that runs out sets the status word and the block ends.
#include "common.cuh"
#include "delta.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int C = kDeltaChunk;
constexpr int THREADS = 384;             // three warpgroups; launched with 168 registers a thread, 504 for one of each
constexpr int MAIN_REGS = 240, SIDE_REGS = 208, REST_REGS = 56;
static_assert(MAIN_REGS + SIDE_REGS + REST_REGS <= 3 * 168, "more registers than the block is launched with");
constexpr int SQUARE = DeltaRecord::kSquare;
// tensor memory columns
constexpr uint32_t kX = 0, kY = 128, kAcc = 256, kAcc2 = 320, kNew = 384, kVal = 448;

struct ScanParams {
    aussm_b200_delta_t p;
    const uint8_t* records;
    DeltaRecord rec;
    int n;
    const void* v;                       // forward: V; backward: dO
    long long v_stride[3];
    const float* s0;                     // forward: initial state, backward: gradient of the final state (NULL = 0)
    float* s1;                           // forward: final state, backward: gradient of the initial state (NULL)
    void* out;                           // forward: O; backward: dV
    float* rows;                         // forward: V' of every chunk (NULL = not kept); backward: X
    float* states;                       // forward: entry states (NULL); backward: gradients of the exit states
    int* status;
};

// ---- PTX -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc512(uint32_t* holder) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(holder)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc512(uint32_t t) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// A from tensor memory, B from shared memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
#define R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R4(r, 0), R4(r, 4), R4(r, 8), R4(r, 12), R4(r, 16), R4(r, 20), R4(r, 24), R4(r, 28) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
                 "%15, %16};" ::"r"(t), W4(r, 0), W4(r, 4), W4(r, 8), W4(r, 12) : "memory");
}
#undef R4
#undef W4

// Shared-memory descriptor of 128-byte swizzled rows, and the instruction descriptor (FP16 parts, float32 sums, M = 128)
__device__ __forceinline__ uint64_t row_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// D (128 x N) (+)= A (128 x 16 STEPS, hi and lo parts in tensor memory) * B: three products of parts.
// MN: B's rows (64 of 128 bytes a panel) are the contraction and N runs along them, in panels of 64; otherwise the rows
// are N and the contraction runs along them.
template <int N, int STEPS, bool MN>
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, int b_lo) {
    constexpr uint32_t id = idesc(N, MN);
    constexpr uint32_t A_LO = STEPS * 8;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const uint32_t at = MN ? b + k * 2048 : b + (k >> 2) * 8192 + (k & 3) * 32;
        const uint64_t bh = row_desc(at, MN ? 8192 : 16), bl = row_desc(at + b_lo, MN ? 8192 : 16);
        mma_ts(d, a + A_LO + k * 8, bh, id, k > 0);
        mma_ts(d, a + k * 8, bl, id, 1);
        mma_ts(d, a + k * 8, bh, id, 1);
    }
}

// COUNT values of this thread's row, scaled by s, as hi parts (COUNT / 2 columns) and lo parts behind them
template <int COUNT>
__device__ __forceinline__ void store_parts(uint32_t t, const float (&x)[COUNT], float s) {
#pragma unroll
    for (int i = 0; i < COUNT; i += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) split2(x[i + 2 * j] * s, x[i + 2 * j + 1] * s, hi[j], lo[j]);
        tmem_st16(t + i / 2, hi);
        tmem_st16(t + COUNT / 2 + i / 2, lo);
    }
}
template <int COUNT>
__device__ __forceinline__ int row_exponent(const float (&x)[COUNT]) {
    float m0 = 0.f, m1 = 0.f, m2 = 0.f, m3 = 0.f;
#pragma unroll
    for (int i = 0; i < COUNT; i += 4) {
        m0 = fmaxf(m0, fabsf(x[i]));
        m1 = fmaxf(m1, fabsf(x[i + 1]));
        m2 = fmaxf(m2, fabsf(x[i + 2]));
        m3 = fmaxf(m3, fabsf(x[i + 3]));
    }
    return part_exponent(fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)));
}

// the same answer in all lanes: what follows is executed by whole warps
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, status));
}

template <int KEY>
struct ScanSmem {
    static constexpr int kTile = KEY * 256;
    // phase 1 operands twice (tile, square), then the two tiles and the square of the later phases
    static constexpr int kA = 0, kB = 2 * (kTile + SQUARE), kC = kB + kTile, kE = kC + kTile, kBytes = kE + SQUARE + 1024;
};

template <typename T, int KEY, bool BWD>
__global__ void __launch_bounds__(THREADS, 1) delta_scan_kernel(const ScanParams a) {
    using Smem = ScanSmem<KEY>;
    constexpr int TILE = Smem::kTile, LO = KEY * 128, SQ_LO = 8192;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full_a[2], full_b, full_c, full_e, empty_a[2], empty_b, empty_c, empty_e;
    __shared__ uint64_t s_ready, v_ready, v_done, n_ready, a_done, y_free, d_done, o_done, o_free;
    __shared__ uint32_t holder;
    __shared__ float un_s[2][128], un_v[128], un_n[128];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const aussm_b200_delta_t& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bh = blockIdx.x, b = bh / p.HV, h = bh % p.HV;
    const int v = blockIdx.y * 128 + (threadIdx.x & 127);             // value column of warps 0-3 and of warps 4-7
    const bool mine = v < p.DV;
    const int count = a.n;                                            // chunks this block walks
    auto chunk_at = [&](int i) { return BWD ? a.n - 1 - i : i; };
    auto record = [&](int i) { return a.records + ((size_t)bh * a.n + chunk_at(i)) * a.rec.bytes(); };

    if (threadIdx.x == 0) {
        for (uint64_t* x : {&full_a[0], &full_a[1], &full_b, &full_c, &full_e, &empty_a[0], &empty_a[1], &empty_b, &empty_c,
                            &empty_e, &v_done, &a_done, &d_done, &o_done})
            mbar_init(x, 1);
        for (uint64_t* x : {&s_ready, &v_ready, &n_ready, &y_free, &o_free}) mbar_init(x, 128);
        fence_mbar_init();
        fence_proxy_async();
    }
    if (warp == 9) tmem_alloc512(&holder);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = holder, lanes = tm + ((uint32_t)((warp & 3) * 32) << 16);

    if (warp < 4) {
        // ---- the state -----------------------------------------------------------------------------------------
        more_registers<MAIN_REGS>();
        float s[KEY];
#pragma unroll
        for (int x = 0; x < KEY; ++x) s[x] = a.s0 && mine && x < p.DK ? a.s0[((size_t)bh * p.DK + x) * p.DV + v] : 0.f;
        for (int i = 0; i < count; ++i) {
            const uint32_t ph = i & 1, X = lanes + (ph ? kY : kX), Y = lanes + (ph ? kX : kY);
            const float* head = reinterpret_cast<const float*>(record(i));
            const int es = row_exponent(s);
            const float uns = pow2_float(-es);
            store_parts(X, s, pow2_float(es));
            un_s[ph][threadIdx.x] = uns;
            tc_wait_st();
            tc_before();
            arrive(&s_ready);
            const float un1 = head[BWD ? kUnKt : kUnW], un2 = head[BWD ? kUnP : kUnT], un3 = head[BWD ? kUnW : kUnKt],
                        unq = head[kUnQ], gamma = head[kGamma];
            if (a.states && mine) {
                float* dst = a.states + ((size_t)bh * a.n + chunk_at(i)) * p.DK * p.DV + v;
#pragma unroll
                for (int x = 0; x < KEY; ++x)
                    if (x < p.DK) dst[(size_t)x * p.DV] = s[x];
            }
            // V' (dV')
            if (!warp_wait(&v_done, ph, a.status) || !warp_wait(&v_ready, ph, a.status)) break;
            tc_after();
            const float f1 = (BWD ? uns : -uns) * un1, f2 = un_v[threadIdx.x] * un2;
            float w[C];
#pragma unroll
            for (int x = 0; x < C; x += 32) {
                uint32_t r1[32], r2[32];
                tmem_ld32(lanes + kAcc + x, r1);
                tmem_ld32(lanes + kAcc2 + x, r2);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; ++y) w[x + y] = fmaf(__uint_as_float(r1[y]), f1, __uint_as_float(r2[y]) * f2);
            }
            const int en = row_exponent(w);
            const float unn = pow2_float(-en);
            store_parts(lanes + kNew, w, pow2_float(en));
            un_n[threadIdx.x] = unn;
            tc_wait_st();
            tc_before();
            arrive(&n_ready);
            if (!BWD && a.rows && mine) {
                float* dst = a.rows + ((size_t)bh * a.n + chunk_at(i)) * C * p.DV + v;
#pragma unroll
                for (int x = 0; x < C; ++x) dst[(size_t)x * p.DV] = w[x];
            }
            if (BWD) {
                if (!warp_wait(&a_done, ph, a.status)) break;
                tc_after();
                const float f = un_v[threadIdx.x] * unq;
#pragma unroll
                for (int x = 0; x < KEY; x += 32) {
                    uint32_t r[32];
                    tmem_ld32(Y + x, r);
                    tc_wait_ld();
#pragma unroll
                    for (int y = 0; y < 32; ++y) s[x + y] = fmaf(gamma, s[x + y], __uint_as_float(r[y]) * f);
                }
                tc_before();
                arrive(&y_free);
            }
            if (!warp_wait(&d_done, ph, a.status)) break;
            tc_after();
            const float f = (BWD ? -unn : unn) * un3;
#pragma unroll
            for (int x = 0; x < KEY; x += 32) {
                uint32_t r[32];
                tmem_ld32(Y + x, r);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; ++y) s[x + y] = fmaf(__uint_as_float(r[y]), f, BWD ? s[x + y] : gamma * s[x + y]);
            }
        }
        if (a.s1 && mine) {
#pragma unroll
            for (int x = 0; x < KEY; ++x)
                if (x < p.DK) a.s1[((size_t)bh * p.DK + x) * p.DV + v] = s[x];
        }
    } else if (warp < 8) {
        // ---- V (dO) in, O (X) out --------------------------------------------------------------------------------
        more_registers<SIDE_REGS>();
        const int me = threadIdx.x & 127;
        const T* src = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2] + v;
        T* dst = static_cast<T*>(a.out) + ((long long)b * p.L * p.HV + h) * p.DV + v;
        auto fetch = [&](int i, float (&x)[C]) {
            const int t0 = chunk_at(i) * C, rows = min(C, p.L - t0);
#pragma unroll
            for (int t = 0; t < C; ++t) x[t] = mine && t < rows ? to_f32(src[(long long)(t0 + t) * a.v_stride[1]]) : 0.f;
        };
        auto hand_over = [&](int i, float (&x)[C]) {
            if (!BWD) {
                const float4* be = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(record(i)) + kBeta);
#pragma unroll
                for (int t = 0; t < C / 4; ++t) {
                    const float4 f = be[t];
                    x[4 * t] *= f.x; x[4 * t + 1] *= f.y; x[4 * t + 2] *= f.z; x[4 * t + 3] *= f.w;
                }
            }
            const int e = row_exponent(x);
            store_parts(lanes + kVal, x, pow2_float(e));
            un_v[me] = pow2_float(-e);
            tc_wait_st();
            tc_before();
            arrive(&v_ready);
        };
        float x[C];
        fetch(0, x);
        hand_over(0, x);
        for (int i = 0; i < count; ++i) {
            const uint32_t ph = i & 1;
            const float* head = reinterpret_cast<const float*>(record(i));
            const float unq = head[kUnQ], un2 = head[BWD ? kUnT : kUnP];
            if (i + 1 < count) fetch(i + 1, x);
            if (!warp_wait(&n_ready, ph, a.status) || !warp_wait(&o_done, ph, a.status)) break;
            tc_after();
            const float f1 = un_s[ph][me] * unq, f2 = un_n[me] * un2;
            float y[C];
#pragma unroll
            for (int t = 0; t < C; t += 32) {
                uint32_t r1[32], r2[32];
                if (!BWD) tmem_ld32(lanes + kAcc + t, r1);
                tmem_ld32(lanes + kAcc2 + t, r2);
                tc_wait_ld();
#pragma unroll
                for (int u = 0; u < 32; ++u)
                    y[t + u] = BWD ? __uint_as_float(r2[u]) * f2 : fmaf(__uint_as_float(r1[u]), f1, __uint_as_float(r2[u]) * f2);
            }
            tc_before();
            arrive(&o_free);
            if (i + 1 < count) hand_over(i + 1, x);
            if (mine) {
                const int t0 = chunk_at(i) * C, rows = min(C, p.L - t0);
                if (BWD) {
                    float* keep = a.rows + ((size_t)bh * a.n + chunk_at(i)) * C * p.DV + v;
#pragma unroll
                    for (int t = 0; t < C; ++t) {
                        keep[(size_t)t * p.DV] = y[t];
                        y[t] *= head[kBeta + t];
                    }
                }
#pragma unroll
                for (int t = 0; t < C; ++t)
                    if (t < rows) dst[(long long)(t0 + t) * p.HV * p.DV] = from_f32<T>(y[t]);
            }
        }
    } else {
        fewer_registers<REST_REGS>();
        if (warp == 8 && lane == 0) {
            // ---- copies ------------------------------------------------------------------------------------------
            const int tile_a = BWD ? a.rec.kt() : a.rec.w(), square_a = BWD ? a.rec.p() : a.rec.t();
            const int tile_b = BWD ? a.rec.w() : a.rec.kt(), square_e = BWD ? a.rec.t() : a.rec.p();
            int done_a = 0, done_b = 0;
            for (int i = 0; i < count; ++i) {
                const uint8_t* rec = record(i);
                const int st = i & 1;
                if (i >= 2 && !mbar_wait_bounded(&empty_a[st], ((i >> 1) - 1) & 1, a.status)) break;
                uint8_t* to = sm + Smem::kA + st * (TILE + SQUARE);
                mbar_arrive_expect_tx(&full_a[st], TILE + SQUARE);
                bulk_g2s(to, rec + tile_a, TILE, &full_a[st]);
                bulk_g2s(to + TILE, rec + square_a, SQUARE, &full_a[st]);
                done_a = i + 1;
                if (i >= 1 && (!mbar_wait_bounded(&empty_b, (i - 1) & 1, a.status) || !mbar_wait_bounded(&empty_c, (i - 1) & 1, a.status) ||
                               !mbar_wait_bounded(&empty_e, (i - 1) & 1, a.status)))
                    break;
                mbar_arrive_expect_tx(&full_b, TILE);
                bulk_g2s(sm + Smem::kB, rec + tile_b, TILE, &full_b);
                mbar_arrive_expect_tx(&full_c, TILE);
                bulk_g2s(sm + Smem::kC, rec + a.rec.q(), TILE, &full_c);
                mbar_arrive_expect_tx(&full_e, SQUARE);
                bulk_g2s(sm + Smem::kE, rec + square_e, SQUARE, &full_e);
                done_b = i + 1;
            }
            // no copy may be in flight when the block ends, also not when a wait ran out
            for (int i = max(0, done_a - 2); i < done_a; ++i) mbar_wait_bounded(&full_a[i & 1], (i >> 1) & 1, a.status);
            if (done_b) {
                mbar_wait_bounded(&full_b, (done_b - 1) & 1, a.status);
                mbar_wait_bounded(&full_c, (done_b - 1) & 1, a.status);
                mbar_wait_bounded(&full_e, (done_b - 1) & 1, a.status);
            }
        } else if (warp == 9 && lane == 0) {
            // ---- MMAs --------------------------------------------------------------------------------------------
            const uint32_t base = smem_addr(sm);
            auto wait = [&](uint64_t* bar, uint32_t ph) { return mbar_wait_bounded(bar, ph, a.status); };
            for (int i = 0; i < count; ++i) {
                const uint32_t ph = i & 1, X = tm + (ph ? kY : kX), Y = tm + (ph ? kX : kY);
                const uint32_t ta = base + Smem::kA + ph * (TILE + SQUARE);
                if (!wait(&full_a[ph], (i >> 1) & 1) || !wait(&v_ready, ph) || (i && !wait(&o_free, ph ^ 1)) || !wait(&s_ready, ph)) break;
                tc_after();
                product<C, KEY / 16, false>(tm + kAcc, X, ta, LO);
                product<C, C / 16, BWD>(tm + kAcc2, tm + kVal, ta + TILE, SQ_LO);
                commit(&v_done);
                commit(&empty_a[ph]);
                if (BWD) {
                    if (!wait(&full_c, ph)) break;
                    product<KEY, C / 16, true>(Y, tm + kVal, base + Smem::kC, LO);
                    commit(&a_done);
                    commit(&empty_c);
                    if (!wait(&y_free, ph)) break;
                }
                if (!wait(&full_b, ph) || !wait(&n_ready, ph)) break;
                tc_after();
                product<KEY, C / 16, true>(Y, tm + kNew, base + Smem::kB, LO);
                commit(&d_done);
                commit(&empty_b);
                if (!BWD) {
                    if (!wait(&full_c, ph)) break;
                    product<C, KEY / 16, false>(tm + kAcc, X, base + Smem::kC, LO);
                    commit(&empty_c);
                }
                if (!wait(&full_e, ph)) break;
                product<C, C / 16, BWD>(tm + kAcc2, tm + kNew, base + Smem::kE, SQ_LO);
                commit(&o_done);
                commit(&empty_e);
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 9) tmem_dealloc512(tm);
}

template <typename T, int KEY, bool BWD>
cudaError_t scan(const ScanParams& a, cudaStream_t st) {
    constexpr int smem = ScanSmem<KEY>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(delta_scan_kernel<T, KEY, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    delta_scan_kernel<T, KEY, BWD><<<dim3(a.p.B * a.p.HV, (a.p.DV + 127) / 128), THREADS, smem, st>>>(a);
    count_launch();
    return cudaGetLastError();
}
template <typename T, bool BWD>
cudaError_t scan_key(const ScanParams& a, cudaStream_t st) {
    return a.rec.key == 64 ? scan<T, 64, BWD>(a, st) : scan<T, 128, BWD>(a, st);
}
template <bool BWD>
cudaError_t scan_typed(const ScanParams& a, cudaStream_t st) {
    return a.p.dtype == AUSSM_FLOAT32 ? scan_key<float, BWD>(a, st)
           : a.p.dtype == AUSSM_BFLOAT16 ? scan_key<__nv_bfloat16, BWD>(a, st) : scan_key<__half, BWD>(a, st);
}

}  // namespace

cudaError_t launch_delta_scan(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaScan& io, bool backward,
                              cudaStream_t st) {
    ScanParams a = {};
    a.p = p; a.records = static_cast<const uint8_t*>(io.records); a.rec = plan.rec; a.n = plan.n;
    a.v = io.v; a.s0 = io.s0; a.s1 = io.s1; a.out = io.out; a.rows = io.rows; a.states = io.states;
    for (int i = 0; i < 3; ++i) a.v_stride[i] = backward ? p.go_stride[i] : p.v_stride[i];
    a.status = device_status_ptr();
    if (!a.status) return cudaErrorUnknown;
    return backward ? scan_typed<true>(a, st) : scan_typed<false>(a, st);
}

}  // namespace aussm
