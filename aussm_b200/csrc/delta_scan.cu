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
// Warps 0-7 own the state, two threads a row, each half of its columns (the chain: convert S, product, convert V',
// product, add); warps 8-11 bring V (dO) in, a chunk ahead, through shared memory; warps 12-15 take everything out (O or X;
// the parts of S and V' that a backward pass reads, as they lie in tensor memory); warp 16 copies the records' tiles (bulk
// copies), warp 17 issues the MMAs (18 and 19 fill their warpgroup, which hands its registers to the others).  Tensor memory, 512
// columns: [X | Y] take turns as the parts of S and as the product that updates it, two accumulators of 64 columns, the
// parts of V' and of V.  Every wait is bounded: one that runs out sets the status word and the block ends.
//
// The roles walk different code, chunk after chunk, out of one instruction cache: with every loop unrolled the issue of 36
// MMAs took 4700 cycles instead of 2500.  Only what must be (registers that are indexed) is unrolled, and the state's
// conversions, the longest straight line, are cut into halves that run side by side (quarters take as long).
//
// What bounds it: a chain of conversions (float32 rows to FP16 parts and back) and products.  A training pass of 8 chunks a
// block issues 3800 instructions an SM quarter and chunk at 0.38 a cycle, 10100 cycles a chunk with the start and everything
// kept for the backward pass; the tensor core is busy 30 % of the time (backward 26 %).  Reading 64 chunks a block takes 4.3 us,
// 7900 cycles, a chunk, of which its MMAs alone would take 4000.
#include "common.cuh"
#include "delta.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int C = kDeltaChunk;
constexpr int PARTS = 2;                 // threads that share a row of the state
constexpr int MAIN = PARTS * 4, IN = MAIN, OUT = IN + 4, COPY = OUT + 4, ISSUE = COPY + 1;     // first warp of each role
constexpr int THREADS = (COPY + 4) * 32; // five warpgroups; launched with 96 registers a thread, 480 for one of each
constexpr int LAUNCHED = 96, MAIN_REGS = 136, IN_REGS = 64, OUT_REGS = 104, REST_REGS = 40;
static_assert(PARTS * MAIN_REGS + IN_REGS + OUT_REGS + REST_REGS <= (PARTS + 3) * LAUNCHED, "more registers than the block is launched with");
static_assert(THREADS * LAUNCHED <= 65536 && THREADS * (LAUNCHED + 8) > 65536, "what the compiler takes for the block");
static_assert(MAIN_REGS >= LAUNCHED && OUT_REGS >= LAUNCHED && IN_REGS <= LAUNCHED && REST_REGS <= LAUNCHED,
              "a warpgroup asks for more than it has, or gives some of it back");
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
    // A block walks one of `segs` segments of `span` chunks (in the order of the walk the first is blockIdx.z +
    // first_seg = 0; the boundaries are the forward walk's both ways).  Segment 0 starts from s0, segment z from seg_in + z
    // * seg_stride (NULL: from zero) and leaves its last state at seg_out + z * seg_stride.
    int span, segs, first_seg;
    const float* seg_in;
    float* seg_out;
    size_t seg_stride;
    int transition;                      // 1: V is zero and the state starts as the identity: what a segment does to a state
    uint4* rows;                         // forward: V' of every chunk (NULL = not kept); backward: X
    uint4* states;                       // forward: entry states (NULL); backward: gradients of the exit states
    int vec_v;                           // rows of v can be copied 16 bytes at a time
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
// The issuing warp runs as one, so that addresses and descriptors stay in uniform registers; `one` is set in the lane that
// issues.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t one) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
                 ::"r"(smem_addr(bar)), "r"(one) : "memory");
}
// A from tensor memory, B from shared memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
#define R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                 "[%16];" : R4(r, 0), R4(r, 4), R4(r, 8), R4(r, 12) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t t, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(t), W4(r, 0), W4(r, 4) : "memory");
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
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, int b_lo, uint32_t one) {
    constexpr uint32_t id = idesc(N, MN);
    constexpr uint32_t A_LO = STEPS * 8;
    uint64_t bh = row_desc(b, MN ? 8192 : 16);
    const uint64_t lo = (uint32_t)(b_lo >> 4);
#pragma unroll 1
    for (int k = 0; k < STEPS; ++k) {
        mma_ts(d, a + A_LO, bh, id, k > 0, one);
        mma_ts(d, a, bh + lo, id, 1, one);
        mma_ts(d, a, bh, id, 1, one);
        a += 8;
        bh += MN ? 2048 >> 4 : (k & 3) == 3 ? (8192 - 96) >> 4 : 32 >> 4;
    }
}

// COUNT values of a row, scaled by f, as hi parts (COUNT / 2 columns at t) and lo parts (`lo` columns behind them)
template <int COUNT>
__device__ __forceinline__ void store_parts(uint32_t t, uint32_t lo_cols, const float2 (&x)[COUNT / 2], float f) {
    const float2 f2 = make_float2(f, f), minus = make_float2(-1.f, -1.f);
#pragma unroll
    for (int i = 0; i < COUNT / 2; i += 8) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 v = __fmul2_rn(x[i + j], f2);
            const __half2 h = __float22half2_rn(v);
            const __half2 l = __float22half2_rn(__ffma2_rn(__half22float2(h), minus, v));
            hi[j] = *reinterpret_cast<const uint32_t*>(&h);
            lo[j] = *reinterpret_cast<const uint32_t*>(&l);
        }
        tmem_st8(t + i, hi);
        tmem_st8(t + lo_cols + i, lo);
    }
}
template <int COUNT>
__device__ __forceinline__ float row_max(const float2 (&x)[COUNT]) {
    float m[4] = {};
#pragma unroll
    for (int i = 0; i < COUNT; i += 2) {
        m[0] = fmaxf(m[0], fabsf(x[i].x));
        m[1] = fmaxf(m[1], fabsf(x[i].y));
        m[2] = fmaxf(m[2], fabsf(x[i + 1].x));
        m[3] = fmaxf(m[3], fabsf(x[i + 1].y));
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// mbar_wait_bounded as a loop of one poll (25 unrolled ones were 65 KB of the kernel's code)
__device__ __forceinline__ bool poll(uint64_t* bar, uint32_t parity, int* status) {
#pragma unroll 1
    for (uint32_t it = 0; it < (1u << 22); ++it)
        if (mbar_try_wait(bar, parity)) return true;
    atomicExch(status, kStatusBarrierTimeout);
    return false;
}
// the same answer in all lanes: what follows is executed by whole warps
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
    return __all_sync(0xffffffffu, poll(bar, parity, status));
}

template <typename T, int KEY>
struct ScanSmem {
    static constexpr int kTile = KEY * 256;
    // A: the operands of phase 1 (tile, square), B and E: tile and square of the later phases, twice, C: Qt, then V (dO).
    // A and C are wanted late after they are free again; B and E copied only then were waited for 1200 to 2200 cycles a chunk.
    static constexpr int kA = 0, kB = kTile + SQUARE, kC = kB + 2 * kTile, kE = kC + kTile, kV = kE + 2 * SQUARE,
                         kBytes = kV + C * 128 * (int)sizeof(T) + 1024;
};

template <typename T, int KEY, bool BWD>
__global__ void __launch_bounds__(THREADS, 1) delta_scan_kernel(const ScanParams a) {
    using Smem = ScanSmem<T, KEY>;
    constexpr int TILE = Smem::kTile, LO = KEY * 128, SQ_LO = 8192;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full_a, full_b[2], full_c, full_e[2], empty_a, empty_b[2], empty_c, empty_e[2];
    __shared__ uint64_t s_ready, v_ready[2], v_done, n_ready, a_done, y_free, d_done, o_done, o_free, x_free, v_loaded, v_read;
    __shared__ uint64_t row_s[4], row_n[4];
    __shared__ uint32_t holder;
    __shared__ float un_s[2][128], un_v[2][128], un_n[128], max_s[PARTS][128], max_n[PARTS][128];
    // Factors of the steps: V comes in times beta kappa and O goes out times r, dO times r and dV times beta kappa.  Those
    // of the way out are copied with the ones of the way in, and chunk i + 4 is asked for when v_done (a_done) of i + 2 is
    // seen, which the issuing warp commits after x_free of i: four of them.
    __shared__ __align__(16) float factors[C], out_factors[4][C];
    __shared__ __align__(16) uint32_t idle[4];                        // [2], [3]: steps without a step size, from the header
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const aussm_b200_delta_t& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bh = blockIdx.x, b = bh / p.HV, h = bh % p.HV;
    const int me = threadIdx.x & 127, v = blockIdx.y * 128 + me;      // row (value column) of all threads but the last warpgroup's
    const int width_all = a.transition ? p.DK : p.DV;                 // value columns (a transition: the state's own keys)
    const bool mine = v < width_all;
    const int seg = a.first_seg + (int)blockIdx.z, c0 = (BWD ? a.segs - 1 - seg : seg) * a.span;
    const int count = min(a.span, a.n - c0);                          // chunks this block walks
    const bool full = a.out != nullptr;                               // otherwise only the state at the end is wanted
    auto chunk_at = [&](int i) { return BWD ? c0 + count - 1 - i : c0 + i; };
    auto record = [&](int i) { return a.records + ((size_t)bh * a.n + chunk_at(i)) * a.rec.bytes(); };

    if (threadIdx.x == 0) {
        for (uint64_t* x : {&full_a, &full_b[0], &full_b[1], &full_c, &full_e[0], &full_e[1], &empty_a, &empty_b[0], &empty_b[1],
                            &empty_c, &empty_e[0], &empty_e[1], &v_done, &a_done, &d_done, &o_done})
            mbar_init(x, 1);
        for (uint64_t* x : {&s_ready, &n_ready, &y_free}) mbar_init(x, PARTS * 128);
        for (uint64_t* x : {&v_ready[0], &v_ready[1], &o_free, &x_free, &v_loaded, &v_read}) mbar_init(x, 128);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&row_s[i], PARTS * 32);
            mbar_init(&row_n[i], PARTS * 32);
        }
        fence_mbar_init();
        fence_proxy_async();
    }
    if (warp == ISSUE) tmem_alloc512(&holder);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = holder, lanes = tm + ((uint32_t)((warp & 3) * 32) << 16);

    if (warp < MAIN) {
        // ---- the state: columns [part * COLS, part * COLS + COLS) of row `me` ------------------------------------------
        more_registers<MAIN_REGS>();
        constexpr int COLS = KEY / PARTS, NEWS = C / PARTS;          // columns of S, of V' of a thread
        const int part = warp >> 2;
        const uint32_t sc = part * COLS;                              // first column in a float32 row
        float2 s[COLS / 2];
        const float* from = seg == 0 ? a.s0 : a.seg_in ? a.seg_in + seg * a.seg_stride : nullptr;
        if (from) from += (size_t)bh * p.DK * p.DV + v;
#pragma unroll
        for (int x = 0; x < COLS / 2; ++x) {
            const int k0 = sc + 2 * x;
            s[x] = make_float2(0.f, 0.f);
            if (a.transition) s[x] = make_float2(k0 == me ? 1.f : 0.f, k0 + 1 == me ? 1.f : 0.f);
            else if (from && mine) {
                if (k0 < p.DK) s[x].x = from[(size_t)k0 * p.DV];
                if (k0 + 1 < p.DK) s[x].y = from[(size_t)(k0 + 1) * p.DV];
            }
        }
        auto all_max = [&](const float (&m)[PARTS][128]) {
            float r = m[0][me];
#pragma unroll
            for (int i = 1; i < PARTS; ++i) r = fmaxf(r, m[i][me]);
            return r;
        };
        // s = s * keep + r * f over the columns of a product
        auto add = [&](uint32_t t, float keep, float f) {
            const float2 k2 = make_float2(keep, keep), f2 = make_float2(f, f);
#pragma unroll
            for (int x = 0; x < COLS; x += 16) {
                uint32_t r[16];
                tmem_ld16(t + sc + x, r);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 8; ++y)
                    s[x / 2 + y] = __ffma2_rn(make_float2(__uint_as_float(r[2 * y]), __uint_as_float(r[2 * y + 1])), f2,
                                              __fmul2_rn(s[x / 2 + y], k2));
            }
        };
        for (int i = 0; i < count; ++i) {
            const uint32_t ph = i & 1, X = lanes + (ph ? kY : kX), Y = lanes + (ph ? kX : kY);
            const float* head = reinterpret_cast<const float*>(record(i));
            const float un1 = head[BWD ? kUnKt : kUnW], un2 = head[BWD ? kUnP : kUnT], un3 = head[BWD ? kUnW : kUnKt],
                        unq = head[kUnQ], gamma = head[kGamma];
            // one power of two for the whole row: its threads tell each other their maxima
            max_s[part][me] = row_max(s);
            arrive(&row_s[warp & 3]);
            if (!warp_wait(&row_s[warp & 3], ph, a.status)) break;
            const int es = part_exponent(all_max(max_s));
            const float uns = pow2_float(-es);
            store_parts<COLS>(X + part * (COLS / 2), KEY / 2, s, pow2_float(es));
            if (part == 0) un_s[ph][me] = uns;
            tc_wait_st();
            tc_before();
            arrive(&s_ready);
            // V' (dV'), columns [NEWS part, NEWS part + NEWS).  v_ready has a barrier for each of two chunks: the next V may
            // be in before a warp that saw v_done has come to this wait, and a single one would be two phases on by then.
            if (!warp_wait(&v_done, ph, a.status) || !warp_wait(&v_ready[ph], (i >> 1) & 1, a.status)) break;
            tc_after();
            const float unv = un_v[ph][me], f1 = (BWD ? uns : -uns) * un1, f2 = unv * un2;
            float2 w[NEWS / 2];
#pragma unroll
            for (int x = 0; x < NEWS; x += 16) {
                uint32_t r1[16], r2[16];
                tmem_ld16(lanes + kAcc + part * NEWS + x, r1);
                tmem_ld16(lanes + kAcc2 + part * NEWS + x, r2);
                tc_wait_ld();
#pragma unroll
                for (int y = 0; y < 8; ++y)
                    w[x / 2 + y] = __ffma2_rn(make_float2(__uint_as_float(r1[2 * y]), __uint_as_float(r1[2 * y + 1])), make_float2(f1, f1),
                                              __fmul2_rn(make_float2(__uint_as_float(r2[2 * y]), __uint_as_float(r2[2 * y + 1])), make_float2(f2, f2)));
            }
            max_n[part][me] = row_max(w);
            arrive(&row_n[warp & 3]);
            if (!warp_wait(&row_n[warp & 3], ph, a.status)) break;
            const int en = part_exponent(all_max(max_n));
            const float unn = pow2_float(-en);
            if (full && i && !warp_wait(&x_free, ph ^ 1, a.status)) break;      // the last V' has been taken out
            store_parts<NEWS>(lanes + kNew + part * (NEWS / 2), C / 2, w, pow2_float(en));
            if (part == 0) un_n[me] = unn;
            tc_wait_st();
            tc_before();
            arrive(&n_ready);
            if (BWD) {
                if (!warp_wait(&a_done, ph, a.status)) break;
                tc_after();
                add(Y, gamma, unv * unq);
                tc_before();
                arrive(&y_free);
            }
            if (!warp_wait(&d_done, ph, a.status)) break;
            tc_after();
            add(Y, BWD ? 1.f : gamma, (BWD ? -unn : unn) * un3);
        }
        float* to = a.seg_out ? a.seg_out + seg * a.seg_stride : seg == a.segs - 1 ? a.s1 : nullptr;
        if (to && mine) {
            const int pitch = a.transition ? KEY : p.DV;
            to += (size_t)bh * (a.transition ? KEY : p.DK) * pitch + v;
#pragma unroll
            for (int x = 0; x < COLS / 2; ++x) {
                const int k0 = sc + 2 * x;
                if (k0 < p.DK) to[(size_t)k0 * pitch] = s[x].x;
                if (k0 + 1 < p.DK) to[(size_t)(k0 + 1) * pitch] = s[x].y;
            }
        }
    } else if (warp < OUT) {
        // ---- V (dO) in -------------------------------------------------------------------------------------------
        fewer_registers<IN_REGS>();
        const T* src = static_cast<const T*>(a.v) + b * a.v_stride[0] + h * a.v_stride[2] + blockIdx.y * 128;
        T* tile = reinterpret_cast<T*>(sm + Smem::kV);
        const int width = a.transition ? 0 : min(128, p.DV - (int)blockIdx.y * 128);
        // rows of chunk i to shared memory, [64][128]: 16-byte pieces in flight, or each lane its own column.  Columns
        // behind the width stay the zeros of the start, rows behind the end are cleared: no selects in the conversions.
        auto fetch = [&](int i) {
            const int t0 = chunk_at(i) * C, rows = min(C, p.L - t0);
            const T* from = src + (long long)t0 * a.v_stride[1];
            if (me < C / 2) {
                const int x = me % (C / 4) * 4;
                const bool out = me >= C / 4;
                cp_async16((out ? out_factors[i & 3] : factors) + x, reinterpret_cast<const float*>(record(i)) + (out != BWD ? kRow : kBeta) + x);
            }
            static_assert(kIdle == 6, "the second half of 16 bytes of the header");
            if (!BWD && me == C / 2) cp_async16(idle, reinterpret_cast<const float*>(record(i)) + 4);
            if (a.vec_v) {
                constexpr int E = 16 / (int)sizeof(T), PIECES = 128 / E, ROWS = 128 / PIECES;      // rows an instruction
                int row = me / PIECES;
                const int col = me % PIECES * E;
                const T* at = from + row * a.v_stride[1] + col;
                uint32_t to = smem_addr(tile + row * 128 + col);
#pragma unroll 2
                for (; row < rows && col < width; row += ROWS) {
                    cp_async16_s(to, at);
                    at += ROWS * a.v_stride[1];
                    to += ROWS * 128 * (uint32_t)sizeof(T);
                }
            } else if (me < width) {
#pragma unroll 4
                for (int row = 0; row < rows; ++row) tile[row * 128 + me] = from[row * a.v_stride[1] + me];
            }
            for (int row = rows; row < C; ++row) tile[row * 128 + me] = from_f32<T>(0.f);
            cp_async_commit();
        };
        for (int row = 0; row < C; ++row) tile[row * 128 + me] = from_f32<T>(0.f);
        arrive(&v_read);
        if (warp_wait(&v_read, 0, a.status)) {
        fetch(0);
        for (int i = 0; i < count; ++i) {
            cp_async_wait<0>();
            arrive(&v_loaded);
            if (!warp_wait(&v_loaded, i & 1, a.status)) break;
            if (!BWD)                             // values that count as zero: each lane clears its column
#pragma unroll 1
                for (int z = 0; z < 2; ++z)
                    for (uint32_t m = idle[2 + z]; m; m &= m - 1) tile[(2 * (__ffs(m) - 1) + z) * 128 + me] = from_f32<T>(0.f);
            // two steps of this lane's column, times their factors
            auto pair = [&](int t) {
                return __fmul2_rn(make_float2(to_f32(tile[t * 128 + me]), to_f32(tile[(t + 1) * 128 + me])),
                                  *reinterpret_cast<const float2*>(factors + t));
            };
            float m0 = 0.f, m1 = 0.f;
#pragma unroll 1
            for (int x = 0; x < C; x += 16)
#pragma unroll
                for (int y = 0; y < 16; y += 2) {
                    const float2 f = pair(x + y);
                    m0 = fmaxf(m0, fabsf(f.x));
                    m1 = fmaxf(m1, fabsf(f.y));
                }
            const int e = part_exponent(fmaxf(m0, m1));
            const float scale = pow2_float(e);
            // the products with chunk i - 1 are done: this one's parts go in
            if (i) {
                if (!warp_wait(BWD ? &a_done : &v_done, (i - 1) & 1, a.status)) break;
                tc_after();
            }
#pragma unroll 1
            for (int x = 0; x < C; x += 16) {
                float2 f[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) f[y] = pair(x + 2 * y);
                store_parts<16>(lanes + kVal + x / 2, C / 2, f, scale);
            }
            un_v[i & 1][me] = pow2_float(-e);
            tc_wait_st();
            tc_before();
            arrive(&v_ready[i & 1]);
            if (i + 1 < count) {
                arrive(&v_read);
                if (!warp_wait(&v_read, (i + 1) & 1, a.status)) break;       // all lanes have read their rows
                fetch(i + 1);
            }
        }
        }
        cp_async_wait<0>();
    } else if (warp < COPY) {
        // ---- O (X), states and V' out ------------------------------------------------------------------------------
        more_registers<OUT_REGS>();
        T* dst = static_cast<T*>(a.out) + ((long long)b * p.L * p.HV + h) * p.DV + v;
        const long long out_step = (long long)p.HV * p.DV;
        // `words` columns of tensor memory, 16 bytes a lane and store: [words / 4][128 lanes]
        auto dump = [&](uint32_t t, int words, uint4* to) {
            to += me;
#pragma unroll 1
            for (int x = 0; x < words; x += 16) {
                uint32_t r[16];
                tmem_ld16(t + x, r);
                tc_wait_ld();
#pragma unroll
                for (int z = 0; z < 4; ++z)
                    if (mine) to[(x / 4 + z) * 128] = make_uint4(r[4 * z], r[4 * z + 1], r[4 * z + 2], r[4 * z + 3]);
            }
        };
        for (int i = 0; full && i < count; ++i) {
            const uint32_t ph = i & 1;
            const float* head = reinterpret_cast<const float*>(record(i));
            const float unq = head[kUnQ], un2 = head[BWD ? kUnT : kUnP];
            const int t0 = chunk_at(i) * C, rows = mine ? min(C, p.L - t0) : 0;
            const size_t at = ((size_t)bh * a.n + chunk_at(i)) * gridDim.y + blockIdx.y;
            if (!warp_wait(&n_ready, ph, a.status) || !warp_wait(&o_done, ph, a.status)) break;
            tc_after();
            const float uns = un_s[ph][me], f1 = uns * unq, unn = un_n[me], f2 = unn * un2;
            T* to = dst + (long long)t0 * p.HV * p.DV;
            float4* keep = reinterpret_cast<float4*>(a.rows) + at * (C / 4 * 128) + me;
            const float4* out_factor = reinterpret_cast<const float4*>(out_factors[i & 3]);
#pragma unroll 1
            for (int t = 0; t < C; t += 16) {
                uint32_t r1[16], r2[16];
                float y[16];
                if (!BWD) tmem_ld16(lanes + kAcc + t, r1);
                tmem_ld16(lanes + kAcc2 + t, r2);
                tc_wait_ld();
                if (t + 16 == C) {               // the accumulators are wanted back
                    tc_before();
                    arrive(&o_free);
                }
#pragma unroll
                for (int u = 0; u < 16; u += 2) {
                    const float2 v = __fmul2_rn(make_float2(__uint_as_float(r2[u]), __uint_as_float(r2[u + 1])), make_float2(f2, f2));
                    const float2 w = BWD ? v : __ffma2_rn(make_float2(__uint_as_float(r1[u]), __uint_as_float(r1[u + 1])), make_float2(f1, f1), v);
                    y[u] = w.x;
                    y[u + 1] = w.y;
                }
#pragma unroll
                for (int u = 0; u < 16; u += 4) {
                    if (BWD && mine) keep[(t + u) / 4 * 128] = make_float4(y[u], y[u + 1], y[u + 2], y[u + 3]);
                    const float4 f = out_factor[(t + u) / 4];
                    y[u] *= f.x; y[u + 1] *= f.y; y[u + 2] *= f.z; y[u + 3] *= f.w;
                }
                if (t + 16 <= rows) {
#pragma unroll
                    for (int u = 0; u < 16; ++u, to += out_step) *to = from_f32<T>(y[u]);
                } else {
#pragma unroll
                    for (int u = 0; u < 16; ++u, to += out_step)
                        if (t + u < rows) *to = from_f32<T>(y[u]);
                }
            }
            if (a.states) {
                uint4* st = a.states + at * (KEY / 4 * 128 + 32);
                dump(lanes + (ph ? kY : kX), KEY, st);
                reinterpret_cast<float*>(st + KEY / 4 * 128)[me] = uns;
            }
            if (!BWD && a.rows) {
                uint4* st = a.rows + at * (C / 4 * 128 + 32);
                dump(lanes + kNew, C, st);
                reinterpret_cast<float*>(st + C / 4 * 128)[me] = unn;
            }
            tc_before();
            arrive(&x_free);
        }
    } else {
        fewer_registers<REST_REGS>();
        if (warp == COPY && lane == 0) {
            // ---- copies ------------------------------------------------------------------------------------------
            const int tile_a = BWD ? a.rec.kt() : a.rec.w(), square_a = BWD ? a.rec.p() : a.rec.t();
            const int tile_b = BWD ? a.rec.w() : a.rec.kt(), square_e = BWD ? a.rec.t() : a.rec.p();
            const bool c = full || BWD;                         // Qt: for O, or for the backward state
            auto copy = [&](uint64_t* bar, int to, const uint8_t* from, int bytes) {
                mbar_arrive_expect_tx(bar, bytes);
                bulk_g2s(sm + to, from, bytes, bar);
            };
            int na = 0, nb = 0, nc = 0;                         // copies under way or done
            for (int i = 0; i < count; ++i) {
                const uint8_t* rec = record(i);
                const int st = i & 1;
                if (i && !poll(&empty_a, (i - 1) & 1, a.status)) break;
                mbar_arrive_expect_tx(&full_a, TILE + SQUARE);
                bulk_g2s(sm + Smem::kA, rec + tile_a, TILE, &full_a);
                bulk_g2s(sm + Smem::kA + TILE, rec + square_a, SQUARE, &full_a);
                na = i + 1;
                if (i >= 2 && (!poll(&empty_b[st], ((i >> 1) - 1) & 1, a.status) || (full && !poll(&empty_e[st], ((i >> 1) - 1) & 1, a.status)))) break;
                copy(&full_b[st], Smem::kB + st * TILE, rec + tile_b, TILE);
                if (full) copy(&full_e[st], Smem::kE + st * SQUARE, rec + square_e, SQUARE);
                nb = i + 1;
                if (c) {
                    if (i && !poll(&empty_c, (i - 1) & 1, a.status)) break;
                    copy(&full_c, Smem::kC, rec + a.rec.q(), TILE);
                    nc = i + 1;
                }
            }
            // no copy may be in flight when the block ends, also not when a wait ran out
            if (na) poll(&full_a, (na - 1) & 1, a.status);
            if (nc) poll(&full_c, (nc - 1) & 1, a.status);
            for (int i = max(0, nb - 2); i < nb; ++i) {
                poll(&full_b[i & 1], (i >> 1) & 1, a.status);
                if (full) poll(&full_e[i & 1], (i >> 1) & 1, a.status);
            }
        } else if (warp == ISSUE) {
            // ---- MMAs --------------------------------------------------------------------------------------------
            const uint32_t base = smem_addr(sm), one = elect_one(), tm = __shfl_sync(0xffffffffu, holder, 0);
            auto wait = [&](uint64_t* bar, uint32_t ph) { return warp_wait(bar, ph, a.status); };
            for (int i = 0; i < count; ++i) {
                const uint32_t ph = i & 1, X = tm + (ph ? kY : kX), Y = tm + (ph ? kX : kY);
                const uint32_t ta = base + Smem::kA, half = (i >> 1) & 1;
                if (!wait(&full_a, ph) || !wait(&v_ready[ph], half) || (full && i && !wait(&o_free, ph ^ 1))) break;
                tc_after();
                product<C, C / 16, BWD>(tm + kAcc2, tm + kVal, ta + TILE, SQ_LO, one);       // no state in it
                if (!wait(&s_ready, ph)) break;
                tc_after();
                product<C, KEY / 16, false>(tm + kAcc, X, ta, LO, one);
                commit(&v_done, one);
                commit(&empty_a, one);
                if (BWD) {
                    if (!wait(&full_c, ph) || (full && i && !wait(&x_free, ph ^ 1))) break;
                    product<KEY, C / 16, true>(Y, tm + kVal, base + Smem::kC, LO, one);
                    commit(&a_done, one);
                    commit(&empty_c, one);
                    if (!wait(&y_free, ph)) break;
                }
                // Y held the parts of the state before this one: they have been taken out.  V' comes last.
                if (!wait(&full_b[ph], half) || (full && (!wait(&full_e[ph], half) || (!BWD && !wait(&full_c, ph)) || (i && !wait(&x_free, ph ^ 1)))) ||
                    !wait(&n_ready, ph))
                    break;
                tc_after();
                product<KEY, C / 16, true>(Y, tm + kNew, base + Smem::kB + ph * TILE, LO, one);
                commit(&d_done, one);
                commit(&empty_b[ph], one);
                if (!full) continue;
                if (!BWD) {
                    product<C, KEY / 16, false>(tm + kAcc, X, base + Smem::kC, LO, one);
                    commit(&empty_c, one);
                }
                product<C, C / 16, BWD>(tm + kAcc2, tm + kNew, base + Smem::kE + ph * SQUARE, SQ_LO, one);
                commit(&o_done, one);
                commit(&empty_e[ph], one);
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == ISSUE) tmem_dealloc512(tm);
}

// States at the segments' boundaries, from what each segment makes of a zero state and what it does to a state:
//     S_1 = N_0,   S_{z+1} = M_z S_z + N_z     (backward M^T of the mirrored segment),
// S_{z+1} in the place of N_z.  A block owns CHAIN_COLS value columns of a head and keeps their states in shared memory, where the
// next M is on its way (M is stored with KEY columns a row) while this one is worked on: a thread adds up some
// rows of two columns in float32.
template <int KEY, int CHAIN_COLS>
struct ChainSmem {
    static constexpr int kPitch = KEY + 4;               // floats of a row of M: neighbouring rows in other banks
    static constexpr int kBytes = (2 * KEY * kPitch + KEY * CHAIN_COLS) * 4;
};
template <int KEY, bool BWD, int CHAIN_COLS>
__global__ void __launch_bounds__(256) delta_chain_kernel(const float* m, float* ends, int dk, int dv, int segs, size_t m_stride,
                                                          size_t end_stride) {
    constexpr int PITCH = ChainSmem<KEY, CHAIN_COLS>::kPitch, LANES = CHAIN_COLS / 2, STEP = 256 / LANES, ROWS = KEY / STEP;
    extern __shared__ __align__(16) float chain[];
    float* s = chain + 2 * KEY * PITCH;                  // [KEY][CHAIN_COLS]
    const int bh = blockIdx.x, v0 = blockIdx.y * CHAIN_COLS, col = threadIdx.x % LANES * 2, row = threadIdx.x / LANES;
    float* end = ends + (size_t)bh * dk * dv + v0 + col;
    const bool in0 = v0 + col < dv, in1 = v0 + col + 1 < dv;
    auto fetch = [&](int z) {
        const float* from = m + (size_t)(BWD ? segs - 1 - z : z) * m_stride + (size_t)bh * KEY * KEY;
        float* to = chain + (z & 1) * KEY * PITCH;
        for (int e = threadIdx.x; e < dk * (KEY / 4); e += 256)
            cp_async16(to + e / (KEY / 4) * PITCH + e % (KEY / 4) * 4, from + e * 4);
        cp_async_commit();
    };
    fetch(1);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int x = row + STEP * i;
        const bool there = x < dk;
        *reinterpret_cast<float2*>(s + x * CHAIN_COLS + col) =
            make_float2(there && in0 ? end[(size_t)x * dv] : 0.f, there && in1 ? end[(size_t)x * dv + 1] : 0.f);
    }
    for (int z = 1; z < segs - 1; ++z) {
        float* to = end + z * end_stride;
        float2 acc[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int x = row + STEP * i;
            acc[i] = make_float2(x < dk && in0 ? to[(size_t)x * dv] : 0.f, x < dk && in1 ? to[(size_t)x * dv + 1] : 0.f);
        }
        cp_async_wait<0>();
        __syncthreads();                                 // M and the states are there, the other M is free
        if (z + 1 < segs - 1) fetch(z + 1);
        const float* M = chain + (z & 1) * KEY * PITCH;
#pragma unroll 2
        for (int x = 0; x + 4 <= dk; x += 4) {
            float w[ROWS][4];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if (BWD) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) w[i][y] = M[(x + y) * PITCH + row + STEP * i];
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(M + (row + STEP * i) * PITCH + x);
                    w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                }
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float2 f = *reinterpret_cast<const float2*>(s + (x + y) * CHAIN_COLS + col);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) acc[i] = __ffma2_rn(make_float2(w[i][y], w[i][y]), f, acc[i]);
            }
        }
        for (int x = dk & ~3; x < dk; ++x) {             // what is behind dk in M was never written
            const float2 f = *reinterpret_cast<const float2*>(s + x * CHAIN_COLS + col);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float w = BWD ? M[x * PITCH + row + STEP * i] : M[(row + STEP * i) * PITCH + x];
                acc[i] = __ffma2_rn(make_float2(w, w), f, acc[i]);
            }
        }
        __syncthreads();                                 // the states have been read
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int x = row + STEP * i;
            if (x >= dk) continue;
            *reinterpret_cast<float2*>(s + x * CHAIN_COLS + col) = acc[i];
            if (in0) to[(size_t)x * dv] = acc[i].x;
            if (in1) to[(size_t)x * dv + 1] = acc[i].y;
        }
    }
}

template <int KEY, bool BWD, int CHAIN_COLS>
cudaError_t chain(const float* m, float* ends, int heads, int dk, int dv, int segs, cudaStream_t st) {
    constexpr int smem = ChainSmem<KEY, CHAIN_COLS>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(delta_chain_kernel<KEY, BWD, CHAIN_COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    delta_chain_kernel<KEY, BWD, CHAIN_COLS><<<dim3(heads, (dv + CHAIN_COLS - 1) / CHAIN_COLS), 256, smem, st>>>(
        m, ends, dk, dv, segs, (size_t)heads * KEY * KEY, (size_t)heads * dk * dv);
    count_launch();
    return cudaGetLastError();
}

template <typename T, int KEY, bool BWD>
cudaError_t scan(ScanParams a, const DeltaPlan& plan, float* m, float* ends, cudaStream_t st) {
    constexpr int smem = ScanSmem<T, KEY>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(delta_scan_kernel<T, KEY, BWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int heads = a.p.B * a.p.HV, segs = plan.segs;
    a.span = plan.span;
    a.segs = segs;
    if (segs > 1) {                          // three or more
        const size_t m_stride = (size_t)heads * KEY * KEY, end_stride = (size_t)heads * a.p.DK * a.p.DV;
        ScanParams q = a;
        q.out = nullptr; q.rows = nullptr; q.states = nullptr;
        if (!BWD) {                          // what the segments between the first and the last do to a state
            q.transition = 1; q.first_seg = 1; q.seg_out = m; q.seg_stride = m_stride;
            delta_scan_kernel<T, KEY, BWD><<<dim3(heads, 1, segs - 2), THREADS, smem, st>>>(q);
            count_launch();
        }
        q.transition = 0; q.first_seg = 0; q.seg_out = ends; q.seg_stride = end_stride;
        delta_scan_kernel<T, KEY, BWD><<<dim3(heads, plan.slices, segs - 1), THREADS, smem, st>>>(q);
        count_launch();
        // 8 columns a block are quicker than 16 while each has an SM (4 heads of 128, 36 segments: 102 against 125 us,
        // 32 heads, 4 segments: 29 against 18 us)
        e = heads * ((a.p.DV + 7) / 8) <= 148 ? chain<KEY, BWD, 8>(m, ends, heads, a.p.DK, a.p.DV, segs, st)
                                              : chain<KEY, BWD, 16>(m, ends, heads, a.p.DK, a.p.DV, segs, st);
        if (e != cudaSuccess) return e;
        a.seg_in = ends - end_stride;        // segment z starts from the state behind segment z - 1
        a.seg_stride = end_stride;
    }
    delta_scan_kernel<T, KEY, BWD><<<dim3(heads, plan.slices, segs), THREADS, smem, st>>>(a);
    count_launch();
    return cudaGetLastError();
}
template <typename T, bool BWD>
cudaError_t scan_key(ScanParams& a, const DeltaPlan& plan, float* m, float* ends, cudaStream_t st) {
    const long long* vs = a.v_stride;
    a.vec_v = reinterpret_cast<uintptr_t>(a.v) % 16 == 0 && vs[0] * sizeof(T) % 16 == 0 && vs[1] * sizeof(T) % 16 == 0 &&
              vs[2] * sizeof(T) % 16 == 0 && a.p.DV * sizeof(T) % 16 == 0;
    return a.rec.key == 64 ? scan<T, 64, BWD>(a, plan, m, ends, st) : scan<T, 128, BWD>(a, plan, m, ends, st);
}
template <bool BWD>
cudaError_t scan_typed(ScanParams& a, const DeltaPlan& plan, float* m, float* ends, cudaStream_t st) {
    return a.p.dtype == AUSSM_FLOAT32 ? scan_key<float, BWD>(a, plan, m, ends, st)
           : a.p.dtype == AUSSM_BFLOAT16 ? scan_key<__nv_bfloat16, BWD>(a, plan, m, ends, st)
                                         : scan_key<__half, BWD>(a, plan, m, ends, st);
}

}  // namespace

cudaError_t launch_delta_scan(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaScan& io, bool backward,
                              cudaStream_t st) {
    ScanParams a = {};
    a.p = p; a.records = static_cast<const uint8_t*>(io.records); a.rec = plan.rec; a.n = plan.n;
    a.v = io.v; a.s0 = io.s0; a.s1 = io.s1; a.out = io.out; a.rows = static_cast<uint4*>(io.rows); a.states = static_cast<uint4*>(io.states);
    for (int i = 0; i < 3; ++i) a.v_stride[i] = backward ? p.go_stride[i] : p.v_stride[i];
    a.status = device_status_ptr();
    if (!a.status) return cudaErrorUnknown;
    float *m = static_cast<float*>(io.transitions), *ends = static_cast<float*>(io.ends);
    return backward ? scan_typed<true>(a, plan, m, ends, st) : scan_typed<false>(a, plan, m, ends, st);
}

}  // namespace aussm
