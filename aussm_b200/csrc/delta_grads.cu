// Gated delta rule, the gradients of q, k, g and beta of a chunk (formulas in delta.cuh), from what the two recurrences
// left: V' and the entry state S forward, X and the gradient dS of the exit state backward.
//
// One block per chunk and key head, 16 warps; the value heads of the key head follow each other and add up in shared
// memory (no atomics: a fixed order).  The products with a contraction over the value columns (dO V'^T, X V'^T, dO S^T,
// X S^T, V' dS^T) take them 64 at a time: the operands come in as the recurrences left them (a value column's 8 keys or
// steps in 16 bytes, so V', X and the states lie transposed and are read with transposing fragment loads), their FP16 parts
// go to shared memory under one power of two per tile, of dO per row (it only shrinks from slice to slice: sums in one unit)
// and mma.sync runs the three products of parts.  Then K K^T, and dO V'^T and X V'^T, masked and decayed, meet Q and K.
// What bounds it: 6800 instructions a warp (conversions, fragments, 490 of them MMAs) at 0.34 a cycle and SM quarter, loads
// and work taking turns: 46 us a block of 64 x 128 x 128, of which 9 are its 384 KB at the DRAM's pace.  Spills gone, operands
// by asynchronous copies or the next block's brought to the L2: 633, 699, 673 us against 638 (2048 chunk heads of 128).
// The gradient of g_t is summed over just the pairs and states it stands for (see the end): sums over all pairs of which
// most cancel would lose the small gradients of a strongly decayed head.
#include "delta_tiles.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int C = kDeltaChunk;
constexpr int NT = 512, WARPS = NT / 32;
constexpr int VS = 64;                   // value columns of a slice
constexpr int FP = 68;                   // floats of a row of F

struct GradParams {
    aussm_b200_delta_t p;
    DeltaInputs in;
    const void* go;
    const uint8_t* records;
    DeltaRecord rec;
    int n;
    const uint8_t *news, *x, *states, *dstates;    // V', X, S, dS
    int slices;
    void *dq, *dk;
    float *dg, *dbeta;
    int vec_q, vec_k, vec_v, vec_go, vec_out;      // rows can be taken 16 bytes at a time
};

template <int KEY>
struct GradSmem {
    static constexpr int kSq = 16384;                    // 64 x 64 tile, hi and lo
    static constexpr int kSt = KEY * 256;                // KEY x 64 tile of a state; 64 x KEY tile of K or Q
    static constexpr int kGo = 0, kX = kSq, kNew = 2 * kSq, kS = 3 * kSq, kDs = kS + kSt;
    static constexpr int kE1 = kGo, kE2 = kX, kK = kS, kQ = kDs;          // second half
    static constexpr int kF = kDs + kSt, kAcc = kF + C * FP * 4, kVec = kAcc + 2 * C * KEY * 4, kBytes = kVec + 4096 + 1024;
};

template <typename T, int KEY>
__global__ void __launch_bounds__(NT, 1) delta_grads_kernel(const GradParams a) {
    using Smem = GradSmem<KEY>;
    constexpr int SQ_LO = 8192, ST_LO = KEY * 128;
    constexpr int NW = KEY / 32;                         // 8-column tiles of a warp in a 64 x KEY product
    extern __shared__ uint8_t raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float *F = reinterpret_cast<float*>(sm + Smem::kF), *accq = reinterpret_cast<float*>(sm + Smem::kAcc), *acck = accq + C * KEY;
    float* vec = reinterpret_cast<float*>(sm + Smem::kVec);
    float *ghi = vec, *glo = vec + 64, *be = vec + 128, *rowa = vec + 192 /* (4, 64) */, *rowk = vec + 448 /* (4, 64) */,
          *rowz = vec + 704 /* (4, 64) */;
    __shared__ uint32_t red[6 * WARPS];
    __shared__ uint32_t e1max[4][C];
    __shared__ int eo[C], eqs[C];                        // exponents of the rows of dO, of Q
    __shared__ float kappa[C], go_shrink[C], xv[8][C], ssum[WARPS], am[C], kkt[C];
    const aussm_b200_delta_t& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rb = warp & 3, cq = warp >> 2;             // 16 rows, a quarter of the columns
    const int r = p.HV / p.HK, c = blockIdx.x % a.n, bk = blockIdx.x / a.n, b = bk / p.HK, hk = bk % p.HK;
    const int t0 = c * C, rows = min(C, p.L - t0), DV = p.DV;
    const uint32_t base = smem_addr(sm);

    for (int e = tid; e < 2 * C * KEY; e += NT) accq[e] = 0.f;

    for (int h = hk * r; h < hk * r + r; ++h) {
        const size_t at = ((size_t)b * p.HV + h) * a.n + c;
        const float* head = reinterpret_cast<const float*>(a.records + at * a.rec.bytes());
        const T* go = static_cast<const T*>(a.go) + b * p.go_stride[0] + t0 * p.go_stride[1] + h * p.go_stride[2];
        const T* v = static_cast<const T*>(a.in.v) + b * p.v_stride[0] + t0 * p.v_stride[1] + h * p.v_stride[2];
        __syncthreads();                                 // the last head is done with shared memory
        if (tid < C) { ghi[tid] = head[kGHi + tid]; glo[tid] = head[kGLo + tid]; kappa[tid] = head[kKey + tid]; be[tid] = head[kBeta + tid] * kappa[tid]; }

        // ---- products over the value columns -------------------------------------------------------------------
        float dp[2][4] = {}, xn[2][4] = {}, dqt[NW][4] = {}, zz[NW][4] = {}, dkt[NW][4] = {};
        int e[5] = {115, 115, 115, 115, 115};            // exponents of dO (this thread's row), X, V', S, dS
        float dotv = 0.f, dots = 0.f;
        for (int v0 = 0; v0 < DV; v0 += VS) {
            const int cols = DV - v0;
            // dO by rows; V', X and the states by value column `dv` and groups of 8 steps or keys
            const int row = tid >> 3, col = (tid & 7) * 8, dv = tid & 63, grp = tid >> 6, l = (v0 & 64) + dv;
            const size_t piece = at * a.slices + (v0 >> 7);
            const bool there = dv < cols;
            float shrink[5];
            auto unit = [&](int y, uint32_t m) {         // exponent of operand y, and what its sums so far shrink by
                const int now = min(e[y], rank_exponent(m));
                shrink[y] = v0 ? pow2_float(max(-126, now - e[y])) : 0.f;
                e[y] = now;
            };
            const int pt = panel_at(dv, 8 * grp);
            {
            float f[3][8], s[KEY / 64][8];
            uint32_t m[3] = {};
            if (row < rows) load8(go + row * p.go_stride[1] + v0, col, cols, a.vec_go, f[0]); else zero8(f[0]);
            auto parts = [&](const uint8_t* base, int groups, int g8, float (&o)[8]) {
                const uint8_t* x = base + ((size_t)g8 * 128 + l) * 16;
                join8(x, x + (size_t)groups * 2048, reinterpret_cast<const float*>(base + (size_t)groups * 4096)[l], o);
            };
            if (there) {
                const float4* x4 = reinterpret_cast<const float4*>(a.x + piece * DeltaPlan::x_bytes()) + l;
                const float4 x0 = x4[2 * grp * 128], x1 = x4[(2 * grp + 1) * 128];
                f[1][0] = x0.x; f[1][1] = x0.y; f[1][2] = x0.z; f[1][3] = x0.w;
                f[1][4] = x1.x; f[1][5] = x1.y; f[1][6] = x1.z; f[1][7] = x1.w;
                parts(a.news + piece * DeltaPlan::news_bytes(), C / 8, grp, f[2]);
            } else {
                zero8(f[1]);
                zero8(f[2]);
            }
#pragma unroll
            for (int y = 0; y < KEY / 64; ++y) {
                if (there) parts(a.states + piece * DeltaPlan::state_bytes(KEY), KEY / 8, grp + 8 * y, s[y]);
                else zero8(s[y]);
                m[2] = max8(s[y], m[2]);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) m[y] = max8(f[1 + y], 0u);
            unit(0, row_max<8>(max8(f[0], 0u)));         // a row of dO meets no other: it has an exponent of its own
            if (col == 0) { eo[row] = e[0]; go_shrink[row] = shrink[0]; }
            block_max<WARPS>(m, red);
#pragma unroll
            for (int y = 0; y < 3; ++y) unit(1 + y, m[y]);
            put8(sm + Smem::kGo + panel_at(row, col), SQ_LO, f[0], pow2_float(e[0]));
            put8(sm + Smem::kX + pt, SQ_LO, f[1], pow2_float(e[1]));
            put8(sm + Smem::kNew + pt, SQ_LO, f[2], pow2_float(e[2]));
#pragma unroll
            for (int y = 0; y < KEY / 64; ++y)
                put8(sm + Smem::kS + panel_at(dv, 8 * grp + 64 * y), ST_LO, s[y], pow2_float(e[3]));
            }
            if (v0) {                                    // the sums so far, in the new unit
                const float go_row[2] = {go_shrink[rb * 16 + g], go_shrink[rb * 16 + g + 8]};
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) { dp[y][i] *= go_row[i >> 1] * shrink[2]; xn[y][i] *= shrink[1] * shrink[2]; }
#pragma unroll
                for (int y = 0; y < NW; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        dqt[y][i] *= go_row[i >> 1] * shrink[3];
                        zz[y][i] *= shrink[1] * shrink[3];
                    }
            }
            __syncthreads();
            // dS is asked for here and taken up behind the products without it
            uint4 raw_d[KEY / 64][2];
            float un_d = 0.f;
            if (there) {
                const uint8_t* base_d = a.dstates + piece * DeltaPlan::state_bytes(KEY);
                un_d = reinterpret_cast<const float*>(base_d + (size_t)KEY * 512)[l];
#pragma unroll
                for (int y = 0; y < KEY / 64; ++y) {
                    const uint8_t* x = base_d + ((size_t)(grp + 8 * y) * 128 + l) * 16;
                    raw_d[y][0] = *reinterpret_cast<const uint4*>(x);
                    raw_d[y][1] = *reinterpret_cast<const uint4*>(x + (size_t)KEY * 256);
                }
            } else {
#pragma unroll
                for (int y = 0; y < KEY / 64; ++y) raw_d[y][0] = raw_d[y][1] = make_uint4(0, 0, 0, 0);
            }
            if (dv < rows) {                             // X.V of step dv over the columns of group grp
                float w[8];
                load8(v + dv * p.v_stride[1] + v0, 8 * grp, cols, a.vec_v, w);
                auto dot = [&]() {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint8_t* x = sm + Smem::kX + panel_at(8 * grp + i, dv);
                        sum = fmaf(__half2float(*reinterpret_cast<const __half*>(x)) + __half2float(*reinterpret_cast<const __half*>(x + SQ_LO)), w[i], sum);
                    }
                    return sum;
                };
                float sum = dot();
                if (be[dv] == 0.f && rank_of(sum) < 0x01000000u) {
                    keep_finite8(w);
                    sum = dot();
                }
                dotv = fmaf(sum, pow2_float(-e[1]), dotv);
            }
#pragma unroll
            for (int k0 = 0; k0 < VS; k0 += 16) {
                if (k0 >= cols) break;
                uint32_t gh[4], gl[4], xh[4], xl[4], bh[4], bl[4];
                const int fa = frag_a(rb * 16, k0);
                ldmatrix4(gh, base + Smem::kGo + fa);
                ldmatrix4(gl, base + Smem::kGo + SQ_LO + fa);
                const int fx = frag_at(k0, rb * 16);
                ldmatrix4_trans(xh, base + Smem::kX + fx);
                ldmatrix4_trans(xl, base + Smem::kX + SQ_LO + fx);
                if (cq <= rb) {                          // on and below the diagonal
                    const int fb = frag_bt(k0, cq * 16);
                    ldmatrix4_trans(bh, base + Smem::kNew + fb);
                    ldmatrix4_trans(bl, base + Smem::kNew + SQ_LO + fb);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mma16816(dp[y], gl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(xn[y], xl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(dp[y], gh, bl[2 * y], bl[2 * y + 1]);
                        mma16816(xn[y], xh, bl[2 * y], bl[2 * y + 1]);
                        mma16816(dp[y], gh, bh[2 * y], bh[2 * y + 1]);
                        mma16816(xn[y], xh, bh[2 * y], bh[2 * y + 1]);
                    }
                }
#pragma unroll
                for (int x = 0; x < NW / 2; ++x) {
                    const int fb = frag_bt(k0, cq * (KEY / 4) + x * 16);
                    ldmatrix4_trans(bh, base + Smem::kS + fb);
                    ldmatrix4_trans(bl, base + Smem::kS + ST_LO + fb);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mma16816(dqt[2 * x + y], gl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(zz[2 * x + y], xl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(dqt[2 * x + y], gh, bl[2 * y], bl[2 * y + 1]);
                        mma16816(zz[2 * x + y], xh, bl[2 * y], bl[2 * y + 1]);
                        mma16816(dqt[2 * x + y], gh, bh[2 * y], bh[2 * y + 1]);
                        mma16816(zz[2 * x + y], xh, bh[2 * y], bh[2 * y + 1]);
                    }
                }
            }
            {
                float d[KEY / 64][8];
                uint32_t m[1] = {};
#pragma unroll
                for (int y = 0; y < KEY / 64; ++y) {
                    join8(reinterpret_cast<const uint8_t*>(&raw_d[y][0]), reinterpret_cast<const uint8_t*>(&raw_d[y][1]), un_d, d[y]);
                    m[0] = max8(d[y], m[0]);
                }
                block_max<WARPS>(m, red + 4 * WARPS);
                unit(4, m[0]);
                const float un_s = pow2_float(-e[3]);
#pragma unroll
                for (int y = 0; y < KEY / 64; ++y) {
                    const int ps = panel_at(dv, 8 * grp + 64 * y);
                    float v8[8];                         // S of the same places
                    put8(sm + Smem::kDs + ps, ST_LO, d[y], pow2_float(e[4]));
                    join8(sm + Smem::kS + ps, sm + Smem::kS + ST_LO + ps, un_s, v8);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dots = fmaf(v8[i], d[y][i], dots);
                }
                if (v0) {
#pragma unroll
                    for (int y = 0; y < NW; ++y)
#pragma unroll
                        for (int i = 0; i < 4; ++i) dkt[y][i] *= shrink[2] * shrink[4];
                }
            }
            __syncthreads();
#pragma unroll
            for (int k0 = 0; k0 < VS; k0 += 16) {
                if (k0 >= cols) break;
                uint32_t gh[4], gl[4], bh[4], bl[4];
                const int fx = frag_at(k0, rb * 16);
                ldmatrix4_trans(gh, base + Smem::kNew + fx);
                ldmatrix4_trans(gl, base + Smem::kNew + SQ_LO + fx);
#pragma unroll
                for (int x = 0; x < NW / 2; ++x) {
                    const int fb = frag_bt(k0, cq * (KEY / 4) + x * 16);
                    ldmatrix4_trans(bh, base + Smem::kDs + fb);
                    ldmatrix4_trans(bl, base + Smem::kDs + ST_LO + fb);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mma16816(dkt[2 * x + y], gl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(dkt[2 * x + y], gh, bl[2 * y], bl[2 * y + 1]);
                        mma16816(dkt[2 * x + y], gh, bh[2 * y], bh[2 * y + 1]);
                    }
                }
            }
            __syncthreads();
        }
        // X.V of a step (a thread for every 8 columns), the product of the states
        xv[tid >> 6][tid & 63] = dotv;
#pragma unroll
        for (int m = 16; m; m >>= 1) dots += __shfl_xor_sync(0xffffffffu, dots, m);
        if (lane == 0) ssum[warp] = dots;

        // ---- K, Q; K K^T ----------------------------------------------------------------------------------------
        int ek;
        {
            constexpr int PIECES = C * KEY / 8 / NT;
            const T* q = static_cast<const T*>(a.in.q) + b * p.q_stride[0] + t0 * p.q_stride[1] + hk * p.q_stride[2];
            const T* k = static_cast<const T*>(a.in.k) + b * p.k_stride[0] + t0 * p.k_stride[1] + hk * p.k_stride[2];
            float fk[PIECES][8], fq[PIECES][8];
            uint32_t m[1] = {}, mq[PIECES];
#pragma unroll
            for (int y = 0; y < PIECES; ++y) {
                const int piece = tid + y * NT, row = piece / (KEY / 8), col = piece % (KEY / 8) * 8;
                if (row < rows) {
                    load8(k + row * p.k_stride[1], col, p.DK, a.vec_k, fk[y]);
                    if (!finite8(fk[y]) && all_idle(a.in.beta + ((long long)b * p.L + t0 + row) * p.HV + hk * r, r)) keep_finite8(fk[y]);
                    load8(q + row * p.q_stride[1], col, p.DK, a.vec_q, fq[y]);
                } else {
                    zero8(fk[y]);
                    zero8(fq[y]);
                }
                m[0] = max(m[0], rank_less(max8(fk[y], 0u), key_exponent_of(kappa[row])));
                mq[y] = row_max<KEY / 8>(max8(fq[y], 0u));
            }
            block_max<WARPS>(m, red);
            ek = rank_exponent(m[0]);
#pragma unroll
            for (int y = 0; y < PIECES; ++y) {
                const int piece = tid + y * NT, row = piece / (KEY / 8), col = piece % (KEY / 8) * 8, pk = panel_at(row, col), eq = rank_exponent(mq[y]);
                put8(sm + Smem::kK + pk, ST_LO, fk[y], pow2_float(ek) * pow2_inverse(kappa[row]));
                put8(sm + Smem::kQ + pk, ST_LO, fq[y], pow2_float(eq));
                if (col == 0) eqs[row] = eq;
            }
        }
        __syncthreads();
        const float unk = pow2_float(-ek);
        float kk[2][4] = {};
        if (cq <= rb) {
#pragma unroll
            for (int k0 = 0; k0 < KEY; k0 += 16) {
                uint32_t ah[4], al[4], bh[4], bl[4];
                const int fa = frag_a(rb * 16, k0), fb = frag_b(cq * 16, k0);
                ldmatrix4(ah, base + Smem::kK + fa);
                ldmatrix4(al, base + Smem::kK + ST_LO + fa);
                ldmatrix4(bh, base + Smem::kK + fb);
                ldmatrix4(bl, base + Smem::kK + ST_LO + fb);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    mma16816(kk[y], al, bh[2 * y], bh[2 * y + 1]);
                    mma16816(kk[y], ah, bl[2 * y], bl[2 * y + 1]);
                    mma16816(kk[y], ah, bh[2 * y], bh[2 * y + 1]);
                }
            }
        }
        // the terms with states: dQt and dKt - beta Gamma Z (they take the places of dqt and dkt), their products with Q and K
        {
            const float fz = pow2_float(-e[1]) * pow2_float(-e[3]), fk = pow2_float(-e[2]) * pow2_float(-e[4]);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int i = rb * 16 + g + 8 * z;
                const float since = expf(ghi[i] + glo[i]), until = expf((ghi[C - 1] - ghi[i]) + (glo[C - 1] - glo[i]));
                const float fq = pow2_float(-eo[i]) * pow2_float(-e[3]), unq = pow2_float(-eqs[i]);
                float sumq = 0.f, sumz = 0.f, sumk = 0.f;
#pragma unroll
                for (int y = 0; y < NW; ++y) {
                    const int col = cq * (KEY / 4) + 8 * y + 2 * t, pa = panel_at(i, col);
                    const float2 kh = __half22float2(*reinterpret_cast<const __half2*>(sm + Smem::kK + pa)),
                                 kl = __half22float2(*reinterpret_cast<const __half2*>(sm + Smem::kK + ST_LO + pa)),
                                 qh = __half22float2(*reinterpret_cast<const __half2*>(sm + Smem::kQ + pa)),
                                 ql = __half22float2(*reinterpret_cast<const __half2*>(sm + Smem::kQ + ST_LO + pa));
                    const float kv[2] = {(kh.x + kl.x) * unk, (kh.y + kl.y) * unk}, qv[2] = {(qh.x + ql.x) * unq, (qh.y + ql.y) * unq};
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float dqv = p.scale * since * (dqt[y][2 * z + w] * fq), zv = since * (zz[y][2 * z + w] * fz),
                                    dkv = until * (dkt[y][2 * z + w] * fk);
                        sumq = fmaf(dqv, qv[w], sumq);
                        sumz = fmaf(zv, kv[w], sumz);
                        sumk = fmaf(dkv, kv[w], sumk);
                        dqt[y][2 * z + w] = dqv;
                        dkt[y][2 * z + w] = dkv - be[i] * zv;
                    }
                }
#pragma unroll
                for (int mm = 1; mm < 4; mm *= 2) {
                    sumq += __shfl_xor_sync(0xffffffffu, sumq, mm);
                    sumz += __shfl_xor_sync(0xffffffffu, sumz, mm);
                    sumk += __shfl_xor_sync(0xffffffffu, sumk, mm);
                }
                if (t == 0) {
                    rowa[cq * 64 + i] = sumq - be[i] * sumz;
                    rowz[cq * 64 + i] = -sumz;
                    rowk[cq * 64 + i] = sumk;
                }
            }
        }
        // E1 = scale D dO V'^T (gradient of Q K^T), E = -beta D X V'^T (gradient of K K^T), F = their part in G_i - G_j
        uint32_t m[1] = {}, mrow[2] = {};
        float bsum[2] = {};                              // dbeta of rows g and g + 8: sum of -D X V'^T K K^T
        {
            const uint8_t* pt = reinterpret_cast<const uint8_t*>(head) + a.rec.p();
            const float unp = head[kUnP], fx = pow2_float(-e[1]) * pow2_float(-e[2]);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int i = rb * 16 + g + 8 * z, j = cq * 16 + 8 * y + 2 * t;
                    const int pa = panel_at(i, j);
                    const float fp = pow2_float(-eo[i]) * pow2_float(-e[2]), unit_q = pow2_float(13 - eqs[i]);     // r_i
                    float2 ph = make_float2(0.f, 0.f), pl = ph;
                    if (cq <= rb) {
                        ph = __half22float2(*reinterpret_cast<const __half2*>(pt + pa));
                        pl = __half22float2(*reinterpret_cast<const __half2*>(pt + 8192 + pa));
                    }
                    const float pv[2] = {(ph.x + pl.x) * unp * unit_q, (ph.y + pl.y) * unp * unit_q};
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const bool in = j + w <= i, below = j + w < i;
                        const float d = in ? expf((ghi[i] - ghi[j + w]) + (glo[i] - glo[j + w])) : 0.f;
                        const float dpv = in ? dp[y][2 * z + w] * fp : 0.f, mx = below ? -d * (xn[y][2 * z + w] * fx) : 0.f;
                        const float kkv = kk[y][2 * z + w] * unk * unk;
                        bsum[z] = fmaf(mx, kkv, bsum[z]);
                        F[i * FP + j + w] = below ? fmaf(dpv, pv[w], be[i] * mx * kkv) : 0.f;
                        dp[y][2 * z + w] = p.scale * d * dpv;
                        xn[y][2 * z + w] = be[i] * mx;
                        mrow[z] = max(mrow[z], rank_of(dp[y][2 * z + w]));
                        m[0] = max(m[0], rank_of(xn[y][2 * z + w]));
                    }
                }
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            bsum[z] += __shfl_xor_sync(0xffffffffu, bsum[z], 1);
            bsum[z] += __shfl_xor_sync(0xffffffffu, bsum[z], 2);
            mrow[z] = row_max<4>(mrow[z]);
            if (t == 0) {
                rowz[cq * 64 + rb * 16 + g + 8 * z] += bsum[z];
                e1max[cq][rb * 16 + g + 8 * z] = mrow[z];
            }
        }
        block_max<WARPS>(m, red + 2 * WARPS);
        // E1's rows have exponents e1 of their own in E1 K, where they meet no other; in E1^T Q the rows of Q make up for them,
        // as q 2^(-e1 - top) with the largest of these in the usual range (in two steps where 2^down is no FP16 number).
        const int e2 = rank_exponent(m[0]);
        auto e1_of = [&](int i) { return rank_exponent(max(max(e1max[0][i], e1max[1][i]), max(e1max[2][i], e1max[3][i]))); };
        const int e1[2] = {e1_of(rb * 16 + g), e1_of(rb * 16 + g + 8)};
        const int top = __reduce_max_sync(0xffffffffu, max(-e1_of(lane) - eqs[lane], -e1_of(lane + 32) - eqs[lane + 32]));
#pragma unroll
        for (int y = 0; y < C * KEY / 8 / NT; ++y) {
            const int piece = tid + y * NT, row = piece / (KEY / 8), down = -e1_of(row) - eqs[row] - top;
            const __half2 f = __float2half2_rn(pow2_float(max(-24, down))), f2 = __float2half2_rn(pow2_float(max(-24, down + 24)));
#pragma unroll
            for (int lo = 0; lo <= ST_LO; lo += ST_LO) {
                uint4* at_q = reinterpret_cast<uint4*>(sm + Smem::kQ + lo + panel_at(row, piece % (KEY / 8) * 8));
                uint4 x = *at_q;
                __half2* h2 = reinterpret_cast<__half2*>(&x);
#pragma unroll
                for (int i = 0; i < 4; ++i) h2[i] = down < -24 ? __hmul2(__hmul2(h2[i], f), f2) : __hmul2(h2[i], f);
                *at_q = x;
            }
        }
        {
            const float s1[2] = {pow2_float(e1[0]), pow2_float(e1[1])}, s2 = pow2_float(e2);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int i = rb * 16 + g + 8 * z, j = cq * 16 + 8 * y + 2 * t, pa = panel_at(i, j);
                    uint32_t hi, lo;
                    split2(dp[y][2 * z] * s1[z], dp[y][2 * z + 1] * s1[z], hi, lo);
                    *reinterpret_cast<uint32_t*>(sm + Smem::kE1 + pa) = hi;
                    *reinterpret_cast<uint32_t*>(sm + Smem::kE1 + SQ_LO + pa) = lo;
                    // E + E^T: the strictly lower triangle and its mirror image (the diagonal is zero)
                    split2(xn[y][2 * z] * s2, xn[y][2 * z + 1] * s2, hi, lo);
                    const __half2 h2 = *reinterpret_cast<const __half2*>(&hi), l2 = *reinterpret_cast<const __half2*>(&lo);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        if (j + w > i) continue;
                        const __half hv = w ? __high2half(h2) : __low2half(h2), lv = w ? __high2half(l2) : __low2half(l2);
                        const int lower = panel_at(i, j + w), upper = panel_at(j + w, i);
                        *reinterpret_cast<__half*>(sm + Smem::kE2 + lower) = hv;
                        *reinterpret_cast<__half*>(sm + Smem::kE2 + SQ_LO + lower) = lv;
                        *reinterpret_cast<__half*>(sm + Smem::kE2 + upper) = hv;
                        *reinterpret_cast<__half*>(sm + Smem::kE2 + SQ_LO + upper) = lv;
                    }
                }
        }
        __syncthreads();
        // ---- dQ = E1 K + since dQt,  dK = E1^T Q + (E + E^T) K + until dKt - beta Gamma Z ---------------------------
        float sq[NW][4] = {}, sk[NW][4] = {}, se[NW][4] = {};
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
            uint32_t ah[4], al[4], th[4], tl[4], eh[4], el[4];
            const int fa = frag_a(rb * 16, jb * 16), ft = frag_at(jb * 16, rb * 16);
            ldmatrix4(eh, base + Smem::kE2 + fa);
            ldmatrix4(el, base + Smem::kE2 + SQ_LO + fa);
            if (jb <= rb) {
                ldmatrix4(ah, base + Smem::kE1 + fa);
                ldmatrix4(al, base + Smem::kE1 + SQ_LO + fa);
            }
            if (jb >= rb) {
                ldmatrix4_trans(th, base + Smem::kE1 + ft);
                ldmatrix4_trans(tl, base + Smem::kE1 + SQ_LO + ft);
            }
#pragma unroll
            for (int x = 0; x < NW / 2; ++x) {
                uint32_t bh[4], bl[4];
                const int fb = frag_bt(jb * 16, cq * (KEY / 4) + x * 16);
                ldmatrix4_trans(bh, base + Smem::kK + fb);
                ldmatrix4_trans(bl, base + Smem::kK + ST_LO + fb);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    mma16816(se[2 * x + y], el, bh[2 * y], bh[2 * y + 1]);
                    mma16816(se[2 * x + y], eh, bl[2 * y], bl[2 * y + 1]);
                    mma16816(se[2 * x + y], eh, bh[2 * y], bh[2 * y + 1]);
                    if (jb <= rb) {
                        mma16816(sq[2 * x + y], al, bh[2 * y], bh[2 * y + 1]);
                        mma16816(sq[2 * x + y], ah, bl[2 * y], bl[2 * y + 1]);
                        mma16816(sq[2 * x + y], ah, bh[2 * y], bh[2 * y + 1]);
                    }
                }
                if (jb >= rb) {
                    ldmatrix4_trans(bh, base + Smem::kQ + fb);
                    ldmatrix4_trans(bl, base + Smem::kQ + ST_LO + fb);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mma16816(sk[2 * x + y], tl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(sk[2 * x + y], th, bl[2 * y], bl[2 * y + 1]);
                        mma16816(sk[2 * x + y], th, bh[2 * y], bh[2 * y + 1]);
                    }
                }
            }
        }
        {
            const float f2 = pow2_float(-e2), fk = pow2_float(top >> 1), fk2 = pow2_float(top - (top >> 1));
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int i = rb * 16 + g + 8 * z;
                const float f1 = pow2_float(-e1[z]);
#pragma unroll
                for (int y = 0; y < NW; ++y) {
                    const int col = cq * (KEY / 4) + 8 * y + 2 * t;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        accq[i * KEY + col + w] += fmaf(sq[y][2 * z + w] * f1, unk, dqt[y][2 * z + w]);
                        acck[i * KEY + col + w] += sk[y][2 * z + w] * fk * fk2 + se[y][2 * z + w] * f2 * unk + dkt[y][2 * z + w];
                    }
                }
            }
        }
        __syncthreads();
        // ---- dg_t: g_t stands in G_i for i >= t, in G_i - G_j for j < t <= i, in G_C - G_i for i < t and in G_C -----------
        const long long o = ((long long)b * p.L + t0) * p.HV + h;
        if (tid < C) {
            am[tid] = (rowa[tid] + rowa[64 + tid]) + (rowa[128 + tid] + rowa[192 + tid]);
            kkt[tid] = (rowk[tid] + rowk[64 + tid]) + (rowk[128 + tid] + rowk[192 + tid]);
            float dotx = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) dotx += xv[w][tid];
            if (tid < rows)
                a.dbeta[o + (long long)tid * p.HV] = kappa[tid] * dotx + kappa[tid] * kappa[tid] * ((rowz[tid] + rowz[64 + tid]) + (rowz[128 + tid] + rowz[192 + tid]));
        }
        const int i = tid >> 3, seg = tid & 7;           // eight threads a row: sums of F up to and with each column
        {
            float* f = F + i * FP + seg * 8;
            float run[8], s = 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) { s += f[x]; run[x] = s; }
            float before = s;
#pragma unroll
            for (int mm = 1; mm < 8; mm *= 2) {
                const float w = __shfl_up_sync(0xffffffffu, before, mm);
                if (seg >= mm) before += w;
            }
            before -= s;
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = before + run[x];
        }
        __syncthreads();
        {
            float s = 0.f;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int row = seg * 8 + x;
                s += row >= i ? am[row] + (i ? F[row * FP + i - 1] : 0.f) : kkt[row];
            }
#pragma unroll
            for (int mm = 1; mm < 8; mm *= 2) s += __shfl_xor_sync(0xffffffffu, s, mm);
            if (seg == 0 && i < rows) {
                float ss = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) ss += ssum[w];
                a.dg[o + (long long)i * p.HV] = fmaf(head[kGamma], ss, s);
            }
        }
    }
    __syncthreads();
    T* dq = static_cast<T*>(a.dq) + (((long long)b * p.L + t0) * p.HK + hk) * p.DK;
    T* dk = static_cast<T*>(a.dk) + (((long long)b * p.L + t0) * p.HK + hk) * p.DK;
    const long long step = (long long)p.HK * p.DK;
    for (int e = tid; e < rows * KEY / 4; e += NT) {
        const int row = e / (KEY / 4), col = e % (KEY / 4) * 4;
        const float of_key = pow2_inverse(kappa[row]);
        if (a.vec_out) {
            struct alignas(4 * sizeof(T)) Raw { T v[4]; } x, y;
#pragma unroll
            for (int w = 0; w < 4; ++w) { x.v[w] = from_f32<T>(accq[row * KEY + col + w]); y.v[w] = from_f32<T>(acck[row * KEY + col + w] * of_key); }
            if (col < p.DK) {
                *reinterpret_cast<Raw*>(dq + row * step + col) = x;
                *reinterpret_cast<Raw*>(dk + row * step + col) = y;
            }
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (col + w < p.DK) {
                    dq[row * step + col + w] = from_f32<T>(accq[row * KEY + col + w]);
                    dk[row * step + col + w] = from_f32<T>(acck[row * KEY + col + w] * of_key);
                }
        }
    }
}

template <typename T, int KEY>
cudaError_t grads(const GradParams& a, cudaStream_t st) {
    constexpr int smem = GradSmem<KEY>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(delta_grads_kernel<T, KEY>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    delta_grads_kernel<T, KEY><<<(unsigned)(a.p.B * a.p.HK * a.n), NT, smem, st>>>(a);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t grads_typed(GradParams& a, cudaStream_t st) {
    auto vec = [&](const void* x, const long long* s, int width) {
        return reinterpret_cast<uintptr_t>(x) % 16 == 0 && s[0] * sizeof(T) % 16 == 0 && s[1] * sizeof(T) % 16 == 0 &&
               s[2] * sizeof(T) % 16 == 0 && width % 8 == 0;
    };
    a.vec_q = vec(a.in.q, a.p.q_stride, a.p.DK);
    a.vec_k = vec(a.in.k, a.p.k_stride, a.p.DK);
    a.vec_v = vec(a.in.v, a.p.v_stride, a.p.DV);
    a.vec_go = vec(a.go, a.p.go_stride, a.p.DV);
    a.vec_out = a.p.DK % 4 == 0 && (reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk)) % (4 * sizeof(T)) == 0;
    return a.rec.key == 64 ? grads<T, 64>(a, st) : grads<T, 128>(a, st);
}

}  // namespace

cudaError_t launch_delta_grads(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaInputs& in, const DeltaGrads& io,
                               cudaStream_t st) {
    GradParams a = {};
    a.p = p; a.in = in; a.go = io.go; a.records = static_cast<const uint8_t*>(io.records); a.rec = plan.rec; a.n = plan.n;
    a.news = static_cast<const uint8_t*>(io.news); a.x = static_cast<const uint8_t*>(io.x); a.slices = plan.slices;
    a.states = static_cast<const uint8_t*>(io.states); a.dstates = static_cast<const uint8_t*>(io.dstates);
    a.dq = io.dq; a.dk = io.dk; a.dg = io.dg; a.dbeta = io.dbeta;
    return p.dtype == AUSSM_FLOAT32 ? grads_typed<float>(a, st)
           : p.dtype == AUSSM_BFLOAT16 ? grads_typed<__nv_bfloat16>(a, st) : grads_typed<__half>(a, st);
}

}  // namespace aussm
