// Gated delta rule, what a chunk of 64 steps needs and no state enters: A, T = (I + A)^-1, W, P and the operand tiles
// of Kt and Q (formulas in delta.cuh), written as the records that the recurrences read.
//
// One block per chunk and key head; K K^T and Q K^T serve all value heads of the key head.  All products run on the
// FP16 parts with mma.sync (two blocks an SM, 8 warps each, warp = 16 rows x half of the columns), skipping the 16 x 16
// blocks above the diagonal.  Differences of the sums of g are taken from pairs of floats: sums reach thousands, and
// e^(G_i - G_j) has to be right to 24 bits where G_i - G_j is small.
//
// What bounds it: 4200 instructions a warp at 0.42 a cycle and SM quarter, barriers and shared memory between them.  2048
// chunk heads of 128: 147 us, 272 MB of records written (1.9 TB/s); 8192 that share 4096 key heads: 471 us.
#include "delta_tiles.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int C = kDeltaChunk;
constexpr int NT = 256;
constexpr int PITCH = 68;                // floats of a row of A / T: rows start on 16 bytes

struct PrepareParams {
    aussm_b200_delta_t p;
    DeltaInputs in;
    uint8_t* records;
    DeltaRecord rec;
    int n;
    int vec_q, vec_k;                    // rows can be read 16 bytes at a time
};

// 4 x 4 words of a quad of lanes change places: lane t comes to hold word t of lanes 0..3
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4], int t) {
    const bool o = t & 1, u = t & 2;
    const uint32_t a = __shfl_xor_sync(0xffffffffu, o ? w[0] : w[1], 1), b = __shfl_xor_sync(0xffffffffu, o ? w[2] : w[3], 1);
    if (o) { w[0] = a; w[2] = b; } else { w[1] = a; w[3] = b; }
    const uint32_t c = __shfl_xor_sync(0xffffffffu, u ? w[0] : w[2], 2), d = __shfl_xor_sync(0xffffffffu, u ? w[1] : w[3], 2);
    if (u) { w[0] = c; w[1] = d; } else { w[2] = c; w[3] = d; }
}

// Accumulator fragments of four neighbouring 8-column tiles (columns col0..col0+31) to a tile in memory: each lane puts
// together the 16-byte pieces of one of the four.
__device__ __forceinline__ void store_fragments(uint8_t* tile, int lo_off, int row0, int col0, const float (&c)[4][4], float s) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) split2(c[x][2 * half] * s, c[x][2 * half + 1] * s, hi[x], lo[x]);
        quad_transpose(hi, t);
        quad_transpose(lo, t);
        uint8_t* at = tile + panel_at(row0 + g + 8 * half, col0 + 8 * t);
        *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(at + lo_off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// T = (I + A)^-1 in place of the strictly lower triangular A (zeros elsewhere): 16 x 16 diagonal blocks by forward
// substitution, then twice by halves, T21 = -T22 A21 T11.
__device__ __forceinline__ void invert(float* A, float* tmp) {
    const int tid = threadIdx.x;
    if (tid < C) {
        const int d = (tid >> 4) * 16, j = tid & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == j ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < i; ++m) s = fmaf(-A[(d + i) * PITCH + d + m], x[m], s);
            x[i] = s;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) A[(d + i) * PITCH + d + j] = x[i];
    }
    __syncthreads();
    {   // 32 x 32: two pairs of blocks, 128 threads each, two rows of one column per thread
        const int e = (tid >> 7) * 32, j = tid & 15, i = (tid & 127) >> 4;
        float s[2] = {};
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            const float t = A[(e + m) * PITCH + e + j];
            s[0] = fmaf(A[(e + 16 + i) * PITCH + e + m], t, s[0]);
            s[1] = fmaf(A[(e + 24 + i) * PITCH + e + m], t, s[1]);
        }
        tmp[(e + i) * 33 + j] = s[0];
        tmp[(e + i + 8) * 33 + j] = s[1];
        __syncthreads();
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            const float t = tmp[(e + m) * 33 + j];
            s[0] = fmaf(A[(e + 16 + i) * PITCH + e + 16 + m], t, s[0]);
            s[1] = fmaf(A[(e + 24 + i) * PITCH + e + 16 + m], t, s[1]);
        }
        A[(e + 16 + i) * PITCH + e + j] = -s[0];
        A[(e + 24 + i) * PITCH + e + j] = -s[1];
    }
    __syncthreads();
    {   // 64 x 64: 2 x 2 elements per thread
        const int j = (tid & 15) * 2, i = (tid >> 4) * 2;
        float s[2][2] = {};
#pragma unroll 8
        for (int m = 0; m < 32; ++m) {
            const float2 t = *reinterpret_cast<const float2*>(A + m * PITCH + j);
            const float a = A[(32 + i) * PITCH + m], b = A[(33 + i) * PITCH + m];
            s[0][0] = fmaf(a, t.x, s[0][0]); s[0][1] = fmaf(a, t.y, s[0][1]);
            s[1][0] = fmaf(b, t.x, s[1][0]); s[1][1] = fmaf(b, t.y, s[1][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) { tmp[(i + x) * 34 + j] = s[x][0]; tmp[(i + x) * 34 + j + 1] = s[x][1]; }
        __syncthreads();
        s[0][0] = s[0][1] = s[1][0] = s[1][1] = 0.f;
#pragma unroll 8
        for (int m = 0; m < 32; ++m) {
            const float2 t = *reinterpret_cast<const float2*>(tmp + m * 34 + j);
            const float a = A[(32 + i) * PITCH + 32 + m], b = A[(33 + i) * PITCH + 32 + m];
            s[0][0] = fmaf(a, t.x, s[0][0]); s[0][1] = fmaf(a, t.y, s[0][1]);
            s[1][0] = fmaf(b, t.x, s[1][0]); s[1][1] = fmaf(b, t.y, s[1][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) { A[(32 + i + x) * PITCH + j] = -s[x][0]; A[(32 + i + x) * PITCH + j + 1] = -s[x][1]; }
    }
    __syncthreads();
}

template <int KEY>
struct PrepareSmem {
    static constexpr int kTile = KEY * 256;
    static constexpr int kBytes = 2 * kTile + DeltaRecord::kSquare + C * PITCH * 4 + 64 * 34 * 4 + 8 * C * 4 + 4 * 4 + 32 * 4;
};

template <typename T, int KEY>
__global__ void __launch_bounds__(NT, 2) delta_prepare_kernel(const PrepareParams a) {
    using Smem = PrepareSmem<KEY>;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t *kr = sm, *qr = sm + Smem::kTile;
    uint8_t* tr = qr + Smem::kTile;                                   // T beta e^G
    float* A = reinterpret_cast<float*>(tr + DeltaRecord::kSquare);
    float *tmp = A + C * PITCH, *ghi = tmp + 64 * 34, *glo = ghi + C, *be = glo + C, *until = be + C, *left = until + C, *since = left + C, *unit = since + C, *kappa = unit + C, *bound = kappa + C;
    uint32_t* red = reinterpret_cast<uint32_t*>(bound + 4);
    constexpr int LO = KEY * 128;                                     // lo panels behind the hi panels
    const aussm_b200_delta_t& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = p.HV / p.HK, c = blockIdx.x % a.n, bk = blockIdx.x / a.n, b = bk / p.HK, hk = bk % p.HK;
    const int t0 = c * C, rows = min(C, p.L - t0);
    const T* q = static_cast<const T*>(a.in.q) + b * p.q_stride[0] + t0 * p.q_stride[1] + hk * p.q_stride[2];
    const T* k = static_cast<const T*>(a.in.k) + b * p.k_stride[0] + t0 * p.k_stride[1] + hk * p.k_stride[2];
    auto record = [&](int h) { return a.records + (((size_t)b * p.HV + h) * a.n + c) * a.rec.bytes(); };

    // warp 0 looks after the decays: two steps a lane, asked for a head ahead
    double g0 = 0., g1 = 0.;
    float b0 = 0.f, b1 = 0.f;
    auto ask = [&](int h) {
        const long long o = ((long long)b * p.L + t0 + 2 * lane) * p.HV + h;
        g0 = 2 * lane < rows ? clamp_log_decay(a.in.g[o]) : 0.f;
        g1 = 2 * lane + 1 < rows ? clamp_log_decay(a.in.g[o + p.HV]) : 0.f;
        b0 = 2 * lane < rows ? a.in.beta[o] : 0.f;
        b1 = 2 * lane + 1 < rows ? a.in.beta[o + p.HV] : 0.f;
    };
    if (warp == 0) ask(hk * r);

    // K and Q: 16-byte pieces of a tile, KEY / 32 of each per thread
    constexpr int PIECES = C * KEY / 8 / NT;
    int ek;
    {
        float fk[PIECES][8], fq[PIECES][8];
        uint32_t m[1] = {}, mq[PIECES];
        int ck[PIECES];                    // exponents of kappa
#pragma unroll
        for (int x = 0; x < PIECES; ++x) {
            const int piece = tid + x * NT, row = piece / (KEY / 8), col = piece % (KEY / 8) * 8;
            if (row < rows) {
                load8(k + row * p.k_stride[1], col, p.DK, a.vec_k, fk[x]);
                load8(q + row * p.q_stride[1], col, p.DK, a.vec_q, fq[x]);
            } else {
                zero8(fk[x]);
                zero8(fq[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < PIECES; ++x) {
            const uint32_t mk = row_max<KEY / 8>(max8(fk[x], 0u));
            ck[x] = key_exponent(mk);
            m[0] = max(m[0], rank_less(mk, ck[x]));
            mq[x] = row_max<KEY / 8>(max8(fq[x], 0u));
        }
        block_max<8>(m, red);
        ek = rank_exponent(m[0]);
#pragma unroll
        for (int x = 0; x < PIECES; ++x) {
            const int piece = tid + x * NT, row = piece / (KEY / 8), col = piece % (KEY / 8) * 8, at = panel_at(row, col);
            const int eq = rank_exponent(mq[x]);
            put8(kr + at, LO, fk[x], pow2_float(ek - ck[x]));      // (12 or 13 less 126 at least: kappa > 1 leaves K / kappa >= 1)
            put8(qr + at, LO, fq[x], pow2_float(eq));              // 2^13 Q / r
            if (col == 0) {
                unit[row] = pow2_float(13 - eq);
                kappa[row] = pow2_float(ck[x]);
            }
        }
    }
    __syncthreads();

    // K K^T and Q K^T on and below the diagonal blocks: warp = rows rb*16.., columns half*32..
    const int rb = warp & 3, half = warp >> 2;
    const uint32_t ks = smem_addr(kr), qs = smem_addr(qr), ts = smem_addr(tr);
    float kk[4][4], qk[4][4];
    for (bool again = false;; again = true) {
#pragma unroll
        for (int x = 0; x < 16; ++x) kk[x >> 2][x & 3] = qk[x >> 2][x & 3] = 0.f;
#pragma unroll
        for (int k0 = 0; k0 < KEY; k0 += 16) {
            uint32_t kh[4], kl[4], qh[4], ql[4];
            const int at = frag_a(rb * 16, k0);
            ldmatrix4(kh, ks + at);
            ldmatrix4(kl, ks + LO + at);
            ldmatrix4(qh, qs + at);
            ldmatrix4(ql, qs + LO + at);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n0 = half * 32 + x * 16;
                if (n0 > rb * 16) continue;
                uint32_t bh[4], bl[4];
                const int bt = frag_b(n0, k0);
                ldmatrix4(bh, ks + bt);
                ldmatrix4(bl, ks + LO + bt);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    mma16816(kk[2 * x + y], kl, bh[2 * y], bh[2 * y + 1]);
                    mma16816(qk[2 * x + y], ql, bh[2 * y], bh[2 * y + 1]);
                    mma16816(kk[2 * x + y], kh, bl[2 * y], bl[2 * y + 1]);
                    mma16816(qk[2 * x + y], qh, bl[2 * y], bl[2 * y + 1]);
                    mma16816(kk[2 * x + y], kh, bh[2 * y], bh[2 * y + 1]);
                    mma16816(qk[2 * x + y], qh, bh[2 * y], bh[2 * y + 1]);
                }
            }
        }
        // |k_i|^2 tells of a key that is not finite: once more without it, if it is one that counts as zero.  (Looking at the
        // elements before they are stored takes 3 % longer.)
        bool bad = false;
#pragma unroll
        for (int x = 0; x < 16; ++x) bad = bad || rank_of(kk[x >> 2][x & 3]) < 0x01000000u;
        if (again || !__syncthreads_or(bad)) break;
        for (int piece = tid; piece < C * KEY / 8; piece += NT) {
            const int row = piece / (KEY / 8);
            if (row >= rows || !all_idle(a.in.beta + ((long long)b * p.L + t0 + row) * p.HV + hk * r, r)) continue;
            __half* at = reinterpret_cast<__half*>(kr + panel_at(row, piece % (KEY / 8) * 8));
            for (int i = 0; i < 8; ++i)
                if (__hisinf(at[i]) || __hisnan(at[i])) at[i] = at[LO / 2 + i] = __float2half(0.f);
        }
        __syncthreads();
    }
    const float unk = pow2_float(-ek), unq = pow2_float(-13);

    for (int h = hk * r; h < hk * r + r; ++h) {
        uint8_t* rec = record(h);
        float* head = reinterpret_cast<float*>(rec);
        __syncthreads();                       // the last value head's T beta e^G and vectors are read
        if (warp == 0) {
            const int i0 = 2 * lane, i1 = i0 + 1;
            b0 *= kappa[i0]; b1 *= kappa[i1];
            be[i0] = b0 * kappa[i0];
            be[i1] = b1 * kappa[i1];
            double s = g0 + g1;
#pragma unroll
            for (int m = 1; m < 32; m *= 2) {
                const double v = __shfl_up_sync(0xffffffffu, s, m);
                if (lane >= m) s += v;
            }
            const double before = s - g1, all = __shfl_sync(0xffffffffu, s, 31);
            const float h0 = (float)before, h1 = (float)s;
            const float u0 = expf((float)(all - before)), u1 = expf((float)(all - s));
            ghi[i0] = h0; ghi[i1] = h1;
            glo[i0] = (float)(before - h0); glo[i1] = (float)(s - h1);
            until[i0] = u0; until[i1] = u1;
            const float e0 = expf((float)before), e1 = expf((float)s);
            left[i0] = be[i0] * e0; left[i1] = be[i1] * e1;                 // what T's columns are multiplied with for W
            since[i0] = p.scale * e0; since[i1] = p.scale * e1;
            head[kBeta + i0] = b0; head[kBeta + i1] = b1;
            head[kGHi + i0] = h0; head[kGHi + i1] = h1;
            head[kGLo + i0] = glo[i0]; head[kGLo + i1] = glo[i1];
            head[kRow + i0] = unit[i0]; head[kRow + i1] = unit[i1];
            head[kKey + i0] = kappa[i0]; head[kKey + i1] = kappa[i1];
            if (lane == 31) head[kGamma] = e1;
            const uint32_t even = __ballot_sync(0xffffffffu, i0 < rows && b0 == 0.f), odd = __ballot_sync(0xffffffffu, i1 < rows && b1 == 0.f);
            if (lane == 0) {
                head[kIdle] = __uint_as_float(even);
                head[kIdle + 1] = __uint_as_float(odd);
            }
            float um = fmaxf(finite_or_zero(u0), finite_or_zero(u1)), em = fabsf(p.scale) * fmaxf(finite_or_zero(e0), finite_or_zero(e1));
#pragma unroll
            for (int m = 16; m; m >>= 1) {
                um = fmaxf(um, __shfl_xor_sync(0xffffffffu, um, m));
                em = fmaxf(em, __shfl_xor_sync(0xffffffffu, em, m));
            }
            if (lane == 0) { bound[0] = um; bound[1] = em; }
            if (h + 1 < hk * r + r) ask(h + 1);
        }
        __syncthreads();
        // A to shared memory, P kept in the fragments
        float pr[4][4];
        uint32_t m[3] = {};
        {
            const int i0 = rb * 16 + (lane >> 2);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int i = i0 + 8 * (y >> 1), j = half * 32 + x * 8 + (lane & 3) * 2 + (y & 1);
                    const float d = j <= i ? expf((ghi[i] - ghi[j]) + (glo[i] - glo[j])) : 0.f;
                    A[i * PITCH + j] = j < i ? be[i] * d * (kk[x][y] * unk * unk) : 0.f;
                    pr[x][y] = j <= i ? p.scale * d * (qk[x][y] * unk * unq) : 0.f;
                    m[0] = max(m[0], rank_of(pr[x][y]));
                }
        }
        // Kt and Qt from the parts of K and Q; their largest magnitudes are at most these
        const int et = part_exponent(bound[0] * pow2_float(min(127, 14 - ek))),
                  eqt = part_exponent(bound[1] * 2.f);
        {
            const float s = unk * pow2_float(et), sq = unq * pow2_float(eqt);
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
                const int piece = tid + x * NT, row = piece / (KEY / 8), at = panel_at(row, piece % (KEY / 8) * 8);
                float f[8];                      // (reading K and Q again takes longer: 509 against 462 us)
                join8(kr + at, kr + LO + at, until[row], f);
                put8(rec + a.rec.kt() + at, LO, f, s);
                join8(qr + at, qr + LO + at, since[row], f);
                put8(rec + a.rec.q() + at, LO, f, sq);
            }
        }
        __syncthreads();
        invert(A, tmp);
        // T and T beta e^G: two 16-byte pieces of each per thread
        float ft[2][8];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int piece = tid + x * NT, row = piece >> 3, col = (piece & 7) * 8;
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(A + row * PITCH + col + i);
                ft[x][i] = v.x; ft[x][i + 1] = v.y; ft[x][i + 2] = v.z; ft[x][i + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m[1] = max(m[1], rank_of(ft[x][i]));
                m[2] = max(m[2], rank_of(ft[x][i] * left[col + i]));
            }
        }
        block_max<8>(m, red);
        const int ep = rank_exponent(m[0]), ett = rank_exponent(m[1]), el = rank_exponent(m[2]);
        store_fragments(rec + a.rec.p(), 8192, rb * 16, half * 32, pr, pow2_float(ep));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int piece = tid + x * NT, row = piece >> 3, col = (piece & 7) * 8, at = panel_at(row, col);
            put8(rec + a.rec.t() + at, 8192, ft[x], pow2_float(ett));
#pragma unroll
            for (int i = 0; i < 8; ++i) ft[x][i] *= left[col + i];
            put8(tr + at, 8192, ft[x], pow2_float(el));
        }
        __syncthreads();
        // W = (T beta e^G) K: warp = 16 rows x half of the columns, steps up to the row block
        constexpr int TILES = KEY / 16;                                    // 8-column tiles of a warp
        float w[TILES][4] = {};
        {
#pragma unroll
            for (int jb = 0; jb < 4; ++jb) {
                if (jb > rb) continue;
                uint32_t th[4], tl[4];
                const int at = frag_a(rb * 16, jb * 16);
                ldmatrix4(th, ts + at);
                ldmatrix4(tl, ts + 8192 + at);
#pragma unroll
                for (int x = 0; x < TILES / 2; ++x) {
                    uint32_t bh[4], bl[4];
                    const int bt = frag_bt(jb * 16, half * (KEY / 2) + x * 16);
                    ldmatrix4_trans(bh, ks + bt);
                    ldmatrix4_trans(bl, ks + LO + bt);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mma16816(w[2 * x + y], tl, bh[2 * y], bh[2 * y + 1]);
                        mma16816(w[2 * x + y], th, bl[2 * y], bl[2 * y + 1]);
                        mma16816(w[2 * x + y], th, bh[2 * y], bh[2 * y + 1]);
                    }
                }
            }
        }
        uint32_t mw[1] = {};
        const float unw = pow2_float(-el) * unk;
#pragma unroll
        for (int x = 0; x < TILES; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                w[x][y] *= unw;
                mw[0] = max(mw[0], rank_of(w[x][y]));
            }
        block_max<8>(mw, red + 24);
        const int ew = rank_exponent(mw[0]);
#pragma unroll
        for (int x = 0; x < TILES / 4; ++x) {
            float f[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int z = 0; z < 4; ++z) f[y][z] = w[4 * x + y][z];
            store_fragments(rec + a.rec.w(), LO, rb * 16, half * (KEY / 2) + x * 32, f, pow2_float(ew));
        }
        if (tid == 0) {
            head[kUnW] = pow2_float(-ew);
            head[kUnKt] = pow2_float(-et);
            head[kUnQ] = pow2_float(-eqt);
            head[kUnT] = pow2_float(-ett);
            head[kUnP] = pow2_float(-ep);
        }
    }
}

template <typename T, int KEY>
cudaError_t prepare(const PrepareParams& a, cudaStream_t st) {
    constexpr int smem = PrepareSmem<KEY>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(delta_prepare_kernel<T, KEY>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    delta_prepare_kernel<T, KEY><<<(unsigned)(a.p.B * a.p.HK * a.n), NT, smem, st>>>(a);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t prepare_typed(PrepareParams& a, cudaStream_t st) {
    auto vec = [&](const void* base, const long long* s) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && s[0] * sizeof(T) % 16 == 0 && s[1] * sizeof(T) % 16 == 0 &&
               s[2] * sizeof(T) % 16 == 0 && a.p.DK % 8 == 0;
    };
    a.vec_q = vec(a.in.q, a.p.q_stride);
    a.vec_k = vec(a.in.k, a.p.k_stride);
    return a.rec.key == 64 ? prepare<T, 64>(a, st) : prepare<T, 128>(a, st);
}

}  // namespace

cudaError_t launch_delta_prepare(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaInputs& in, void* records,
                                 cudaStream_t st) {
    PrepareParams a = {p, in, static_cast<uint8_t*>(records), plan.rec, plan.n, 0, 0};
    return p.dtype == AUSSM_FLOAT32 ? prepare_typed<float>(a, st)
           : p.dtype == AUSSM_BFLOAT16 ? prepare_typed<__nv_bfloat16>(a, st) : prepare_typed<__half>(a, st);
}

}  // namespace aussm
