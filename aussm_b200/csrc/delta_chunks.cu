// Gated delta rule over chunks, the plain way: products of small matrices element by element, operands in global
// memory, float32 throughout.
#include "delta.cuh"
#include "host_common.cuh"

namespace aussm {
namespace {

constexpr int C = kDeltaChunk;
constexpr int NT = 256;
constexpr int SLICE = 32;            // value columns of a block of the recurrences

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// a stored tile as the numbers it stands for
struct Tile {
    const uint8_t* p;
    int lo;
    float un;
    __device__ float operator()(int i, int j) const {
        const uint8_t* at = p + panel_at(i, j);
        return (__half2float(*reinterpret_cast<const __half*>(at)) + __half2float(*reinterpret_cast<const __half*>(at + lo))) * un;
    }
};
struct Header {
    const float* f;
    __device__ float diff(int i, int j) const { return (f[kGHi + i] - f[kGHi + j]) + (f[kGLo + i] - f[kGLo + j]); }
    __device__ float since(int i) const { return expf(f[kGHi + i] + f[kGLo + i]); }
    __device__ float until(int i) const { return expf(diff(C - 1, i)); }
};
struct Record {
    Header G;
    Tile W, Kt, Q, T, P;
    __device__ Record(const uint8_t* base, const DeltaRecord& r, size_t at) {
        const uint8_t* p = base + at * r.bytes();
        const float* f = reinterpret_cast<const float*>(p);
        const int lo = r.key * 128;
        G.f = f;
        W = {p + r.w(), lo, f[kUnW]};
        Kt = {p + r.kt(), lo, f[kUnKt]};
        Q = {p + r.q(), lo, f[kUnQ]};
        T = {p + r.t(), 8192, f[kUnT]};
        P = {p + r.p(), 8192, f[kUnP]};
    }
};

struct Params {
    aussm_b200_delta_t p;
    DeltaInputs in;
    const void* go;
    const float *s0, *gs1;
    void* o;
    float *s1, *ds0;
    const uint8_t* records;
    DeltaRecord rec;
    float *N, *S;              // V' and entry states of every chunk and head
    float *X, *dN, *dS;        // backward: (C, DV) twice, (DK, DV) per chunk and head
    void *dq, *dk, *dv;
    float *dg, *dbeta;
    int n;                     // chunks
};

template <typename T>
struct Rows {                  // rows of one head from step t0 on; zero behind the end
    const T* p;
    long long step;
    int rows;
    __device__ float operator()(int i, int j) const { return i < rows ? to_f32(p[i * step + j]) : 0.f; }
};
template <typename T>
__device__ Rows<T> rows_of(const void* base, const long long (&s)[3], int b, int t0, int h, int L) {
    return {static_cast<const T*>(base) + b * s[0] + t0 * s[1] + h * s[2], s[1], min(C, L - t0)};
}

template <typename F, typename G>
__device__ void products(int M, int N, int K, F term, G store) {
    for (int e = threadIdx.x; e < M * N; e += NT) {
        const int i = e / N, j = e % N;
        float a = 0.f;
        for (int k = 0; k < K; ++k) a += term(i, j, k);
        store(i, j, a);
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) backward_kernel(const Params a) {
    extern __shared__ float dS[];    // (DK, SLICE)
    const aussm_b200_delta_t& p = a.p;
    const int bh = blockIdx.x, b = bh / p.HV, h = bh % p.HV, hk = h / (p.HV / p.HK);
    const int v0 = blockIdx.y * SLICE, nv = min(SLICE, p.DV - v0);
    for (int e = threadIdx.x; e < p.DK * nv; e += NT)
        dS[e / nv * SLICE + e % nv] = a.gs1 ? a.gs1[((size_t)bh * p.DK + e / nv) * p.DV + v0 + e % nv] : 0.f;
    __syncthreads();
    for (int c = a.n - 1; c >= 0; --c) {
        const int t0 = c * C, rows = min(C, p.L - t0);
        const size_t at = (size_t)bh * a.n + c;
        const Record r(a.records, a.rec, at);
        float *dN = a.dN + at * C * p.DV + v0, *X = a.X + at * C * p.DV + v0;
        const Rows<T> q = rows_of<T>(a.in.q, p.q_stride, b, t0, hk, p.L), k = rows_of<T>(a.in.k, p.k_stride, b, t0, hk, p.L),
                      go = rows_of<T>(a.go, p.go_stride, b, t0, h, p.L);
        const float* be = a.in.beta + ((long long)b * p.L + t0) * p.HV + h;
        for (int e = threadIdx.x; e < p.DK * nv; e += NT)
            a.dS[(at * p.DK + e / nv) * p.DV + v0 + e % nv] = dS[e / nv * SLICE + e % nv];
        products(C, nv, C + p.DK, [&](int i, int j, int m) {
            if (m >= C) return r.Kt(i, m - C) * dS[(m - C) * SLICE + j];
            return m >= i ? r.P(m, i) * go(m, v0 + j) : 0.f;
        }, [&](int i, int j, float x) { dN[(size_t)i * p.DV + j] = x; });
        __syncthreads();
        products(C, nv, C, [&](int i, int j, int m) { return m >= i ? r.T(m, i) * dN[(size_t)m * p.DV + j] : 0.f; },
                 [&](int i, int j, float x) {
                     X[(size_t)i * p.DV + j] = x;
                     if (i < rows)
                         static_cast<T*>(a.dv)[(((long long)b * p.L + t0 + i) * p.HV + h) * p.DV + v0 + j] =
                             from_f32<T>(be[(long long)i * p.HV] * x);
                 });
        products(p.DK, nv, C, [&](int x, int j, int i) {
            return r.Q(i, x) * go(i, v0 + j) - r.W(i, x) * dN[(size_t)i * p.DV + j];
        }, [&](int x, int j, float s) { dS[x * SLICE + j] = r.G.f[kGamma] * dS[x * SLICE + j] + s; });
        __syncthreads();
    }
    if (a.ds0)
        for (int e = threadIdx.x; e < p.DK * nv; e += NT)
            a.ds0[((size_t)bh * p.DK + e / nv) * p.DV + v0 + e % nv] = dS[e / nv * SLICE + e % nv];
}

// Gradients of q, k, g and beta of a chunk; a block loops over the value heads of a key head.
template <typename T>
__global__ void __launch_bounds__(NT) gradients_kernel(const Params a) {
    extern __shared__ float sm[];
    const aussm_b200_delta_t& p = a.p;
    const int r = p.HV / p.HK, c = blockIdx.x % a.n, b = blockIdx.x / a.n / p.HK, hk = blockIdx.x / a.n % p.HK;
    const int t0 = c * C, rows = min(C, p.L - t0), DK = p.DK, DV = p.DV;
    float *Ep = sm, *E = Ep + C * C, *F = E + C * C, *dQ = F + C * C, *dK = dQ + C * DK, *dG = dK + C * DK, *dB = dG + C, *dGs = dB + C;
    const Rows<T> q = rows_of<T>(a.in.q, p.q_stride, b, t0, hk, p.L), k = rows_of<T>(a.in.k, p.k_stride, b, t0, hk, p.L);
    for (int e = threadIdx.x; e < 2 * C * DK; e += NT) dQ[e] = 0.f;
    for (int h = hk * r; h < hk * r + r; ++h) {
        const size_t at = ((size_t)b * p.HV + h) * a.n + c;
        const Record rc(a.records, a.rec, at);
        const Header& G = rc.G;
        const float *N = a.N + at * C * DV, *X = a.X + at * C * DV, *S = a.S + at * DK * DV,
                    *dS = a.dS + at * DK * DV;
        const Rows<T> go = rows_of<T>(a.go, p.go_stride, b, t0, h, p.L), v = rows_of<T>(a.in.v, p.v_stride, b, t0, h, p.L);
        const float* beta = a.in.beta + ((long long)b * p.L + t0) * p.HV + h;
        auto be = [&](int i) { return i < rows ? beta[(long long)i * p.HV] : 0.f; };
        __syncthreads();
        for (int e = threadIdx.x; e < 3 * C; e += NT) dG[e] = 0.f;
        __syncthreads();
        products(C, C, DV, [&](int i, int j, int x) { return j <= i ? go(i, x) * N[(size_t)j * DV + x] : 0.f; },
                 [&](int i, int j, float x) { Ep[i * C + j] = j <= i ? p.scale * expf(G.diff(i, j)) * x : 0.f; });
        products(C, C, DV, [&](int i, int j, int x) { return j < i ? X[(size_t)i * DV + x] * N[(size_t)j * DV + x] : 0.f; },
                 [&](int i, int j, float x) { E[i * C + j] = j < i ? -expf(G.diff(i, j)) * x : 0.f; });      // beta follows
        __syncthreads();
        if (threadIdx.x < C) {
            const int i = threadIdx.x;
            float bi = 0.f;
            for (int j = 0; j < i; ++j) {
                float qk = 0.f, kk = 0.f;
                for (int x = 0; x < DK; ++x) {
                    qk += q(i, x) * k(j, x);
                    kk += k(i, x) * k(j, x);
                }
                F[i * C + j] = Ep[i * C + j] * qk + be(i) * E[i * C + j] * kk;      // gradient of G_i - G_j
                bi += E[i * C + j] * kk;
            }
            for (int x = 0; x < DV; ++x) bi += X[(size_t)i * DV + x] * v(i, x);
            dB[i] = bi;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < C; i += NT) {            // row i: the terms with states
            const float since = G.since(i), until = G.until(i);
            float kz = 0.f, kkt = 0.f, qqt = 0.f;
            for (int x = 0; x < DK; ++x) {
                float dqt = 0.f, z = 0.f, dkt = 0.f;
                for (int y = 0; y < DV; ++y) {
                    dqt += go(i, y) * S[(size_t)x * DV + y];
                    z += X[(size_t)i * DV + y] * S[(size_t)x * DV + y];
                    dkt += N[(size_t)i * DV + y] * dS[(size_t)x * DV + y];
                }
                kz += since * z * k(i, x);
                kkt += until * dkt * k(i, x);
                qqt += p.scale * since * dqt * q(i, x);
                float dq = p.scale * since * dqt, dk = until * dkt - be(i) * since * z;
                for (int j = 0; j < C; ++j) {
                    dq += Ep[i * C + j] * k(j, x);
                    dk += Ep[j * C + i] * q(j, x) + (be(i) * E[i * C + j] + be(j) * E[j * C + i]) * k(j, x);
                }
                dQ[i * DK + x] += dq;
                dK[i * DK + x] += dk;
            }
            dG[i] = qqt - be(i) * kz;
            dB[i] -= kz;
            dGs[i] = kkt;
        }
        __syncthreads();
        // g_t stands in G_i for i >= t, in G_i - G_j for j < t <= i, in G_C - G_i for i < t and in G_C: summed over just
        // these pairs, since sums over all of which most cancel would lose a strongly decayed head's small gradients
        if (threadIdx.x < rows) {
            const int t = threadIdx.x;
            float ss = 0.f, sum = 0.f;
            for (int e = 0; e < DK * DV; ++e) ss += dS[e] * S[e];
            sum = G.f[kGamma] * ss;
            for (int i = 0; i < t; ++i) sum += dGs[i];
            for (int i = t; i < C; ++i) {
                sum += dG[i];
                for (int j = 0; j < t; ++j) sum += F[i * C + j];
            }
            const long long o = ((long long)b * p.L + t0 + t) * p.HV + h;
            a.dg[o] = sum;
            a.dbeta[o] = dB[t];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * DK; e += NT) {
        const long long o = (((long long)b * p.L + t0 + e / DK) * p.HK + hk) * DK + e % DK;
        static_cast<T*>(a.dq)[o] = from_f32<T>(dQ[e]);
        static_cast<T*>(a.dk)[o] = from_f32<T>(dK[e]);
    }
}

template <typename T>
cudaError_t backward(const Params& a, cudaStream_t st) {
    backward_kernel<T><<<dim3(a.p.B * a.p.HV, (a.p.DV + SLICE - 1) / SLICE), NT, a.p.DK * SLICE * 4, st>>>(a);
    const int smem = (3 * C * C + 2 * C * a.p.DK + 3 * C) * 4;
    cudaError_t e = cudaFuncSetAttribute(gradients_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    gradients_kernel<T><<<(unsigned)(a.p.B * a.p.HK * a.n), NT, smem, st>>>(a);
    count_launch(2);
    return cudaGetLastError();
}

}  // namespace

DeltaPlan delta_plan(const aussm_b200_delta_t& p) {
    DeltaPlan d;
    d.n = (p.L + C - 1) / C;
    d.heads = (size_t)p.B * p.HV * d.n;
    d.rec.key = p.DK <= 64 ? 64 : 128;
    d.news = d.heads * d.rec.bytes();
    d.states = d.news + up256(d.heads * C * p.DV * sizeof(float));
    d.keep_bytes = d.states + up256(d.heads * p.DK * p.DV * sizeof(float));
    d.bwd_bytes = up256(d.heads * (size_t)(2 * C * p.DV + p.DK * p.DV) * 4);
    return d;
}

static Params params(const aussm_b200_delta_t& p, const DeltaPlan& plan, const DeltaInputs& in, void* keep) {
    Params a = {};
    uint8_t* k = static_cast<uint8_t*>(keep);
    a.p = p; a.in = in; a.n = plan.n; a.rec = plan.rec; a.records = k;
    a.N = reinterpret_cast<float*>(k + plan.news);
    a.S = reinterpret_cast<float*>(k + plan.states);
    return a;
}

cudaError_t launch_delta_fwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* s0, void* o, float* s1,
                             void* keep, bool train, cudaStream_t st) {
    const DeltaPlan plan = delta_plan(p);
    cudaError_t e = launch_delta_prepare(p, plan, in, keep, st);
    if (e != cudaSuccess) return e;
    uint8_t* k = static_cast<uint8_t*>(keep);
    float *news = train ? reinterpret_cast<float*>(k + plan.news) : nullptr, *states = train ? reinterpret_cast<float*>(k + plan.states) : nullptr;
    return launch_delta_scan(p, plan, {keep, in.v, s0, s1, o, news, states}, false, st);
}

cudaError_t launch_delta_bwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const void* go, const float* gs1,
                             const void* keep, void* dq, void* dk, void* dv, float* dg, float* dbeta, float* ds0,
                             void* ws, cudaStream_t st) {
    const DeltaPlan plan = delta_plan(p);
    Params a = params(p, plan, in, const_cast<void*>(keep));
    a.go = go; a.gs1 = gs1;
    a.dq = dq; a.dk = dk; a.dv = dv; a.dg = dg; a.dbeta = dbeta; a.ds0 = ds0;
    a.X = static_cast<float*>(ws);
    a.dN = a.X + plan.heads * C * p.DV;
    a.dS = a.dN + plan.heads * C * p.DV;
    return p.dtype == AUSSM_FLOAT32 ? backward<float>(a, st) : p.dtype == AUSSM_BFLOAT16 ? backward<__nv_bfloat16>(a, st)
                                                                                        : backward<__half>(a, st);
}

}  // namespace aussm
