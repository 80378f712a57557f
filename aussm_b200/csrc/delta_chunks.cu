// Gated delta rule over whole sequences: the order of its kernels and the layout of their buffers (formulas in delta.cuh).
#include "delta.cuh"

namespace aussm {
namespace {

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

DeltaPlan delta_plan(const aussm_b200_delta_t& p) {
    DeltaPlan d;
    d.n = delta_chunks(p.L);
    d.heads = (size_t)p.B * p.HV * d.n;
    d.rec.key = p.DK <= 64 ? 64 : 128;
    d.slices = (p.DV + 127) / 128;
    const size_t pieces = d.heads * d.slices;
    // A block of the recurrences takes an SM; a segment costs a second pass (a third forward) over its chunks and a share of
    // the chain.  One sequence of 4096 steps, heads of 128, forward / training, in segments and whole: 16 heads 213 against
    // 331 / 671 against 1021 us, 32 heads 358 against 402 / 1217 against 1417 us, 48 heads 490 against 474 / 1747 against
    // 1797 us; 64 heads in two segments 540 against 546 / 2185 against 2190 us.  So: from a third of the SMs on, whole.
    const long long blocks = (long long)p.B * p.HV * d.slices;
    long long segs = 1;
    if (blocks * 3 <= 148) {
        segs = 148 / blocks;
        if (segs > d.n / 4) segs = d.n / 4;
        if (segs < 3) segs = 1;        // three segments or more of at least four chunks stay three or more when rounded up
    }
    d.span = (int)((d.n + segs - 1) / segs);
    d.segs = (d.n + d.span - 1) / d.span;
    const size_t bh = (size_t)p.B * p.HV, ends = d.segs > 1 ? up256((d.segs - 1) * bh * p.DK * p.DV * sizeof(float)) : 0;
    d.transitions = d.heads * d.rec.bytes();
    d.ends = d.transitions + (d.segs > 1 ? d.segs * bh * d.rec.key * d.rec.key * sizeof(float) : 0);
    d.fwd_bytes = d.news = d.ends + ends;
    d.states = d.news + up256(pieces * DeltaPlan::news_bytes());
    d.keep_bytes = d.states + up256(pieces * DeltaPlan::state_bytes(d.rec.key));
    d.dstates = up256(pieces * DeltaPlan::x_bytes());
    d.bwd_ends = d.dstates + up256(pieces * DeltaPlan::state_bytes(d.rec.key));
    d.bwd_bytes = d.bwd_ends + ends;
    return d;
}

cudaError_t launch_delta_fwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const float* s0, void* o, float* s1,
                             void* keep, bool train, cudaStream_t st) {
    const DeltaPlan plan = delta_plan(p);
    cudaError_t e = launch_delta_prepare(p, plan, in, keep, st);
    if (e != cudaSuccess) return e;
    uint8_t* k = static_cast<uint8_t*>(keep);
    void *news = train ? k + plan.news : nullptr, *states = train ? k + plan.states : nullptr;
    return launch_delta_scan(p, plan, {keep, in.v, s0, s1, o, news, states, k + plan.transitions, k + plan.ends}, false, st);
}

cudaError_t launch_delta_bwd(const aussm_b200_delta_t& p, const DeltaInputs& in, const void* go, const float* gs1,
                             const void* keep, void* dq, void* dk, void* dv, float* dg, float* dbeta, float* ds0,
                             void* workspace, cudaStream_t st) {
    const DeltaPlan plan = delta_plan(p);
    const uint8_t* k = static_cast<const uint8_t*>(keep);
    uint8_t* w = static_cast<uint8_t*>(workspace);
    cudaError_t e = launch_delta_scan(p, plan, {keep, go, gs1, ds0, dv, w, w + plan.dstates,
                                              const_cast<uint8_t*>(k) + plan.transitions, w + plan.bwd_ends}, true, st);
    if (e != cudaSuccess) return e;
    return launch_delta_grads(p, plan, in, {keep, go, k + plan.news, w, k + plan.states, w + plan.dstates, dq, dk, dg, dbeta}, st);
}

}  // namespace aussm
