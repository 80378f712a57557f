// extern "C" entry points of the gated delta rule (see include/aussm_b200.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include "delta.cuh"
#include "host_common.cuh"

using namespace aussm;

namespace {

int delta_check(const char* who, const aussm_b200_delta_t* p) {
    if (!p) {
        set_error("%s: null problem", who);
        return AUSSM_EINVAL;
    }
    if (p->B <= 0 || p->L <= 0 || p->HK <= 0 || p->HV <= 0 || p->DK <= 0 || p->DV <= 0) {
        set_error("%s: sizes must be positive (B=%d L=%d HK=%d HV=%d DK=%d DV=%d)", who, p->B, p->L, p->HK, p->HV, p->DK,
                  p->DV);
        return AUSSM_EINVAL;
    }
    if (p->HV % p->HK) {
        set_error("%s: %d value heads are not a multiple of %d key heads", who, p->HV, p->HK);
        return AUSSM_EINVAL;
    }
    if (p->DK > AUSSM_MAX_DELTA_KEY || p->DV > AUSSM_MAX_DELTA_VALUE) {
        set_error("%s: heads of %d keys and %d values, at most %d and %d are supported", who, p->DK, p->DV,
                  AUSSM_MAX_DELTA_KEY, AUSSM_MAX_DELTA_VALUE);
        return AUSSM_EINVAL;
    }
    if (p->dtype < AUSSM_FLOAT32 || p->dtype > AUSSM_FLOAT16) {
        set_error("%s: unknown type %d", who, p->dtype);
        return AUSSM_EINVAL;
    }
    // grids are built from the number of chunks and heads
    if ((long long)p->B * p->HV > 0x3fffffffLL / delta_chunks(p->L)) {
        set_error("%s: B*HV*L/%d exceeds 2^30", who, kDeltaChunk);
        return AUSSM_EINVAL;
    }
    return AUSSM_OK;
}

int need(const char* who, const char* what, const void* ptr, size_t have, size_t want) {
    if (want && (!ptr || have < want || (reinterpret_cast<uintptr_t>(ptr) & 255u))) {
        set_error("%s: %s of %zu bytes, 256-byte aligned, required, got %zu", who, what, want, have);
        return AUSSM_EWORKSPACE;
    }
    return AUSSM_OK;
}

int launched(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return AUSSM_OK;
    set_error("%s launch: %s", who, cudaGetErrorString(e));
    return AUSSM_ECUDA;
}

}  // namespace

extern "C" {

size_t aussm_b200_delta_keep_bytes(const aussm_b200_delta_t* p) {
    return delta_check("delta_keep_bytes", p) ? 0 : delta_plan(*p).keep_bytes;
}

size_t aussm_b200_delta_workspace_bytes(const aussm_b200_delta_t* p, int backward) {
    if (delta_check("delta_workspace_bytes", p)) return 0;
    return backward ? delta_plan(*p).bwd_bytes : delta_plan(*p).fwd_bytes;
}

int aussm_b200_delta_fwd(const aussm_b200_delta_t* p, const void* q, const void* k, const void* v, const float* g,
                         const float* beta, const float* s0, void* o, float* s1, void* keep, size_t keep_bytes,
                         void* workspace, size_t workspace_bytes, aussm_stream_t stream) {
    if (int rc = delta_check("delta_fwd", p)) return rc;
    if (!q || !k || !v || !g || !beta || !o) {
        set_error("delta_fwd: null input or output pointer");
        return AUSSM_EINVAL;
    }
    const bool train = keep != nullptr;
    if (train) {
        if (int rc = need("delta_fwd", "keep buffer", keep, keep_bytes, delta_plan(*p).keep_bytes)) return rc;
    } else {
        if (int rc = need("delta_fwd", "workspace", workspace, workspace_bytes, aussm_b200_delta_workspace_bytes(p, 0))) return rc;
        keep = workspace;
    }
    return launched("delta_fwd", launch_delta_fwd(*p, {q, k, v, g, beta}, s0, o, s1, keep, train, (cudaStream_t)stream));
}

int aussm_b200_delta_bwd(const aussm_b200_delta_t* p, const void* go, const float* gs1, const void* q, const void* k,
                         const void* v, const float* g, const float* beta, const void* keep, size_t keep_bytes,
                         void* dq, void* dk, void* dv, float* dg, float* dbeta, float* ds0, void* workspace,
                         size_t workspace_bytes, aussm_stream_t stream) {
    if (int rc = delta_check("delta_bwd", p)) return rc;
    if (!go || !q || !k || !v || !g || !beta || !dq || !dk || !dv || !dg || !dbeta) {
        set_error("delta_bwd: null input or output pointer");
        return AUSSM_EINVAL;
    }
    if (int rc = need("delta_bwd", "keep buffer", keep, keep_bytes, delta_plan(*p).keep_bytes)) return rc;
    if (int rc = need("delta_bwd", "workspace", workspace, workspace_bytes, delta_plan(*p).bwd_bytes)) return rc;
    return launched("delta_bwd", launch_delta_bwd(*p, {q, k, v, g, beta}, go, gs1, keep, dq, dk, dv, dg, dbeta, ds0,
                                                  workspace, (cudaStream_t)stream));
}

int aussm_b200_delta_step(const aussm_b200_delta_t* p, const void* q, const void* k, const void* v, const float* g,
                          const float* beta, const float* state, float* new_state, void* o, aussm_stream_t stream) {
    if (int rc = delta_check("delta_step", p)) return rc;
    if (!q || !k || !v || !g || !beta || !state || !new_state || !o) {
        set_error("delta_step: null input or output pointer");
        return AUSSM_EINVAL;
    }
    return launched("delta_step", launch_delta_step(*p, {q, k, v, g, beta}, state, new_state, o, (cudaStream_t)stream));
}

}  // extern "C"
