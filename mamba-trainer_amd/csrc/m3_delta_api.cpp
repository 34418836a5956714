// C ABI of the gated delta rule (include/mamba3_delta.h): argument checks and
// dispatch.
#include "mamba3_delta.h"

#include <hip/hip_runtime.h>

#include "delta.hpp"
#include "m3_internal.hpp"

namespace m3 {
m3_status api_fail(m3_status st, const char *fmt, ...);
m3_status api_ok();
m3_status api_hip_fail(hipError_t e, const char *what);
void count_launches(uint64_t n);
}  // namespace m3

namespace {

hipStream_t as_stream(void *s) { return static_cast<hipStream_t>(s); }

// A 31-bit count of anything a grid or a kernel's own index runs over.
constexpr size_t kMost = size_t(1) << 31;
bool product_over(size_t a, size_t b, size_t most) { return b != 0 && a > (most - 1) / b; }

// The checks every entry point runs before any device work.
m3_status check(const m3_delta_inputs *in) {
    if (in == nullptr) return m3::api_fail(M3_ERR_ARGUMENT, "delta inputs are NULL");
    if (in->dtype != M3_F32 && in->dtype != M3_BF16 && in->dtype != M3_F16)
        return m3::api_fail(M3_ERR_ARGUMENT, "unknown dtype %d", static_cast<int>(in->dtype));
    if (in->heads == 0 || in->groups == 0 || in->head_dim == 0 || in->d_state == 0)
        return m3::api_fail(M3_ERR_CONFIG, "delta rule dimensions must all be positive");
    if (in->heads % in->groups != 0)
        return m3::api_fail(M3_ERR_CONFIG, "n_heads (%zu) must be a multiple of n_groups (%zu)", in->heads,
                            in->groups);
    if (in->head_dim > m3::kDeltaMaxHeadDim || in->d_state > m3::kDeltaMaxState)
        return m3::api_fail(M3_ERR_UNSUPPORTED, "the delta rule takes head_dim up to %zu and d_state up to %zu "
                            "(got %zu, %zu)", m3::kDeltaMaxHeadDim, m3::kDeltaMaxState, in->head_dim, in->d_state);
    if (in->heads >= 65536 || product_over(in->batch, in->heads, kMost) ||
        product_over(in->batch * in->heads, in->seq, kMost))
        return m3::api_fail(M3_ERR_UNSUPPORTED, "batch x seq x heads must stay below 2^31 and heads below 2^16 "
                            "(got %zu x %zu x %zu)", in->batch, in->seq, in->heads);
    const size_t qk = in->groups * in->d_state, pv = in->heads * in->head_dim;
    if ((in->q_stride != 0 && in->q_stride < qk) || (in->k_stride != 0 && in->k_stride < qk) ||
        (in->v_stride != 0 && in->v_stride < pv))
        return m3::api_fail(M3_ERR_SHAPE, "token strides (%zu, %zu, %zu) are shorter than the rows (%zu, %zu, %zu)",
                            in->q_stride, in->k_stride, in->v_stride, qk, qk, pv);
    return M3_OK;
}

m3_status check_buffers(const m3_delta_inputs *in) {
    if (in->batch * in->seq > 0 && (in->q == nullptr || in->k == nullptr || in->v == nullptr ||
                                    in->g == nullptr || in->beta == nullptr))
        return m3::api_fail(M3_ERR_ARGUMENT, "q, k, v, g and beta are required");
    return M3_OK;
}

m3::DeltaLaunch launch_of(const m3_delta_inputs *in) {
    m3::DeltaLaunch a{};
    a.batch = in->batch; a.seq = in->seq; a.heads = in->heads; a.groups = in->groups;
    a.head_dim = in->head_dim; a.d_state = in->d_state; a.dtype = in->dtype;
    a.q = in->q; a.k = in->k; a.v = in->v;
    a.qs = in->q_stride ? in->q_stride : in->groups * in->d_state;
    a.ks = in->k_stride ? in->k_stride : in->groups * in->d_state;
    a.vs = in->v_stride ? in->v_stride : in->heads * in->head_dim;
    a.g = in->g; a.beta = in->beta; a.lengths = in->lengths; a.state = in->state;
    a.scale = in->scale; a.qk_norm = in->qk_norm;
    return a;
}

m3_status check_workspace(const m3_delta_inputs *in, size_t need) {
    if (need == 0) return M3_OK;
    if (in->workspace == nullptr || in->workspace_bytes < need)
        return m3::api_fail(M3_ERR_ARGUMENT, "the workspace holds %zu bytes of the %zu needed",
                            in->workspace == nullptr ? size_t(0) : in->workspace_bytes, need);
    if ((reinterpret_cast<uintptr_t>(in->workspace) & 255u) != 0)
        return m3::api_fail(M3_ERR_ARGUMENT, "the workspace must be 256-byte aligned");
    return M3_OK;
}

}  // namespace

extern "C" {

m3_status m3_delta_gates(size_t rows, size_t heads, int32_t dtype, const void *a, const void *b, size_t stride,
                         const float *a_log, const float *dt_bias, float *g, float *beta, void *stream) {
    if (dtype != M3_F32 && dtype != M3_BF16 && dtype != M3_F16)
        return m3::api_fail(M3_ERR_ARGUMENT, "unknown dtype %d", static_cast<int>(dtype));
    if (heads == 0) return m3::api_fail(M3_ERR_CONFIG, "delta rule dimensions must all be positive");
    if (stride < heads)
        return m3::api_fail(M3_ERR_SHAPE, "rows (%zu apart) are shorter than the heads (%zu)", stride, heads);
    if (product_over(rows, heads, kMost))
        return m3::api_fail(M3_ERR_UNSUPPORTED, "rows x heads must stay below 2^31 (got %zu x %zu)", rows, heads);
    if (rows == 0) return m3::api_ok();
    if (a == nullptr || b == nullptr || a_log == nullptr || g == nullptr || beta == nullptr)
        return m3::api_fail(M3_ERR_ARGUMENT, "a, b, a_log, g and beta are required");
    const hipError_t e = m3::launch_delta_gates(rows, heads, dtype, a, b, stride, a_log, dt_bias, g, beta,
                                                as_stream(stream));
    if (e != hipSuccess) return m3::api_hip_fail(e, "delta gates launch");
    m3::count_launches(1);
    return m3::api_ok();
}

size_t m3_delta_rule_workspace_bytes(const m3_delta_inputs *in) {
    if (check(in) != M3_OK || in->batch == 0) return 0;
    const m3::DeltaLaunch a = launch_of(in);
    return m3::delta_chunk_wanted(a) ? m3::delta_chunk_workspace(a) : 0;
}

m3_status m3_delta_rule(const m3_delta_inputs *in, void *y, float *state_out, void *stream) {
    m3_status st = check(in);
    if (st == M3_OK) st = check_buffers(in);
    if (st != M3_OK) return st;
    if (in->batch * in->seq > 0 && y == nullptr) return m3::api_fail(M3_ERR_ARGUMENT, "y is required");
    m3::DeltaLaunch a = launch_of(in);
    a.y = y;
    a.state_out = state_out;
    if (in->batch == 0) return m3::api_ok();
    int launches = 1;
    hipError_t e;
    if (m3::delta_chunk_wanted(a)) {
        st = check_workspace(in, m3::delta_chunk_workspace(a));
        if (st != M3_OK) return st;
        launches = 0;
        e = m3::launch_delta_chunk(a, in->workspace, as_stream(stream), launches);
    } else {
        e = m3::launch_delta_recur(a, as_stream(stream));
    }
    if (e != hipSuccess) return m3::api_hip_fail(e, "delta rule launch");
    m3::count_launches(static_cast<uint64_t>(launches));
    return m3::api_ok();
}

m3_status m3_delta_step(const m3_delta_inputs *in, float *state, void *y, void *stream) {
    m3_status st = check(in);
    if (st == M3_OK && in->seq != 1)
        st = m3::api_fail(M3_ERR_SHAPE, "a step takes one token a sequence, got %zu", in->seq);
    if (st == M3_OK) st = check_buffers(in);
    if (st != M3_OK) return st;
    if (in->batch == 0) return m3::api_ok();
    if (state == nullptr || y == nullptr) return m3::api_fail(M3_ERR_ARGUMENT, "state and y are required");
    m3::DeltaLaunch a = launch_of(in);
    a.state = a.state_out = state;
    a.y = y;
    const hipError_t e = m3::launch_delta_recur(a, as_stream(stream));
    if (e != hipSuccess) return m3::api_hip_fail(e, "delta step launch");
    m3::count_launches(1);
    return m3::api_ok();
}

size_t m3_delta_rule_backward_workspace_bytes(const m3_delta_inputs *in) {
    if (check(in) != M3_OK) return 0;
    const m3::DeltaLaunch a = launch_of(in);
    return m3::delta_backward_supported(a) ? m3::delta_backward_workspace(a) : 0;
}

m3_status m3_delta_rule_backward(const m3_delta_inputs *in, const m3_delta_grads *gr, void *stream) {
    m3_status st = check(in);
    if (st == M3_OK) st = check_buffers(in);
    if (st != M3_OK) return st;
    if (gr == nullptr) return m3::api_fail(M3_ERR_ARGUMENT, "delta gradients are NULL");
    if (in->batch * in->seq > 0 && (gr->dy == nullptr || gr->dq == nullptr || gr->dk == nullptr ||
                                    gr->dv == nullptr || gr->dg == nullptr || gr->dbeta == nullptr))
        return m3::api_fail(M3_ERR_ARGUMENT, "dy, dq, dk, dv, dg and dbeta are required");
    if ((in->state != nullptr) != (gr->dstate0 != nullptr))
        return m3::api_fail(M3_ERR_ARGUMENT, "dstate0 goes with the state before the window");
    const m3::DeltaLaunch a = launch_of(in);
    if (!m3::delta_backward_supported(a))
        return m3::api_fail(M3_ERR_UNSUPPORTED, "the delta rule's gradient takes d_state up to 128 (got %zu)",
                            in->d_state);
    if (in->batch == 0) return m3::api_ok();
    st = check_workspace(in, m3::delta_backward_workspace(a));
    if (st != M3_OK) return st;
    const m3::DeltaGrads g{gr->dy, gr->dstate, gr->dq, gr->dk, gr->dv, gr->dg, gr->dbeta, gr->dstate0};
    int launches = 0;
    const hipError_t e = m3::launch_delta_backward(a, g, in->workspace, as_stream(stream), launches);
    if (e != hipSuccess) return m3::api_hip_fail(e, "delta rule backward launch");
    m3::count_launches(static_cast<uint64_t>(launches));
    return m3::api_ok();
}

}  // extern "C"
