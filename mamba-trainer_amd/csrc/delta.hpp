// The gated delta rule's kernels share this: the launch arguments and the
// storage types (bf16, f16, f32; all arithmetic is in f32 or wider).
#pragma once

#include <type_traits>

#include "m3_device.hpp"

namespace m3 {

struct DeltaLaunch {
    size_t batch, seq, heads, groups, head_dim, d_state;
    int dtype;                      // m3_dtype of q, k, v, y
    const void *q, *k, *v;          // [B,T,G,N] x2, [B,T,H,P] at the token strides
    size_t qs, ks, vs;              // elements between tokens
    const float *g, *beta;          // [B,T,H]
    const int32_t *lengths;         // [B] or null
    const float *state;             // [B,H,P,N] or null
    float scale;
    int qk_norm;
    void *y;                        // [B,T,H,P]
    float *state_out;               // [B,H,P,N] or null
};
struct DeltaGrads {
    const void *dy;                 // [B,T,H,P]
    const float *dstate;            // [B,H,P,N] or null
    void *dq, *dk, *dv;             // [B,T,G,N] x2, [B,T,H,P]
    float *dg, *dbeta;              // [B,T,H]
    float *dstate0;                 // [B,H,P,N] or null
};
constexpr size_t kDeltaMaxHeadDim = 1024;
constexpr size_t kDeltaMaxState = 256;

// The recurrence token by token with the state in registers (delta_recur.hip).
hipError_t launch_delta_recur(const DeltaLaunch &a, hipStream_t s);

// g and beta from a projection's columns (delta_recur.hip).
hipError_t launch_delta_gates(size_t rows, size_t heads, int dtype, const void *pa, const void *pb, size_t stride,
                              const float *a_log, const float *dt_bias, float *g, float *beta, hipStream_t s);

// Chunk by chunk on the MFMA (delta_chunk.hip): whether a window takes this
// form, the workspace it needs, and the launch.
bool delta_chunk_wanted(const DeltaLaunch &a);
size_t delta_chunk_workspace(const DeltaLaunch &a);
hipError_t launch_delta_chunk(const DeltaLaunch &a, void *workspace, hipStream_t s, int &launches);

// Gradients (delta_backward.hip): the shapes covered, the workspace, the launch.
bool delta_backward_supported(const DeltaLaunch &a);
size_t delta_backward_workspace(const DeltaLaunch &a);
hipError_t launch_delta_backward(const DeltaLaunch &a, const DeltaGrads &g, void *workspace,
                                 hipStream_t s, int &launches);

namespace delta {

struct f16_t {
    uint16_t bits;
};
__device__ __forceinline__ float ldf(const float *p) { return *p; }
__device__ __forceinline__ float ldf(const bf16_t *p) { return to_f32(*p); }
__device__ __forceinline__ float ldf(const f16_t *p) {
    return static_cast<float>(__builtin_bit_cast(_Float16, p->bits));
}
__device__ __forceinline__ void stf(float *p, float v) { *p = v; }
__device__ __forceinline__ void stf(bf16_t *p, float v) { *p = from_f32<bf16_t>(v); }
__device__ __forceinline__ void stf(f16_t *p, float v) {
    p->bits = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

constexpr float kUnitEps = 1e-6f;   // of qk_norm

// exp(g) is zero in f32 from here on (the smallest subnormal is exp(-103.3)),
// so a log decay below it, -inf among them, stands for it: sums of log decays
// then stay finite.  NaN passes.
__device__ __forceinline__ float clamp_decay(float g) { return g < -128.0f ? -128.0f : g; }

// Tokens of sequence b that count.
__device__ __forceinline__ int valid_len(const int32_t *lengths, size_t b, int seq) {
    if (lengths == nullptr) return seq;
    const int n = lengths[b];
    return n < 0 ? 0 : n > seq ? seq : n;
}

// f(T{}) for the storage type of `dtype` (M3_F32 0, M3_BF16 1, M3_F16 2).
template <typename F>
hipError_t by_type(int dtype, F f) {
    if (dtype == 0) return f(float{});
    if (dtype == 1) return f(bf16_t{});
    return f(f16_t{});
}

}  // namespace delta
}  // namespace m3
