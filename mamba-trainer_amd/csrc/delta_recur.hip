// The gated delta rule token by token on gfx950: the serving step, and short
// windows.
//
// Per sequence and head S~ = exp(g) S, u = beta (v - S~ k), S = S~ + u k^T,
// y = scale S q.  Each row of S [P, N] goes on by itself, so a group of LN
// lanes holds RPL rows in registers, four columns a lane, for all tokens of
// the call: the state is read and written once, which is what a step costs
// (8 P N bytes a head against 2 (2 N + 2 P) of inputs).  One reduction over the
// group's lanes serves both products of a token, as S q = S~ q + u (k . q).
#include "delta.hpp"

namespace m3 {
namespace {

using namespace delta;

// Sum over aligned groups of LN lanes; every lane gets the sum.
template <int LN>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int off = 1; off < LN; off <<= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Four consecutive values from index n on, zero from N on.
template <bool VEC>
__device__ __forceinline__ f32x4 ld4f(const float *row, int n, int N) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
        if (n < N) r = *reinterpret_cast<const f32x4 *>(row + n);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < N) r[j] = row[n + j];
    }
    return r;
}
template <typename T>
__device__ __forceinline__ f32x4 ld4(const T *row, int n, int N) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < N) r[j] = ldf(row + n + j);
    return r;
}
__device__ __forceinline__ float dot4(f32x4 a, f32x4 b) {
    return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}

// VEC: the state's rows are 16-byte aligned (N a multiple of 4).
template <typename T, int LN, int RPL, bool VEC>
__global__ void __launch_bounds__(256) delta_recur_kernel(DeltaLaunch a) {
    constexpr int NG = 256 / LN;   // row groups of the workgroup
    const int tid = threadIdx.x, lane = tid % LN, grp = tid / LN;
    const size_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
    const int N = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const int n0 = 4 * lane, row0 = blockIdx.y * (NG * RPL) + grp;
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    const size_t kg = h / (a.heads / a.groups);
    const float *s_in = a.state ? a.state + bh * P * N : nullptr;
    f32x4 S[RPL];
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const int r = row0 + j * NG;
        S[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s_in && r < P) S[j] = ld4f<VEC>(s_in + static_cast<size_t>(r) * N, n0, N);
    }
    T *yp = static_cast<T *>(a.y) + (b * L * a.heads + h) * P;
    for (int t = 0; t < len; ++t) {
        const size_t tok = b * L + t;
        const T *vp = static_cast<const T *>(a.v) + tok * a.vs + h * P;
        f32x4 k = ld4(static_cast<const T *>(a.k) + tok * a.ks + kg * N, n0, N);
        f32x4 q = ld4(static_cast<const T *>(a.q) + tok * a.qs + kg * N, n0, N);
        const float alpha = expf(clamp_decay(a.g[tok * a.heads + h]));
        const float beta = a.beta[tok * a.heads + h];
        float v[RPL];
#pragma unroll
        for (int j = 0; j < RPL; ++j) v[j] = row0 + j * NG < P ? ldf(vp + row0 + j * NG) : 0.f;
        if (a.qk_norm) {
            const float rk = 1.0f / sqrtf(lanes_sum<LN>(dot4(k, k)) + kUnitEps);
            const float rq = 1.0f / sqrtf(lanes_sum<LN>(dot4(q, q)) + kUnitEps);
            k *= rk;
            q *= rq;
        }
        const float kq = lanes_sum<LN>(dot4(k, q));
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
            S[j] *= alpha;
            const float u = beta * (v[j] - lanes_sum<LN>(dot4(S[j], k)));
            const float y = a.scale * (lanes_sum<LN>(dot4(S[j], q)) + u * kq);
            S[j] += u * k;
            const int r = row0 + j * NG;
            if (lane == 0 && r < P) stf(yp + static_cast<size_t>(t) * a.heads * P + r, y);
        }
    }
    for (int t = len; t < L; ++t)
        for (int j = 0; j < RPL; ++j) {
            const int r = row0 + j * NG;
            if (lane == 0 && r < P) stf(yp + static_cast<size_t>(t) * a.heads * P + r, 0.f);
        }
    if (a.state_out == nullptr) return;
    float *s_out = a.state_out + bh * P * N;
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const int r = row0 + j * NG;
        if (r >= P) continue;
        float *row = s_out + static_cast<size_t>(r) * N;
        if constexpr (VEC) {
            if (n0 < N) *reinterpret_cast<f32x4 *>(row + n0) = S[j];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < N) row[n0 + i] = S[j][i];
        }
    }
}

template <typename T, int LN, int RPL>
hipError_t go(const DeltaLaunch &a, hipStream_t s) {
    const auto aligned = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = a.d_state % 4 == 0 && aligned(a.state) && aligned(a.state_out);
    constexpr unsigned rows = 256 / LN * RPL;
    const dim3 grid(static_cast<unsigned>(a.batch * a.heads),
                    static_cast<unsigned>((a.head_dim + rows - 1) / rows));
    if (vec)
        hipLaunchKernelGGL((delta_recur_kernel<T, LN, RPL, true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((delta_recur_kernel<T, LN, RPL, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename T, int LN>
hipError_t by_rows(const DeltaLaunch &a, hipStream_t s) {
    // eight rows a group keep 128 bytes a lane in flight; few sequences are
    // spread over more workgroups instead
    const size_t wgs = a.batch * a.heads * ((a.head_dim * LN + 2047) / 2048);
    if (wgs >= 1024) return go<T, LN, 8>(a, s);
    if (wgs >= 256) return go<T, LN, 4>(a, s);
    return go<T, LN, 1>(a, s);
}

}  // namespace

hipError_t launch_delta_recur(const DeltaLaunch &a, hipStream_t s) {
    if (a.batch == 0) return hipSuccess;
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.d_state <= 16) return by_rows<T, 4>(a, s);
        if (a.d_state <= 32) return by_rows<T, 8>(a, s);
        if (a.d_state <= 64) return by_rows<T, 16>(a, s);
        if (a.d_state <= 128) return by_rows<T, 32>(a, s);
        return by_rows<T, 64>(a, s);
    });
}

}  // namespace m3
