// The gated delta rule token by token on gfx950: the serving step, and short
// windows.
//
// Per sequence and head S~ = exp(g) S, u = beta (v - S~ k), S = S~ + u k^T,
// y = scale S q.  Each row of S [P, N] goes on by itself, so eight lanes hold RPL
// rows in registers for all tokens of the call: the state is read and written
// once, which is what a step costs (8 P N bytes a head against 2 (2 N + 2 P) of
// inputs).  A lane takes four columns of every 32 (128 contiguous bytes a row),
// so a sum over a row is three DPP steps; one reduction serves both products of a
// token, as S q = S~ q + u (k . q).
//
// A step of 256 sequences of 24 heads (64, 128), bf16, moves 407 MB in 79 us, 5.2
// TB/s, with several states in turn, 61 us on one state again and again; five tokens
// of 64 sequences 106 MB in 30 us, where the tokens' chain counts too.  One sequence:
// 3.7 us, the launch.
#include "delta.hpp"

namespace m3 {
namespace {

using namespace delta;

// Sum over aligned groups of eight lanes, every lane gets it: within quads
// (quad_perm), then across the two (row_half_mirror).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float eight_sum(float v) {
    return dpp_add<0x141>(dpp_add<0x4E>(dpp_add<0xB1>(v)));
}

// Four consecutive stored values from index n on as loaded, zero from N on.  VEC
// (N a multiple of 4, rows aligned to four values): without a branch, so that a
// lane's loads are all on their way together.
template <typename T> struct Four { u32x2 q; };
template <> struct Four<float> { f32x4 q; };
template <bool VEC, typename T>
__device__ __forceinline__ Four<T> load4(const T *row, int n, int N) {
    Four<T> r;
    if constexpr (VEC) {
        r.q = *reinterpret_cast<const decltype(r.q) *>(row + (n < N ? n : 0));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r.q[j] = n + j < N ? row[n + j] : 0.f;
    } else {
        r.q = u32x2{0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < N) r.q[j >> 1] |= static_cast<uint32_t>(row[n + j].bits) << (16 * (j & 1));
    }
    return r;
}
__device__ __forceinline__ f32x4 wide4(const Four<float> &r, bool ok) { return ok ? r.q : f32x4{0.f, 0.f, 0.f, 0.f}; }
template <typename T>
__device__ __forceinline__ f32x4 wide4(const Four<T> &r, bool ok) {
    f32x4 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const T x{static_cast<uint16_t>(r.q[j >> 1] >> (16 * (j & 1)))};
        f[j] = ok ? ldf(&x) : 0.f;
    }
    return f;
}
__device__ __forceinline__ float dot4(f32x4 a, f32x4 b) {
    return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
}

// CH: 32-column pieces of a row; TH: threads.  A token's inputs are loaded while
// the one before is worked on.
template <typename T, int CH, int RPL, int TH, bool VEC>
__global__ void __launch_bounds__(TH) delta_recur_kernel(DeltaLaunch a) {
    constexpr int NG = TH / 8;   // row groups of the workgroup
    const int tid = threadIdx.x, lane = tid % 8, grp = tid / 8;
    const size_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
    const int N = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const int n0 = 4 * lane, row0 = blockIdx.y * (NG * RPL) + grp;
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    const size_t kg = h / (a.heads / a.groups);
    const float *s_in = a.state ? a.state + bh * P * N : nullptr;
    Four<float> s4[RPL][CH];
    f32x4 S[RPL][CH];
    int row[RPL];   // this lane's, clamped: what is past P is not stored
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const int r = row0 + j * NG;
        row[j] = r < P ? r : P - 1;
        if (s_in)
#pragma unroll
            for (int i = 0; i < CH; ++i) s4[j][i] = load4<VEC>(s_in + static_cast<size_t>(row[j]) * N, n0 + 32 * i, N);
    }
    Four<T> k4[CH], q4[CH];
    T v1[RPL];
    float g1 = 0.f, b1 = 0.f;
    const auto load = [&](int t) {
        const size_t tok = b * L + t;
        const T *vp = static_cast<const T *>(a.v) + tok * a.vs + h * P;
        const T *kp = static_cast<const T *>(a.k) + tok * a.ks + kg * N;
        const T *qp = static_cast<const T *>(a.q) + tok * a.qs + kg * N;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            k4[i] = load4<VEC>(kp, n0 + 32 * i, N);
            q4[i] = load4<VEC>(qp, n0 + 32 * i, N);
        }
#pragma unroll
        for (int j = 0; j < RPL; ++j) v1[j] = vp[row[j]];
        g1 = a.g[tok * a.heads + h];
        b1 = a.beta[tok * a.heads + h];
    };
    if (len > 0) load(0);
#pragma unroll
    for (int j = 0; j < RPL; ++j)
#pragma unroll
        for (int i = 0; i < CH; ++i) S[j][i] = s_in ? wide4(s4[j][i], n0 + 32 * i < N) : f32x4{0.f, 0.f, 0.f, 0.f};
    T *yp = static_cast<T *>(a.y) + (b * L * a.heads + h) * P;
    for (int t = 0; t < len; ++t) {
        f32x4 k[CH], q[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            k[i] = wide4(k4[i], n0 + 32 * i < N);
            q[i] = wide4(q4[i], n0 + 32 * i < N);
        }
        const float alpha = expf(clamp_decay(g1)), beta = b1;
        float v[RPL];
#pragma unroll
        for (int j = 0; j < RPL; ++j) v[j] = ldf(&v1[j]);
        if (t + 1 < len) load(t + 1);
        float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            kk += dot4(k[i], k[i]);
            qq += dot4(q[i], q[i]);
            kq += dot4(k[i], q[i]);
        }
        // raw k and q stay as they are: their lengths multiply the sums
        const float rk = a.qk_norm ? 1.0f / sqrtf(eight_sum(kk) + kUnitEps) : 1.0f;
        const float rq = a.scale * (a.qk_norm ? 1.0f / sqrtf(eight_sum(qq) + kUnitEps) : 1.0f);
        kq = eight_sum(kq) * rk;
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
            float sk = 0.f, sq = 0.f;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                S[j][i] *= alpha;
                sk += dot4(S[j][i], k[i]);
                sq += dot4(S[j][i], q[i]);
            }
            const float u = beta * (v[j] - rk * eight_sum(sk));
            const float y = rq * (eight_sum(sq) + u * kq);
            const float uk = u * rk;
#pragma unroll
            for (int i = 0; i < CH; ++i) S[j][i] += uk * k[i];
            const int r = row0 + j * NG;
            if (lane == 0 && r < P) stf(yp + static_cast<size_t>(t) * a.heads * P + r, y);
        }
    }
    for (int t = len; t < L; ++t)
        for (int j = 0; j < RPL; ++j) {
            const int r = row0 + j * NG;
            if (lane == 0 && r < P) stf(yp + static_cast<size_t>(t) * a.heads * P + r, 0.f);
        }
    // an unchanged state in place is not written
    if (a.state_out == nullptr || (len == 0 && a.state_out == a.state)) return;
    float *s_out = a.state_out + bh * P * N;
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const int r = row0 + j * NG;
        if (r >= P) continue;
        float *to = s_out + static_cast<size_t>(r) * N;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int n = n0 + 32 * i;
            if constexpr (VEC) {
                if (n < N) *reinterpret_cast<f32x4 *>(to + n) = S[j][i];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < N) to[n + e] = S[j][i][e];
            }
        }
    }
}

// One thread a (row, head): a few bytes each, bound by the launch.
template <typename T>
__global__ void __launch_bounds__(256)
delta_gates_kernel(size_t n, size_t heads, const T *pa, const T *pb, size_t stride, const float *a_log,
                   const float *dt_bias, float *g, float *beta) {
    const size_t i = blockIdx.x * size_t(256) + threadIdx.x;
    if (i >= n) return;
    const size_t row = i / heads, h = i % heads;
    const float x = ldf(pa + row * stride + h) + (dt_bias ? dt_bias[h] : 0.f);
    // softplus: x + log(1 + exp(-x)) where exp(x) could overflow
    const float sp = (x > 0.f ? x : 0.f) + log1pf(expf(-fabsf(x)));
    g[i] = -expf(a_log[h]) * sp;
    beta[i] = 1.0f / (1.0f + expf(-ldf(pb + row * stride + h)));
}

template <typename T, int CH, int RPL, int TH>
hipError_t go(const DeltaLaunch &a, hipStream_t s) {
    const auto ok = [](const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    const bool vec = a.d_state % 4 == 0 && ok(a.state, 16) && ok(a.state_out, 16) && ok(a.q, 4 * sizeof(T)) &&
                     ok(a.k, 4 * sizeof(T)) && a.qs % 4 == 0 && a.ks % 4 == 0;
    constexpr unsigned rows = TH / 8 * RPL;
    const dim3 grid(static_cast<unsigned>(a.batch * a.heads),
                    static_cast<unsigned>((a.head_dim + rows - 1) / rows));
    if (vec)
        hipLaunchKernelGGL((delta_recur_kernel<T, CH, RPL, TH, true>), grid, dim3(TH), 0, s, a);
    else
        hipLaunchKernelGGL((delta_recur_kernel<T, CH, RPL, TH, false>), grid, dim3(TH), 0, s, a);
    return hipGetLastError();
}

template <typename T, int CH>
hipError_t by_rows(const DeltaLaunch &a, hipStream_t s) {
    // many rows: two a group of lanes; few: a wave each, so that they reach
    // every CU
    if (a.batch * a.heads * a.head_dim >= 32768) return go<T, CH, 2, 256>(a, s);
    return go<T, CH, 1, 64>(a, s);
}

}  // namespace

hipError_t launch_delta_gates(size_t rows, size_t heads, int dtype, const void *pa, const void *pb, size_t stride,
                              const float *a_log, const float *dt_bias, float *g, float *beta, hipStream_t s) {
    const size_t n = rows * heads;
    if (n == 0) return hipSuccess;
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(delta_gates_kernel<T>, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, n,
                           heads, static_cast<const T *>(pa), static_cast<const T *>(pb), stride, a_log, dt_bias, g,
                           beta);
        return hipGetLastError();
    });
}

hipError_t launch_delta_recur(const DeltaLaunch &a, hipStream_t s) {
    if (a.batch == 0) return hipSuccess;
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.d_state <= 32) return by_rows<T, 1>(a, s);
        if (a.d_state <= 64) return by_rows<T, 2>(a, s);
        if (a.d_state <= 128) return by_rows<T, 4>(a, s);
        return by_rows<T, 8>(a, s);
    });
}

}  // namespace m3
