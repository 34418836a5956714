// What stands between two blocks of a residual stack, in one pass (gfx950):
// the norm after a block with its gate and residual scale, the residual add,
// and the norm before the next block.
//   n = post_w x rsqrt(mean x^2 + eps)   (or x)
//   r' = r + scale act(gate) n
//   y = pre_w r' rsqrt(mean r'^2 + eps)
// and the gradients of it.  HBM-bound both ways: each row is read once into
// registers, its sums are taken over the lanes that hold it, and it is written
// once; all arithmetic is f32, and y follows from the r' in registers, not from
// its rounding to the residual's type.
//
// A thread holds E = 8 values of a row per piece.  Which eight is free, as every
// step is a sum over the row or elementwise: 16-byte pieces where the rows allow
// it (VEC), else values a stride apart, so that a wave's scalar loads are
// contiguous.
#include "delta.hpp"
#include "m3_internal.hpp"

namespace m3 {
namespace {

using namespace delta;

constexpr int E = 8;

template <typename T> struct Raw8 {
    uint4 q;
    __device__ __forceinline__ void ld(const T *p) { q = *reinterpret_cast<const uint4 *>(p); }
};
template <> struct Raw8<float> {
    f32x4 a, b;
    __device__ __forceinline__ void ld(const float *p) {
        a = *reinterpret_cast<const f32x4 *>(p);
        b = *reinterpret_cast<const f32x4 *>(p + 4);
    }
};
__device__ __forceinline__ void wide(const Raw8<float> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = r.a[i];
        f[4 + i] = r.b[i];
    }
}
__device__ __forceinline__ void wide(const Raw8<bf16_t> &r, float *f) {
    const uint32_t u[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void wide(const Raw8<f16_t> &r, float *f) {
    const uint32_t u[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u[i])));
        f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u[i] >> 16)));
    }
}
__device__ __forceinline__ void store8(float *p, const float *f) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
}
__device__ __forceinline__ void store8(bf16_t *p, const float *f) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                               pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void store8(f16_t *p, const float *f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i]))) |
               static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i + 1]))) << 16;
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// The eight values of piece c of a row that thread `tid` of NT holds.
template <bool VEC, int NT>
__device__ __forceinline__ int at(int tid, int c, int e) {
    return VEC ? (c * NT + tid) * E + e : (c * E + e) * NT + tid;
}
template <bool VEC, int NT, typename T>
__device__ __forceinline__ void load(const T *row, int tid, int c, int dim, float pad, float *f) {
    if constexpr (VEC) {
        const int i = at<true, NT>(tid, c, 0);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = pad;
        if (i < dim) {
            Raw8<T> r;
            r.ld(row + i);
            wide(r, f);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = at<false, NT>(tid, c, e);
            f[e] = i < dim ? ldf(row + i) : pad;
        }
    }
}
template <bool VEC, int NT, typename T>
__device__ __forceinline__ void store(T *row, int tid, int c, int dim, const float *f) {
    if constexpr (VEC) {
        const int i = at<true, NT>(tid, c, 0);
        if (i < dim) store8(row + i, f);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = at<false, NT>(tid, c, e);
            if (i < dim) stf(row + i, f[e]);
        }
    }
}

// act(z) and, with D, its derivative.
enum { kNone = 0, kSilu = 1, kSigmoid = 2 };
__device__ __forceinline__ float act_of(int act, float z) {
    if (act == kNone) return z;
    const float s = 1.0f / (1.0f + expf(-z));
    return act == kSilu ? z * s : s;
}
__device__ __forceinline__ float dact_of(int act, float z) {
    if (act == kNone) return 1.0f;
    const float s = 1.0f / (1.0f + expf(-z));
    return act == kSilu ? s * (1.0f + z * (1.0f - s)) : s * (1.0f - s);
}

// Sums of K values over the NT threads of a row; `red` is this row's own
// [K][NT / 64] and used once per call site.
template <int NT, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float *red, int tid) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = group_sum(v[k], 64);
    if constexpr (NT > 64) {
        __syncthreads();
        if ((tid & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) red[k * (NT / 64) + (tid >> 6)] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) s += red[k * (NT / 64) + i];
            v[k] = s;
        }
    }
}

// A row on NT threads, NC pieces; waves of a workgroup take rows of their own
// where a row is one wave's.
template <typename T, typename RT, int NT, int NC, bool VEC>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) block_norm_kernel(BlockNormLaunch a) {
    constexpr int RPW = NT < 256 ? 256 / NT : 1;
    __shared__ float red[NT > 64 ? RPW * (NT / 64) : 1];
    const int tid = threadIdx.x % NT, sub = threadIdx.x / NT;
    const size_t row = static_cast<size_t>(blockIdx.x) * RPW + sub;
    const bool live = row < a.rows;   // every thread meets the barriers
    const int dim = live ? static_cast<int>(a.dim) : 0;
    const float inv = 1.0f / static_cast<float>(a.dim);
    float x[NC][E], r[NC][E];
    float sx[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        load<VEC, NT>(static_cast<const T *>(a.x) + row * a.dim, tid, c, dim, 0.f, x[c]);
#pragma unroll
        for (int e = 0; e < E; ++e) sx[0] += x[c][e] * x[c][e];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
        load<VEC, NT>(static_cast<const RT *>(a.residual) + row * a.dim, tid, c, dim, 0.f, r[c]);
    float rx = 1.0f;
    if (a.post_norm) {
        row_sum<NT>(sx, red + sub * (NT / 64), tid);
        rx = 1.0f / sqrtf(sx[0] * inv + a.eps);
    }
    float sr[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float f[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[c][e] *= rx;
        if (a.post_w) {
            load<VEC, NT>(a.post_w, tid, c, dim, 0.f, f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= f[e];
        }
        if (a.gate) {
            load<VEC, NT>(static_cast<const T *>(a.gate) + row * a.gate_stride, tid, c, dim, 0.f, f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= act_of(a.act, f[e]);
        }
        if (a.scale) {
            load<VEC, NT>(a.scale, tid, c, dim, 0.f, f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r[c][e] += x[c][e];
            sr[0] += r[c][e] * r[c][e];
        }
        store<VEC, NT>(static_cast<RT *>(a.residual_out) + row * a.dim, tid, c, dim, r[c]);
    }
    if (a.y == nullptr) return;
    row_sum<NT>(sr, red + sub * (NT / 64), tid);
    const float rho = 1.0f / sqrtf(sr[0] * inv + a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int e = 0; e < E; ++e) r[c][e] *= rho;
        if (a.pre_w) {
            float f[E];
            load<VEC, NT>(a.pre_w, tid, c, dim, 0.f, f);
#pragma unroll
            for (int e = 0; e < E; ++e) r[c][e] *= f[e];
        }
        store<VEC, NT>(static_cast<T *>(a.y) + row * a.dim, tid, c, dim, r[c]);
    }
}

// Gradients.  Workgroup i takes rows i, i + grid, ...; the column sums of the
// three weights stay in its registers and go to partials[i][3][dim] at the end.
template <typename T, typename RT, int NT, int NC, bool VEC>
__global__ void __launch_bounds__(NT) block_norm_backward_kernel(BlockNormLaunch a, BlockNormGrads g, float *partials) {
    __shared__ float red[2 * (NT / 64)];
    const int tid = threadIdx.x, dim = static_cast<int>(a.dim);
    const float inv = 1.0f / static_cast<float>(a.dim);
    float spost[NC][E], sscale[NC][E], spre[NC][E];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) spost[c][e] = sscale[c][e] = spre[c][e] = 0.f;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float x[NC][E], r[NC][E], z[NC][E], dy[NC][E];
        float s1[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load<VEC, NT>(static_cast<const T *>(a.x) + row * a.dim, tid, c, dim, 0.f, x[c]);
            load<VEC, NT>(static_cast<const RT *>(a.residual) + row * a.dim, tid, c, dim, 0.f, r[c]);
            if (a.gate) load<VEC, NT>(static_cast<const T *>(a.gate) + row * a.gate_stride, tid, c, dim, 0.f, z[c]);
            if (g.dy) load<VEC, NT>(static_cast<const T *>(g.dy) + row * a.dim, tid, c, dim, 0.f, dy[c]);
#pragma unroll
            for (int e = 0; e < E; ++e) s1[0] += x[c][e] * x[c][e];
        }
        float rx = 1.0f;
        if (a.post_norm) {
            row_sum<NT>(s1, red, tid);
            rx = 1.0f / sqrtf(s1[0] * inv + a.eps);
        }
        float s2[2] = {0.f, 0.f};
        float rho = 0.f, back = 0.f;
        if (g.dy) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float w[E], sc[E], pw[E];
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] = sc[e] = pw[e] = 1.f;
                if (a.post_w) load<VEC, NT>(a.post_w, tid, c, dim, 0.f, w);
                if (a.scale) load<VEC, NT>(a.scale, tid, c, dim, 0.f, sc);
                if (a.pre_w) load<VEC, NT>(a.pre_w, tid, c, dim, 0.f, pw);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    r[c][e] += x[c][e] * rx * w[e] * (a.gate ? act_of(a.act, z[c][e]) : 1.f) * sc[e];
                    s2[0] += r[c][e] * r[c][e];
                    s2[1] += dy[c][e] * pw[e] * r[c][e];
                }
            }
            row_sum<NT>(s2, red, tid);
            rho = 1.0f / sqrtf(s2[0] * inv + a.eps);
            back = s2[1] * inv * rho * rho * rho;
        }
        float s3[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float d[E], w[E], sc[E], pw[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                w[e] = sc[e] = pw[e] = 1.f;
                d[e] = 0.f;
            }
            if (g.dres) load<VEC, NT>(static_cast<const RT *>(g.dres) + row * a.dim, tid, c, dim, 0.f, d);
            if (a.post_w) load<VEC, NT>(a.post_w, tid, c, dim, 0.f, w);
            if (a.scale) load<VEC, NT>(a.scale, tid, c, dim, 0.f, sc);
            if (a.pre_w) load<VEC, NT>(a.pre_w, tid, c, dim, 0.f, pw);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (g.dy) {
                    spre[c][e] += dy[c][e] * r[c][e] * rho;
                    d[e] += rho * dy[c][e] * pw[e] - r[c][e] * back;
                }
            }
            store<VEC, NT>(static_cast<RT *>(g.dresidual) + row * a.dim, tid, c, dim, d);
            float dz[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float av = a.gate ? act_of(a.act, z[c][e]) : 1.f, n = x[c][e] * rx * w[e];
                sscale[c][e] += av * n * d[e];
                const float m = sc[e] * av * d[e];
                dz[e] = a.gate ? sc[e] * n * d[e] * dact_of(a.act, z[c][e]) : 0.f;
                spost[c][e] += m * x[c][e] * rx;
                r[c][e] = m * w[e];   // r is done with
                s3[0] += r[c][e] * x[c][e];
            }
            if (a.gate) store<VEC, NT>(static_cast<T *>(g.dgate) + row * a.dim, tid, c, dim, dz);
        }
        float mean = 0.f;
        if (a.post_norm) {
            row_sum<NT>(s3, red, tid);
            mean = s3[0] * inv * rx * rx;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int e = 0; e < E; ++e) r[c][e] = rx * (r[c][e] - x[c][e] * mean);
            store<VEC, NT>(static_cast<T *>(g.dx) + row * a.dim, tid, c, dim, r[c]);
        }
    }
    float *p = partials + static_cast<size_t>(blockIdx.x) * 3 * a.dim;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        store<VEC, NT>(p, tid, c, dim, spost[c]);
        store<VEC, NT>(p + a.dim, tid, c, dim, sscale[c]);
        store<VEC, NT>(p + 2 * a.dim, tid, c, dim, spre[c]);
    }
}

// The partial sums of `parts` workgroups, in their order: one column a thread of
// a row of 64, the parts dealt to four rows of threads.
__global__ void __launch_bounds__(256) block_norm_columns(const float *partials, size_t parts, size_t dim, BlockNormGrads g) {
    __shared__ float red[4][64];
    const size_t col = blockIdx.x * size_t(64) + (threadIdx.x & 63);
    const int q = threadIdx.x >> 6;
    const size_t all = 3 * dim;
    float s = 0.f;
    if (col < all)
        for (size_t i = q; i < parts; i += 4) s += partials[i * all + col];
    red[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q != 0 || col >= all) return;
    s = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
    float *out = col < dim ? g.dpost_w : col < 2 * dim ? g.dscale : g.dpre_w;
    if (out) out[col % dim] = s;
}

template <typename F>
hipError_t by_types(const BlockNormLaunch &a, F f) {
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return a.residual_dtype == a.dtype ? f(T{}, T{}) : f(T{}, float{});
    });
}

// f(threads of a row, pieces): up to 2048 values a row is one wave's, past that a
// workgroup's.
template <int NT, typename F>
hipError_t by_pieces(size_t dim, F f) {
    constexpr size_t piece = NT * E;
    using std::integral_constant;
    if (dim <= piece) return f(integral_constant<int, NT>{}, integral_constant<int, 1>{});
    if (dim <= 2 * piece) return f(integral_constant<int, NT>{}, integral_constant<int, 2>{});
    if (dim <= 3 * piece) return f(integral_constant<int, NT>{}, integral_constant<int, 3>{});
    return f(integral_constant<int, NT>{}, integral_constant<int, 4>{});
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool vec_ok(const BlockNormLaunch &a) {
    return a.dim % E == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.residual_out) &&
           aligned16(a.y) && aligned16(a.gate) && a.gate_stride % E == 0 && aligned16(a.post_w) &&
           aligned16(a.scale) && aligned16(a.pre_w);
}

unsigned backward_grid(const BlockNormLaunch &a) {
    return static_cast<unsigned>(a.rows < 1024 ? a.rows : 1024);
}

}  // namespace

hipError_t launch_block_norm(const BlockNormLaunch &a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    const bool vec = vec_ok(a);
    return by_types(a, [&](auto t, auto rt) {
        using T = decltype(t);
        using RT = decltype(rt);
        const auto go = [&](auto nt, auto nc) {
            constexpr int NT = decltype(nt)::value, NC = decltype(nc)::value;
            constexpr unsigned rpw = NT < 256 ? 256 / NT : 1;
            const dim3 grid(static_cast<unsigned>((a.rows + rpw - 1) / rpw)), wg(rpw * NT);
            if (vec)
                hipLaunchKernelGGL((block_norm_kernel<T, RT, NT, NC, true>), grid, wg, 0, s, a);
            else
                hipLaunchKernelGGL((block_norm_kernel<T, RT, NT, NC, false>), grid, wg, 0, s, a);
            return hipGetLastError();
        };
        if (a.dim <= 2048) return by_pieces<64>(a.dim, go);
        if (a.dim <= 8192) return by_pieces<256>(a.dim, go);
        return by_pieces<1024>(a.dim, go);
    });
}

size_t block_norm_backward_workspace(const BlockNormLaunch &a) {
    return static_cast<size_t>(backward_grid(a)) * 3 * a.dim * sizeof(float);
}

hipError_t launch_block_norm_backward(const BlockNormLaunch &a, const BlockNormGrads &g, void *workspace,
                                      hipStream_t s) {
    const unsigned grid = backward_grid(a);
    float *partials = static_cast<float *>(workspace);
    const bool vec = vec_ok(a) && aligned16(g.dres) && aligned16(g.dy) && aligned16(g.dx) &&
                     aligned16(g.dresidual) && aligned16(g.dgate) && aligned16(workspace);
    hipError_t e = hipSuccess;
    if (grid > 0)
        e = by_types(a, [&](auto t, auto rt) {
            using T = decltype(t);
            using RT = decltype(rt);
            const auto go = [&](auto nt, auto nc) {
                constexpr int NT = decltype(nt)::value, NC = decltype(nc)::value;
                if (vec)
                    hipLaunchKernelGGL((block_norm_backward_kernel<T, RT, NT, NC, true>), dim3(grid), dim3(NT), 0,
                                       s, a, g, partials);
                else
                    hipLaunchKernelGGL((block_norm_backward_kernel<T, RT, NT, NC, false>), dim3(grid), dim3(NT), 0,
                                       s, a, g, partials);
                return hipGetLastError();
            };
            if (a.dim <= 8192) return by_pieces<256>(a.dim, go);
            return by_pieces<1024>(a.dim, go);
        });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(block_norm_columns, dim3(static_cast<unsigned>((3 * a.dim + 63) / 64)), dim3(256), 0, s,
                       partials, static_cast<size_t>(grid), a.dim, g);
    return hipGetLastError();
}

}  // namespace m3
