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
//
// 32768 rows of 768 (bf16, residual f32): 352 MB in 69 us, 5.1 TB/s.  16384 rows of
// 1536 (bf16): 252 MB in 50 us; the gradient 403 MB and 19 MB of partial sums in 104 us
// (3.9 TB/s) and 5 more to add those: its vector instructions are the nearer bound, 80 %
// of the issue slots.
#include "delta.hpp"
#include "m3_internal.hpp"
#include "scan_common.hpp"

namespace m3 {
namespace {

using namespace delta;

constexpr int E = 8;

// Eight values as loaded.
template <typename T> struct Raw8 { u32x4 q; };
template <> struct Raw8<float> { f32x4 a, b; };
__device__ __forceinline__ void wide(const Raw8<float> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = r.a[i];
        f[4 + i] = r.b[i];
    }
}
__device__ __forceinline__ void wide(const Raw8<bf16_t> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(r.q[i] << 16);
        f[2 * i + 1] = __uint_as_float(r.q[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void wide(const Raw8<f16_t> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.q[i])));
        f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.q[i] >> 16)));
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
// Without a branch where the loads are whole pieces: a thread past the row reads
// its start, and `wide_row` puts zeros there.
template <bool VEC, int NT, typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T *row, int tid, int c, int dim) {
    Raw8<T> r;
    if constexpr (VEC) {
        const int i = at<true, NT>(tid, c, 0), k = i < dim ? i : 0;
        if constexpr (sizeof(T) == 4) {
            r.a = *reinterpret_cast<const f32x4 *>(row + k);
            r.b = *reinterpret_cast<const f32x4 *>(row + k + 4);
        } else {
            r.q = *reinterpret_cast<const u32x4 *>(row + k);
        }
    } else {
        uint32_t u[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = at<false, NT>(tid, c, e);
            const T x = row[i < dim ? i : 0];
            u[e] = sizeof(T) == 4 ? __builtin_bit_cast(uint32_t, ldf(&x)) : *reinterpret_cast<const uint16_t *>(&x);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r.a[e] = __uint_as_float(u[e]);
                r.b[e] = __uint_as_float(u[4 + e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) r.q[e] = u[2 * e] | u[2 * e + 1] << 16;
        }
    }
    return r;
}
template <bool VEC, int NT, typename T>
__device__ __forceinline__ void wide_row(const Raw8<T> &r, int tid, int c, int dim, float *f) {
    wide(r, f);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (at<VEC, NT>(tid, c, e) >= dim) f[e] = 0.f;
}
template <bool VEC, int NT, typename T>
__device__ __forceinline__ void load(const T *row, int tid, int c, int dim, float *f) {
    wide_row<VEC, NT>(load_raw<VEC, NT>(row, tid, c, dim), tid, c, dim, f);
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

// act(z) and its derivative, from one exponential and one reciprocal (v_rcp_f32,
// within one unit in the last place).
enum { kNone = 0, kSilu = 1, kSigmoid = 2 };
__device__ __forceinline__ float act_of(int act, float z, float &d) {
    if (act == kNone) {
        d = 1.0f;
        return z;
    }
    const float s = __builtin_amdgcn_rcpf(1.0f + expf(-z));
    if (act == kSigmoid) {
        d = s * (1.0f - s);
        return s;
    }
    d = s * (1.0f + z * (1.0f - s));
    return z * s;
}

// Sums of K values over the NT threads of a row; `red` is [K][NT / 64], its
// own for each call site, so that one barrier a sum is enough as long as
// another call's stands between two uses.  Loads on their way stay so.
template <int NT, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float *red, int tid) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(seg_scan<64>(v[k])), 63));
    if constexpr (NT > 64) {
        if ((tid & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) red[k * (NT / 64) + (tid >> 6)] = v[k];
        scan::lds_barrier();
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
    __shared__ float red[2][NT / 64];   // a row of more than a wave is the workgroup's
    const int tid = threadIdx.x % NT, sub = threadIdx.x / NT;
    const size_t row = static_cast<size_t>(blockIdx.x) * RPW + sub;
    if (RPW > 1 && row >= a.rows) return;   // no barrier there
    const int dim = static_cast<int>(a.dim);
    const float inv = 1.0f / static_cast<float>(a.dim);
    // every load of the row, and of the weights, on its way at once
    Raw8<T> x8[NC], z8[NC];
    Raw8<RT> r8[NC];
    Raw8<float> w8[NC], s8[NC], p8[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        x8[c] = load_raw<VEC, NT>(static_cast<const T *>(a.x) + row * a.dim, tid, c, dim);
        r8[c] = load_raw<VEC, NT>(static_cast<const RT *>(a.residual) + row * a.dim, tid, c, dim);
        if (a.gate) z8[c] = load_raw<VEC, NT>(static_cast<const T *>(a.gate) + row * a.gate_stride, tid, c, dim);
        if (a.post_w) w8[c] = load_raw<VEC, NT>(a.post_w, tid, c, dim);
        if (a.scale) s8[c] = load_raw<VEC, NT>(a.scale, tid, c, dim);
        if (a.pre_w) p8[c] = load_raw<VEC, NT>(a.pre_w, tid, c, dim);
    }
    float x[NC][E], r[NC][E];
    float sx[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        wide_row<VEC, NT>(x8[c], tid, c, dim, x[c]);
#pragma unroll
        for (int e = 0; e < E; ++e) sx[0] += x[c][e] * x[c][e];
    }
    float rx = 1.0f;
    if (a.post_norm) {
        row_sum<NT>(sx, red[0], tid);
        rx = 1.0f / sqrtf(sx[0] * inv + a.eps);
    }
    float sr[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float f[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[c][e] *= rx;
        if (a.post_w) {
            wide(w8[c], f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= f[e];
        }
        if (a.gate) {
            wide(z8[c], f);
            float unused;
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= act_of(a.act, f[e], unused);
        }
        if (a.scale) {
            wide(s8[c], f);
#pragma unroll
            for (int e = 0; e < E; ++e) x[c][e] *= f[e];
        }
        wide(r8[c], r[c]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r[c][e] += x[c][e];
            sr[0] += at<VEC, NT>(tid, c, e) < dim ? r[c][e] * r[c][e] : 0.f;
        }
        store<VEC, NT>(static_cast<RT *>(a.residual_out) + row * a.dim, tid, c, dim, r[c]);
    }
    if (a.y == nullptr) return;
    row_sum<NT>(sr, red[1], tid);
    const float rho = 1.0f / sqrtf(sr[0] * inv + a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int e = 0; e < E; ++e) r[c][e] *= rho;
        if (a.pre_w) {
            float f[E];
            wide(p8[c], f);
#pragma unroll
            for (int e = 0; e < E; ++e) r[c][e] *= f[e];
        }
        store<VEC, NT>(static_cast<T *>(a.y) + row * a.dim, tid, c, dim, r[c]);
    }
}

// Gradients.  Workgroup i takes rows i, i + grid, ..., the next one's loads on
// their way during this one's sums; the weights and the column sums of their
// gradients stay in its registers (the sums go to partials[i][3][dim] at the
// end).
template <typename T, typename RT, int NT, int NC, bool VEC>
__global__ void __launch_bounds__(NT) block_norm_backward_kernel(BlockNormLaunch a, BlockNormGrads g, float *partials) {
    __shared__ float red[4][NT / 64];
    const int tid = threadIdx.x, dim = static_cast<int>(a.dim);
    const float inv = 1.0f / static_cast<float>(a.dim);
    float spost[NC][E], sscale[NC][E], spre[NC][E], w[NC][E], sc[NC][E], pw[NC][E];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            spost[c][e] = sscale[c][e] = spre[c][e] = 0.f;
            w[c][e] = sc[c][e] = pw[c][e] = 1.f;
        }
        if (a.post_w) load<VEC, NT>(a.post_w, tid, c, dim, w[c]);
        if (a.scale) load<VEC, NT>(a.scale, tid, c, dim, sc[c]);
        if (a.pre_w) load<VEC, NT>(a.pre_w, tid, c, dim, pw[c]);
    }
    Raw8<T> rx8[NC], rz8[NC], ry8[NC];
    Raw8<RT> rr8[NC], rd8[NC];
    const auto fetch = [&](size_t row) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            rx8[c] = load_raw<VEC, NT>(static_cast<const T *>(a.x) + row * a.dim, tid, c, dim);
            rr8[c] = load_raw<VEC, NT>(static_cast<const RT *>(a.residual) + row * a.dim, tid, c, dim);
            if (a.gate) rz8[c] = load_raw<VEC, NT>(static_cast<const T *>(a.gate) + row * a.gate_stride, tid, c, dim);
            if (g.dy) ry8[c] = load_raw<VEC, NT>(static_cast<const T *>(g.dy) + row * a.dim, tid, c, dim);
            if (g.dres) rd8[c] = load_raw<VEC, NT>(static_cast<const RT *>(g.dres) + row * a.dim, tid, c, dim);
        }
    };
    if (blockIdx.x < a.rows) fetch(blockIdx.x);
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float x[NC][E], r[NC][E], dy[NC][E], d[NC][E];
        float av[NC][E], dav[NC][E];   // the gate and its derivative
        float s1[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            wide_row<VEC, NT>(rx8[c], tid, c, dim, x[c]);
            wide_row<VEC, NT>(rr8[c], tid, c, dim, r[c]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dy[c][e] = d[c][e] = dav[c][e] = 0.f;
                av[c][e] = 1.f;
            }
            if (a.gate) {
                float z[E];
                wide_row<VEC, NT>(rz8[c], tid, c, dim, z);
#pragma unroll
                for (int e = 0; e < E; ++e) av[c][e] = act_of(a.act, z[e], dav[c][e]);
            }
            if (g.dy) wide_row<VEC, NT>(ry8[c], tid, c, dim, dy[c]);
            if (g.dres) wide_row<VEC, NT>(rd8[c], tid, c, dim, d[c]);
#pragma unroll
            for (int e = 0; e < E; ++e) s1[0] += x[c][e] * x[c][e];
        }
        if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
        float rx = 1.0f;
        if (a.post_norm) {
            row_sum<NT>(s1, red[0], tid);
            rx = 1.0f / sqrtf(s1[0] * inv + a.eps);
        }
        float s2[2] = {0.f, 0.f};
        float rho = 0.f, back = 0.f;
        if (g.dy) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    r[c][e] += x[c][e] * rx * w[c][e] * av[c][e] * sc[c][e];
                    s2[0] += r[c][e] * r[c][e];
                    s2[1] += dy[c][e] * pw[c][e] * r[c][e];
                }
            row_sum<NT>(s2, red[1], tid);
            rho = 1.0f / sqrtf(s2[0] * inv + a.eps);
            back = s2[1] * inv * rho * rho * rho;
        }
        float s3[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float dz[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (g.dy) {
                    spre[c][e] += dy[c][e] * r[c][e] * rho;
                    d[c][e] += rho * dy[c][e] * pw[c][e] - r[c][e] * back;
                }
                const float n = x[c][e] * rx * w[c][e];
                sscale[c][e] += av[c][e] * n * d[c][e];
                const float m = sc[c][e] * av[c][e] * d[c][e];
                dz[e] = sc[c][e] * n * d[c][e] * dav[c][e];
                spost[c][e] += m * x[c][e] * rx;
                r[c][e] = m * w[c][e];   // r is done with
                s3[0] += r[c][e] * x[c][e];
            }
            store<VEC, NT>(static_cast<RT *>(g.dresidual) + row * a.dim, tid, c, dim, d[c]);
            if (a.gate) store<VEC, NT>(static_cast<T *>(g.dgate) + row * a.dim, tid, c, dim, dz);
        }
        float mean = 0.f;
        if (a.post_norm) {
            row_sum<NT>(s3, red[3], tid);
            mean = s3[0] * inv * rx * rx;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int e = 0; e < E; ++e) r[c][e] = rx * (r[c][e] - x[c][e] * mean);
            store<VEC, NT>(static_cast<T *>(g.dx) + row * a.dim, tid, c, dim, r[c]);
        }
        // without a norm on either side of the add the loop has one sum or none
        if (!(a.post_norm && g.dy)) scan::lds_barrier();
    }
    float *p = partials + static_cast<size_t>(blockIdx.x) * 3 * a.dim;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        store<VEC, NT>(p, tid, c, dim, spost[c]);
        store<VEC, NT>(p + a.dim, tid, c, dim, sscale[c]);
        store<VEC, NT>(p + 2 * a.dim, tid, c, dim, spre[c]);
    }
}

// The partial sums of `parts` workgroups in a fixed order: 64 columns a
// workgroup, the parts dealt to its 16 waves, eight on their way at once.
__global__ void __launch_bounds__(1024) block_norm_columns(const float *partials, size_t parts, size_t dim, BlockNormGrads g) {
    __shared__ float red[16][64];
    const size_t all = 3 * dim, at = blockIdx.x * size_t(64) + (threadIdx.x & 63), col = at < all ? at : 0;
    const size_t q = threadIdx.x >> 6;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    size_t i = q;
    for (; i + 7 * 16 < parts; i += 8 * 16)
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += partials[(i + 16 * k) * all + col];
    for (; i < parts; i += 16) s[0] += partials[i * all + col];
    red[q][threadIdx.x & 63] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (q != 0 || at >= all) return;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][threadIdx.x];
    float *out = col < dim ? g.dpost_w : col < 2 * dim ? g.dscale : g.dpre_w;
    if (out) out[col % dim] = t;
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
            // one piece a thread as far as 2048 values: few enough registers for
            // three waves a SIMD
            using std::integral_constant;
            constexpr integral_constant<int, 1> one{};
            if (a.dim <= 512) return go(integral_constant<int, 64>{}, one);
            if (a.dim <= 1024) return go(integral_constant<int, 128>{}, one);
            if (a.dim <= 1536) return go(integral_constant<int, 192>{}, one);
            if (a.dim <= 8192) return by_pieces<256>(a.dim, go);
            return by_pieces<1024>(a.dim, go);
        });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(block_norm_columns, dim3(static_cast<unsigned>((3 * a.dim + 63) / 64)), dim3(1024), 0, s,
                       partials, static_cast<size_t>(grid), a.dim, g);
    return hipGetLastError();
}

}  // namespace m3
