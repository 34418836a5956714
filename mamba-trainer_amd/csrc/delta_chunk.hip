// The gated delta rule over a window, chunk by chunk on the MFMA (gfx950); the
// mathematics, the numbers and the register layout are in delta_chunk.hpp.
#include "delta_chunk.hpp"

namespace m3 {
namespace {

using namespace delta;

// One workgroup a (sequence, head, chunk): the chunk's row factors, T and the
// attention within the chunk.
template <typename T, int N, bool VEC>
__global__ void __launch_bounds__(256) delta_prep(DeltaLaunch a, unsigned char *records, int chunks) {
    constexpr int KP = Parts<T>::in, LP = kC + 4;
    using R = Record<T>;
    __shared__ double G[kC];
    __shared__ float beta[kC], rq[kC], rk[kC];
    __shared__ __attribute__((aligned(16))) float A[kC][LP], X[kC][LP];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const size_t rec = blockIdx.x, bh = rec / chunks, b = bh / a.heads, h = bh % a.heads;
    const int t0 = static_cast<int>(rec % chunks) * kC;
    const int L = static_cast<int>(a.seq), live = valid_len(a.lengths, b, L) - t0;   // of this chunk
    if (live <= 0) return;
    const size_t kg = h / (a.heads / a.groups);
    const int n_of = static_cast<int>(a.d_state);
    const Rows<T, VEC> kp(static_cast<const T *>(a.k) + (b * L + t0) * a.ks + kg * n_of, a.ks, live, n_of);
    const Rows<T, VEC> qp(static_cast<const T *>(a.q) + (b * L + t0) * a.qs + kg * n_of, a.qs, live, n_of);
    if (w == 0) {
        const size_t th = (b * L + t0 + lane) * a.heads + h;
        double s = 0.0;
        float bt = 0.f;
        if (lane < live) {
            s = clamp_decay(a.g[th]);
            bt = a.beta[th];
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(s, off, 64);
            if (lane >= off) s += o;
        }
        G[lane] = s;
        beta[lane] = bt;
    }
    // Q and K rows of this wave's 16 tokens as operands, their lengths
    bf16x8 qa[N / 32][KP], ka[N / 32][KP];
    const int my = 16 * w + c;
    float sq = 0.f, sk = 0.f;
#pragma unroll
    for (int kk = 0; kk < N / 32; ++kk) {
        const Eight<T> q8 = load_eight(qp, my, 32 * kk + 8 * g);
        const Eight<T> k8 = load_eight(kp, my, 32 * kk + 8 * g);
        float f[8];
        widen(q8, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += f[i] * f[i];
        widen(k8, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sk += f[i] * f[i];
        to_parts(q8, qa[kk]);
        to_parts(k8, ka[kk]);
    }
    sq += __shfl_xor(sq, 16, 64);
    sk += __shfl_xor(sk, 16, 64);
    sq += __shfl_xor(sq, 32, 64);
    sk += __shfl_xor(sk, 32, 64);
    if (g == 0) {
        rq[my] = a.scale * (a.qk_norm ? 1.0f / sqrtf(sq + kUnitEps) : 1.0f);
        rk[my] = a.qk_norm ? 1.0f / sqrtf(sk + kUnitEps) : 1.0f;
    }
    // tiles j <= w of K K^T and Q K^T
    f32x4 kkt[4], qkt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kkt[j] = qkt[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (j > w) continue;
        const int row = 16 * j + c;
#pragma unroll
        for (int kk = 0; kk < N / 32; ++kk) {
            bf16x8 kb[KP];
            to_parts(load_eight(kp, row, 32 * kk + 8 * g), kb);
            kkt[j] = mma_parts<KP, KP>(ka[kk], kb, kkt[j]);
            qkt[j] = mma_parts<KP, KP>(qa[kk], kb, qkt[j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * w + 4 * g + r, jj = 16 * j + c;
            float m = 0.f, p = 0.f;
            if (jj <= i) {
                const float d = expf(static_cast<float>(G[i] - G[jj])) * rk[jj] * beta[jj];
                p = d * rq[i] * qkt[j][r];
                if (jj < i) m = d * rk[i] * kkt[j][r];
            }
            A[i][jj] = m;
            X[i][jj] = p;
        }
    unsigned char *out = records + rec * R::bytes;
    if (w == 0) {
        float *f = reinterpret_cast<float *>(out);
        const float eg = expf(static_cast<float>(G[lane]));
        f[R::kK + lane] = eg * rk[lane];
        f[R::kQ + lane] = eg * rq[lane];
        f[R::kU + lane] = beta[lane] * expf(static_cast<float>(G[kC - 1] - G[lane])) * rk[lane];
        if (lane == 0) f[R::kEnd] = expf(static_cast<float>(G[kC - 1]));
    }
    __syncthreads();
    // a triangle of X or A as operand blocks: wave w writes those of rows 16 w
    const auto emit = [&](const float(*src)[LP], unsigned char *dst, auto parts) {
        constexpr int NP = decltype(parts)::value;
        for (int kk = 0; kk < lower_steps(w); ++kk) {
            float x[8];
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(&src[my][32 * kk + 4 * g]);
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(&src[my][32 * kk + 16 + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = lo[i];
                x[4 + i] = hi[i];
            }
            bf16x8 o[NP];
            split8<NP>(x, o);
#pragma unroll
            for (int p = 0; p < NP; ++p)
                *reinterpret_cast<bf16x8 *>(dst + ((lower_block(w, kk) * NP + p) * 64 + lane) * 16) = o[p];
        }
    };
    emit(X, out + R::p_at, std::integral_constant<int, Parts<T>::out>{});
    // T = (I + A)^-1.  The diagonal blocks by substitution, wave w block w, a
    // column a lane (the four lane groups alike)
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == c ? 1.0f : 0.0f;
#pragma unroll
            for (int l = 0; l < i; ++l) s -= A[16 * w + i][16 * w + l] * x[l];
            x[i] = s;
        }
        __syncthreads();   // X has been emitted
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((i >> 2) == g) X[16 * w + i][16 * w + c] = x[i];
    }
    // the rest block column by block column: T_ij = -T_ii sum_l A_il T_lj, the
    // products in f32 (MFMA 16x16x4, k-step r takes rows 4g + r)
    __syncthreads();
    if (w < 3) {
        f32x4 t[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) t[0][r] = X[16 * w + 4 * g + r][16 * w + c];
#pragma unroll
        for (int d = 1; d < 4; ++d) {
            if (w + d > 3) break;
            const int i = w + d;
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int l = 0; l < d; ++l) {
                const f32x4 av = *reinterpret_cast<const f32x4 *>(&A[16 * i + c][16 * (w + l) + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) s = mfma_f32(av[r], t[l][r], s);
            }
            const f32x4 tv = *reinterpret_cast<const f32x4 *>(&X[16 * i + c][16 * i + 4 * g]);
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) o = mfma_f32(-tv[r], s[r], o);
            t[d] = o;
        }
#pragma unroll
        for (int d = 1; d < 4; ++d)
            if (w + d <= 3)
#pragma unroll
                for (int r = 0; r < 4; ++r) X[16 * (w + d) + 4 * g + r][16 * w + c] = t[d][r];
    }
    // above the diagonal T is zero where a block row's operands reach past it
    if (w < 4) {
        const int j = w ^ 1;   // the other half of this row's last block pair
        if (j > w)
#pragma unroll
            for (int r = 0; r < 4; ++r) X[16 * w + 4 * g + r][16 * j + c] = 0.f;
    }
    __syncthreads();
    emit(X, out + R::t_at, std::integral_constant<int, kNP>{});
}

// One workgroup a (sequence, head, 64 columns of P), a wave 16 of them, the
// chunks in turn; the next chunk's operands are on their way to registers while
// this one's are multiplied.
template <typename T, int N, bool VEC>
__global__ void __launch_bounds__(256) delta_chunks(DeltaLaunch a, const unsigned char *records, int chunks) {
    constexpr int KP = Parts<T>::in, YP = Parts<T>::out, KS = N / 32, NT = N / 16;
    using R = Record<T>;
    constexpr int pieces = kC * N / 8 / 256, rpieces = (R::bytes / 16 + 255) / 256;
    __shared__ __attribute__((aligned(16))) __bf16 sk[KP * Tile<N>::size], sq[KP * Tile<N>::size];
    __shared__ __attribute__((aligned(16))) unsigned char sr[R::bytes];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const size_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, kg = h / (a.heads / a.groups);
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    const int n_of = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const int p = blockIdx.y * 64 + 16 * w + c;      // this lane's column
    const T *kp = static_cast<const T *>(a.k) + b * L * a.ks + kg * n_of;
    const T *qp = static_cast<const T *>(a.q) + b * L * a.qs + kg * n_of;
    const T *vp = static_cast<const T *>(a.v) + b * L * a.vs + h * P;
    T *yp = static_cast<T *>(a.y) + (b * L * a.heads + h) * P + p;
    const size_t ystep = a.heads * P;
    f32x4 S[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = 16 * nt + 4 * g + r;
            S[nt][r] = a.state && p < P && n < n_of ? a.state[(bh * P + p) * n_of + n] : 0.f;
        }
    const int live = (len + kC - 1) / kC;
    Eight<T> k8[pieces], q8[pieces];
    u32x4 r8[rpieces];
    uint32_t v[4][4];
    const auto fetch = [&](int ck) {
        const size_t t0 = static_cast<size_t>(ck) * kC;
        const int left = len - ck * kC;
        const Rows<T, VEC> kr(kp + t0 * a.ks, a.ks, left, n_of), qr(qp + t0 * a.qs, a.qs, left, n_of);
        const Rows<T, VEC> vr(vp + t0 * a.vs, a.vs, left, P);
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            const int id = tid + 256 * i, t = id / (N / 8), n = id % (N / 8) * 8;
            k8[i] = load_eight(kr, t, n);
            q8[i] = load_eight(qr, t, n);
        }
        const rsrc_t rec = make_rsrc(records + (bh * chunks + ck) * R::bytes, R::bytes);
#pragma unroll
        for (int i = 0; i < rpieces; ++i) r8[i] = bld16(rec, (tid + 256 * i) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[i][r] = load_one(vr, 16 * i + 4 * g + r, p);
    };
    if (live > 0) fetch(0);
    for (int ck = 0; ck < live; ++ck) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            const int id = tid + 256 * i, t = id / (N / 8), n = id % (N / 8) * 8;
            bf16x8 x[KP];
            const auto put = [&](const Eight<T> &e, __bf16 *tile) {
                to_parts(e, x);
#pragma unroll
                for (int q = 0; q < KP; ++q) {
                    __bf16 *row = tile + q * Tile<N>::size + t * Tile<N>::pitch;
                    *reinterpret_cast<bf16x4 *>(row + slot(n)) = __builtin_shufflevector(x[q], x[q], 0, 1, 2, 3);
                    *reinterpret_cast<bf16x4 *>(row + slot(n + 4)) = __builtin_shufflevector(x[q], x[q], 4, 5, 6, 7);
                }
            };
            put(k8[i], sk);
            put(q8[i], sq);
        }
#pragma unroll
        for (int i = 0; i < rpieces; ++i)
            if (tid + 256 * i < static_cast<int>(R::bytes / 16)) reinterpret_cast<u32x4 *>(sr)[tid + 256 * i] = r8[i];
        f32x4 e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) e[i][r] = value_of<T>(v[i][r]);
        __syncthreads();
        if (ck + 1 < live) fetch(ck + 1);
        const float *fac = reinterpret_cast<const float *>(sr);
        f32x4 y[4];
        // R and the state's part of Y
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 ks[4] = {y[0], y[0], y[0], y[0]};
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            bf16x8 s[kNP];
            split_tiles<kNP>(S[2 * kk], S[2 * kk + 1], s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x8 x[KP];
#pragma unroll
                for (int q = 0; q < KP; ++q) x[q] = tile_rows<N>(sk + q * Tile<N>::size, i, kk, lane);
                ks[i] = mma_parts<KP, kNP>(x, s, ks[i]);
#pragma unroll
                for (int q = 0; q < KP; ++q) x[q] = tile_rows<N>(sq + q * Tile<N>::size, i, kk, lane);
                y[i] = mma_parts<KP, YP>(x, s, y[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 fk = *reinterpret_cast<const f32x4 *>(fac + R::kK + 16 * i + 4 * g);
            const f32x4 fq = *reinterpret_cast<const f32x4 *>(fac + R::kQ + 16 * i + 4 * g);
            e[i] -= fk * ks[i];
            y[i] *= fq;
        }
        // E = T R
        const auto tri = [&](size_t at, int np, int blk, int q) {
            return *reinterpret_cast<const bf16x8 *>(sr + at + ((blk * np + q) * 64 + lane) * 16);
        };
        bf16x8 x[2][kNP];
        split_tiles<kNP>(e[0], e[1], x[0]);
        split_tiles<kNP>(e[2], e[3], x[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < lower_steps(i); ++kk) {
                bf16x8 t[kNP];
#pragma unroll
                for (int q = 0; q < kNP; ++q) t[q] = tri(R::t_at, kNP, lower_block(i, kk), q);
                e[i] = mma_parts<kNP, kNP>(t, x[kk], e[i]);
            }
        }
        // Y
        split_tiles<YP>(e[0], e[1], x[0]);
        split_tiles<YP>(e[2], e[3], x[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int kk = 0; kk < lower_steps(i); ++kk) {
                bf16x8 t[YP];
#pragma unroll
                for (int q = 0; q < YP; ++q) t[q] = tri(R::p_at, YP, lower_block(i, kk), q);
                y[i] = mma_parts<YP, YP>(t, x[kk], y[i]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = ck * kC + 16 * i + 4 * g + r;
                if (t < len && p < P) stf(yp + t * ystep, y[i][r]);
            }
        }
        // S
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] *= *reinterpret_cast<const f32x4 *>(fac + R::kU + 16 * i + 4 * g);
        split_tiles<kNP>(e[0], e[1], x[0]);
        split_tiles<kNP>(e[2], e[3], x[1]);
        const float end = fac[R::kEnd];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            S[nt] *= end;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                bf16x8 kt[KP];
#pragma unroll
                for (int q = 0; q < KP; ++q) kt[q] = tile_cols<N>(sk + q * Tile<N>::size, nt, kk, lane);
                S[nt] = mma_parts<KP, kNP>(kt, x[kk], S[nt]);
            }
        }
    }
    if (p >= P) return;
    for (int t = len + g; t < L; t += 4) stf(yp + t * ystep, 0.f);
    if (a.state_out == nullptr) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = 16 * nt + 4 * g + r;
            if (n < n_of) a.state_out[(bh * P + p) * n_of + n] = S[nt][r];
        }
}

template <typename F>
hipError_t by_state(size_t d_state, F f) {
    if (d_state <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

// 16-byte loads of q and k rows: whole pieces of eight, every row aligned; a
// chunk's offsets below 2^31.
bool qk_vec(const DeltaLaunch &a, size_t size) {
    const size_t most = (size_t(1) << 31) / (kC * size) - 1024;
    return a.d_state % 8 == 0 && a.qs < most && a.ks < most && a.vs < most && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(a.k) & 15) == 0 && a.qs * size % 16 == 0 && a.ks * size % 16 == 0;
}

size_t chunks_of(const DeltaLaunch &a) { return (a.seq + kC - 1) / kC; }

}  // namespace

bool delta_chunk_wanted(const DeltaLaunch &a) { return a.d_state <= 128 && a.seq > 16; }

size_t delta_chunk_workspace(const DeltaLaunch &a) {
    size_t bytes = 0;
    (void)by_type(a.dtype, [&](auto t) {
        bytes = a.batch * a.heads * chunks_of(a) * Record<decltype(t)>::bytes;
        return hipSuccess;
    });
    return bytes;
}

hipError_t launch_delta_chunk(const DeltaLaunch &a, void *workspace, hipStream_t s, int &launches) {
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_state(a.d_state, [&](auto n) {
            constexpr int N = decltype(n)::value;
            const int chunks = static_cast<int>(chunks_of(a));
            unsigned char *rec = static_cast<unsigned char *>(workspace);
            const dim3 prep(static_cast<unsigned>(a.batch * a.heads * chunks));
            const dim3 main(static_cast<unsigned>(a.batch * a.heads), static_cast<unsigned>((a.head_dim + 63) / 64));
            const auto go = [&](auto vec) {
                constexpr bool VEC = decltype(vec)::value;
                hipLaunchKernelGGL((delta_prep<T, N, VEC>), prep, dim3(256), 0, s, a, rec, chunks);
                hipLaunchKernelGGL((delta_chunks<T, N, VEC>), main, dim3(256), 0, s, a, rec, chunks);
                launches += 2;
                return hipGetLastError();
            };
            return qk_vec(a, sizeof(T)) ? go(std::true_type{}) : go(std::false_type{});
        });
    });
}

}  // namespace m3
