// Gradients of the gated delta rule, chunk by chunk on the MFMA (gfx950); the
// chunk's notation, numbers and layouts are in delta_chunk.hpp.
//
// Given dY and the gradient dS1 of the state after a chunk, with P the attention
// scale (tril(Q K^T) . D), row factors fQ = scale exp(G) rq, fK = exp(G) rk and
// fU = beta exp(G_C - G) rk on raw rows q, k:
//   dR = T^T ((P diag(beta))^T dY + diag(fU) K dS1^T);  dV = dR
//   dS0 = exp(G_C) dS1 + (diag(fQ) dY)^T Q - (diag(fK) dR)^T K
// passes from the last chunk to the first, column by column of P as the forward
// does (delta_reverse: bound by its chain of products as the window, 129 us at 8 x
// 2048 tokens, 12 heads (64, 128), bf16).  The rest is each chunk's own (delta_grads): with F = dY
// E^T and Z = dR E^T,
//   X_ij = scale rq_i rk_j D_ij beta_j F_ij (j <= i),  Y_ij = rk_i rk_j D_ij beta_j Z_ij (j < i)
//   rq dq^ = diag(fQ) dY S0 + X K
//   rk dk^ = diag(fU) E dS1 - diag(fK) dR S0 + X^T Q - (Y + Y^T) K
//   V_ij = X_ij / beta_j (q_i.k_j) - Y_ij / beta_j (k_i.k_j)
//   dbeta_j = sum_i V_ij + (fU_j / beta_j) k_j.(E dS1)_j
//   dg_t = sum_{j<t<=i} beta_j V_ij + sum_{i>=t} a_i + sum_{j<t} b_j + exp(G_C) <dS1, S0>
//     a_i = fQ_i q_i.(dY S0)_i - fK_i k_i.(dR S0)_i,  b_j = fU_j k_j.(E dS1)_j
// (nothing is divided by beta), and through the unit-length norm dq = rq dq^ - q
// rq^2 (q . rq dq^), dk alike.  The first sum of dg_t is over a rectangle of the
// triangle: as the suffix sum of row sums less column sums, in f64, where the
// entries outside the rectangle cancel exactly.
#include "delta_chunk.hpp"

namespace m3 {
namespace {

using namespace delta;

// One workgroup a (sequence, head, 32 columns of P), the chunks from the last to
// the first, in pairs of waves as delta_chunks: a wave has half of N of its
// sixteen columns of the state's gradient.
template <typename T, int N, bool VEC>
__global__ void __launch_bounds__((kChunkThreads<T, VEC>))
delta_reverse(DeltaLaunch a, DeltaGrads gr, const unsigned char *records, int chunks, float *kept) {
    constexpr int KP = Parts<T>::in, KS = N / 64, NT = N / 32;   // of this wave
    using St = Stage<T, N, VEC, true, 1 + 2 * kTriT, kTriT>;
    constexpr bool DMA = St::DMA;
    constexpr int BUFS = DMA ? 2 : 1;
    constexpr size_t rec_bytes = BackRecord::units * 1024;
    __shared__ __attribute__((aligned(1024))) typename St::Rows1 sk[BUFS], sq[BUFS];
    __shared__ __attribute__((aligned(1024))) typename St::Rec sr[BUFS];
    __shared__ __attribute__((aligned(1024))) typename St::V sv;
    __shared__ f32x4 meet[4][4][64];
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave >> 1, half = wave & 1;
    const size_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    const int n_of = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const int p0 = blockIdx.y * kCols, p = p0 + 16 * w + c;      // this lane's column
    const size_t pv = a.heads * P, row0 = (b * L * a.heads + h) * P;
    T *dvp = static_cast<T *>(gr.dv) + row0;
    const uint32_t dv_at = row_off<T>(pv, P, 4 * g, p);
    const Kept kd(a);
    const int nt0 = half * NT, kk0 = half * KS;
    const int live = (len + kC - 1) / kC;
    St in(a, b, h, len, static_cast<const T *>(gr.dy) + row0, pv, p0, records + bh * chunks * rec_bytes, rec_bytes);
    if constexpr (DMA) {
        if (wave == 4) {
            const auto bring = [&](int ck) {
                in.dma_k(sk[ck & 1], ck);
                in.dma_q(sq[ck & 1], ck);
                in.template dma_rec<0, 1 + 2 * kTriT>(sr[ck & 1].at, ck);
            };
            if (live > 0) {
                bring(live - 1);
                in.dma_v(sv, live - 1);
            }
            for (int ck = live - 1; ck >= 0; --ck) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                scan::lds_barrier();   // the chunk is there, the one after it is done with
                if (ck > 0) bring(ck - 1);
                scan::lds_barrier();   // dY is done with
                if (ck > 0) in.dma_v(sv, ck - 1);
            }
            return;
        }
    } else {
        if (live > 0) in.fetch(live - 1);
    }
    // the gradient of the state after the chunk (the fifth wave has no columns)
    f32x4 S[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = state_n(nt0 + nt, g, r);
            S[nt][r] = gr.dstate && p < P && n < n_of ? gr.dstate[(bh * P + p) * n_of + n] : 0.f;
        }
    // rows 32 half .. of a chunk's dR: written a chunk later, so that the wait for
    // the operands does not wait for them
    f32x4 late[2];
    const auto write = [&](int ck) {
        float *keep = kept + (bh * chunks + ck) * kd.floats();
        const Rows<T, VEC> dvr(dvp + static_cast<size_t>(ck) * kC * pv, pv, len - ck * kC, P);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                keep[kd.dr() + (32 * half + 16 * i + 4 * g + r) * kd.p64 + p] = late[i][r];
                store_one(dvr, dv_at, 4 * g, p, 32 * half + 16 * i + r, late[i][r]);
            }
    };
    for (int ck = live - 1; ck >= 0; --ck) {
        const int now = DMA ? ck & 1 : 0;
        const typename St::Rows1 &k = sk[now], &q1 = sq[now];
        const unsigned char *rec = sr[now].at;
        f32x4 dy[4];
        if constexpr (DMA) {
            scan::lds_barrier();
        } else {
            __syncthreads();
            in.put(sk[0], sq[0], sr[0]);
            in.values(sv, dy);
            __syncthreads();
            if (ck > 0) in.fetch(ck - 1);
        }
        if (ck + 1 < live) write(ck + 1);
        float *keep = kept + (bh * chunks + ck) * kd.floats();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<f32x4 *>(keep + kd.s1() + kd.tile(p, nt0 + nt, lane)) = S[nt];
        const float *fac = reinterpret_cast<const float *>(rec);
        f32x4 ks[4], x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ks[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        bf16x8 kf[2][4][KP], sp[2][kNP], t4[4][kNP], t2[2][kNP], p4[4][kNP], p2[2][kNP];
        const auto rows = [&](int kk) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < KP; ++q) kf[kk & 1][i][q] = tile_rows<N>(k.part[q], i, kk0 + kk, lane);
        };
        rows(0);
        split_tiles<kNP>(S[0], S[1], sp[0]);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            if (kk + 1 < KS) {
                rows(kk + 1);
            } else {
                tri_load<kNP>(rec + (1 + kTriT) * 1024, lane, p4, p2, true);
                if constexpr (DMA) in.values(sv, dy);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (kk + 1 < KS) split_tiles<kNP>(S[2 * kk + 2], S[2 * kk + 3], sp[(kk + 1) & 1]);
            mma_rows<4, KP, kNP>(kf[kk & 1], sp[kk & 1], ks);
            interleave<4 * 3, 5>();
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) meet[wave][i][lane] = ks[i];
        {
            bf16x8 d[2][KP];
            split_tiles<KP>(dy[0], dy[1], d[0]);
            split_tiles<KP>(dy[2], dy[3], d[1]);
            mma_rows<2, kNP, KP>(p2, d[0], x);
            mma_rows<4, kNP, KP>(p4, d[1], x);
        }
        tri_load<kNP>(rec + 1024, lane, t4, t2, true);
        scan::lds_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ks[i] += meet[wave ^ 1][i][lane];
            x[i] += *reinterpret_cast<const f32x4 *>(fac + kFacU + 16 * i + 4 * g) * ks[i];
        }
        bf16x8 xs[2][kNP], ys[2][kNP];
        split_tiles<kNP>(x[0], x[1], xs[0]);
        split_tiles<kNP>(x[2], x[3], xs[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        mma_rows<2, kNP, kNP>(t2, xs[0], x);
        mma_rows<4, kNP, kNP>(t4, xs[1], x);
        bf16x8 kt[2][NT][KP], qt[2][NT][KP];
        const auto cols = [&](int j) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int q = 0; q < KP; ++q) {
                    kt[j][i][q] = tile_cols<N>(k.part[q], nt0 + i, j, lane);
                    qt[j][i][q] = tile_cols<N>(q1.part[q], nt0 + i, j, lane);
                }
        };
        cols(0);
        // x is dR
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (half)
                late[i] = x[2 + i];
            else
                late[i] = x[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] *= -*reinterpret_cast<const f32x4 *>(fac + kFacK + 16 * i + 4 * g);
            dy[i] *= *reinterpret_cast<const f32x4 *>(fac + kFacQ + 16 * i + 4 * g);
        }
        split_tiles<kNP>(x[0], x[1], xs[0]);
        split_tiles<kNP>(x[2], x[3], xs[1]);
        split_tiles<kNP>(dy[0], dy[1], ys[0]);
        split_tiles<kNP>(dy[2], dy[3], ys[1]);
        const float end = fac[kFacEnd];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] *= end;
        cols(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mma_rows<NT, KP, kNP>(kt[j], xs[j], S);
            mma_rows<NT, KP, kNP>(qt[j], ys[j], S);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (live > 0) write(0);
    if (p >= P) return;
    if (half == 0)
        for (int t = len + g; t < L; t += 4) stf(dvp + t * pv + p, 0.f);
    if (gr.dstate0 == nullptr) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = state_n(nt0 + nt, g, r);
            if (n < n_of) gr.dstate0[(bh * P + p) * n_of + n] = S[nt][r];
        }
}

// Sums over the sixteen lanes that hold a row of an accumulator tile.
__device__ __forceinline__ float row16(float v) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) v += __shfl_xor(v, off, 64);
    return v;
}
template <int DIR>   // inclusive, 1: from lane 0 on, -1: from lane 63 down
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = DIR > 0 ? __shfl_up(v, off, 64) : __shfl_down(v, off, 64);
        if (DIR > 0 ? lane >= off : lane + off < 64) v += o;
    }
    return v;
}

// One workgroup a (sequence, group, chunk), a wave sixteen of its tokens; the
// heads that share the group's q and k in turn.  First the triangles (F, Z, V and
// the sums of V), then the products with the states, then those within the
// chunk: what each holds in registers is gone before the next, so that two
// workgroups fit a CU and one's loads pass behind the other's products.  At 8 x 2048
// tokens, 12 heads (64, 128), bf16: 222 us, 3.1 TB/s of 556 MB read and 141 written; the
// vector instructions are busy 47 % of the time, LDS 43, the matrix unit 17 (the
// splitting of f32 operands costs more than their products).  One workgroup a CU of
// twice the waves took 480 us, the states' products before the triangles 281 (then 260).
// MANY:
// more than one head a group, whose dq and dk add up in further registers.
template <typename T, int N, bool VEC, bool MANY>
__global__ void __launch_bounds__(256, !MANY && Parts<T>::in == 1 ? 2 : 1)
delta_grads(DeltaLaunch a, DeltaGrads gr, const unsigned char *records, int chunks, const float *kept) {
    constexpr int KP = Parts<T>::in, OP = Parts<T>::out, NT = N / 16, per = N / 8;
    constexpr int s_bytes = kNP * Tile<N>::bytes / 2, xy_bytes = 2 * OP * Tile<64>::bytes, LW = kC + 1;
    constexpr int region = s_bytes > xy_bytes ? s_bytes : xy_bytes;
    static_assert(region >= kC * LW * 4 && region >= 2 * Tile<N>::bytes, "V and the outputs share the region");
    __shared__ __attribute__((aligned(16))) unsigned char sk[KP][Tile<N>::bytes], sq[KP][Tile<N>::bytes];
    __shared__ __attribute__((aligned(16))) unsigned char area[region];
    __shared__ __attribute__((aligned(16))) float fac[256];
    __shared__ double G[kC], sum_up[4][kC], sum_all[4][kC];
    __shared__ float beta[kC], rq[kC], rk[kC], da[kC], db[kC], dots[4];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t id = blockIdx.x, ck = id % chunks, kg = id / chunks % a.groups, b = id / chunks / a.groups;
    const int L = static_cast<int>(a.seq), t0 = static_cast<int>(ck) * kC, left = L - t0;
    const int live = valid_len(a.lengths, b, L) - t0;
    const int n_of = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const size_t rep = a.heads / a.groups, qk = a.groups * n_of, tok = b * L + t0, out0 = tok * qk + kg * n_of;
    T *dqp = static_cast<T *>(gr.dq) + out0, *dkp = static_cast<T *>(gr.dk) + out0;
    if (live <= 0) {   // padding: zeros
        const int rows = left < kC ? left : kC;
        for (int i = tid; i < rows * n_of; i += 256) {
            stf(dqp + (i / n_of) * qk + i % n_of, 0.f);
            stf(dkp + (i / n_of) * qk + i % n_of, 0.f);
        }
        for (int i = tid; i < rows * static_cast<int>(rep); i += 256) {
            const size_t th = (tok + i / rep) * a.heads + kg * rep + i % rep;
            gr.dg[th] = gr.dbeta[th] = 0.f;
        }
        return;
    }
    const Kept kd(a);
    const int my = 16 * w + c;
    // the group's rows, and the factors that bring them to unit length
    constexpr int own_rows = kC * per / 256;
    Eight<T> k8[own_rows], q8[own_rows];
    {
        const Rows<T, VEC> kr(static_cast<const T *>(a.k) + tok * a.ks + kg * n_of, a.ks, live, n_of);
        const Rows<T, VEC> qr(static_cast<const T *>(a.q) + tok * a.qs + kg * n_of, a.qs, live, n_of);
#pragma unroll
        for (int i = 0; i < own_rows; ++i) {
            k8[i] = load_eight(kr, tid / per + i * (256 / per), tid % per * 8);
            q8[i] = load_eight(qr, tid / per + i * (256 / per), tid % per * 8);
        }
    }
    const auto put_row = [&](const Eight<T> &x8, unsigned char(*to)[Tile<N>::bytes], float *unit, int t) {
        const int n = tid % per * 8;
        float f[8], ss = 0.f;
        widen(x8, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
#pragma unroll
        for (int off = 1; off < per; off <<= 1) ss += __shfl_xor(ss, off, 64);
        if (n == 0) unit[t] = a.qk_norm ? 1.0f / sqrtf(ss + kUnitEps) : 1.0f;
        bf16x8 x[KP];
        to_parts(x8, x);
#pragma unroll
        for (int q = 0; q < KP; ++q) *reinterpret_cast<bf16x8 *>(to[q] + tile_at<N>(t, n / 8)) = x[q];
    };
    const auto put_rows = [&]() {
#pragma unroll
        for (int i = 0; i < own_rows; ++i) {
            put_row(k8[i], sk, rk, tid / per + i * (256 / per));
            put_row(q8[i], sq, rq, tid / per + i * (256 / per));
        }
    };
    if constexpr (MANY) put_rows();
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    // q (or k) at row r, column state_n(nt, c >> 2, c & 3), from its parts
    const int own = (16 * w + 4 * g) * (2 * N) + ((g ^ (c >> 2)) << 4) + 2 * (c & 3);
    const auto value = [&](const unsigned char(*t)[Tile<N>::bytes], int nt, int r) {
        const int at = own + r * (2 * N) + (((nt >> 1) ^ (N == 128 ? r : r >> 1)) << 6) + 8 * (nt & 1);
        float v = 0.f;
#pragma unroll
        for (int q = KP - 1; q >= 0; --q) v += bf16_bits_to_f32(*reinterpret_cast<const uint16_t *>(t[q] + at));
        return v;
    };
    f32x4 dq[NT], dk[NT], tq[MANY ? NT : 1], tk[MANY ? NT : 1];
    if constexpr (MANY)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) tq[nt] = tk[nt] = zero;
    for (size_t hr = 0; hr < (MANY ? rep : 1); ++hr) {
        const size_t h = kg * rep + hr, rec = (b * a.heads + h) * chunks + ck;
        const float *keep = kept + rec * kd.floats();
        const Rows<T, VEC> dyr(static_cast<const T *>(gr.dy) + (tok * a.heads + h) * P, a.heads * P, live, P);
        // rows of dY, dR, E as loaded: columns pb + 4g .. and pb + 16 + 4g ..
        const auto kept_row = [&](size_t at, int t, int pb, f32x4 *out) {
            const float *s = keep + at + t * kd.p64 + pb + 4 * g;
            out[0] = *reinterpret_cast<const f32x4 *>(s);
            out[1] = *reinterpret_cast<const f32x4 *>(s + 16);
        };
        // dY's, four columns in one load where the rows allow it
        constexpr int words = VEC ? 2 * sizeof(T) : 8;
        const auto dy_row = [&](int pb, uint32_t *out) {
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t at = row_off<T>(dyr.stride, P, my, pb + 16 * j + 4 * g);
                    if constexpr (sizeof(T) == 4)
                        *reinterpret_cast<u32x4 *>(out + 4 * j) = bld16(dyr.r, at);
                    else
                        *reinterpret_cast<u32x2 *>(out + 2 * j) = bld8(dyr.r, at);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int n = pb + 16 * (j >> 2) + 4 * g + (j & 3);
                    out[j] = load_one(dyr, row_off<T>(dyr.stride, P, my, n), my, n, 0);
                }
            }
        };
        const auto dy_parts = [&](const uint32_t *y, bf16x8 *out) {
            float y8[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y8[j] = words == 8 ? value_of<T>(y[j]) : value_of<T>(y[j >> 1] >> (16 * (j & 1)) & 0xFFFFu);
            split8<KP>(y8, out);
        };
        // this head's decays, steps and factors, on their way while the rows are put down
        const size_t th = (tok + lane) * a.heads + h;
        float g1 = 0.f, b1 = 0.f;
        f32x4 fac1 = zero;
        if (w == 0 && lane < live) {
            g1 = a.g[th];
            b1 = a.beta[th];
        }
        if (w == 1) fac1 = *reinterpret_cast<const f32x4 *>(records + rec * (BackRecord::units * 1024) + 16 * lane);
        f32x4 f[4] = {zero, zero, zero, zero}, z[4] = {zero, zero, zero, zero};
        {
            __attribute__((aligned(16))) uint32_t y1[words];
            f32x4 r1[2], e1[4][2];
            const auto load = [&](int pb) {
                dy_row(pb, y1);
                kept_row(kd.dr(), my, pb, r1);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j <= w) kept_row(kd.e(), 16 * j + c, pb, e1[j]);
            };
            load(0);
            if constexpr (!MANY) put_rows();
            if (w == 0) {
                G[lane] = wave_scan<1>(static_cast<double>(clamp_decay(g1)), lane);
                beta[lane] = b1;
            }
            if (w == 1) *reinterpret_cast<f32x4 *>(fac + 4 * lane) = fac1;
#pragma unroll 1
            for (int pb = 0; pb < static_cast<int>(kd.p64); pb += 32) {
                bf16x8 ya[KP], ra[kNP], eb[4][kNP];
                dy_parts(y1, ya);
                split_tiles<kNP>(r1[0], r1[1], ra);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j <= w) split_tiles<kNP>(e1[j][0], e1[j][1], eb[j]);
                if (pb + 32 < static_cast<int>(kd.p64)) load(pb + 32);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j > w) continue;
                    f[j] = mma_parts<KP, kNP>(ya, eb[j], f[j]);
                    z[j] = mma_parts<kNP, kNP>(ra, eb[j], z[j]);
                }
            }
        }
        // what the states' first block takes, on its way during the triangle
        constexpr int pieces = 32 * N / 8 / 256;
        // piece i of this wave: columns 16 (w & 1) .. of the block, n of the pair of tiles i
        const auto pair = [&](int i) { return (w >> 1) + 2 * i; };
        f32x4 st[pieces][2], r1[2];   // S0, then dS1; rows of dR, then of E
        __attribute__((aligned(16))) uint32_t y1[words];
        const auto load_state = [&](size_t at, int pb) {
#pragma unroll
            for (int i = 0; i < pieces; ++i) {
                const float *s = keep + at + kd.tile(pb + 16 * (w & 1), 2 * pair(i), lane);
                st[i][0] = *reinterpret_cast<const f32x4 *>(s);
                st[i][1] = *reinterpret_cast<const f32x4 *>(s + 256);
            }
        };
        const auto load_first = [&](int pb) {
            load_state(kd.s0(), pb);
            dy_row(pb, y1);
            kept_row(kd.dr(), my, pb, r1);
        };
        const auto load_second = [&](int pb) {
            load_state(kd.s1(), pb);
            kept_row(kd.e(), my, pb, r1);
        };
        load_first(0);
        scan::lds_barrier();
        {
            f32x4 qkt[4] = {zero, zero, zero, zero}, kkt[4] = {zero, zero, zero, zero};
#pragma unroll 1
            for (int kk = 0; kk < N / 32; ++kk) {
                bf16x8 qa[KP], ka[KP], kb[KP];
#pragma unroll
                for (int q = 0; q < KP; ++q) {
                    qa[q] = tile_rows<N>(sq[q], w, kk, lane);
                    ka[q] = tile_rows<N>(sk[q], w, kk, lane);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j > w) continue;
#pragma unroll
                    for (int q = 0; q < KP; ++q) kb[q] = tile_rows<N>(sk[q], j, kk, lane);
                    qkt[j] = mma_parts<KP, KP>(qa, kb, qkt[j]);
                    kkt[j] = mma_parts<KP, KP>(ka, kb, kkt[j]);
                }
            }
            float(*V)[LW] = reinterpret_cast<float(*)[LW]>(area);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * w + 4 * g + r, jj = 16 * j + c;
                    float x = 0.f, y = 0.f, v = 0.f;
                    if (j <= w && jj <= i) {
                        const float d = expf(static_cast<float>(G[i] - G[jj])) * rk[jj];
                        x = a.scale * rq[i] * d * f[j][r];
                        if (jj < i) y = rk[i] * d * z[j][r];
                        v = x * qkt[j][r] - y * kkt[j][r];
                    }
                    V[i][jj] = v;
                    f[j][r] = x * beta[jj];
                    z[j][r] = -y * beta[jj];
                }
            scan::lds_barrier();
            // each wave's rows (columns) of every token's sums
            const int t = lane;
            double col = 0.0, all = 0.0, across = 0.0;
#pragma unroll 4
            for (int n = 0; n < 16; ++n) {
                const int i = 16 * w + n;
                const double v = V[i][t];
                if (i > t) col += v;
                if (i >= t) all += v;
                if (i < t) across += static_cast<double>(beta[i]) * V[t][i];
            }
            sum_up[w][t] = across - beta[t] * col;
            sum_all[w][t] = all;
        }
        f32x4 ki[NT], dot4 = zero;   // dq: dY S0, ki: dR S0, dk: E dS1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) dq[nt] = ki[nt] = dk[nt] = zero;
#pragma unroll 1
        for (int pb = 0; pb < static_cast<int>(kd.p64); pb += 32) {
            const auto mine = [&](int i, int q) {
                return reinterpret_cast<bf16x8 *>(area + q * (Tile<N>::bytes / 2) +
                                                  tile_at<N>(16 * (w & 1) + c, 4 * pair(i) + g));
            };
            const auto put = [&]() {
#pragma unroll
                for (int i = 0; i < pieces; ++i) {
                    bf16x8 x[kNP];
                    split_tiles<kNP>(st[i][0], st[i][1], x);
#pragma unroll
                    for (int q = 0; q < kNP; ++q) *mine(i, q) = x[q];
                }
            };
            const auto state = [&](int nt, bf16x8 *out) {
#pragma unroll
                for (int q = 0; q < kNP; ++q) out[q] = tile_cols<N>(area + q * (Tile<N>::bytes / 2), nt, 0, lane);
            };
            bf16x8 ya[KP], ra[kNP];
            dy_parts(y1, ya);
            split_tiles<kNP>(r1[0], r1[1], ra);
            scan::lds_barrier();
            put();
            load_second(pb);
            scan::lds_barrier();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                bf16x8 s[kNP];
                state(nt, s);
                dq[nt] = mma_parts<KP, kNP>(ya, s, dq[nt]);
                ki[nt] = mma_parts<kNP, kNP>(ra, s, ki[nt]);
                if (nt & 1) __builtin_amdgcn_sched_barrier(0);
            }
            split_tiles<kNP>(r1[0], r1[1], ra);
            // <S0, dS1> from S0's parts where this thread put them
#pragma unroll
            for (int i = 0; i < pieces; ++i)
#pragma unroll
                for (int q = kNP - 1; q >= 0; --q) {
                    const bf16x8 x = *mine(i, q);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dot4[j & 3] += static_cast<float>(x[j]) * st[i][j >> 2][j & 3];
                }
            scan::lds_barrier();
            put();
            if (pb + 32 < static_cast<int>(kd.p64)) load_first(pb + 32);
            scan::lds_barrier();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                bf16x8 s[kNP];
                state(nt, s);
                dk[nt] = mma_parts<kNP, kNP>(ra, s, dk[nt]);
                if (nt & 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        const float dot = group_sum(dot4[0] + dot4[1] + dot4[2] + dot4[3], 64);
        if (lane == 0) dots[w] = dot;
        // row by row: what the states contribute
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 16 * w + 4 * g + r;
            const float fq = fac[kFacQ + t], fk = fac[kFacK + t], fu = fac[kFacU + t];
            float x = 0.f, xs = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float kv = value(sk, nt, r), ka = fk * ki[nt][r];
                dq[nt][r] *= fq;
                x += value(sq, nt, r) * dq[nt][r] - kv * ka;
                xs += kv * dk[nt][r];
                dk[nt][r] = fu * dk[nt][r] - ka;
            }
            x = row16(x);
            xs = row16(xs);
            if (c == 0) {
                da[t] = x;
                db[t] = xs;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        scan::lds_barrier();
        // X and -Y as parts, then the products within the chunk
        const auto place = [&](int which, int q) { return area + (which * OP + q) * Tile<64>::bytes; };
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * w + 4 * g + r;
                const int at = tile_at<64>(i, 2 * j + (c >> 3)) + 2 * (c & 7);
                float x = f[j][r], y = z[j][r];
#pragma unroll
                for (int q = 0; q < OP; ++q) {
                    const bf16_t xb = from_f32<bf16_t>(x), yb = from_f32<bf16_t>(y);
                    *reinterpret_cast<uint16_t *>(place(0, q) + at) = xb.bits;
                    *reinterpret_cast<uint16_t *>(place(1, q) + at) = yb.bits;
                    x -= to_f32(xb);
                    y -= to_f32(yb);
                }
            }
        if (w == 0) {
            const int t = lane;
            const double up = wave_scan<-1>(sum_up[0][t] + sum_up[1][t] + sum_up[2][t] + sum_up[3][t] + da[t], lane);
            const double all = sum_all[0][t] + sum_all[1][t] + sum_all[2][t] + sum_all[3][t];
            const double bt = fac[kFacU + t] * db[t], down = wave_scan<1>(bt, lane) - bt;
            const float dot_all = dots[0] + dots[1] + dots[2] + dots[3];
            const size_t th = (tok + t) * a.heads + h;
            if (t < left) {
                const bool ok = t < live;
                gr.dg[th] = ok ? static_cast<float>(up + down + static_cast<double>(fac[kFacEnd]) * dot_all) : 0.f;
                gr.dbeta[th] = ok ? static_cast<float>(all + expf(static_cast<float>(G[kC - 1] - G[t])) * rk[t] * db[t]) : 0.f;
            }
        }
        scan::lds_barrier();
#pragma unroll 1
        for (int kk = 0; kk < 2; ++kk) {
            // rows 16 w of X and Y (tokens 32 kk + 4g .., + 16 + 4g ..), and of their transposes
            bf16x8 xr[OP], yr[OP], xt[OP], yt[OP];
#pragma unroll
            for (int q = 0; q < OP; ++q) {
                const int piece = 4 * kk + (g >> 1), off = 8 * (g & 1);
                const auto four = [&](int which, int pc) {
                    return *reinterpret_cast<const bf16x4 *>(place(which, q) + tile_at<64>(my, pc) + off);
                };
                xr[q] = __builtin_shufflevector(four(0, piece), four(0, piece + 2), 0, 1, 2, 3, 4, 5, 6, 7);
                yr[q] = __builtin_shufflevector(four(1, piece), four(1, piece + 2), 0, 1, 2, 3, 4, 5, 6, 7);
                const auto acc = [&](int which, int i) { return tile_acc<64>(place(which, q), i, w, lane); };
                xt[q] = __builtin_shufflevector(acc(0, 2 * kk), acc(0, 2 * kk + 1), 0, 1, 2, 3, 4, 5, 6, 7);
                yt[q] = __builtin_shufflevector(acc(1, 2 * kk), acc(1, 2 * kk + 1), 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                bf16x8 kc[KP], qc[KP];
#pragma unroll
                for (int q = 0; q < KP; ++q) {
                    kc[q] = tile_cols<N>(sk[q], nt, kk, lane);
                    qc[q] = tile_cols<N>(sq[q], nt, kk, lane);
                }
                if (kk <= (w >> 1)) {
                    dq[nt] = mma_parts<OP, KP>(xr, kc, dq[nt]);
                    dk[nt] = mma_parts<OP, KP>(yr, kc, dk[nt]);
                }
                if (kk >= (w >> 1)) {
                    dk[nt] = mma_parts<OP, KP>(xt, qc, dk[nt]);
                    dk[nt] = mma_parts<OP, KP>(yt, kc, dk[nt]);
                }
                if (nt & 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        scan::lds_barrier();
        if constexpr (MANY)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                tq[nt] += dq[nt];
                tk[nt] += dk[nt];
            }
    }
    if constexpr (MANY)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            dq[nt] = tq[nt];
            dk[nt] = tk[nt];
        }
    // through the norm, and out
    const Rows<T, VEC> dqr(dqp, qk, left, n_of), dkr(dkp, qk, left, n_of);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = 16 * w + 4 * g + r;
        float xq = 0.f, xk = 0.f;
        if (a.qk_norm) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                xq += value(sq, nt, r) * dq[nt][r];
                xk += value(sk, nt, r) * dk[nt][r];
            }
            xq = row16(xq) * rq[t] * rq[t];
            xk = row16(xk) * rk[t] * rk[t];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int n = state_n(nt, c >> 2, c & 3);
            const float q = dq[nt][r] - value(sq, nt, r) * xq, k = dk[nt][r] - value(sk, nt, r) * xk;
            if constexpr (VEC && sizeof(T) == 2) {
                T *at = reinterpret_cast<T *>(area + tile_at<N>(t, n / 8) + 2 * (n % 8));
                stf(at, q);
                stf(at + Tile<N>::bytes / 2, k);
            } else {
                const uint32_t at = row_off<T>(qk, n_of, t, n);
                store_one(dqr, at, t, n, 0, q);
                store_one(dkr, at, t, n, 0, k);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (VEC && sizeof(T) == 2) {
        scan::lds_barrier();
#pragma unroll
        for (int i = 0; i < kC * per / 256; ++i) {
            const int t = tid / per + i * (256 / per), n = tid % per * 8;
            const uint32_t at = row_off<T>(qk, n_of, t, n);
            const unsigned char *s = area + tile_at<N>(t, n / 8);
            bst16(*reinterpret_cast<const u32x4 *>(s), dqr.r, at);
            bst16(*reinterpret_cast<const u32x4 *>(s + Tile<N>::bytes), dkr.r, at);
        }
    }
}

}  // namespace

bool delta_backward_supported(const DeltaLaunch &a) { return a.d_state <= 128; }

size_t delta_backward_workspace(const DeltaLaunch &a) {
    size_t kept_at = 0;
    return delta_states_workspace(a, kept_at);
}

hipError_t launch_delta_backward(const DeltaLaunch &a, const DeltaGrads &g, void *workspace, hipStream_t s,
                                 int &launches) {
    unsigned char *records = static_cast<unsigned char *>(workspace);
    size_t kept_at = 0;
    delta_states_workspace(a, kept_at);
    float *kept = reinterpret_cast<float *>(records + kept_at);
    if (a.seq > 0) {
        const hipError_t e = launch_delta_states(a, records, s, launches);
        if (e != hipSuccess) return e;
    }
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_state(a.d_state, [&](auto n) {
            constexpr int N = decltype(n)::value;
            const int chunks = static_cast<int>(chunks_of(a));
            const dim3 rev(static_cast<unsigned>(a.batch * a.heads), static_cast<unsigned>(kept_cols(a)));
            const dim3 own(static_cast<unsigned>(a.batch * a.groups * chunks));
            const auto go = [&](auto vec) {
                constexpr bool VEC = decltype(vec)::value;
                constexpr unsigned threads = kChunkThreads<T, VEC>;
                hipLaunchKernelGGL((delta_reverse<T, N, VEC>), rev, dim3(threads), 0, s, a, g, records, chunks, kept);
                ++launches;
                if (chunks > 0) {
                    if (a.heads == a.groups)
                        hipLaunchKernelGGL((delta_grads<T, N, VEC, false>), own, dim3(256), 0, s, a, g, records, chunks, kept);
                    else
                        hipLaunchKernelGGL((delta_grads<T, N, VEC, true>), own, dim3(256), 0, s, a, g, records, chunks, kept);
                    ++launches;
                }
                return hipGetLastError();
            };
            // the gradients' rows are as v's and y's, q's and k's contiguous ones
            DeltaLaunch o = a;
            o.y = const_cast<void *>(g.dy);
            bool vec = rows_vec(o, sizeof(T));
            o.y = g.dv;
            o.q = g.dq;
            o.k = g.dk;
            o.qs = o.ks = a.groups * a.d_state;
            vec = vec && rows_vec(o, sizeof(T));
            return vec ? go(std::true_type{}) : go(std::false_type{});
        });
    });
}

}  // namespace m3
