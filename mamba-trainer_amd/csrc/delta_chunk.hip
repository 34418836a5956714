// The gated delta rule over a window, chunk by chunk on the MFMA (gfx950); the
// mathematics, the numbers and the register layout are in delta_chunk.hpp.
#include "delta_chunk.hpp"

namespace m3 {
namespace {

using namespace delta;

// One workgroup a (sequence, head, chunk): the chunk's row factors, T and the
// attention within the chunk.  What the chunks' chain would else redo for every
// column block of P is done once here and left as ready operands.  Near a copy's
// rate: 8 x 2048 tokens, 12 heads (64, 128), bf16: 101 MB of q and k read and 97 of
// records written in 46 us, 4.3 TB/s (BACK: 172 written in 56 us).
template <typename T, int N, bool VEC, bool BACK>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && N == 128 ? 2 : 4) delta_prep(DeltaLaunch a, unsigned char *records, int chunks) {
    constexpr int KP = Parts<T>::in, LP = kC + 4;
    using R = Record<T>;
    constexpr size_t bytes = (BACK ? BackRecord::units : R::units) * 1024;
    // the rows as loaded, then (in the same place) the triangles
    constexpr int row_bytes = N * sizeof(T), rows_bytes = kC * row_bytes, tri_bytes = kC * LP * 4;
    __shared__ __attribute__((aligned(16))) unsigned char area[2 * (rows_bytes > tri_bytes ? rows_bytes : tri_bytes)];
    __shared__ double G[kC];
    __shared__ float beta[kC], rq[kC], rk[kC];
    float(*A)[LP] = reinterpret_cast<float(*)[LP]>(area), (*X)[LP] = A + kC;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t rec = blockIdx.x, bh = rec / chunks, b = bh / a.heads, h = bh % a.heads;
    const int t0 = static_cast<int>(rec % chunks) * kC;
    const int L = static_cast<int>(a.seq), live = valid_len(a.lengths, b, L) - t0;   // of this chunk
    if (live <= 0) return;
    const size_t kg = h / (a.heads / a.groups);
    const int n_of = static_cast<int>(a.d_state);
    const Rows<T, VEC> kp(static_cast<const T *>(a.k) + (b * L + t0) * a.ks + kg * n_of, a.ks, live, n_of);
    const Rows<T, VEC> qp(static_cast<const T *>(a.q) + (b * L + t0) * a.qs + kg * n_of, a.qs, live, n_of);
    // eight values of row t from n on: 16-byte pieces, permuted against bank conflicts
    const auto at = [&](int which, int t, int n) {
        const int piece = n * sizeof(T) / 16, perm = sizeof(T) == 4 ? t & 15 : swizzle<N>(t);
        return area + which * rows_bytes + t * row_bytes + ((piece ^ perm) << 4);
    };
    const auto put = [&](int which, int t, int n, const Eight<T> &e) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<u32x4 *>(at(which, t, n)) = e.a;
            *reinterpret_cast<u32x4 *>(at(which, t, n + 4)) = e.b;
        } else {
            *reinterpret_cast<u32x4 *>(at(which, t, n)) = e.q;
        }
    };
    const auto get = [&](int which, int t, int n, bf16x8 *out) {
        Eight<T> e;
        if constexpr (sizeof(T) == 4) {
            e.a = *reinterpret_cast<const u32x4 *>(at(which, t, n));
            e.b = *reinterpret_cast<const u32x4 *>(at(which, t, n + 4));
        } else {
            e.q = *reinterpret_cast<const u32x4 *>(at(which, t, n));
        }
        to_parts(e, out);
    };
    constexpr int per = N / 8, pieces = kC * per / 256;   // threads of a row
    Eight<T> k8[pieces], q8[pieces];
#pragma unroll
    for (int i = 0; i < pieces; ++i) {
        k8[i] = load_eight(kp, tid / per + i * (256 / per), tid % per * 8);
        q8[i] = load_eight(qp, tid / per + i * (256 / per), tid % per * 8);
    }
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
#pragma unroll
    for (int i = 0; i < pieces; ++i) {
        const int t = tid / per + i * (256 / per), n = tid % per * 8;
        float f[8], sq = 0.f, sk = 0.f;
        widen(q8[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sq += f[e] * f[e];
        widen(k8[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sk += f[e] * f[e];
#pragma unroll
        for (int off = 1; off < per; off <<= 1) {
            sq += __shfl_xor(sq, off, 64);
            sk += __shfl_xor(sk, off, 64);
        }
        if (n == 0) {
            rq[t] = a.scale * (a.qk_norm ? 1.0f / sqrtf(sq + kUnitEps) : 1.0f);
            rk[t] = a.qk_norm ? 1.0f / sqrtf(sk + kUnitEps) : 1.0f;
        }
        put(0, t, n, k8[i]);
        put(1, t, n, q8[i]);
    }
    __syncthreads();
    // the ten lower tiles of K K^T and Q K^T, two or three a wave: (0,0) (3,0) (3,1);
    // (1,0) (1,1); (2,0) (2,1) (2,2); (3,2) (3,3)
    const int count = w & 1 ? 2 : 3;
    const auto row_of = [&](int s) { return w == 0 && s > 0 ? 3 : w; };
    const auto col_of = [&](int s) { return w == 0 ? (s > 0 ? s - 1 : 0) : w == 3 ? 2 + s : s; };
    f32x4 kkt[3], qkt[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        kkt[s] = qkt[s] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s >= count) continue;
        const int ri = 16 * row_of(s) + c, rj = 16 * col_of(s) + c;
#pragma unroll
        for (int kk = 0; kk < N / 32; ++kk) {
            bf16x8 qa[KP], ka[KP], kb[KP];
            get(1, ri, 32 * kk + 8 * g, qa);
            get(0, ri, 32 * kk + 8 * g, ka);
            get(0, rj, 32 * kk + 8 * g, kb);
            kkt[s] = mma_parts<KP, KP>(ka, kb, kkt[s]);
            qkt[s] = mma_parts<KP, KP>(qa, kb, qkt[s]);
        }
    }
    __syncthreads();   // the rows are done with
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        if (s >= count) continue;
        const int jj = 16 * col_of(s) + c;
        const float f = rk[jj] * beta[jj];
        const double gj = G[jj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * row_of(s) + 4 * g + r;
            float m = 0.f, p = 0.f;
            if (jj <= i) {
                const float d = expf(static_cast<float>(G[i] - gj)) * f;
                p = d * rq[i] * qkt[s][r];
                if (jj < i) m = d * rk[i] * kkt[s][r];
            }
            A[i][jj] = m;
            X[i][jj] = p;
        }
    }
    // the tiles above the diagonal that an operand block takes in: zero
    if ((w & 1) == 0)
#pragma unroll
        for (int r = 0; r < 4; ++r) X[16 * w + 4 * g + r][16 * (w + 1) + c] = 0.f;
    const int my = 16 * w + c;
    unsigned char *out = records + rec * bytes;
    if (w == 0) {
        float *f = reinterpret_cast<float *>(out);
        const float eg = expf(static_cast<float>(G[lane]));
        f[kFacK + lane] = eg * rk[lane];
        f[kFacQ + lane] = eg * rq[lane];
        f[kFacU + lane] = beta[lane] * expf(static_cast<float>(G[kC - 1] - G[lane])) * rk[lane];
        if (lane == 0) f[kFacEnd] = expf(static_cast<float>(G[kC - 1]));
    }
    __syncthreads();
    // a triangle of X as operand blocks, or of its transpose: wave w writes those
    // of rows 16 w
    const auto emit = [&](int unit, auto parts, auto upper) {
        constexpr int NP = decltype(parts)::value;
        constexpr bool UP = decltype(upper)::value;
        for (int kk = UP ? w >> 1 : 0; kk < (UP ? 2 : 1 + (w >> 1)); ++kk) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = 32 * kk + 16 * (i >> 2) + 4 * g + (i & 3);
                x[i] = UP ? X[k][my] : X[my][k];
            }
            bf16x8 o[NP];
            split8<NP>(x, o);
            const int blk = UP ? upper_block(w, kk) : lower_block(w, kk);
#pragma unroll
            for (int p = 0; p < NP; ++p)
                *reinterpret_cast<bf16x8 *>(out + unit * 1024 + ((blk * NP + p) * 64 + lane) * 16) = o[p];
        }
    };
    constexpr std::integral_constant<int, kNP> full{};
    if constexpr (BACK)
        emit(BackRecord::pt, full, std::true_type{});
    else
        emit(R::p, std::integral_constant<int, Parts<T>::out>{}, std::false_type{});
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
    __syncthreads();
    emit(R::t, full, std::false_type{});
    if constexpr (BACK) emit(BackRecord::tt, full, std::true_type{});
}

// One workgroup a (sequence, head, 32 columns of P), the chunks in turn.  A pair
// of waves has sixteen columns, each half of the state's N: their halves of K S0^T
// (and of Q S0^T) meet in LDS, then both form E, and each its half of S and of
// Y's rows.  DMA: what is read first in a chunk (K, v, the record) goes to a
// second buffer while the one before is multiplied, Q to the buffer it has left
// (without Q: v and T to theirs).
// KEEP is the backward's way in: no y, but the state before each chunk and its E
// are kept.
//
// Bound by its own chain: a workgroup a CU, one chunk after another, each some
// 5500 cycles of products that wait for each other (the matrix unit is busy 29 % of
// them, vector instructions 35 %).  So what stood beside the chain was moved off
// it, 8 x 2048 tokens, 12 heads (64, 128), bf16: pairs of waves a column tile instead of one
// 149 -> 117 us, the fetch in a fifth wave 117 -> 92.  The passes without outputs
// fetch less: there the four waves do it (KEEP 97 -> 89 us), and as five waves of
// their registers would not, two workgroups of four fit a CU (CARRY 162 -> 139 us at 16384
// tokens of one sequence).
//
// Few sequences leave most CUs idle while their chunks pass one by one; then the
// window is cut into segments that run side by side.  As S [P, N] passes through
// a segment it becomes S Phi + Psi, with Phi [N, N] of the keys alone, so a CARRY
// pass finds Psi (the segment on v from a zero state) and Phi (on v = 0 from the
// rows of the identity, as further columns of P), delta_join the state before
// each segment, and the window's pass (or KEEP) runs each from there: some
// (2 P + N) / P times the work, in segments' time.
enum { kWindow, kKeep, kCarry };
template <typename T, int N, bool VEC, int MODE, bool BACK>
__global__ void __launch_bounds__((kChunkThreads<T, VEC, MODE != kWindow>), (kDma<T, VEC> && MODE != kWindow ? 2 : 1))
delta_chunks(DeltaLaunch a, const unsigned char *records, int chunks, float *kept, Segments sg) {
    constexpr bool KEEP = MODE == kKeep, Y = MODE == kWindow;
    constexpr int KP = Parts<T>::in, YP = Parts<T>::out, KS = N / 64, NT = N / 32;   // of this wave
    using R = Record<T>;
    constexpr size_t rec_bytes = (BACK ? BackRecord::units : R::units) * 1024;
    using St = Stage<T, N, VEC, Y, Y ? R::units : R::p, 0, !Y>;
    constexpr bool DMA = St::DMA;
    constexpr int BUFS = DMA ? 2 : 1;
    __shared__ __attribute__((aligned(1024))) typename St::Rows1 sk[BUFS];
    constexpr bool TWO = DMA && Y;   // else only K and the record's factors lie there twice
    __shared__ __attribute__((aligned(1024))) typename St::Rec sr[TWO ? 2 : 1];
    __shared__ __attribute__((aligned(1024))) typename St::V sv[TWO ? 2 : 1];
    __shared__ __attribute__((aligned(1024))) unsigned char odd_fac[DMA && !Y ? 1024 : 16];
    __shared__ __attribute__((aligned(1024))) unsigned char sq_[!Y ? 16 : sizeof(typename St::Rows1)];
    __shared__ f32x4 meet[4][Y ? 6 : 4][64];
    __shared__ __attribute__((aligned(16))) uint16_t sy[DMA && Y ? 4 : 1][DMA && Y ? 32 : 1][16];
    typename St::Rows1 &sq = reinterpret_cast<typename St::Rows1 &>(sq_);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave >> 1, half = wave & 1;
    const size_t bh = blockIdx.x / sg.count, b = bh / a.heads, h = bh % a.heads;
    const int seg = static_cast<int>(blockIdx.x % sg.count);
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    const int n_of = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim);
    const int p0 = blockIdx.y * kCols, p = p0 + 16 * w + c;      // this lane's column
    const int unit_row = p - static_cast<int>(sg.cols);           // CARRY: of the identity, if not below 0
    T *yp = static_cast<T *>(a.y) + (b * L * a.heads + h) * P;
    const size_t ystep = a.heads * P;
    const uint32_t y_at = row_off<T>(ystep, P, 4 * g, p);
    const Kept kd(a);
    const int nt0 = half * NT, kk0 = half * KS;
    const int all = (len + kC - 1) / kC, first = seg * sg.chunks;
    const int live = sg.chunks < all - first ? first + sg.chunks : all;   // the segment's end
    St in(a, b, h, len, static_cast<const T *>(a.v) + b * L * a.vs + h * P, a.vs, p0,
          records + bh * chunks * rec_bytes, rec_bytes);
    const auto first_half = [&](int ck) {
        in.dma_k(sk[ck & 1], ck);
        if constexpr (Y) {
            in.dma_v(sv[ck & 1], ck);
            in.template dma_rec<0, R::units>(sr[ck & 1].at, ck);
        } else {
            in.template dma_rec<0, 1>(ck & 1 ? odd_fac : sr[0].at, ck);
        }
    };
    const auto second_half = [&](int ck) {
        if constexpr (Y) {
            in.dma_q(sq, ck);
        } else {
            in.dma_v(sv[0], ck);
            in.template dma_rec<R::t, R::p>(sr[0].at, ck);
        }
    };
    if constexpr (DMA) {
        if (Y ? wave == 4 : true)
            if (first < live) {
                first_half(first);
                second_half(first);
            }
        if (Y && wave == 4) {
            for (int ck = first; ck < live; ++ck) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                scan::lds_barrier();   // the chunk is there, the one before is done with
                if (ck + 1 < live) first_half(ck + 1);
                scan::lds_barrier();   // Q is done with
                if (ck + 1 < live) second_half(ck + 1);
            }
            return;
        }
    } else {
        if (first < live) in.fetch(first);
    }
    // (after the fifth wave has gone its way: it has no columns)
    f32x4 S[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int n4 = state_n(nt0 + nt, g, 0);
        if constexpr (MODE != kCarry)
            if (sg.count > 1) {
                S[nt] = *reinterpret_cast<const f32x4 *>(sg.starts + ((bh * sg.count + seg) * sg.cols + p) * N + n4);
                continue;
            }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = n4 + r;
            if constexpr (MODE == kCarry)
                S[nt][r] = n == unit_row ? 1.f : 0.f;
            else
                S[nt][r] = a.state && p < P && n < n_of ? a.state[(bh * P + p) * n_of + n] : 0.f;
        }
    }
    // rows 32 half .. of a chunk's Y (KEEP: E): written a chunk later, so that the
    // wait for the operands does not wait for them
    f32x4 late[2];
    const auto write = [&](int ck) {
        if constexpr (KEEP) {
            float *to = kept + (bh * chunks + ck) * kd.floats() + kd.e() + (32 * half + 4 * g) * kd.p64 + p;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(16 * i + r) * kd.p64] = late[i][r];
        }
        if constexpr (Y) {
            // padding rows past the buffer's end are dropped
            const Rows<T, VEC> yrow(yp + static_cast<size_t>(ck) * kC * ystep, ystep, len - ck * kC, P);
            if constexpr (DMA) {
                // the wave's 32 x 16 through LDS to 16-byte stores
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        sy[wave][16 * i + 4 * g + r][c] = from_f32<bf16_t>(late[i][r]).bits;
                bst16(*reinterpret_cast<const u32x4 *>(&sy[wave][lane >> 1][8 * (lane & 1)]), yrow.r,
                      row_off<T>(ystep, P, 32 * half + (lane >> 1), p0 + 16 * w + 8 * (lane & 1)));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) store_one(yrow, y_at, 4 * g, p, 32 * half + 16 * i + r, late[i][r]);
            }
        }
    };
    for (int ck = first; ck < live; ++ck) {
        const int now = DMA ? ck & 1 : 0;
        const typename St::Rows1 &k = sk[now];
        const unsigned char *rec = sr[TWO ? now : 0].at;
        f32x4 e[4];
        if constexpr (DMA) {
            if constexpr (!Y) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            scan::lds_barrier();
        } else {
            __syncthreads();
            in.put(sk[0], sq, sr[0]);
            in.values(sv[0], e);
            __syncthreads();
            if (ck + 1 < live) in.fetch(ck + 1);
        }
        if (ck > first) write(ck - 1);
        if constexpr (KEEP) {
            float *keep = kept + (bh * chunks + ck) * kd.floats();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                *reinterpret_cast<f32x4 *>(keep + kd.s0() + kd.tile(p, nt0 + nt, lane)) = S[nt];
        }
        const float *fac = reinterpret_cast<const float *>(DMA && !Y && now ? odd_fac : rec);
        // this half of K S0^T and Q S0^T: while a k-step is multiplied, the next
        // one's operands are read and its columns of S are split
        f32x4 y[4], ks[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = ks[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        bf16x8 kf[2][4][KP], qf[2][4][KP], sp[2][kNP];
        const auto rows = [&](int kk) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < KP; ++q) {
                    kf[kk & 1][i][q] = tile_rows<N>(k.part[q], i, kk0 + kk, lane);
                    if constexpr (Y) qf[kk & 1][i][q] = tile_rows<N>(sq.part[q], i, kk0 + kk, lane);
                }
        };
        bf16x8 t4[4][kNP], t2[2][kNP];
        rows(0);
        split_tiles<kNP>(S[0], S[1], sp[0]);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            if (kk + 1 < KS) {
                rows(kk + 1);
            } else {
                if constexpr (DMA) in.values(sv[TWO ? now : 0], e);
            }
            if constexpr (DMA && !Y)
                if (kk == 0 && ck + 1 < live) first_half(ck + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (kk + 1 < KS) split_tiles<kNP>(S[2 * kk + 2], S[2 * kk + 3], sp[(kk + 1) & 1]);
            mma_rows<4, KP, kNP>(kf[kk & 1], sp[kk & 1], ks);
            if constexpr (Y) mma_rows<4, KP, YP>(qf[kk & 1], sp[kk & 1], y);
            interleave<4 * (3 + 2), 3>();
            __builtin_amdgcn_sched_barrier(0);
        }
        // the other half
#pragma unroll
        for (int i = 0; i < 4; ++i) meet[wave][i][lane] = ks[i];
        if constexpr (Y)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (half)
                    meet[wave][4 + i][lane] = y[i];
                else
                    meet[wave][4 + i][lane] = y[2 + i];
            }
        tri_load<kNP>(rec + R::t * 1024, lane, t4, t2, false);
        scan::lds_barrier();
        if constexpr (DMA && !Y)
            if (ck + 1 < live) second_half(ck + 1);   // v and T are done with
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ks[i] += meet[wave ^ 1][i][lane];
            e[i] -= *reinterpret_cast<const f32x4 *>(fac + kFacK + 16 * i + 4 * g) * ks[i];
        }
        // E = T R
        bf16x8 x[2][kNP];
        split_tiles<kNP>(e[0], e[1], x[0]);
        split_tiles<kNP>(e[2], e[3], x[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        mma_rows<4, kNP, kNP>(t4, x[0], e);
        mma_rows<2, kNP, kNP>(t2, x[1], e + 2);
        // S, and Y's part within the chunk: rows 32 half ..
        bf16x8 pb[2][2][YP], xe[2][YP];
        f32x4 yr[2];
        bf16x8 kt[2][NT][KP];
        const auto cols = [&](int j) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int q = 0; q < KP; ++q) kt[j][i][q] = tile_cols<N>(k.part[q], nt0 + i, j, lane);
        };
        cols(0);
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (half)
                    late[i] = e[2 + i];
                else
                    late[i] = e[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (half)
                    yr[i] = y[2 + i];
                else
                    yr[i] = y[i];
                yr[i] = (yr[i] + meet[wave ^ 1][4 + i][lane]) *
                        *reinterpret_cast<const f32x4 *>(fac + kFacQ + 32 * half + 16 * i + 4 * g);
            }
            split_tiles<YP>(e[0], e[1], xe[0]);
            split_tiles<YP>(e[2], e[3], xe[1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] *= *reinterpret_cast<const f32x4 *>(fac + kFacU + 16 * i + 4 * g);
        split_tiles<kNP>(e[0], e[1], x[0]);
        split_tiles<kNP>(e[2], e[3], x[1]);
        const float end = fac[kFacEnd];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] *= end;
        cols(1);
        if constexpr (Y)
#pragma unroll
            for (int q = 0; q < YP; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    pb[0][i][q] = tri_block<YP>(rec + R::p * 1024, half ? 2 + 2 * i : i, q, lane);
                    pb[1][i][q] = tri_block<YP>(rec + R::p * 1024, 3 + 2 * i, q, lane);   // rows 32 .. only
                }
        __builtin_amdgcn_sched_barrier(0);
        mma_rows<NT, KP, kNP>(kt[0], x[0], S);
        mma_rows<NT, KP, kNP>(kt[1], x[1], S);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!Y) continue;
        mma_rows<2, YP, YP>(pb[0], xe[0], yr);
        if (half) mma_rows<2, YP, YP>(pb[1], xe[1], yr);
        late[0] = yr[0];
        late[1] = yr[1];
    }
    if (first < live) write(live - 1);
    if constexpr (MODE == kCarry) {
        float *to = sg.carry + ((bh * sg.count + seg) * (sg.cols + N) + p) * N;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<f32x4 *>(to + state_n(nt0 + nt, g, 0)) = S[nt];
        return;
    }
    if (KEEP || p >= P) return;
    if (half == 0 && seg == 0)
        for (int t = len + g; t < L; t += 4) stf(yp + t * ystep + p, 0.f);
    if (a.state_out == nullptr || seg + 1 < static_cast<int>(sg.count)) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = state_n(nt0 + nt, g, r);
            if (n < n_of) a.state_out[(bh * P + p) * n_of + n] = S[nt][r];
        }
}

// The state before each segment: one workgroup a (sequence, head, 16 rows of S),
// a wave 16 columns, S_s Phi_s + Psi_s segment by segment in f32 (MFMA 16x16x4);
// the next segment's Phi and Psi are on their way meanwhile.  A chain of loads and
// products: 20 us for ten segments of 12 heads (64, 128).
template <int N>
__global__ void __launch_bounds__(4 * N) delta_join(DeltaLaunch a, Segments sg) {
    constexpr int KS = N / 4;
    __shared__ float s[2][16][N + 4];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const size_t bh = blockIdx.x;
    const int p0 = blockIdx.y * 16, P = static_cast<int>(a.head_dim), n_of = static_cast<int>(a.d_state);
    const int n = 16 * w + c;
    float phi[KS], psi[4];
    const auto load = [&](size_t seg) {
        const float *at = sg.carry + (bh * sg.count + seg) * (sg.cols + N) * N;
#pragma unroll
        for (int r = 0; r < 4; ++r) psi[r] = at[(p0 + 4 * g + r) * N + n];
#pragma unroll
        for (int k = 0; k < KS; ++k) phi[k] = at[(sg.cols + 4 * k + g) * N + n];
    };
    load(0);
    for (int i = tid; i < 16 * N; i += 4 * N) {
        const int p = p0 + i / N, m = i % N;
        const float v = a.state && p < P && m < n_of ? a.state[(bh * P + p) * n_of + m] : 0.f;
        s[0][i / N][m] = v;
        sg.starts[(bh * sg.count * sg.cols + p) * N + m] = v;
    }
    scan::lds_barrier();
    for (size_t seg = 0; seg + 1 < sg.count; ++seg) {
        const float(*from)[N + 4] = s[seg & 1];
        f32x4 acc[2] = {f32x4{psi[0], psi[1], psi[2], psi[3]}, f32x4{0.f, 0.f, 0.f, 0.f}};
        float m[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) m[k] = phi[k];
        if (seg + 2 < sg.count) load(seg + 1);
#pragma unroll
        for (int k = 0; k < KS; ++k) acc[k & 1] = mfma_f32(from[c][4 * k + g], m[k], acc[k & 1]);
        float *out = sg.starts + (bh * sg.count + seg + 1) * sg.cols * N;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = acc[0][r] + acc[1][r];
            s[(seg + 1) & 1][4 * g + r][n] = v;
            out[(p0 + 4 * g + r) * N + n] = v;
        }
        scan::lds_barrier();
    }
}

// Segments of a window, by the time its chunk passes take in chunks (256 CUs, a
// workgroup each; the carry pass is counted alike, though two fit and take 1.4 times
// one's time; each segment joined 3/4 of a chunk, the launches four).  Measured on MI355X,
// one sequence of 12 heads (64, 128), bf16, with and without: 16384 tokens 255 against 655
// us, 4096 94 against 173, 2048 66 against 97; 1024 tokens 58 either way, and two
// sequences of 2048 are left whole (98).
size_t segments_of(const DeltaLaunch &a) {
    const size_t chunks = chunks_of(a), heads = a.batch * a.heads, n = a.d_state <= 64 ? 64 : 128;
    const size_t tiles = (a.head_dim + kCols - 1) / kCols;
    const auto rounds = [](size_t wgs) { return (wgs + 255) / 256; };
    size_t best = 1, least = rounds(heads * tiles) * chunks;
    for (size_t count = 2; count <= 32 && count * 4 <= chunks; ++count) {
        const size_t each = (chunks + count - 1) / count;
        const size_t time = each * (rounds(heads * count * (tiles + n / kCols)) + rounds(heads * count * tiles)) + 4 + count * 3 / 4;
        if (time < least) {
            least = time;
            best = count;
        }
    }
    return best;
}
size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Where a call's segments lie in its workspace from byte `at` on.
struct SegmentPlan {
    size_t count, cols, n, carry, starts, bytes;
    SegmentPlan(const DeltaLaunch &a, size_t at) : count(segments_of(a)), cols(Kept(a).p64), n(Kept(a).n) {
        const size_t heads = a.batch * a.heads;
        carry = align256(at);
        starts = carry + (count > 1 ? heads * count * (cols + n) * n * sizeof(float) : 0);
        bytes = starts + (count > 1 ? heads * count * cols * n * sizeof(float) : 0);
    }
};

template <bool BACK>
size_t record_units(const DeltaLaunch &a) {
    size_t units = BackRecord::units;
    if (!BACK)
        (void)by_type(a.dtype, [&](auto t) {
            units = Record<decltype(t)>::units;
            return hipSuccess;
        });
    return units;
}
template <bool BACK>
size_t records_bytes(const DeltaLaunch &a) {
    return align256(a.batch * a.heads * chunks_of(a) * record_units<BACK>(a) * 1024);
}

// delta_prep, the segments' states where there is more than one, and the window's
// pass (BACK: the backward's way in).
template <bool BACK>
hipError_t launch(const DeltaLaunch &a, unsigned char *workspace, size_t segments_at, float *kept, hipStream_t s,
                  int &launches) {
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_state(a.d_state, [&](auto n) {
            constexpr int N = decltype(n)::value, MODE = BACK ? kKeep : kWindow;
            const int chunks = static_cast<int>(chunks_of(a));
            const unsigned heads = static_cast<unsigned>(a.batch * a.heads);
            const SegmentPlan plan(a, segments_at);
            const Segments sg{plan.count, (chunks + static_cast<int>(plan.count) - 1) / static_cast<int>(plan.count),
                              plan.cols, reinterpret_cast<float *>(workspace + plan.carry),
                              reinterpret_cast<float *>(workspace + plan.starts)};
            const unsigned tiles = static_cast<unsigned>(BACK ? kept_cols(a) : (a.head_dim + kCols - 1) / kCols);
            const auto go = [&](auto vec) {
                constexpr bool VEC = decltype(vec)::value;
                constexpr unsigned threads = kChunkThreads<T, VEC, MODE != kWindow>;
                constexpr unsigned carry_threads = kChunkThreads<T, VEC, true>;
                hipLaunchKernelGGL((delta_prep<T, N, VEC, BACK>), dim3(heads * chunks), dim3(256), 0, s, a, workspace,
                                   chunks);
                if (plan.count > 1) {
                    const dim3 carry(heads * static_cast<unsigned>(plan.count),
                                     static_cast<unsigned>((plan.cols + N) / kCols));
                    hipLaunchKernelGGL((delta_chunks<T, N, VEC, kCarry, BACK>), carry, dim3(carry_threads), 0, s, a, workspace,
                                       chunks, kept, sg);
                    hipLaunchKernelGGL((delta_join<N>), dim3(heads, static_cast<unsigned>(plan.cols / 16)), dim3(4 * N), 0,
                                       s, a, sg);
                    launches += 2;
                }
                hipLaunchKernelGGL((delta_chunks<T, N, VEC, MODE, BACK>),
                                   dim3(heads * static_cast<unsigned>(plan.count), tiles), dim3(threads), 0, s, a,
                                   workspace, chunks, kept, sg);
                launches += 2;
                return hipGetLastError();
            };
            return rows_vec(a, sizeof(T)) ? go(std::true_type{}) : go(std::false_type{});
        });
    });
}

}  // namespace

// 16-byte access to the rows of q, k, v and y: whole pieces of eight, every row
// aligned; a chunk's offsets below 2^31.
bool delta::rows_vec(const DeltaLaunch &a, size_t size) {
    const auto ok = [&](const void *p, size_t stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0 &&
               (stride + 1024) * size * kC < size_t(1) << 31;
    };
    return a.d_state % 8 == 0 && a.head_dim % 8 == 0 && ok(a.q, a.qs) && ok(a.k, a.ks) && ok(a.v, a.vs) &&
           ok(a.y, a.heads * a.head_dim);
}

size_t delta::delta_states_workspace(const DeltaLaunch &a, size_t &kept_at) {
    const size_t records = records_bytes<true>(a);
    kept_at = records;
    return SegmentPlan(a, records + a.batch * a.heads * chunks_of(a) * Kept(a).floats() * sizeof(float)).bytes;
}

hipError_t delta::launch_delta_states(const DeltaLaunch &a, unsigned char *workspace, hipStream_t s, int &launches) {
    size_t kept_at = 0;
    delta_states_workspace(a, kept_at);
    return launch<true>(a, workspace, kept_at + a.batch * a.heads * chunks_of(a) * Kept(a).floats() * sizeof(float),
                        reinterpret_cast<float *>(workspace + kept_at), s, launches);
}

// Against the recurrence token by token, which reads and writes the state once and
// then takes its tokens one by one.  Measured on MI355X, heads of (64, 128) bf16,
// recurrence and chunks: 96 heads 16 tokens 17.2 and 19.7 us a call, 24 tokens 23.5
// and 19.4; 1536 heads 16 tokens 61 and 118, 32 tokens 112 and 123, 48 tokens 165 and
// 127.
bool delta_chunk_wanted(const DeltaLaunch &a) {
    return a.d_state <= 128 && a.seq > (a.batch * a.heads >= 1024 ? 32u : 16u);
}

size_t delta_chunk_workspace(const DeltaLaunch &a) { return SegmentPlan(a, records_bytes<false>(a)).bytes; }

hipError_t launch_delta_chunk(const DeltaLaunch &a, void *workspace, hipStream_t s, int &launches) {
    return launch<false>(a, static_cast<unsigned char *>(workspace), records_bytes<false>(a), nullptr, s, launches);
}

}  // namespace m3
