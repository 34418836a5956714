// The chunked form of the gated delta rule: what its forward and backward
// kernels share.
//
// A chunk is C = 64 tokens.  With G the running sum of its log decays (taken in
// f64, so that a difference of two is exact to f32 however large they are),
// D_ij = exp(G_i - G_j), M_ij = D_ij k_i.k_j (j < i) and T = (I + M diag(beta))^-1:
//   R = V - diag(exp G) K S0^T        what the state before the chunk leaves of v
//   E = T R                           each token's prediction error
//   Y = scale (diag(exp G) Q S0^T + (tril(Q K^T) . D) diag(beta) E)
//   S1 = exp(G_C) S0 + (diag(beta exp(G_C - G)) E)^T K
// T depends on the keys alone, so every chunk's is formed at once (delta_prep);
// only S passes from chunk to chunk.
//
// Numbers.  Products run on the bf16 MFMA.  An f32 operand goes in as a sum of
// bf16 parts, x = x0 + x1 + x2 (each rounding what the ones before left), which
// is exact to 24 bits in three and to 16 in two; products of parts whose order
// falls below the last are left out.  bf16 inputs are one part, f16 two, f32
// three.  Row factors (decay, beta, the unit-length norm's) multiply f32
// accumulators, never an operand before its rounding.
//
// Registers.  A 16x16 accumulator tile holds rows 4g + r in lane group g, and a
// 16x16x32 operand takes eight k a lane in any order that both operands share:
// two accumulator tiles (rows 4g .. 4g+3 of each) are an operand as they lie.
// So a wave that owns 16 columns of P takes its columns of S, R and E from
// product to product in registers; what it reads from LDS are the chunk's own
// operands.  Rows of S's tiles are n = 32 (nt / 2) + 8g + 4 (nt % 2) + r, so that
// the pair of them takes eight consecutive n of a K row; rows of R's and E's
// tiles are tokens 16 i + 4g + r.
#pragma once

#include "delta.hpp"
#include "scan_common.hpp"

namespace m3 {
namespace delta {

constexpr int kC = 64;          // tokens of a chunk
constexpr int kTri = 6;         // 16 x 32 blocks of a triangular 64 x 64 operand

// bf16 parts of a stored value.
template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int in = 1, out = 2; };
template <> struct Parts<f16_t> { static constexpr int in = 2, out = 2; };
template <> struct Parts<float> { static constexpr int in = 3, out = 3; };
constexpr int kNP = 3;          // of an f32 value on the way of the state

// x = out[0] + out[1] + ...
template <int NP>
__device__ __forceinline__ void split8(const float *x, bf16x8 *out) {
    typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        u32x4v w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
            if (p + 1 < NP) {
                r[2 * i] -= __uint_as_float(w[i] << 16);
                r[2 * i + 1] -= __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
        out[p] = __builtin_bit_cast(bf16x8, w);
    }
}
// Two accumulator tiles as an operand.
template <int NP>
__device__ __forceinline__ void split_tiles(f32x4 lo, f32x4 hi, bf16x8 *out) {
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    split8<NP>(x, out);
}

// acc[m] + A[m] B for M tiles over the products of parts up to order max(NA, NB)
// - 1, the smallest first.  The tiles take turns, so that no product waits for
// the one before it.
template <int M, int NA, int NB>
__device__ __forceinline__ void mma_rows(const bf16x8 (*a)[NA], const bf16x8 *b, f32x4 *acc) {
    constexpr int top = (NA > NB ? NA : NB) - 1;
#pragma unroll
    for (int o = top; o >= 0; --o)
#pragma unroll
        for (int i = 0; i <= o; ++i)
            if (i < NA && o - i < NB)
#pragma unroll
                for (int m = 0; m < M; ++m) acc[m] = mfma_bf16(a[m][i], b[o - i], acc[m]);
}
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma_parts(const bf16x8 *a, const bf16x8 *b, f32x4 acc) {
    mma_rows<1, NA, NB>(reinterpret_cast<const bf16x8(*)[NA]>(a), b, &acc);
    return acc;
}
// Matrix products of a region in turn with the vector work beside them: `n`
// times one MFMA and `valu` VALU instructions.
template <int n, int valu>
__device__ __forceinline__ void interleave() {
#pragma unroll
    for (int i = 0; i < n; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, valu, 0);
    }
}

// The rows of a chunk's q, k or v (or dy): `live` tokens `stride` elements apart.
// VEC: through a buffer resource that ends with the last of them, so that a
// load past it gives zeros without a branch (loads behind branches wait for one
// another); the host sees to it that a chunk's offsets fit 31 bits.  Else by
// pointer, element by element.
template <typename T, bool VEC>
struct Rows {
    rsrc_t r;
    const T *p;
    uint32_t step;      // bytes between tokens
    size_t stride;
    int live, width;
    __device__ __forceinline__ Rows(const T *base, size_t st, int lv, int w)
        : p(base), step(static_cast<uint32_t>(st * sizeof(T))), stride(st), live(lv < kC ? lv : kC), width(w) {
        if constexpr (VEC) r = make_rsrc(base, live > 0 ? (live - 1) * step + w * sizeof(T) : 0u);
    }
};

// Byte offset of values n, n + 1, .. of token t in such rows, past any range from
// `width` on.
template <typename T>
__device__ __forceinline__ uint32_t row_off(size_t stride, int width, int t, int n) {
    return n < width ? (t * static_cast<uint32_t>(stride) + n) * static_cast<uint32_t>(sizeof(T)) : 0x80000000u;
}

// Eight consecutive stored values of token t + dt as loaded; zero from `live` and
// from `width` on.  VEC reads at off + dt * step, off = row_off(t, n): what does
// not change from chunk to chunk stays with the caller.
template <typename T> struct Eight { u32x4 q; };
template <> struct Eight<float> { u32x4 a, b; };

template <typename T, bool VEC>
__device__ __forceinline__ Eight<T> load_eight(const Rows<T, VEC> &rows, uint32_t off, int t, int n, int dt) {
    Eight<T> e;
    if constexpr (VEC) {
        const uint32_t o = off + dt * rows.step;
        if constexpr (sizeof(T) == 4) {
            e.a = bld16(rows.r, o);
            e.b = bld16(rows.r, o + 16);
        } else {
            e.q = bld16(rows.r, o);
        }
    } else {
        const T *row = rows.p + (t + dt) * rows.stride;
        uint32_t u[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (t + dt >= rows.live || n + i >= rows.width) continue;
            if constexpr (sizeof(T) == 4)
                u[i] = __float_as_uint(row[n + i]);
            else
                u[i >> 1] |= static_cast<uint32_t>(row[n + i].bits) << (16 * (i & 1));
        }
        if constexpr (sizeof(T) == 4) {
            e.a = u32x4{u[0], u[1], u[2], u[3]};
            e.b = u32x4{u[4], u[5], u[6], u[7]};
        } else {
            e.q = u32x4{u[0], u[1], u[2], u[3]};
        }
    }
    return e;
}
template <typename T, bool VEC>
__device__ __forceinline__ Eight<T> load_eight(const Rows<T, VEC> &rows, int t, int n) {
    return load_eight(rows, row_off<T>(rows.stride, rows.width, t, n), t, n, 0);
}
// One stored value as loaded (its bits), and what it stands for.
template <typename T, bool VEC>
__device__ __forceinline__ uint32_t load_one(const Rows<T, VEC> &rows, uint32_t off, int t, int n, int dt) {
    if constexpr (VEC) {
        const uint32_t o = off + dt * rows.step;
        if constexpr (sizeof(T) == 4) return bld4(rows.r, o);
        else return __builtin_amdgcn_raw_buffer_load_b16(rows.r, o, 0, 0);
    } else {
        if (t + dt >= rows.live || n >= rows.width) return 0u;
        if constexpr (sizeof(T) == 4) return __float_as_uint(rows.p[(t + dt) * rows.stride + n]);
        else return rows.p[(t + dt) * rows.stride + n].bits;
    }
}
// The same rows written: a value past their range is dropped.
template <typename T, bool VEC>
__device__ __forceinline__ void store_one(const Rows<T, VEC> &rows, uint32_t off, int t, int n, int dt, float v) {
    T x;
    stf(&x, v);
    if constexpr (VEC) {
        const uint32_t o = off + dt * rows.step;
        if constexpr (sizeof(T) == 4) bst4(__float_as_uint(x), rows.r, o);
        else bst2(x.bits, rows.r, o);
    } else {
        if (t + dt < rows.live && n < rows.width) const_cast<T *>(rows.p)[(t + dt) * rows.stride + n] = x;
    }
}
template <typename T>
__device__ __forceinline__ float value_of(uint32_t bits) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(bits);
    } else {
        const T v{static_cast<uint16_t>(bits)};
        return ldf(&v);
    }
}
__device__ __forceinline__ void widen(const Eight<float> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = __uint_as_float(r.a[i]);
        f[4 + i] = __uint_as_float(r.b[i]);
    }
}
__device__ __forceinline__ void widen(const Eight<bf16_t> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(r.q[i] << 16);
        f[2 * i + 1] = __uint_as_float(r.q[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void widen(const Eight<f16_t> &r, float *f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.q[i])));
        f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.q[i] >> 16)));
    }
}
template <typename T>
__device__ __forceinline__ void to_parts(const Eight<T> &r, bf16x8 *out) {
    if constexpr (sizeof(T) == 2 && Parts<T>::in == 1) {
        out[0] = __builtin_bit_cast(bf16x8, r.q);
    } else {
        float f[8];
        widen(r, f);
        split8<Parts<T>::in>(f, out);
    }
}

// Rows of a chunk in LDS, [token][N] of 16-bit values, a row's 16-byte pieces
// permuted so that both ways of reading them fall on different banks: sixteen
// rows' pieces at one place (an operand's rows), and four rows' by four pieces
// (a transposed operand).
template <int N>
__device__ __forceinline__ constexpr int swizzle(int t) {
    return N == 128 ? (t & 3) << 2 | ((t >> 2) & 3) : N == 64 ? ((t >> 1) & 1) << 2 | ((t >> 2) & 3) : 0;
}
template <int N> struct Tile {
    static constexpr int bytes = kC * N * 2;
};
template <int N>
__device__ __forceinline__ int tile_at(int t, int piece) {
    return t * (2 * N) + ((piece ^ swizzle<N>(t)) << 4);
}
// Operand rows 16 i + c, columns 32 kk + 8g ..
template <int N>
__device__ __forceinline__ bf16x8 tile_rows(const unsigned char *t, int i, int kk, int lane) {
    return *reinterpret_cast<const bf16x8 *>(t + 16 * i * (2 * N) + tile_at<N>(lane & 15, 4 * kk + (lane >> 4)));
}
// The tile transposed: operand rows are the n of tile nt, k runs over the tokens
// of k-step kk in the order of two accumulator tiles.
template <int N>
__device__ __forceinline__ bf16x8 tile_cols(const unsigned char *t, int nt, int kk, int lane) {
    const int l = lane & 15, g = lane >> 4;
    const unsigned char *p = t + 32 * kk * (2 * N) + tile_at<N>(4 * g + (l >> 2), 4 * (nt >> 1) + (l & 3)) + 8 * (nt & 1);
    const bf16x4 lo = scan::lds_read_tr16(reinterpret_cast<const __bf16 *>(p));
    const bf16x4 hi = scan::lds_read_tr16(reinterpret_cast<const __bf16 *>(p + 16 * (2 * N)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Sixteen columns from 16 w on of an M-wide tile as accumulator tile i holds them.
template <int M>
__device__ __forceinline__ bf16x4 tile_acc(const unsigned char *t, int i, int w, int lane) {
    const int l = lane & 15, g = lane >> 4, q = l & 3;
    const unsigned char *p = t + 16 * i * (2 * M) + tile_at<M>(4 * g + (l >> 2), 2 * w + (q >> 1)) + 8 * (q & 1);
    return scan::lds_read_tr16(reinterpret_cast<const __bf16 *>(p));
}
// The n of row r of lane group g of S's tile nt.
__device__ __forceinline__ constexpr int state_n(int nt, int g, int r) {
    return 32 * (nt >> 1) + 8 * g + 4 * (nt & 1) + r;
}

// A tile's rows straight from memory to LDS by one of four waves: kilobytes w, w
// + 4, ..  `at` is this lane's place (dma_at), the same for all of them.
template <typename T, int N>
__device__ __forceinline__ uint32_t dma_at(size_t stride, int width, int n0, int w, int lane) {
    const int t = w * (512 / N) + lane / (N / 8);
    const int n = n0 + ((lane % (N / 8)) ^ swizzle<N>(t)) * 8;
    return row_off<T>(stride, width, t, n);
}
template <int N, typename R>
__device__ __forceinline__ void dma_tile(const R &rows, uint32_t at, unsigned char *tile, int w) {
#pragma unroll
    for (int i = 0; i < N / 32; ++i)
        scan::lds_dma16(rows.r, scan::lds_addr(tile + (w + 4 * i) * 1024), at + i * (2048 / N) * rows.step);
}

// Block (i, kk) of a lower- or upper-triangular 64 x 64 operand (rows 16 i,
// columns 32 kk) among its kTri stored ones, row by row.
__device__ __forceinline__ constexpr int lower_block(int i, int kk) { return i < 2 ? i : 2 * (i - 1) + kk; }
__device__ __forceinline__ constexpr int upper_block(int i, int kk) { return i < 2 ? 2 * i + kk : i + 2; }

// What delta_prep leaves for a chunk of a head, in kilobytes: row factors, then
// triangular operands block by block, part by part, sixteen bytes a lane.  The
// window's kernel takes T and the attention scale (tril(Q K^T) . D) diag(beta);
// the backward's T for the states on the way in and both transposed for the way
// back.
constexpr int kFacK = 0, kFacQ = 64, kFacU = 128, kFacEnd = 192;   // floats: exp(G) rk, scale exp(G) rq,
                                                                   // beta exp(G_C - G) rk, exp(G_C)
constexpr int kTriT = kTri * kNP;                                  // kilobytes of T
template <typename T> struct Record {
    static constexpr int t = 1, p = t + kTriT, units = p + kTri * Parts<T>::out;
};
struct BackRecord {
    static constexpr int t = 1, tt = t + kTriT, pt = tt + kTriT, units = pt + kTriT;
};

// Columns of P that a workgroup of the chunk kernels takes: two tiles, each a
// pair of waves' whose halves of N meet in LDS.
constexpr int kCols = 32;

// The fetch of a chunk's operands to LDS: K, Q, a tile of v (or dy), and UNITS
// kilobytes of its record (unit u > 0 from kilobyte u + GAP).  bf16 with aligned
// rows (DMA): straight from memory, by a fifth wave that does nothing else (issuing
// them stalls a wave some 100 cycles a kilobyte), or by the four waves themselves
// (SELF).  Other inputs become their bf16 parts on the way, through registers; v stays
// there.
template <typename T, bool VEC> constexpr bool kDma = VEC && std::is_same<T, bf16_t>::value;
template <typename T, bool VEC, bool SELF = false> constexpr unsigned kChunkThreads = kDma<T, VEC> && !SELF ? 320 : 256;
template <typename T, int N, bool VEC, bool WITHQ, int UNITS, int GAP, bool SELF = false>
struct Stage {
    static constexpr int KP = Parts<T>::in;
    static constexpr bool DMA = kDma<T, VEC>;
    static constexpr int pieces = kC * N / 8 / 256, rpieces = UNITS / 4 + 1;
    struct Rows1 { unsigned char part[KP][Tile<N>::bytes]; };
    struct Rec { unsigned char at[UNITS * 1024]; };
    struct V { unsigned char at[DMA ? Tile<kCols>::bytes : 16]; };
    const T *kp, *qp, *vp;              // the sequence's rows of this head
    size_t ks, qs, vs, rec_bytes;
    const unsigned char *rec;           // the sequence's records
    int len, n_of, P, wave, w, lane;    // wave: 4 is the DMA's, unless SELF; w: its tile of columns
    static constexpr int own = SELF ? 1 : 4;
    uint32_t dk[own], dq[own], dv[own];   // DMA: places in a kilobyte, by kilobyte modulo 4
    int kt, kn, vt, vn;                 // else: this thread's places
    uint32_t k_at, q_at, v_at;
    Eight<T> k8[pieces], q8[WITHQ ? pieces : 1];
    u32x4 r8[rpieces];
    uint32_t v1[4][4];

    __device__ __forceinline__ Stage(const DeltaLaunch &a, size_t b, size_t h, int length, const T *v, size_t vstride,
                                     int p0, const unsigned char *records, size_t record_bytes) {
        const int tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        w = wave >> 1;
        len = length;
        n_of = static_cast<int>(a.d_state);
        P = static_cast<int>(a.head_dim);
        const size_t kg = h / (a.heads / a.groups);
        ks = a.ks;
        qs = a.qs;
        vs = vstride;
        kp = static_cast<const T *>(a.k) + b * a.seq * ks + kg * n_of;
        qp = static_cast<const T *>(a.q) + b * a.seq * qs + kg * n_of;
        vp = v;
        rec = records;
        rec_bytes = record_bytes;
        kt = tid / (N / 8);
        kn = tid % (N / 8) * 8;
        vt = 4 * (lane >> 4);
        vn = p0 + 16 * w + (lane & 15);
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < own; ++i) {
                dk[i] = dma_at<T, N>(ks, n_of, 0, nth(i), lane);
                dq[i] = dma_at<T, N>(qs, n_of, 0, nth(i), lane);
                dv[i] = dma_at<T, kCols>(vs, P, p0, nth(i), lane);
            }
        } else {
            k_at = row_off<T>(ks, n_of, kt, kn);
            q_at = row_off<T>(qs, n_of, kt, kn);
            v_at = row_off<T>(vs, P, vt, vn);
        }
    }
    __device__ __forceinline__ int nth(int i) const { return SELF ? wave : i; }
    __device__ __forceinline__ rsrc_t record(int ck) const { return make_rsrc(rec + ck * rec_bytes, static_cast<uint32_t>(rec_bytes)); }
    static __device__ __forceinline__ constexpr int unit(int u) { return u == 0 ? 0 : u + GAP; }
    __device__ __forceinline__ Rows<T, VEC> rows_of(const T *p, size_t stride, int ck, int width) const {
        return Rows<T, VEC>(p + static_cast<size_t>(ck) * kC * stride, stride, len - ck * kC, width);
    }

    __device__ __forceinline__ void dma_k(Rows1 &to, int ck) const {
        const Rows<T, VEC> rows = rows_of(kp, ks, ck, n_of);
#pragma unroll
        for (int i = 0; i < own; ++i) dma_tile<N>(rows, dk[i], to.part[0], nth(i));
    }
    __device__ __forceinline__ void dma_q(Rows1 &to, int ck) const {
        const Rows<T, VEC> rows = rows_of(qp, qs, ck, n_of);
#pragma unroll
        for (int i = 0; i < own; ++i) dma_tile<N>(rows, dq[i], to.part[0], nth(i));
    }
    __device__ __forceinline__ void dma_v(V &to, int ck) const {
        const Rows<T, VEC> rows = rows_of(vp, vs, ck, P);
#pragma unroll
        for (int i = 0; i < own; ++i) dma_tile<kCols>(rows, dv[i], to.at, nth(i));
    }
    template <int FROM, int END>   // kilobytes FROM .. of the record, to where its first would lie at `to`
    __device__ __forceinline__ void dma_rec(unsigned char *to, int ck) const {
        const rsrc_t r = record(ck);
#pragma unroll
        for (int i = 0; i < (END - FROM + 4 / own - 1) / (4 / own); ++i) {
            const int u = FROM + (SELF ? wave + 4 * i : i);
            if (u < END) scan::lds_dma16(r, scan::lds_addr(to + u * 1024), unit(u) * 1024 + lane * 16);
        }
    }
    __device__ __forceinline__ void fetch(int ck) {
        const Rows<T, VEC> kr = rows_of(kp, ks, ck, n_of), qr = rows_of(qp, qs, ck, n_of), vr = rows_of(vp, vs, ck, P);
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            k8[i] = load_eight(kr, k_at, kt, kn, i * (2048 / N));
            if constexpr (WITHQ) q8[i] = load_eight(qr, q_at, kt, kn, i * (2048 / N));
        }
        const rsrc_t r = record(ck);
#pragma unroll
        for (int i = 0; i < rpieces; ++i) r8[i] = bld16(r, unit(wave + 4 * i) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r1 = 0; r1 < 4; ++r1) v1[i][r1] = load_one(vr, v_at, vt, vn, 16 * i + r1);
    }
    __device__ __forceinline__ void put(Rows1 &k, Rows1 &q, Rec &to) const {
#pragma unroll
        for (int i = 0; i < pieces; ++i) {
            bf16x8 x[KP];
            const int at = tile_at<N>(kt + i * (2048 / N), kn / 8);
            to_parts(k8[i], x);
#pragma unroll
            for (int p = 0; p < KP; ++p) *reinterpret_cast<bf16x8 *>(k.part[p] + at) = x[p];
            if constexpr (WITHQ) {
                to_parts(q8[i], x);
#pragma unroll
                for (int p = 0; p < KP; ++p) *reinterpret_cast<bf16x8 *>(q.part[p] + at) = x[p];
            }
        }
#pragma unroll
        for (int i = 0; i < rpieces; ++i)
            if (wave + 4 * i < UNITS) *reinterpret_cast<u32x4 *>(to.at + (wave + 4 * i) * 1024 + lane * 16) = r8[i];
    }
    // v as accumulator tiles
    __device__ __forceinline__ void values(const V &from, f32x4 *e) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DMA) {
                const bf16x4 x = tile_acc<kCols>(from.at, i, w, lane);
#pragma unroll
                for (int r = 0; r < 4; ++r) e[i][r] = static_cast<float>(x[r]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) e[i][r] = value_of<T>(v1[i][r]);
            }
        }
    }
};

// Blocks of a lower (upper) triangle that take the first k-step, then those that
// take the second, with the accumulator tile each adds to.
template <int NP>
__device__ __forceinline__ bf16x8 tri_block(const unsigned char *base, int blk, int q, int lane) {
    return *reinterpret_cast<const bf16x8 *>(base + ((blk * NP + q) * 64 + lane) * 16);
}
template <int NP>
__device__ __forceinline__ void tri_load(const unsigned char *base, int lane, bf16x8 (*all)[NP], bf16x8 (*part)[NP],
                                         bool upper) {
    // lower: block 0: (0, 0), 1: (1, 0), 2: (2, 0), 3: (2, 1), 4: (3, 0), 5: (3, 1)
    // upper: 0: (0, 0), 1: (0, 1), 2: (1, 0), 3: (1, 1), 4: (2, 1), 5: (3, 1)
    const int al[4] = {0, 1, 2, 4}, pl[2] = {3, 5}, au[4] = {1, 3, 4, 5}, pu[2] = {0, 2};
#pragma unroll
    for (int q = 0; q < NP; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) all[i][q] = tri_block<NP>(base, upper ? au[i] : al[i], q, lane);
#pragma unroll
        for (int i = 0; i < 2; ++i) part[i][q] = tri_block<NP>(base, upper ? pu[i] : pl[i], q, lane);
    }
}

// The chunk kernels' launches for the other passes (delta_chunk.hip).
bool rows_vec(const DeltaLaunch &a, size_t size);
inline size_t chunks_of(const DeltaLaunch &a) { return (a.seq + kC - 1) / kC; }

template <typename F>
hipError_t by_state(size_t d_state, F f) {
    if (d_state <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

// What the backward keeps of each chunk of a head, f32: the state before it and
// the gradient of the state after it [P64][N] (P64: head_dim to the next multiple
// of 64, N: 64 or 128) as the accumulators hold them, tile by tile of 16 columns
// and 16 of N, a lane's four together, so that a wave's store is one kilobyte; E
// and dR [64][P64].
struct Kept {
    size_t p64, n;
    __host__ __device__ Kept(const DeltaLaunch &a) : p64((a.head_dim + 63) / 64 * 64), n(a.d_state <= 64 ? 64 : 128) {}
    // a lane's part of tile nt of columns p ..
    __device__ __forceinline__ size_t tile(int p, int nt, int lane) const {
        return ((p / 16) * (n / 16) + nt) * 256 + 4 * lane;
    }
    __host__ __device__ size_t s0() const { return 0; }
    __host__ __device__ size_t s1() const { return p64 * n; }
    __host__ __device__ size_t e() const { return 2 * p64 * n; }
    __host__ __device__ size_t dr() const { return 2 * p64 * n + kC * p64; }
    __host__ __device__ size_t floats() const { return 2 * p64 * (n + kC); }
};

// The backward's chunk kernels write all of P64.
inline size_t kept_cols(const DeltaLaunch &a) { return Kept(a).p64 / kCols; }

// A window's segments: how many, chunks of each, and where their states are, f32:
// carry [heads][count][cols + N][N] (Psi, then Phi), starts [heads][count][cols][N].
struct Segments {
    size_t count;
    int chunks;
    size_t cols;
    float *carry, *starts;
};

// delta_prep and the forward states of the backward (delta_chunk.hip): the
// workspace of both, with the records first and what is kept from byte kept_at on.
size_t delta_states_workspace(const DeltaLaunch &a, size_t &kept_at);
hipError_t launch_delta_states(const DeltaLaunch &a, unsigned char *workspace, hipStream_t s, int &launches);

}  // namespace delta
}  // namespace m3
