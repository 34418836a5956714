// Gradients of the gated delta rule on gfx950, by the reverse of its
// recurrence (S~ = exp(g) S, e = v - S~ k, u = beta e, S' = S~ + u k^T,
// y = scale S' q):
//   dS' += scale dy q^T;  dq = scale S'^T dy;  du = dS' k;  dk = dS'^T u
//   dbeta = du . e;  de = beta du;  dv = de
//   dS~ = dS' - de k^T;  dk -= S~^T de;  dg = <dS~, S~>;  dS = exp(g) dS~
// Two launches a sequence walk: forward, leaving every S~ in the workspace,
// and back; a third sums dq and dk over the heads of a group and takes them
// through the unit-length norm.
#include "delta.hpp"

namespace m3 {
namespace {

using namespace delta;

constexpr int kThreads = 256;

__device__ float block_sum(float v, float *red) {
    v = group_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < kThreads / 64; ++i) s += red[i];
    return s;
}

// One workgroup a (sequence, head): thread i holds rows of P through LDS
// vectors of k and q; S lives in global memory (states).
template <typename T>
__global__ void __launch_bounds__(kThreads)
delta_backward_walk(DeltaLaunch a, DeltaGrads gr, float *states, float *dqh, float *dkh, float *dS) {
    extern __shared__ float lds[];
    __shared__ float red[kThreads / 64];
    const int tid = threadIdx.x;
    const int N = static_cast<int>(a.d_state), P = static_cast<int>(a.head_dim), PN = P * N;
    float *kv = lds, *qv = kv + N, *ev = qv + N, *uv = ev + P, *yv = uv + P;
    const size_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads, kg = h / (a.heads / a.groups);
    const int L = static_cast<int>(a.seq), len = valid_len(a.lengths, b, L);
    float *st = states + bh * L * PN;
    float *ds = dS + bh * PN;
    const auto load_kq = [&](size_t tok) {
        __syncthreads();
        const T *kp = static_cast<const T *>(a.k) + tok * a.ks + kg * N;
        const T *qp = static_cast<const T *>(a.q) + tok * a.qs + kg * N;
        float sk = 0.f, sq = 0.f;
        for (int i = tid; i < N; i += kThreads) {
            const float x = ldf(kp + i), y = ldf(qp + i);
            kv[i] = x;
            qv[i] = y;
            sk += x * x;
            sq += y * y;
        }
        if (a.qk_norm) {
            const float rk = 1.0f / sqrtf(block_sum(sk, red) + kUnitEps);
            const float rq = 1.0f / sqrtf(block_sum(sq, red) + kUnitEps);
            for (int i = tid; i < N; i += kThreads) {
                kv[i] *= rk;
                qv[i] *= rq;
            }
        }
        __syncthreads();
    };
    // forward: st[t] = S~ of token t
    for (int t = 0; t < len; ++t) {
        const size_t tok = b * L + t;
        const float al = expf(clamp_decay(a.g[tok * a.heads + h]));
        float *cur = st + static_cast<size_t>(t) * PN;
        if (t > 0) {
            const float *pre = cur - PN;
            for (int i = tid; i < PN; i += kThreads) cur[i] = al * (pre[i] + uv[i / N] * kv[i % N]);
        } else {
            for (int i = tid; i < PN; i += kThreads) cur[i] = a.state ? al * a.state[bh * PN + i] : 0.f;
        }
        load_kq(tok);
        const float beta = a.beta[tok * a.heads + h];
        for (int p = tid; p < P; p += kThreads) {
            float d = 0.f;
            for (int i = 0; i < N; ++i) d += cur[p * N + i] * kv[i];
            uv[p] = beta * (ldf(static_cast<const T *>(a.v) + tok * a.vs + h * P + p) - d);
        }
        __syncthreads();
    }
    for (int i = tid; i < PN; i += kThreads) ds[i] = gr.dstate ? gr.dstate[bh * PN + i] : 0.f;
    for (int t = L - 1; t >= len; --t) {
        const size_t tok = b * L + t;
        for (int i = tid; i < N; i += kThreads)
            dqh[(tok * a.heads + h) * N + i] = dkh[(tok * a.heads + h) * N + i] = 0.f;
        for (int p = tid; p < P; p += kThreads) stf(static_cast<T *>(gr.dv) + (tok * a.heads + h) * P + p, 0.f);
        if (tid == 0) gr.dg[tok * a.heads + h] = gr.dbeta[tok * a.heads + h] = 0.f;
    }
    for (int t = len - 1; t >= 0; --t) {
        const size_t tok = b * L + t, th = tok * a.heads + h;
        const float *cur = st + static_cast<size_t>(t) * PN;
        load_kq(tok);
        const float beta = a.beta[th], al = expf(clamp_decay(a.g[th]));
        float sb = 0.f;
        for (int p = tid; p < P; p += kThreads) {
            const float dy = a.scale * ldf(static_cast<const T *>(gr.dy) + th * P + p);
            float d = 0.f, du = 0.f;
            for (int i = 0; i < N; ++i) {
                d += cur[p * N + i] * kv[i];
                ds[p * N + i] += dy * qv[i];
                du += ds[p * N + i] * kv[i];
            }
            const float e = ldf(static_cast<const T *>(a.v) + tok * a.vs + h * P + p) - d;
            sb += du * e;
            uv[p] = beta * e;
            ev[p] = beta * du;
            yv[p] = dy;
            stf(static_cast<T *>(gr.dv) + th * P + p, beta * du);
        }
        sb = block_sum(sb, red);   // its barriers also publish uv, ev, yv and dS
        for (int i = tid; i < N; i += kThreads) {
            float dq = 0.f, dk = 0.f;
            for (int p = 0; p < P; ++p) {
                dq += yv[p] * (cur[p * N + i] + uv[p] * kv[i]);
                dk += ds[p * N + i] * uv[p] - cur[p * N + i] * ev[p];
            }
            dqh[th * N + i] = dq;
            dkh[th * N + i] = dk;
        }
        __syncthreads();
        float sg = 0.f;
        for (int p = tid; p < P; p += kThreads)
            for (int i = 0; i < N; ++i) {
                const float x = ds[p * N + i] - ev[p] * kv[i];
                sg += x * cur[p * N + i];
                ds[p * N + i] = al * x;
            }
        sg = block_sum(sg, red);
        if (tid == 0) {
            gr.dg[th] = sg;
            gr.dbeta[th] = sb;
        }
    }
    __syncthreads();
    if (gr.dstate0)
        for (int i = tid; i < PN; i += kThreads) gr.dstate0[bh * PN + i] = ds[i];
}

// One wave a (token, group).
template <typename T>
__global__ void __launch_bounds__(64) delta_backward_heads(DeltaLaunch a, DeltaGrads gr, const float *dqh, const float *dkh) {
    const size_t tg = blockIdx.x, tok = tg / a.groups, kg = tg % a.groups, rep = a.heads / a.groups;
    const int N = static_cast<int>(a.d_state), lane = threadIdx.x;
    for (int which = 0; which < 2; ++which) {
        const float *src = (which ? dkh : dqh) + (tok * a.heads + kg * rep) * N;
        const T *x = which ? static_cast<const T *>(a.k) + tok * a.ks + kg * N
                           : static_cast<const T *>(a.q) + tok * a.qs + kg * N;
        T *out = static_cast<T *>(which ? gr.dk : gr.dq) + tg * N;
        float d[4], xv[4], ss = 0.f, sd = 0.f;
        for (int j = 0; j < 4; ++j) {
            const int n = lane + 64 * j;
            d[j] = xv[j] = 0.f;
            if (n >= N) continue;
            for (size_t r = 0; r < rep; ++r) d[j] += src[r * N + n];
            xv[j] = ldf(x + n);
            ss += xv[j] * xv[j];
            sd += xv[j] * d[j];
        }
        float r = 1.f, c = 0.f;
        if (a.qk_norm) {
            r = 1.0f / sqrtf(group_sum(ss, 64) + kUnitEps);
            c = group_sum(sd, 64) * r * r;
        }
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < N)
                // d == 0: a padding token, whatever it holds
                stf(out + lane + 64 * j, d[j] == 0.f && c != c ? 0.f : r * (d[j] - xv[j] * c));
    }
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

size_t delta_backward_workspace(const DeltaLaunch &a) {
    const size_t pn = a.head_dim * a.d_state, bh = a.batch * a.heads;
    return align256(bh * a.seq * pn * 4) + 2 * align256(bh * a.seq * a.d_state * 4) + align256(bh * pn * 4);
}

hipError_t launch_delta_backward(const DeltaLaunch &a, const DeltaGrads &g, void *workspace,
                                 hipStream_t s, int &launches) {
    const size_t pn = a.head_dim * a.d_state, bh = a.batch * a.heads;
    char *w = static_cast<char *>(workspace);
    float *states = reinterpret_cast<float *>(w);
    w += align256(bh * a.seq * pn * 4);
    float *dqh = reinterpret_cast<float *>(w);
    w += align256(bh * a.seq * a.d_state * 4);
    float *dkh = reinterpret_cast<float *>(w);
    w += align256(bh * a.seq * a.d_state * 4);
    float *dS = reinterpret_cast<float *>(w);
    const size_t lds = (2 * a.d_state + 3 * a.head_dim) * 4;
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (bh == 0) return hipSuccess;
        hipLaunchKernelGGL(delta_backward_walk<T>, dim3(static_cast<unsigned>(bh)), dim3(kThreads), lds, s, a,
                           g, states, dqh, dkh, dS);
        ++launches;
        if (a.seq > 0) {
            hipLaunchKernelGGL(delta_backward_heads<T>, dim3(static_cast<unsigned>(a.batch * a.seq * a.groups)),
                               dim3(64), 0, s, a, g, dqh, dkh);
            ++launches;
        }
        return hipGetLastError();
    });
}

}  // namespace m3
