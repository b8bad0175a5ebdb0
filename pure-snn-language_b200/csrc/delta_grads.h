// delta_grads.h - gradients of a delta-rule scan, what is left beside the states'.
#pragma once
#include "delta_tile.h"

namespace snnb_delta {
// For all chunks at once.  With S before a chunk, D behind it, U and R as above, G the decays between steps:
//   p = G (Z U^T) (j <= i),   x = -b G (R U^T) (j < i)
//   dQ = since Z S^T + p K,   dK = -since b R S^T + until U D^T + x K + x^T K + p^T Q
//   db_i = R_i.V_i - since_i k_i.(S R_i) + sum_j x_ij k_i.k_j / b_i
// and for the logarithm of a decay all terms that it is a factor of: their sum over
// i >= t > j, as sums over rows less sums over columns from t on.
// Products over the values' columns have bf16 operands for bf16 tensors (as the results
// are rounded), otherwise f32 in two tf32 pieces; those over steps the keys' type, p and x in
// one piece of f16 for bf16 tensors, two for f16.  16 warps: 16 rows and a quarter
// of the columns each; half of an SM's registers are accumulators, so that S, D, U, R and dy are
// read once.  That leaves one CTA an SM, whose phases wait for one another: 8,192 chunks of 128 x 128
// bf16: kernel 911 us (280 at the copy rate; 800 with U and R in one piece, whose gradients are off by
// 2.5e-3 of their norm where these are by 1.9e-3 and the rounding alone makes 1.7e-3).
struct Ops16 {                 // one piece of a 16-bit type E
    template <typename E>
    static __device__ __forceinline__ void rows_of(unsigned (&a)[4], const E* m, int st) {  // A[i][k] = m[i][k]
        const int l = threadIdx.x & 31;
        ldsm4(a, m + (l & 15) * st + (l >> 4) * 8);
    }
    template <typename E>
    static __device__ __forceinline__ void columns_of(unsigned (&a)[4], const E* m, int st) {  // A[i][k] = m[k][i]
        const int l = threadIdx.x & 31;
        ldsm4t(a, m + ((l >> 4) * 8 + (l & 7)) * st + ((l >> 3) & 1) * 8);
    }
};
template <typename E> struct GradOps {
    struct A {
        unsigned v[4];
    };
    struct B {
        unsigned v[2];
    };
    static __device__ __forceinline__ A rows_of(const E* m, int st) {
        A a;
        Ops16::rows_of(a.v, m, st);
        return a;
    }
    static __device__ __forceinline__ A columns_of(const E* m, int st) {
        A a;
        Ops16::columns_of(a.v, m, st);
        return a;
    }
    static __device__ __forceinline__ void by_rows(B (&b)[2], const E* m, int st) {
        const int l = threadIdx.x & 31;
        unsigned r[4];
        ldsm4(r, m + ((l & 7) + (l >> 4) * 8) * st + ((l >> 3) & 1) * 8);
        b[0] = {{r[0], r[1]}};
        b[1] = {{r[2], r[3]}};
    }
    static __device__ __forceinline__ void by_columns(B (&b)[2], const E* m, int st) {
        const int l = threadIdx.x & 31;
        unsigned r[4];
        ldsm4t(r, m + ((l & 7) + ((l >> 3) & 1) * 8) * st + (l >> 4) * 8);
        b[0] = {{r[0], r[1]}};
        b[1] = {{r[2], r[3]}};
    }
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) {
        mma16<E>(d0, a.v, b[0].v);
        mma16<E>(d1, a.v, b[1].v);
    }
    template <int N>  // N pieces, planes of C * MS
    static __device__ __forceinline__ void put(E* m, float x, float y) {
#pragma unroll
        for (int p = 0; p < N; ++p) *reinterpret_cast<unsigned*>(m + p * C * MS) = piece<E>(x, y);
    }
};
template <> struct GradOps<float> : Path32 {
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) { full(d0, d1, a, b); }
    template <int N>
    static __device__ __forceinline__ void put(float* m, float x, float y) { *reinterpret_cast<float2*>(m) = make_float2(x, y); }
};

// A tile of R rows of W columns of F as E, r and w of them there, zeros in the others, by
// all threads: where rows are words of 16 bytes each thread takes the same places of every tile
constexpr int GRADS = 512;
template <typename E, int R, int W, typename F>
__device__ __forceinline__ void load_tile(E* to, const F* from, long long st, int r, int w, int word) {
    constexpr int V = 16 / (int)sizeof(E), N = W / V, STEP = GRADS / N;
    if (std::is_same<E, F>::value && word == 16) {
        const int c = threadIdx.x % N * V, row = threadIdx.x / N;
        to += row * (W + PAD) + c;
        const F* p = from + row * st + c;
#pragma unroll
        for (int a = 0; a < R; a += STEP) {
            const bool there = row + a < r && c < w;
            copy16(to + a * (W + PAD), there ? p + a * st : from, there);
        }
    } else {
        if constexpr (std::is_same<E, F>::value) {
            if (word == 8) return load_by<E, R, W, 8>(to, from, st, r, w, threadIdx.x, GRADS);
            if (word == 4) return load_by<E, R, W, 4>(to, from, st, r, w, threadIdx.x, GRADS);
        }
        for (int i = threadIdx.x; i < R * W; i += GRADS) {
            const int a = i / W, c = i - a * W;
            to[a * (W + PAD) + c] = from_f32<E>(a < r && c < w ? to_f32(from[a * st + c]) : 0.0f);
        }
    }
}
// the sum of products of the elements of two words of 16 bytes
__device__ __forceinline__ float word_dot(const float* a, const float* b, float sum) {
    const float4 x = *reinterpret_cast<const float4*>(a), y = *reinterpret_cast<const float4*>(b);
    return fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, sum))));
}
__device__ __forceinline__ float word_dot(const __nv_bfloat16* a, const __nv_bfloat16* b, float sum) {
    const uint4 x = *reinterpret_cast<const uint4*>(a), y = *reinterpret_cast<const uint4*>(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = of_pair<__nv_bfloat16>((&x.x)[i]), v = of_pair<__nv_bfloat16>((&y.x)[i]);
        sum = fmaf(u.x, v.x, fmaf(u.y, v.y, sum));
    }
    return sum;
}

template <typename T, int KD>
struct GradTile {
    using E = typename Kept<T>::K;             // of the blocks
    using KE = typename PathOf<T>::P::KE;      // of keys, p and x
    static constexpr int GW = sizeof(E) == 2 ? 64 : 32;  // columns of the values taken at a time
    static constexpr int STAGES = sizeof(E) == 2 ? 2 : 1, PIECES = sizeof(E) == 4 && sizeof(KE) == 2 ? 2 : 1;
    static constexpr int KEYS = C * (KD + PAD), ROWS = C * (GW + PAD), STATE = GW * (KD + PAD);
    static constexpr int PLANES = Kept<T>::PLANES;            // of U and R
    static constexpr int BLOCK = (2 + 2 * PLANES) * ROWS + 2 * STATE, SQ = PIECES * C * MS;
    // p and x take the blocks' place
    static constexpr int BLOCKS = STAGES * BLOCK * (int)sizeof(E), SQUARES = 2 * SQ * (int)sizeof(KE);
    static constexpr int BYTES = 2 * KEYS * (int)sizeof(KE) + SC * 4 + (BLOCKS > SQUARES ? BLOCKS : SQUARES);
};

template <typename T, int KD>
__global__ void __launch_bounds__(GRADS, 1) k_delta_grads(const __grid_constant__ DeltaArgs A) {
    using G = GradTile<T, KD>;
    using E = typename G::E;
    using KE = typename G::KE;
    using Op = GradOps<E>;
    using KOp = GradOps<KE>;
    constexpr bool SCALED = PathOf<T>::P::SCALED;
    constexpr int KS = KD + PAD, GW = G::GW, RS = GW + PAD, NQ = KD / 32, PIECES = G::PIECES;  // NQ: tiles of 8 columns of a warp
    extern __shared__ __align__(16) char smem[];
    KE *Ks = reinterpret_cast<KE*>(smem), *Qs = Ks + G::KEYS;
    float* F = reinterpret_cast<float*>(Qs + G::KEYS);
    E* blocks = reinterpret_cast<E*>(F + SC);
    KE *Ps = reinterpret_cast<KE*>(blocks), *Xs = Ps + G::SQ;
    __shared__ float rows[4][4][C], cols[4][C], more[GRADS / 32], dots[C], top[4][GRADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int wr = warp & 3, wc = warp >> 2, kh = blockIdx.y;
    const long long slot = blockIdx.x, s = sequence_of(A, slot);
    const Span sp = span_of(A, s);
    const long long first = (slot - sp.chunk) * C;
    if (first < 0 || first >= sp.len) return;
    const int t0 = (int)first, n = min(C, sp.len - t0);
    const KE* keys = (const KE*)A.keys + (slot * A.hk + kh) * 2 * G::KEYS;
    float tq[NQ][4] = {}, tk[NQ][4] = {};
    const int n_blocks = (A.vdim + GW - 1) / GW;
#pragma unroll 1
    for (int gi = 0; gi < A.group; ++gi) {
        const int head = kh * A.group + gi;
        const long long unit = slot * A.heads + head;
        auto load = [&](int b) {
            E* m = blocks + (G::STAGES == 2 ? (b & 1) * G::BLOCK : 0);
            const int c0 = b * GW, w = A.vdim - c0;
            load_tile<E, C, GW>(m, (const T*)A.dy.p + row_at(A, A.dy, s, sp, t0) + head * A.dy.hs + c0, A.dy.st, A.dy.p ? n : 0, w, A.dy.word);
            load_tile<E, C, GW>(m + G::ROWS, (const E*)A.u + unit * G::PLANES * C * A.vpad + c0, A.vpad, C, A.vpad - c0, 16);
            load_tile<E, C, GW>(m + 2 * G::ROWS, (const E*)A.dr + unit * G::PLANES * C * A.vpad + c0, A.vpad, C, A.vpad - c0, 16);
            if constexpr (G::PLANES == 2) {
                E* rest = m + 4 * G::ROWS + 2 * G::STATE;
                load_tile<E, C, GW>(rest, (const E*)A.u + (unit * 2 + 1) * C * A.vpad + c0, A.vpad, C, A.vpad - c0, 16);
                load_tile<E, C, GW>(rest + G::ROWS, (const E*)A.dr + (unit * 2 + 1) * C * A.vpad + c0, A.vpad, C, A.vpad - c0, 16);
            }
            load_tile<E, C, GW>(m + 3 * G::ROWS, (const T*)A.v.p + row_at(A, A.v, s, sp, t0) + head * A.v.hs + c0, A.v.st, n, w, A.v.word);
            load_tile<E, GW, KD>(m + 4 * G::ROWS, (const E*)A.states + (unit * A.vdim + c0) * KS, KS, w, KD, 16);
            load_tile<E, GW, KD>(m + 4 * G::ROWS + G::STATE, (const E*)A.dstates + (unit * A.vdim + c0) * KS, KS, w, KD, 16);
        };
        if (gi == 0) load_words(Ks, keys, 2 * G::KEYS * (int)sizeof(KE), tid, GRADS);
        load_words(F, A.factors + unit * SC, SC * 4, tid, GRADS);
        load(0);
        copies_end();
        float zq[NQ][4] = {}, zk[NQ][4] = {}, zm[NQ][4] = {}, p[2][4] = {}, x[2][4] = {};
        float inner = 0.0f, rv = 0.0f;  // <S, D>; R_i.V_i of row tid / 8
#pragma unroll 1
        for (int b = 0; b < n_blocks; ++b) {
            if (G::STAGES == 2 && b + 1 < n_blocks) load(b + 1);
            copies_end();
            copies_wait<G::STAGES == 2 ? 1 : 0>();
            __syncthreads();
            const E* m = blocks + (G::STAGES == 2 ? (b & 1) * G::BLOCK : 0);
            const E *Z = m, *U = m + G::ROWS, *R = m + 2 * G::ROWS, *V = m + 3 * G::ROWS, *S = m + 4 * G::ROWS, *D = S + G::STATE;
            [[maybe_unused]] const E *UL = D + G::STATE, *RL = UL + G::ROWS;  // the second pieces
#pragma unroll
            for (int k = 0; k < GW; k += 16) {
                const typename Op::A az = Op::rows_of(Z + wr * 16 * RS + k, RS), ar = Op::rows_of(R + wr * 16 * RS + k, RS);
                const typename Op::A au = Op::rows_of(U + wr * 16 * RS + k, RS);
                typename Op::A rl, ul;
                if constexpr (G::PLANES == 2) {
                    rl = Op::rows_of(RL + wr * 16 * RS + k, RS);
                    ul = Op::rows_of(UL + wr * 16 * RS + k, RS);
                }
                typename Op::B bb[2];
#pragma unroll
                for (int j = 0; j < NQ; j += 2) {
                    Op::by_columns(bb, S + k * KS + wc * (KD / 4) + j * 8, KS);
                    Op::mma(zq[j], zq[j + 1], az, bb);
                    if constexpr (G::PLANES == 2) Op::mma(zk[j], zk[j + 1], rl, bb);
                    Op::mma(zk[j], zk[j + 1], ar, bb);
                    Op::by_columns(bb, D + k * KS + wc * (KD / 4) + j * 8, KS);
                    if constexpr (G::PLANES == 2) Op::mma(zm[j], zm[j + 1], ul, bb);
                    Op::mma(zm[j], zm[j + 1], au, bb);
                }
                if (wc <= wr) {
                    if constexpr (G::PLANES == 2) {
                        Op::by_rows(bb, UL + wc * 16 * RS + k, RS);
                        Op::mma(p[0], p[1], az, bb);
                        Op::mma(x[0], x[1], ar, bb);
                    }
                    Op::by_rows(bb, U + wc * 16 * RS + k, RS);
                    Op::mma(p[0], p[1], az, bb);
                    if constexpr (G::PLANES == 2) Op::mma(x[0], x[1], rl, bb);
                    Op::mma(x[0], x[1], ar, bb);
                }
            }
            constexpr int V4 = 16 / (int)sizeof(E);
            static_assert(C * GW / V4 == GRADS, "a word of R and V to a thread");
            const int at = (tid >> 3) * RS + (tid & 7) * V4;
            rv = word_dot(R + at, V + at, rv);
            if constexpr (G::PLANES == 2) rv = word_dot(RL + at, V + at, rv);
#pragma unroll
            for (int i = tid; i < GW * KD / V4; i += GRADS) {
                const int e = i / (KD / V4) * KS + i % (KD / V4) * V4;
                inner = word_dot(S + e, D + e, inner);
            }
            __syncthreads();
            if (G::STAGES == 1 && b + 1 < n_blocks) load(b + 1);
        }
        copies_wait<0>();
        // the products' sums of rows and columns, for the decays and rates
        const float *since = F, *until = F + C, *rate = F + 2 * C;
        const float *up = F + UP, *low = F + UP_LOW;
        const int* cut = reinterpret_cast<const int*>(F + CUT);
        const float ks = SCALED ? F[K_SCALE] : 1.0f, qs = SCALED ? F[Q_SCALE] : 1.0f, ik = inverse_of(ks), iq = inverse_of(qs);
        float kk[2][4] = {}, qk[2][4] = {};
        if (wc <= wr) {
#pragma unroll 4
            for (int d = 0; d < KD; d += 16) {
                typename KOp::B bb[2];
                KOp::by_rows(bb, Ks + wc * 16 * KS + d, KS);
                KOp::mma(kk[0], kk[1], KOp::rows_of(Ks + wr * 16 * KS + d, KS), bb);
                KOp::mma(qk[0], qk[1], KOp::rows_of(Qs + wr * 16 * KS + d, KS), bb);
            }
        }
        float by_row[4][2] = {}, by_col[2][2] = {};  // q.dQ + b k.., k..until, R part of db, sum of x k.k / b; columns
        float tp = 0.0f, tx = 0.0f, tq1 = 0.0f, tk1 = 0.0f;  // the largest of p, x, zq and zk
        if (wc <= wr)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = wr * 16 + g + (e >> 1) * 8, jj = wc * 16 + j * 8 + 2 * t4 + (e & 1);
                    const float d = jj <= i ? decay_between(up, low, cut, i, jj) : 0.0f;
                    const float pv = d != 0.0f ? A.scale * d * p[j][e] : 0.0f, xv = d != 0.0f && jj < i ? -d * x[j][e] : 0.0f;
                    const float xr = xv * (kk[j][e] * ik * ik), mp = pv * (qk[j][e] * ik * iq), both = fmaf(rate[i], xr, mp);
                    by_row[0][e >> 1] += both;
                    by_row[3][e >> 1] += xr;
                    by_col[j][e & 1] += both;
                    p[j][e] = pv;
                    x[j][e] = rate[i] * xv;
                    tp = fmaxf(tp, finite_size(p[j][e]));
                    tx = fmaxf(tx, finite_size(x[j][e]));
                }
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = wr * 16 + g + h * 8, c = wc * (KD / 4) + j * 8 + 2 * t4;
                float2 kv, qv;
                if constexpr (sizeof(KE) == 2) {
                    kv = of_pair<KE>(*reinterpret_cast<const unsigned*>(Ks + i * KS + c));
                    qv = of_pair<KE>(*reinterpret_cast<const unsigned*>(Qs + i * KS + c));
                } else {
                    kv = *reinterpret_cast<const float2*>(Ks + i * KS + c);
                    qv = *reinterpret_cast<const float2*>(Qs + i * KS + c);
                }
                // (divided by the scales of the keys and queries that they meet here)
                const float fq1 = A.scale * since[i] * iq, fk1 = -since[i] * ik, fm1 = until[i] * ik, ra = rate[i];
                float *q2 = zq[j] + 2 * h, *k2 = zk[j] + 2 * h, *m2 = zm[j] + 2 * h;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    q2[e] *= fq1;
                    k2[e] *= fk1;
                    m2[e] *= fm1;
                }
                by_row[0][h] += fmaf(qv.x, q2[0], qv.y * q2[1]);
                by_row[2][h] += fmaf(kv.x, k2[0], kv.y * k2[1]);
                by_row[1][h] += fmaf(kv.x, m2[0], kv.y * m2[1]);
                k2[0] = fmaf(ra, k2[0], m2[0]);
                k2[1] = fmaf(ra, k2[1], m2[1]);
                if constexpr (SCALED) {
                    tq1 = fmaxf(tq1, fmaxf(fabsf(q2[0]), fabsf(q2[1])));
                    tk1 = fmaxf(tk1, fmaxf(fabsf(k2[0]), fabsf(k2[1])));
                }
            }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v = by_row[q][h];
                v += __shfl_xor_sync(~0u, v, 1);
                v += __shfl_xor_sync(~0u, v, 2);
                if (t4 == 0) rows[q][wc][wr * 16 + g + h * 8] = v;
            }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v = by_col[j][h];
                v += __shfl_xor_sync(~0u, v, 4);
                v += __shfl_xor_sync(~0u, v, 8);
                v += __shfl_xor_sync(~0u, v, 16);
                if (g == 0) cols[wr][wc * 16 + j * 8 + 2 * t4 + h] = v;
            }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) rv += __shfl_xor_sync(~0u, rv, o);
        if ((tid & 7) == 0) dots[tid >> 3] = rv;
#pragma unroll
        for (int o = 16; o; o >>= 1) inner += __shfl_xor_sync(~0u, inner, o);
        auto most = [](float v) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v))); };
        if constexpr (SCALED) {
            tp = most(tp);
            tx = most(tx);
            tq1 = most(finite_size(tq1));
            tk1 = most(finite_size(tk1));
        }
        if (lane == 0) {
            more[warp] = inner;
            top[0][warp] = tp;
            top[1][warp] = tx;
            top[2][warp] = tq1;
            top[3][warp] = tk1;
        }
        float ps = 1.0f, xs = 1.0f, fq = 1.0f, fk = 1.0f;  // scales of p, x and of what they are added to
        if constexpr (SCALED) {
            __syncthreads();
            tp = most(top[0][lane % (GRADS / 32)]);
            tx = most(top[1][lane % (GRADS / 32)]);
            tq1 = most(top[2][lane % (GRADS / 32)]);
            tk1 = most(top[3][lane % (GRADS / 32)]);
            // (held so that a product with both keys' scales is finite, and so are zq and zk times these)
            xs = scale_within(scale_for(tx), fminf(0x1p100f * scale_for(tk1), 0x1p120f) * ik * ik);
            ps = scale_within(scale_for(tp), fminf(0x1p100f * scale_for(tq1), 0x1p120f) * ik * iq);
            fk = scale_of_both(xs, ks);
            fq = scale_of_both(ps, ks);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    zq[j][e] *= fq * qs;
                    zk[j][e] *= fk * ks;
                }
        }
        if (wc <= wr)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = (wr * 16 + g + h * 8) * MS + wc * 16 + j * 8 + 2 * t4;
                    KOp::template put<PIECES>(Ps + at, p[j][2 * h] * ps, p[j][2 * h + 1] * ps);
                    KOp::template put<PIECES>(Xs + at, x[j][2 * h] * xs, x[j][2 * h + 1] * xs);
                }
        __syncthreads();
        // dQ += p K, dK += x K + x^T K, then p^T Q, which has a scale of its own
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            typename KOp::B bk[NQ / 2][2];
#pragma unroll
            for (int j = 0; j < NQ / 2; ++j) KOp::by_columns(bk[j], Ks + d * 16 * KS + wc * (KD / 4) + j * 16, KS);
#pragma unroll
            for (int i = PIECES - 1; i >= 0; --i) {
                if (d <= wr) {
                    const typename KOp::A ap = KOp::rows_of(Ps + i * C * MS + wr * 16 * MS + d * 16, MS);
                    const typename KOp::A ax = KOp::rows_of(Xs + i * C * MS + wr * 16 * MS + d * 16, MS);
#pragma unroll
                    for (int j = 0; j < NQ / 2; ++j) {
                        KOp::mma(zq[2 * j], zq[2 * j + 1], ap, bk[j]);
                        KOp::mma(zk[2 * j], zk[2 * j + 1], ax, bk[j]);
                    }
                }
                if (d >= wr) {
                    const typename KOp::A xt = KOp::columns_of(Xs + i * C * MS + d * 16 * MS + wr * 16, MS);
#pragma unroll
                    for (int j = 0; j < NQ / 2; ++j) KOp::mma(zk[2 * j], zk[2 * j + 1], xt, bk[j]);
                }
            }
        }
        const float bq1 = inverse_of(fq), bk1 = inverse_of(fk), bp1 = inverse_of(SCALED ? scale_of_both(ps, qs) : 1.0f);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tq[j][e] = fmaf(zq[j][e], bq1, tq[j][e]);
                tk[j][e] = fmaf(zk[j][e], bk1, tk[j][e]);
                zq[j][e] = 0.0f;
            }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (d < wr) continue;
            typename KOp::B bq[NQ / 2][2];
#pragma unroll
            for (int j = 0; j < NQ / 2; ++j) KOp::by_columns(bq[j], Qs + d * 16 * KS + wc * (KD / 4) + j * 16, KS);
#pragma unroll
            for (int i = PIECES - 1; i >= 0; --i) {
                const typename KOp::A pt = KOp::columns_of(Ps + i * C * MS + d * 16 * MS + wr * 16, MS);
#pragma unroll
                for (int j = 0; j < NQ / 2; ++j) KOp::mma(zq[2 * j], zq[2 * j + 1], pt, bq[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) tk[j][e] = fmaf(zq[j][e], bp1, tk[j][e]);
        if (warp == 0) {
            // rows 2 lane, 2 lane + 1: what each adds to the decays up to it
            float d[2], whole = 0.0f, edge = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * lane + h;
                float a = 0.0f, m = 0.0f, r = 0.0f, xk = 0.0f, c = 0.0f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    a += rows[0][q][i];
                    m += rows[1][q][i];
                    r += rows[2][q][i];
                    xk += rows[3][q][i];
                    c += cols[q][i];
                }
                d[h] = a + rate[i] * r - m - c;
                edge += m;
                if (i < n) {
                    float db = dots[i] + r + xk;
                    if (A.logit) db *= rate[i] * (1.0f - rate[i]);
                    ((T*)A.dbeta.p)[row_at(A, A.dbeta, s, sp, t0 + i) + head * A.dbeta.hs] = from_f32<T>(db);
                }
            }
            if (lane < GRADS / 32) whole = more[lane];
            // (since at the chunk's end is 0 where a decay is)
            whole *= since[C - 1];
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                whole += __shfl_xor_sync(~0u, whole, o);
                edge += __shfl_xor_sync(~0u, edge, o);
            }
            float sum = d[0] + d[1];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const float v = __shfl_down_sync(~0u, sum, o);
                if (lane + o < 32) sum += v;
            }
            whole += edge;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * lane + h;
                float dg = whole + sum - (h ? d[0] : 0.0f);
                if (i < n) {
                    const T gate = ((const T*)A.gate.p)[row_at(A, A.gate, s, sp, t0 + i) + head * A.gate.hs];
                    if (A.logit) dg *= 1.0f / (1.0f + expf(to_f32(gate)));
                    if (cut[i] != (i ? cut[i - 1] : 0)) dg = 0.0f;  // a decay of 0
                    ((T*)A.dgate.p)[row_at(A, A.dgate, s, sp, t0 + i) + head * A.dgate.hs] = from_f32<T>(dg);
                }
            }
        }
        __syncthreads();
    }
    // dQ, dK as rows of T, through the keys' and queries' place
    T *oq = reinterpret_cast<T*>(Qs), *ok = reinterpret_cast<T*>(Ks);
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = (wr * 16 + g + h * 8) * KS + wc * (KD / 4) + j * 8 + 2 * t4;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<unsigned*>(oq + at) = pair_of<T>(tq[j][2 * h], tq[j][2 * h + 1]);
                *reinterpret_cast<unsigned*>(ok + at) = pair_of<T>(tk[j][2 * h], tk[j][2 * h + 1]);
            } else {
                *reinterpret_cast<float2*>(oq + at) = make_float2(tq[j][2 * h], tq[j][2 * h + 1]);
                *reinterpret_cast<float2*>(ok + at) = make_float2(tk[j][2 * h], tk[j][2 * h + 1]);
            }
        }
    __syncthreads();
    auto store = [&](const Heads& h, const T* from) {
        T* to = (T*)h.p + row_at(A, h, s, sp, t0) + kh * h.hs;
        if (h.word == 16) {
            constexpr int V = 16 / (int)sizeof(T), N = KD / V;
            for (int i = tid; i < n * N; i += GRADS) {
                const int r = i / N, c = i % N * V;
                if (c < A.kdim) *reinterpret_cast<uint4*>(to + r * h.st + c) = *reinterpret_cast<const uint4*>(from + r * KS + c);
            }
        } else {
            for (int i = tid; i < n * KD; i += GRADS) {
                const int r = i / KD, c = i % KD;
                if (c < A.kdim) to[r * h.st + c] = from[r * KS + c];
            }
        }
    };
    store(A.dq, oq);
    store(A.dk, ok);
}

}  // namespace snnb_delta
