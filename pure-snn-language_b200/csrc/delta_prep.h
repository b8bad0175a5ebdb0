// delta_prep.h - keys, T, P and the factors of every chunk of a delta-rule scan.
//
// A CTA of four warps for a chunk and head, 16 rows to a warp.  T by blocks of 16: a
// warp inverts its block on the diagonal by substitution, a column to a lane, then
// with N = -T_ii A_im:  T_ij = sum of N_im T_mj, one row of blocks after the other, in f32
// by two tf32 pieces.
#pragma once
#include "delta_tile.h"

namespace snnb_delta {
constexpr int PREP = 128;
template <class P, int KD>
constexpr int prep_smem() {
    const int keys = 2 * C * (KD + PAD) * (int)sizeof(typename P::KE), m = C * MS * 4;
    return keys > m ? keys : m;  // A and T take the place of K and Q
}
// Scale of a chunk's keys or queries.  At most 2^40, and that where all are zero: what
// they are multiplied with shares the scale of the product and must not lose bits to nothing.
__device__ __forceinline__ float key_scale(float top) { return top == 0.0f ? 0x1p40f : fminf(scale_for(top), 0x1p40f); }
// rows of keys or queries into registers, words of V elements; their largest magnitude
template <typename T, int KD, int N>
__device__ __forceinline__ float read_keys(uint4 (&w)[N], const T* from, long long st, int n, const DeltaArgs& A, int word) {
    constexpr int V = 16 / (int)sizeof(T), L = KD / V;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int k = threadIdx.x + i * PREP, r = k / L, c = (k - r * L) * V;
        w[i] = make_uint4(0, 0, 0, 0);
        if (r >= n || c >= A.kdim) continue;
        const T* p = from + r * st + c;
        if (word == 16) {
            w[i] = *reinterpret_cast<const uint4*>(p);
        } else {
            T e[V];
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = c + j < A.kdim ? p[j] : from_f32<T>(0.0f);
            memcpy(&w[i], e, 16);
        }
    }
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = of_pair<T>((&w[i].x)[j]);
                top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
    return top;
}
// the same times s as KE, rows of stride KD + PAD, to shared memory and, unless null, to memory
template <typename T, typename KE, int KD, int N>
__device__ __forceinline__ void write_keys(const uint4 (&w)[N], KE* sm, KE* copy, float s) {
    constexpr int V = 16 / (int)sizeof(T), L = KD / V;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int k = threadIdx.x + i * PREP, r = k / L, c = (k - r * L) * V;
        uint4 o = w[i];
        if constexpr (sizeof(T) == 2)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = of_pair<T>((&w[i].x)[j]);
                (&o.x)[j] = pair_of<KE>(f.x * s, f.y * s);
            }
        *reinterpret_cast<uint4*>(sm + r * (KD + PAD) + c) = o;
        if (copy) *reinterpret_cast<uint4*>(copy + r * (KD + PAD) + c) = o;
    }
}
template <class P, int KD>
__global__ void __launch_bounds__(PREP, 4) k_delta_prep(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using KE = typename P::KE;
    constexpr int KS = KD + PAD, WORDS = C * KD * (int)sizeof(T) / 16 / PREP;
    extern __shared__ __align__(16) char smem[];
    KE *K = reinterpret_cast<KE*>(smem), *Q = K + C * KS;
    float* M = reinterpret_cast<float*>(smem);  // [C][MS]
    __shared__ float up[C], low[C], rate[C], top[2][4];
    __shared__ int cut[C];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.y, kh = head / A.group;
    const int g = lane >> 2, t4 = lane & 3;
    const long long slot = blockIdx.x, s = sequence_of(A, slot);
    const Span sp = span_of(A, s);
    const long long first = (slot - sp.chunk) * C;
    if (first < 0 || first >= sp.len) return;
    const int t0 = (int)first, n = min(C, sp.len - t0);
    float ks = 1.0f, qs = 1.0f;
    {
        uint4 wk[WORDS], wq[WORDS];
        float a = read_keys<T, KD>(wk, (const T*)A.k.p + row_at(A, A.k, s, sp, t0) + kh * A.k.hs, A.k.st, n, A, A.k.word);
        float b = read_keys<T, KD>(wq, (const T*)A.q.p + row_at(A, A.q, s, sp, t0) + kh * A.q.hs, A.q.st, n, A, A.q.word);
        if (warp == 0) chunk_decays<T>(A, s, sp, t0, n, head, lane, up, low, cut, rate);
        if constexpr (P::SCALED) {
            a = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(a)));
            b = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(b)));
            if (lane == 0) {
                top[0][warp] = a;
                top[1][warp] = b;
            }
            __syncthreads();
            ks = key_scale(fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3])));
            qs = key_scale(fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3])));
        }
        KE* copy = head % A.group == 0 ? (KE*)A.keys + (slot * A.hk + kh) * 2 * C * KS : nullptr;
        write_keys<T, KE, KD>(wk, K, copy, ks);
        write_keys<T, KE, KD>(wq, Q, copy ? copy + C * KS : nullptr, qs);
    }
    __syncthreads();
    const long long unit = slot * A.heads + head;
    float* F = A.factors + unit * SC;
    KE *Tm = reinterpret_cast<KE*>(A.squares + unit * P::SQUARES) + low_at(warp), *Pm = Tm + P::PIECES * LOW;
    const int st = low_stride(warp);
    if (tid < C) {
        F[tid] = cut[tid] ? 0.0f : expf(up[tid]) * (1.0f + low[tid]);
        F[C + tid] = decay_between(up, low, cut, C - 1, tid);
        F[2 * C + tid] = rate[tid];
        F[UP + tid] = up[tid];
        F[UP_LOW + tid] = low[tid];
        reinterpret_cast<int*>(F + CUT)[tid] = cut[tid];
        if (tid == 0) {
            F[LOST] = cut[C - 1] ? 1.0f : fmaf(-low[C - 1], expf(up[C - 1]), -expm1f(up[C - 1]));
            F[K_SCALE] = ks;
            F[Q_SCALE] = qs;
        }
    }
    // This warp's rows of the products of queries with keys, and of keys.  (A decay
    // of 0 takes all: what lies above the diagonal may be anything.)
    const float ik = inverse_of(ks), iq = inverse_of(qs);
    float x2[8][4] = {}, p2[8][4] = {};
#pragma unroll
    for (int np = 0; np < 4; ++np) {
        if (np > warp) break;  // above the diagonal
#pragma unroll 4
        for (int d = 0; d < KD; d += 16) {
            P::gram(x2[2 * np], x2[2 * np + 1], K + warp * 16 * KS + d, K + np * 16 * KS + d, KS);
            P::gram(p2[2 * np], p2[2 * np + 1], Q + warp * 16 * KS + d, K + np * 16 * KS + d, KS);
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = warp * 16 + g + (e >> 1) * 8, j = nt * 8 + 2 * t4 + (e & 1);
            const float G = j <= i ? decay_between(up, low, cut, i, j) : 0.0f, a = rate[i] * G;
            p2[nt][e] = G != 0.0f ? G * (p2[nt][e] * ik * iq) : 0.0f;
            x2[nt][e] = j < i && a != 0.0f ? a * (x2[nt][e] * ik * ik) : 0.0f;
            most = fmaxf(most, fabsf(p2[nt][e]));
        }
    }
    float scale = 1.0f;
    if constexpr (P::SCALED) {
        scale = scale_for(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most))));
        if (lane == 0) F[P_SCALE + warp] = scale;
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) P::put(Pm + (g + h * 8) * st + nt * 8 + 2 * t4, p2[nt][2 * h], p2[nt][2 * h + 1], scale);
    }
    __syncthreads();  // K and Q are no longer read
    float* rows = M + warp * 16 * MS;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2*>(rows + (g + h * 8) * MS + nt * 8 + 2 * t4) = make_float2(x2[nt][2 * h], x2[nt][2 * h + 1]);
    }
    __syncwarp();
    // the block on the diagonal
    float* own = rows + warp * 16;
    {
        const int c = lane & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
            for (int m = 0; m < i; m += 2) {
                const float2 r = *reinterpret_cast<const float2*>(own + i * MS + m);
                a0 = fmaf(r.x, x[m], a0);
                if (m + 1 < i) a1 = fmaf(r.y, x[m + 1], a1);
            }
            x[i] = i < c ? 0.0f : (i == c ? 1.0f : 0.0f) - (a0 + a1);
        }
        __syncwarp();
        if (lane < 16)
#pragma unroll
            for (int i = 0; i < 16; ++i) own[i * MS + c] = x[i];
    }
    __syncwarp();
    float N[3][2][4] = {};
    {
        const Path32::A a = Path32::rows_of(own, MS);
#pragma unroll
        for (int m = 0; m < 3; ++m)
            if (m < warp) {
                Path32::B b[2];
                Path32::by_columns(b, rows + m * 16, MS);
                Path32::full(N[m][0], N[m][1], a, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    N[m][0][e] = -N[m][0][e];
                    N[m][1][e] = -N[m][1][e];
                }
            }
    }
#pragma unroll 1
    for (int i = 1; i < 4; ++i) {
        __syncthreads();  // the rows of blocks above are there
        if (warp != i) continue;
        float t[3][2][4] = {};
#pragma unroll
        for (int m = 0; m < 3; ++m) {
            if (m >= i) break;
            const Path32::A a = Path32::split(N[m][0], N[m][1], 1.0f);
#pragma unroll
            for (int j = 0; j <= m; ++j) {
                Path32::B b[2];
                Path32::by_columns(b, M + m * 16 * MS + j * 16, MS);
                Path32::full(t[j][0], t[j][1], a, b);
            }
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            if (j >= i) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<float2*>(rows + (g + e * 8) * MS + j * 16 + h * 8 + 2 * t4) = make_float2(t[j][h][2 * e], t[j][h][2 * e + 1]);
        }
        __syncwarp();
    }
    // out, this warp's rows
    float2 v[16];
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)  // row i, a lane a pair of columns
        if (2 * lane < 16 * (warp + 1)) {
            v[i] = *reinterpret_cast<const float2*>(rows + i * MS + 2 * lane);
            big = fmaxf(big, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        }
    scale = 1.0f;
    if constexpr (P::SCALED) {
        scale = scale_for(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big))));
        if (lane == 0) F[T_SCALE + warp] = scale;
    }
    if (2 * lane < 16 * (warp + 1))
#pragma unroll
        for (int i = 0; i < 16; ++i) P::put(Tm + i * st + 2 * lane, v[i].x, v[i].y, scale);
}
}  // namespace snnb_delta
