// delta_prep.h - keys, T, P and the factors of every chunk of a delta-rule scan.
//
// A CTA of four warps for a chunk and head, 16 rows to a warp.  T by blocks of 16: a
// warp inverts its block on the diagonal by substitution, a column to a lane, then
// with N = -T_ii A_im:  T_ij = sum of N_im T_mj, one row of blocks after the other, in f32
// by two tf32 pieces.  Bound by latency (half of it loads, scaling and
// decays, half products and the inversion), which four CTAs on an SM hide in part: 8,192 chunks
// of 128 bf16: kernel 277 us, 117 at the copy rate.  Five CTAs of 96 registers: 290; eight warps,
// queries and keys apart: 322.
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
// The largest magnitude of this thread's words of a [C, KD] tile (stride KD + PAD), and the tile
// times s as KE in its place and, unless null, in memory
template <typename T, int KD>
__device__ __forceinline__ float top_of_tile(const T* m) {
    constexpr int V = 16 / (int)sizeof(T), L = KD / V;
    // (magnitudes of 16 bits order as their bits)
    constexpr unsigned INFINITE = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
    unsigned top = 0;
#pragma unroll
    for (int i = threadIdx.x; i < C * L; i += PREP) {
        const uint4 w = *reinterpret_cast<const uint4*>(m + i / L * (KD + PAD) + i % L * V);
        top = __vmaxu2(__vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)), top);
    }
    if (__vcmpgeu2(top, INFINITE)) {  // infinities and NaN do not set the scale of the others
        top = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < C * L * 4; i += PREP) {  // the same words, a quarter at a time
            const int k = threadIdx.x + i / (4 * PREP) * PREP, q = (i / PREP) % 4;
            const unsigned size = *reinterpret_cast<const unsigned*>(m + k / L * (KD + PAD) + k % L * V + q * (V / 4)) & 0x7fff7fffu;
            top = __vmaxu2(top, size & __vcmpltu2(size, INFINITE));
        }
    }
    const float2 f = of_pair<T>(top);
    return fmaxf(f.x, f.y);
}
template <typename T, typename KE, int KD>
__device__ __forceinline__ void scale_tile(KE* m, KE* copy, float s) {
    constexpr int V = 16 / (int)sizeof(T), L = KD / V;
#pragma unroll 4
    for (int i = threadIdx.x; i < C * L; i += PREP) {
        const int at = i / L * (KD + PAD) + i % L * V;
        uint4 w = *reinterpret_cast<const uint4*>(m + at);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = of_pair<T>((&w.x)[j]);
                (&w.x)[j] = pair_of<KE>(f.x * s, f.y * s);
            }
            *reinterpret_cast<uint4*>(m + at) = w;
        }
        if (copy) *reinterpret_cast<uint4*>(copy + at) = w;
    }
}
template <class P, int KD>
__global__ void __launch_bounds__(PREP, 4) k_delta_prep(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using KE = typename P::KE;
    constexpr int KS = KD + PAD;
    extern __shared__ __align__(16) char smem[];
    KE *K = reinterpret_cast<KE*>(smem), *Q = K + C * KS;
    float* M = reinterpret_cast<float*>(smem);  // [C][MS]
    __shared__ __align__(16) float up[C], low[C], rate[C], top[2][4];
    __shared__ int cut[C];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.y, kh = head / A.group;
    const int g = lane >> 2, t4 = lane & 3;
    const long long slot = blockIdx.x, s = sequence_of(A, slot);
    const Span sp = span_of(A, s);
    const long long first = (slot - sp.chunk) * C;
    if (first < 0 || first >= sp.len) return;
    const int t0 = (int)first, n = min(C, sp.len - t0);
    float ks = 1.0f, qs = 1.0f;
    float lost = 0.0f;
    load_rows<T, C, KD>(reinterpret_cast<T*>(K), (const T*)A.k.p + row_at(A, A.k, s, sp, t0) + kh * A.k.hs, A.k.st, n, A.kdim, A.k.word, tid, PREP);
    load_rows<T, C, KD>(reinterpret_cast<T*>(Q), (const T*)A.q.p + row_at(A, A.q, s, sp, t0) + kh * A.q.hs, A.q.st, n, A.kdim, A.q.word, tid, PREP);
    copies_end();
    if (warp == 0) chunk_decays<T>(A, s, sp, t0, n, head, lane, up, low, cut, rate, lost);
    copies_wait<0>();
    __syncthreads();
    if constexpr (P::SCALED) {
        const float a = top_of_tile<T, KD>(reinterpret_cast<T*>(K)), b = top_of_tile<T, KD>(reinterpret_cast<T*>(Q));
        const unsigned ka = __reduce_max_sync(~0u, __float_as_uint(a)), qa = __reduce_max_sync(~0u, __float_as_uint(b));
        if (lane == 0) {
            top[0][warp] = __uint_as_float(ka);
            top[1][warp] = __uint_as_float(qa);
        }
        __syncthreads();
        ks = key_scale(fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3])));
        qs = key_scale(fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3])));
    }
    KE* copy = head % A.group == 0 ? (KE*)A.keys + (slot * A.hk + kh) * 2 * C * KS : nullptr;
    if (P::SCALED || copy) {
        scale_tile<T, KE, KD>(K, copy, ks);
        scale_tile<T, KE, KD>(Q, copy ? copy + C * KS : nullptr, qs);
    }
    __syncthreads();
    const long long unit = slot * A.heads + head;
    float* F = A.factors + unit * SC;
    KE *Tm = reinterpret_cast<KE*>(A.squares + unit * P::SQUARES) + low_at(warp), *Pm = Tm + P::PIECES * LOW;
    const int st = low_stride(warp);
    if (tid < C) {
        F[tid] = cut[tid] ? 0.0f : power_of_2(up[tid] + low[tid]);
        F[C + tid] = decay_between(up, low, cut, C - 1, tid);
        F[2 * C + tid] = rate[tid];
        F[UP + tid] = up[tid];
        F[UP_LOW + tid] = low[tid];
        reinterpret_cast<int*>(F + CUT)[tid] = cut[tid];
        if (tid == 31) {  // (the last lane of the warp that summed)
            F[LOST] = lost;
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
    const bool cuts = cut[C - 1] != 0;
    const float iqk = P::SCALED ? ik * iq : 1.0f;
    float upi[2], lowi[2], ri[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = warp * 16 + g + 8 * h;
        upi[h] = up[i];
        lowi[h] = low[i];
        ri[h] = rate[i];
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
        const float2 upj = *reinterpret_cast<const float2*>(up + nt * 8 + 2 * t4), lowj = *reinterpret_cast<const float2*>(low + nt * 8 + 2 * t4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int h = e >> 1, i = warp * 16 + g + h * 8, j = nt * 8 + 2 * t4 + (e & 1);
            float G = power_of_2((upi[h] - (e & 1 ? upj.y : upj.x)) + (lowi[h] - (e & 1 ? lowj.y : lowj.x)));
            if (nt / 2 == warp && j > i) G = 0.0f;
            if (cuts && cut[i] != cut[j]) G = 0.0f;
            const float a = ri[h] * G;
            p2[nt][e] = G != 0.0f ? G * (p2[nt][e] * iqk) : 0.0f;
            x2[nt][e] = a != 0.0f && (nt / 2 < warp || j < i) ? a * (x2[nt][e] * ik * ik) : 0.0f;
            most = fmaxf(most, finite_size(p2[nt][e]));
        }
    }
    float scale = 1.0f;
    if constexpr (P::SCALED) {
        scale = fminf(scale_for(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most)))), 0x1p40f);
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
            big = fmaxf(big, fmaxf(finite_size(v[i].x), finite_size(v[i].y)));
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
