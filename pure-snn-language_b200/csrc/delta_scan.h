// delta_scan.h - a delta-rule scan along the sequences, forward (k_delta_scan) and, for
// the states' gradients, back (k_delta_back).  Bound by the chain of products of a chunk: a warp
// has 400 (back 504) matrix instructions and 2,500 others for its 16 columns of 64 steps,
// and a scheduler two warps at most, since a warp takes 250 registers.  8 x 4,096 steps x 16 heads of
// 128 x 128 bf16: kernel 560 us, 480 without what the gradient wants, back 615; tensor pipe 39 %, issue
// 30 %.  Columns could not be cut finer (16 is the instruction's height), and a second warp for the same
// columns would have to exchange half of K S, of the answers and of U in every chunk.
#pragma once
#include "delta_tile.h"

namespace snnb_delta {
// A chunk in shared memory: K, Q, T and the first PP planes of P, the factors and the
// columns of V (or dy), two chunks where they fit.  All but the last are copied as they
// lie in the workspace.
template <class P, int KD, int NW, int PP>
struct Stage {
    using T = typename P::T;
    using KE = typename P::KE;
    static constexpr int VW = 16 * NW;
    static constexpr int KEYS = C * (KD + PAD) * (int)sizeof(KE), VALUES = C * (VW + PAD) * (int)sizeof(T);
    static constexpr int SQUARES = (P::PIECES + PP) * LOW * (int)sizeof(KE);
    static constexpr int BYTES = 2 * KEYS + VALUES + SQUARES + SCAN_FACTORS * 4;
    using K = typename Kept<T>::K;
    static constexpr int KEEP = sizeof(K) == 2 ? 16 * (KD + PAD) * 2 : 0;  // a warp's stage of its state
    static constexpr int STAGES = 2 * BYTES + NW * KEEP <= 227 * 1024 - 1024 ? 2 : 1;
    static constexpr int SMEM = STAGES * BYTES + NW * KEEP;
    static __device__ __forceinline__ K* keep(char* m, int warp) { return reinterpret_cast<K*>(m + STAGES * BYTES + warp * KEEP); }
    KE *k, *q, *t, *p;
    T* v;
    float* f;
    __device__ __forceinline__ explicit Stage(char* m) {
        k = reinterpret_cast<KE*>(m);
        q = reinterpret_cast<KE*>(m + KEYS);
        v = reinterpret_cast<T*>(m + 2 * KEYS);
        t = reinterpret_cast<KE*>(m + 2 * KEYS + VALUES);
        p = t + P::PIECES * LOW;
        f = reinterpret_cast<float*>(m + 2 * KEYS + VALUES + SQUARES);
    }
    // chunk c of sequence s; vals: the values' rows or, backward, those of dy (or none)
    __device__ __forceinline__ void load(const DeltaArgs& A, const Heads& vals, long long s, const Span& sp, int c, int head,
                                         int col0, int vdim, int tid) {
        const int n = min(C, sp.len - c * C);
        const long long slot = sp.chunk + c, unit = slot * A.heads + head;
        load_words(k, A.keys + (slot * A.hk + head / A.group) * 2 * KEYS, 2 * KEYS, tid, NW * 32);
        load_rows<T, C, VW>(v, (const T*)vals.p + row_at(A, vals, s, sp, c * C) + head * vals.hs + col0, vals.st,
                            vals.p ? n : 0, vdim - col0, vals.p ? vals.word : 16, tid, NW * 32);
        load_words(t, A.squares + unit * P::SQUARES, SQUARES, tid, NW * 32);
        load_words(f, A.factors + unit * SC, SCAN_FACTORS * 4, tid, NW * 32);
    }
};

// a warp's columns of the values' tile [C][ST] as accumulators [16 columns, C steps]
template <typename T, int ST>
__device__ __forceinline__ void values_of(float (&o)[8][4], const T* v) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            unsigned r[4];
            ldsm4t(r, v + (i * 8 + (lane >> 4) * 8 + (lane & 7)) * ST + ((lane >> 3) & 1) * 8);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = of_pair<T>(r[k]);
                o[i + (k >> 1)][2 * (k & 1)] = f.x;
                o[i + (k >> 1)][2 * (k & 1) + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = v[(i * 8 + 2 * t4 + (e & 1)) * ST + g + (e >> 1) * 8];
    }
}
// accumulators [16 columns, C steps] as n rows of T, the first w columns: through the warp's columns
// of `stage` [C][ST]
template <typename T, int ST, bool REST = false>  // REST: what rounding to T leaves of them
__device__ __forceinline__ void store_tile(const float (&o)[8][4], T* stage, T* to, long long st, int n, int w, int word) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    auto pair = [](float x, float y) {
        if constexpr (REST) piece<T>(x, y);
        return pair_of<T>(x, y);
    };
    __syncwarp();
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            stsm4t(stage + (i * 8 + (lane >> 4) * 8 + (lane & 7)) * ST + ((lane >> 3) & 1) * 8, pair(o[i][0], o[i][1]),
                   pair(o[i][2], o[i][3]), pair(o[i + 1][0], o[i + 1][1]), pair(o[i + 1][2], o[i + 1][3]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) stage[(i * 8 + 2 * t4 + (e & 1)) * ST + g + (e >> 1) * 8] = o[i][e];
    }
    __syncwarp();
    auto words = [&](auto z) {
        using W = decltype(z);
        constexpr int V = (int)(sizeof(W) / sizeof(T)), N = 16 / V;
        const int c = lane % N * V;
        if (c < w)
#pragma unroll 4
            for (int r = lane / N; r < n; r += 32 / N)
                *reinterpret_cast<W*>(to + r * st + c) = *reinterpret_cast<const W*>(stage + r * ST + c);
    };
    if (word == 16) words(uint4());
    else if (word == 8) words(uint2());
    else if (word == 4) words(unsigned());
    else {
        for (int i = lane; i < n * 16; i += 32) {
            const int r = i >> 4, c = i & 15;
            if (c < w) to[r * st + c] = stage[r * ST + c];
        }
    }
    __syncwarp();
}
// accumulators as C rows of what is kept, w columns (whole words of 16 bytes)
template <typename T, typename K, int ST>
__device__ __forceinline__ void keep_tile(const float (&o)[8][4], T* stage, K* to, long long st, int w) {
    if constexpr (std::is_same<T, K>::value) {
        store_tile<T, ST>(o, stage, to, st, C, w, 16);
        if constexpr (Kept<T>::PLANES == 2) store_tile<T, ST, true>(o, stage, to + C * st, st, C, w, 16);
    } else {  // f32 of f16 tensors
        const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = g + (e >> 1) * 8;
                if (c < w) to[(long long)(i * 8 + 2 * t4 + (e & 1)) * st + c] = from_f32<K>(o[i][e]);
            }
    }
}
// S^T [16 columns, KD] of a warp, divided by its scale, as w rows of KD elements (stride KD +
// PAD).  bf16: through the warp's `stage` [16][KD + PAD], from where it is copied while the
// warp goes on (stores from registers, of 16 bytes to a row, took 2 us of 9.5 a chunk).
template <typename K, int NT>
__device__ __forceinline__ void keep_state(const float (&S)[NT][4], float back, K* stage, K* to, int w) {
    constexpr int KS = NT * 8 + PAD;
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    if constexpr (sizeof(K) == 2) {
        if (lane == 0) store_read();  // what was kept before has left the stage
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NT; i += 2)
            stsm4(stage + ((lane & 7) + ((lane >> 3) & 1) * 8) * KS + (i + (lane >> 4)) * 8, pair_of<K>(S[i][0] * back, S[i][1] * back),
                  pair_of<K>(S[i][2] * back, S[i][3] * back), pair_of<K>(S[i + 1][0] * back, S[i + 1][1] * back),
                  pair_of<K>(S[i + 1][2] * back, S[i + 1][3] * back));
        store_fence();
        __syncwarp();
        if (lane == 0) store_bulk(to, stage, min(w, 16) * KS * 2);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (g + 8 * h < w)
#pragma unroll
                for (int i = 0; i < NT; ++i)
                    *reinterpret_cast<float2*>(to + (g + 8 * h) * KS + i * 8 + 2 * t4) = make_float2(S[i][2 * h] * back, S[i][2 * h + 1] * back);
    }
}
// f32 states [kdim, vdim] from and to a warp's columns
template <int NT>
__device__ __forceinline__ void read_state(float (&S)[NT][4], const float* h, const DeltaArgs& A, int col, int vdim) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = col + g + (e >> 1) * 8, d = i * 8 + 2 * t4 + (e & 1);
            S[i][e] = h && c < vdim && d < A.kdim ? h[(long long)d * vdim + c] : 0.0f;
        }
}
template <int NT>
__device__ __forceinline__ void write_state(const float (&S)[NT][4], float back, float* h, const DeltaArgs& A, int col, int vdim) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = col + g + (e >> 1) * 8, d = i * 8 + 2 * t4 + (e & 1);
            if (c < vdim && d < A.kdim) h[(long long)d * vdim + c] = S[i][e] * back;
        }
}


// Accumulators that are the first operand of products as they are, in pieces: times a
// power of two (scale) that keeps their largest magnitude (top) in 2^6 .. 2^15, changed
// only where it leaves that.
template <int NT>
__device__ __forceinline__ void recentre(float (&S)[NT][4], float& scale, float& top) {
    top = warp_top(S);
    if (top >= 0x1p15f || (top < 0x1p6f && top > 0.0f && scale < MOST_SCALE)) {
        const float f = fminf(scale_for(top), MOST_SCALE * inverse_of(scale));
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] *= f;
        scale *= f;
        top *= f;
    }
}
// The same before products of x and y, which are already times their part of the scale to be
// pieces, are added to what a chunk leaves of S (at most top): neither is too large for
// a piece, nor all of them so small that pieces lose bits.  `held` is the scale as x and y have it: less than S's
// where they would not be finite otherwise.
template <int NT>
__device__ __forceinline__ void make_room(float (&S)[NT][4], float (&x)[8][4], float (&y)[8][4], float& scale, float held, float top) {
    const float part = held * inverse_of(scale), both = fmaxf(warp_top(x), &x != &y ? warp_top(y) : 0.0f), all = fmaxf(both, top * part);
    if (held < scale || both >= 0x1p15f || (all < 0x1p6f && all > 0.0f && scale < MOST_SCALE)) {
        const float f = fminf(scale_for(both >= 0x1p15f ? both : all), MOST_SCALE * inverse_of(held)), fs = part * f;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] *= fs;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[i][e] *= f;
                if (&x != &y) y[i][e] *= f;
            }
        scale = held * f;
    }
}
// S times the decays of a chunk: by what they take off where that is little, since 1 - lost keeps its
// bits there (and S those that it has)
template <int NT>
__device__ __forceinline__ void decay_state(float (&S)[NT][4], float lost, float kept) {
    if (lost < 0.5f) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = fmaf(-lost, S[i][e], S[i][e]);
    } else {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] *= kept;
    }
}
// acc [16, 64] += x m^T (ROWS; m lower triangular: steps k <= n) or x m (k >= n), in N pieces
template <class P, int N, bool ROWS, typename F>
__device__ __forceinline__ void times_square(float (&acc)[8][4], const float (&x)[8][4], F scale, const typename P::KE* m) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const typename P::A a = P::split(x[2 * d], x[2 * d + 1], scale(d));
        auto plane = [&](auto jj) {
            constexpr int j = decltype(jj)::value;
            typename P::B b[4][2];
#pragma unroll
            for (int np = 0; np < 4; ++np) {
                if (ROWS && np >= d) P::by_rows(b[np], m + j * LOW + low_at(np) + 16 * d, low_stride(np));
                if (!ROWS && np <= d) P::by_columns(b[np], m + j * LOW + low_at(d) + 16 * np, low_stride(d));
            }
            if constexpr (N - 1 - j >= 1)
#pragma unroll
                for (int np = 0; np < 4; ++np)
                    if (ROWS ? np >= d : np <= d) P::template mma<1>(acc[2 * np], acc[2 * np + 1], a, b[np]);
#pragma unroll
            for (int np = 0; np < 4; ++np)
                if (ROWS ? np >= d : np <= d) P::template mma<0>(acc[2 * np], acc[2 * np + 1], a, b[np]);
        };
        if constexpr (N == 2) plane(std::integral_constant<int, 1>());
        plane(std::integral_constant<int, 0>());
    }
}
// S^T [16, KD] += x [16, 64] m [64, KD], x in all pieces
template <class P, int KD>
__device__ __forceinline__ void add_outer(float (&S)[KD / 8][4], const float (&x)[8][4], const typename P::KE* m) {
    constexpr int KS = KD + PAD;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const typename P::A a = P::split(x[2 * d], x[2 * d + 1], 1.0f);
#pragma unroll
        for (int h = 0; h < KD / 64; ++h) {
            typename P::B b[4][2];
#pragma unroll
            for (int np = 0; np < 4; ++np) P::by_columns(b[np], m + d * 16 * KS + (h * 4 + np) * 16, KS);
            if constexpr (P::PIECES == 2)
#pragma unroll
                for (int np = 0; np < 4; ++np) P::template mma<1>(S[2 * (h * 4 + np)], S[2 * (h * 4 + np) + 1], a, b[np]);
#pragma unroll
            for (int np = 0; np < 4; ++np) P::template mma<0>(S[2 * (h * 4 + np)], S[2 * (h * 4 + np) + 1], a, b[np]);
        }
    }
}
// acc [16, 64] += S^T [16, KD] m^T for m [64, KD], piece d of 16 of the depth
template <class P, int N, int KD>
__device__ __forceinline__ void read_with(float (&acc)[8][4], const typename P::A& a, const typename P::KE* m, int d) {
    constexpr int KS = KD + PAD;
    typename P::B b[4][2];
#pragma unroll
    for (int np = 0; np < 4; ++np) P::by_rows(b[np], m + np * 16 * KS + d * 16, KS);
    if constexpr (N == 2)
#pragma unroll
        for (int np = 0; np < 4; ++np) P::template mma<1>(acc[2 * np], acc[2 * np + 1], a, b[np]);
#pragma unroll
    for (int np = 0; np < 4; ++np) P::template mma<0>(acc[2 * np], acc[2 * np + 1], a, b[np]);
}
__device__ __forceinline__ float2 pair_at(const float* f, int i) {  // of an accumulator tile's two steps
    return *reinterpret_cast<const float2*>(f + i * 8 + 2 * (threadIdx.x & 3));
}

template <class P, int KD, int NW>
__global__ void __launch_bounds__(NW * 32, 1) k_delta_scan(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using St = Stage<P, KD, NW, P::OUT>;
    using K = typename Kept<T>::K;
    constexpr int NT = KD / 8, VS = St::VW + PAD;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5;
    // (of the runs that make the segments' starts, those behind the values' columns take the unit matrix along, with
    // no values: what comes out is the product of the steps)
    const bool unit_run = A.only && (int)blockIdx.z >= A.tiles;
    const int head = blockIdx.y, col0 = ((int)blockIdx.z - (unit_run ? A.tiles : 0)) * St::VW, col = col0 + warp * 16;
    const int vdim = unit_run ? A.kdim : A.vdim, w = vdim - col;  // w: this warp's columns (16 and more: all; none: it only loads)
    Heads values = A.v;
    if (unit_run) values = {nullptr, 0, 0, 0, 16};  // (copies of nothing have an aligned address all the same)
    for (long long item = blockIdx.x; item < A.items; item += gridDim.x) {
        const long long s = sequence_of_item(A, item);
        const Span sp = span_of(A, s);
        const int segment = (int)(item - item_at(A, s, sp));
        if (segment < 0) continue;  // of no sequence
        const int all = (sp.len + C - 1) / C, first = segment * A.seg;
        const int chunks = A.seg ? min(all, first + A.seg) : all;  // the first one that is not this segment's
        const bool last = segment == (A.seg ? max(0, (all + A.seg - 1) / A.seg - 1) : 0);
        if ((!last && chunks <= first) || (A.only && (last || (unit_run && segment == 0)))) continue;
        float S[NT][4], sigma = 1.0f;  // S times sigma
        const long long size = (long long)A.kdim * A.vdim;
        if (unit_run) {
            const int lane = tid & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][e] = col + g + (e >> 1) * 8 == i * 8 + 2 * t4 + (e & 1) ? 1.0f : 0.0f;
        } else {
            // (h may be h0: where another CTA writes h, that is, behind other segments, segment 0 takes what the first run left
            // of h0 for it)
            float* start = A.seg ? A.starts + (item * A.heads + head) * size : nullptr;
            const bool from_h0 = segment == 0 && (A.only || last);
            read_state<NT>(S, from_h0 ? (A.h0 ? A.h0 + (s * A.heads + head) * size : nullptr) : (A.only ? nullptr : start), A, col, vdim);
            if (A.only && segment == 0 && w > 0) write_state<NT>(S, 1.0f, start, A, col, vdim);
        }
        if (St::STAGES == 2 && chunks > first) St(smem + (first & 1) * St::BYTES).load(A, values, s, sp, first, head, col0, vdim, tid);
        copies_end();
        for (int c = first; c < chunks; ++c) {
            const St st(smem + (St::STAGES == 2 ? (c & 1) * St::BYTES : 0));
            if (St::STAGES == 1) St(smem).load(A, values, s, sp, c, head, col0, vdim, tid);
            else if (c + 1 < chunks) St(smem + ((c + 1) & 1) * St::BYTES).load(A, values, s, sp, c + 1, head, col0, vdim, tid);
            copies_end();
            copies_wait<St::STAGES - 1>();
            __syncthreads();
            if (w > 0) {
                const int n = min(C, sp.len - c * C);
                const long long unit = (sp.chunk + c) * A.heads + head;
                float top = 0.0f;
                if constexpr (P::SCALED) recentre(S, sigma, top);
                float back = inverse_of(sigma), ik = 1.0f, iq = 1.0f;
                if constexpr (P::SCALED) {
                    ik = inverse_of(st.f[K_SCALE]);
                    iq = inverse_of(st.f[Q_SCALE]);
                }
                if (A.states && !A.only) keep_state<K, NT>(S, back, St::keep(smem, warp), (K*)A.states + (unit * A.vdim + col) * (KD + PAD), w);
                float r[8][4] = {}, o[8][4] = {}, u[8][4];
#pragma unroll
                for (int d = 0; d < KD / 16; ++d) {
                    const typename P::A a = P::split(S[2 * d], S[2 * d + 1], 1.0f);
                    read_with<P, P::PIECES, KD>(r, a, st.k, d);
                    if (!A.only) read_with<P, P::OUT, KD>(o, a, st.q, d);
                }
                // r = b (v - since K S)
                values_of<T, VS>(u, st.v + warp * 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 since = pair_at(st.f, i), rate = pair_at(st.f + 2 * C, i);
                    const float f0 = -since.x * back * ik, f1 = -since.y * back * ik;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        r[i][e] = (e & 1 ? rate.y : rate.x) * fmaf(e & 1 ? f1 : f0, r[i][e], u[i][e]);
                        u[i][e] = 0.0f;
                    }
                }
                // u = T r
                float ss = 1.0f, held = sigma;
                if constexpr (P::SCALED) ss = warp_scale(r);
                times_square<P, P::PIECES, true>(u, r, [&](int) { return ss; }, st.t);
                if constexpr (P::SCALED) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = inverse_of(ss) * inverse_of(st.f[T_SCALE + i / 2]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[i][e] *= f;
                    }
                    // (times the state's scale u is 2^74 at most; the answers' sum of state and queries, 2^35 / (their scales)
                    // at most, is taken times ss and P's scale, which is 2^40 at most)
                    ss = warp_scale(u);
                    held = scale_within(sigma, 0x1p60f * ss * st.f[K_SCALE]);
                    ss = scale_within(ss, 0x1p45f * sigma * st.f[Q_SCALE]);
                }
                if (!A.only) {
                // o = since Q S + P u, times the pieces' scales
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 since = pair_at(st.f, i);
                    const float f = P::SCALED ? ss * st.f[P_SCALE + i / 2] : 1.0f, f0 = since.x * back * iq, f1 = since.y * back * iq;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] = o[i][e] * (e & 1 ? f1 : f0) * f;
                }
                times_square<P, P::OUT, true>(o, u, [&](int) { return ss; }, st.p);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float f = P::SCALED ? A.scale * (inverse_of(ss) * inverse_of(st.f[P_SCALE + i / 2])) : A.scale;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] *= f;
                }
                store_tile<T, VS>(o, st.v + warp * 16, (T*)A.y.p + row_at(A, A.y, s, sp, c * C) + head * A.y.hs + col, A.y.st, n, w, A.y.word);
                }
                if (A.u && !A.only) keep_tile<T, K, VS>(u, st.v + warp * 16, (K*)A.u + unit * Kept<T>::PLANES * C * A.vpad + col, A.vpad, A.vpad - col);
                // S = since_64 S + (until u)^T K; 1 - since_64 keeps its bits where decays are near 1
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 until = pair_at(st.f + C, i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[i][e] *= (e & 1 ? until.y : until.x) * held * ik;
                }
                if constexpr (P::SCALED) make_room(S, u, u, sigma, held, top * st.f[C - 1]);
                decay_state(S, st.f[LOST], st.f[C - 1]);
                add_outer<P, KD>(S, u, st.k);
            }
            __syncthreads();
        }
        float* to = unit_run ? A.maps + (item * A.heads + head) * A.kdim * A.kdim
                             : A.only ? A.starts + ((item + 1) * A.heads + head) * size : A.h && last ? A.h + (s * A.heads + head) * size : nullptr;
        if (to && w > 0) write_state<NT>(S, inverse_of(sigma), to, A, col, vdim);
        copies_wait<0>();
        __syncthreads();
    }
    store_done();
    if (A.zero && !A.only) zero_rest<T>(A, A.y, A.heads, A.vdim, ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x,
                             (long long)gridDim.x * gridDim.y * gridDim.z);
}

// The states' gradients, from the last chunk.  With D the gradient of the state behind a
// chunk, Z = scale dy:
//   dU = P^T Z + until K D,   R = T^T dU,   dV = b R,
//   D <- since_64 D + (since Z)^T Q - (since b R)^T K   (the transposed scan, in the same layout)
template <class P, int KD, int NW>
__global__ void __launch_bounds__(NW * 32, 1) k_delta_back(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using St = Stage<P, KD, NW, P::PIECES>;
    using K = typename Kept<T>::K;
    constexpr int NT = KD / 8, VS = St::VW + PAD;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5;
    const int head = blockIdx.y, col0 = (int)blockIdx.z * St::VW, col = col0 + warp * 16;
    const int w = A.vdim - col;
    for (long long s = blockIdx.x; s < A.n_seq; s += gridDim.x) {
        const Span sp = span_of(A, s);
        const int chunks = (sp.len + C - 1) / C;
        float D[NT][4], sigma = 1.0f;
        read_state<NT>(D, A.dh ? A.dh + (s * A.heads + head) * A.kdim * A.vdim : nullptr, A, col, A.vdim);
        if (St::STAGES == 2 && chunks) St(smem).load(A, A.dy, s, sp, chunks - 1, head, col0, A.vdim, tid);
        copies_end();
        for (int i = 0; i < chunks; ++i) {
            const int c = chunks - 1 - i;
            const St st(smem + (St::STAGES == 2 ? (i & 1) * St::BYTES : 0));
            if (St::STAGES == 1) St(smem).load(A, A.dy, s, sp, c, head, col0, A.vdim, tid);
            else if (c > 0) St(smem + ((i + 1) & 1) * St::BYTES).load(A, A.dy, s, sp, c - 1, head, col0, A.vdim, tid);
            copies_end();
            copies_wait<St::STAGES - 1>();
            __syncthreads();
            if (w > 0) {
                const int n = min(C, sp.len - c * C);
                const long long unit = (sp.chunk + c) * A.heads + head;
                float top = 0.0f;
                if constexpr (P::SCALED) recentre(D, sigma, top);
                float back = inverse_of(sigma), ik = 1.0f, iq = 1.0f;
                if constexpr (P::SCALED) {
                    ik = inverse_of(st.f[K_SCALE]);
                    iq = inverse_of(st.f[Q_SCALE]);
                }
                keep_state<K, NT>(D, back, St::keep(smem, warp), (K*)A.dstates + (unit * A.vdim + col) * (KD + PAD), w);
                float u[8][4] = {}, r[8][4] = {}, z[8][4];
#pragma unroll
                for (int d = 0; d < KD / 16; ++d) {
                    const typename P::A a = P::split(D[2 * d], D[2 * d + 1], 1.0f);
                    read_with<P, P::PIECES, KD>(u, a, st.k, d);
                }
                values_of<T, VS>(z, st.v + warp * 16);
                // u = P^T Z + until K D, times c; the scales of row blocks are made up for in Z, R's in u
                float c1 = 1.0f, c2 = 1.0f, cz = 1.0f, held = sigma;
                if constexpr (P::SCALED) {
                    const float least_p = fminf(fminf(st.f[P_SCALE], st.f[P_SCALE + 1]), fminf(st.f[P_SCALE + 2], st.f[P_SCALE + 3]));
                    cz = scale_for(fabsf(A.scale) * warp_top(z));
                    // (K D, 2^35 / (their scales) at most, is taken times c1)
                    c1 = scale_of_both(scale_within(cz, 0x1p85f * sigma * st.f[K_SCALE] * inverse_of(least_p)), least_p);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 until = pair_at(st.f + C, j);
                    const float f0 = until.x * back * ik, f1 = until.y * back * ik;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[j][e] = u[j][e] * (e & 1 ? f1 : f0) * c1;
                        z[j][e] *= A.scale;
                    }
                }
                times_square<P, P::PIECES, false>(u, z, [&](int d) { return P::SCALED ? c1 * inverse_of(st.f[P_SCALE + d]) : 1.0f; }, st.p);
                if constexpr (P::SCALED)
                    c2 = scale_of_both(warp_scale(u), fminf(fminf(st.f[T_SCALE], st.f[T_SCALE + 1]), fminf(st.f[T_SCALE + 2], st.f[T_SCALE + 3])));
                times_square<P, P::PIECES, false>(r, u, [&](int d) { return P::SCALED ? c2 * inverse_of(st.f[T_SCALE + d]) : 1.0f; }, st.t);
                if constexpr (P::SCALED) {
                    // (R is 2^35 / (c1 c2) at most, Z 2^14 / cz: times D's scale they are finite)
                    held = scale_within(sigma, 0x1p60f * cz * st.f[Q_SCALE], 0x1p70f * c1 * c2 * st.f[K_SCALE]);
                    const float f1 = inverse_of(c1), f2 = inverse_of(c2);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[j][e] = r[j][e] * f2 * f1;
                }
                // (dy's tile is not read any more)
                keep_tile<T, K, VS>(r, st.v + warp * 16, (K*)A.dr + unit * Kept<T>::PLANES * C * A.vpad + col, A.vpad, A.vpad - col);
                // r = b R, u = -since b R, z = since Z, the last two times sigma / ks, sigma / qs
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 since = pair_at(st.f, j), rate = pair_at(st.f + 2 * C, j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float si = (e & 1 ? since.y : since.x) * held;
                        r[j][e] *= e & 1 ? rate.y : rate.x;
                        u[j][e] = r[j][e] * (-si * ik);
                        z[j][e] *= si * iq;
                    }
                }
                store_tile<T, VS>(r, st.v + warp * 16, (T*)A.dv.p + row_at(A, A.dv, s, sp, c * C) + head * A.dv.hs + col, A.dv.st, n, w, A.dv.word);
                if constexpr (P::SCALED) make_room(D, u, z, sigma, held, top * st.f[C - 1]);
                decay_state(D, st.f[LOST], st.f[C - 1]);
                add_outer<P, KD>(D, z, st.q);
                add_outer<P, KD>(D, u, st.k);
            }
            __syncthreads();
        }
        if (A.dh0 && w > 0) write_state<NT>(D, inverse_of(sigma), A.dh0 + (s * A.heads + head) * A.kdim * A.vdim, A, col, A.vdim);
        copies_wait<0>();
        __syncthreads();
    }
    store_done();
}
}  // namespace snnb_delta
