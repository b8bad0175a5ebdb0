// delta_tile.h - kernels of the delta-rule scan (snn_delta_scan) over chunks of 64
// steps, included by one file per element type.
//
// With S the state [dk, dv] before a chunk, a_t the decays, G_ij = a_{j+1} .. a_i,
// since_i = a_1 .. a_i and until_j = a_{j+1} .. a_64 (steps counted in the chunk):
//   A_ij = b_i G_ij k_i.k_j (j < i),   T = (1 + A)^-1,   P_ij = G_ij q_i.k_j (j <= i)
//   U = T b (V - since K S),   Y = scale (since Q S + P U),   S <- since_64 S + (until K)^T U
// which is the recurrence's own sum, reordered (the chunked form of the gated delta
// rule).  T and P do not depend on the state: k_delta_prep makes them for all chunks at
// once.  k_delta_scan then runs along the sequence.  Columns of the state are
// independent, so a warp takes 16 of them, alone: it holds S^T [16, dk] in registers
// as accumulators of the matrix instruction, whose layout (a thread has columns 2t,
// 2t+1 of rows g, g+8) is that of the instruction's first operand again.  So
// every product takes its first operand from the accumulators of the one before it and the
// second (K, Q, T, P; by rows or transposed) from shared memory, and the state never leaves
// the registers.  Tensor memory would hold a state per SM only and pay a round trip
// through shared memory for each of the three products that follow one another in a
// chunk; warps that need not wait for one another hide each other's latency.
//
// Numbers: states, U and sums are f32.  The matrix instruction takes 16-bit (or tf32)
// operands, so an f32 operand is split into pieces that are summed: two of f16 times a
// power of two (22 bits; three of bf16 would be 24), for f32 tensors two of tf32 (22 bits).
// K and Q of 16 bits are exact in one piece of f16, times a power of two a chunk: bf16 has
// fewer bits, and what is below 2^-27 of the chunk's largest element is off by 2^-39 of it
// at most.  What only reaches bf16 Y takes one piece (2^-12).
#pragma once
#include <algorithm>
#include <cfloat>
#include <type_traits>
#include "elem.h"

namespace snnb_delta {
using snnb::from_f32;
using snnb::to_f32;
constexpr int C = 64;         // steps of a chunk
constexpr int MS = C + 8;     // row stride of T and P in shared memory
constexpr int PAD = 8;        // elements behind a row in shared memory: eight rows lie in different banks
// floats of a chunk's factors: since, until, rate, those of Factor; for the gradients
// the logarithms' sums (64 bits) and the counts of decays of 0
constexpr int SCAN_FACTORS = 3 * C + 8, SC = SCAN_FACTORS + 3 * C;
enum Factor { LOST = 3 * C, T_SCALE, P_SCALE, K_SCALE, Q_SCALE, UP = SCAN_FACTORS, CUT = UP + 2 * C };
constexpr int SMS = 148;

struct Heads {                // rows of heads: strides in elements
    void* p;
    long long ss, st, hs;
    int word;                 // bytes of the widest word that rows and heads consist of, 16 at most
};
struct DeltaArgs {
    Heads q, k, v, y, dy, dq, dk, dv;
    Heads gate, beta, dgate, dbeta;
    const float *h0, *dh;
    float *h, *dh0;
    const int64_t* off;
    long long n_seq, slots;   // chunks in all (packed: at most)
    int n_steps, hk, heads, group, kdim, vdim;
    int logit, zero;
    float scale;
    char* keys;               // [slots, hk, 2, C, KD] of Path::KE: K and Q times their scales
    char* squares;            // [slots, heads] of Path::SQUARES bytes: planes [C, C] of T, of P
    float* factors;           // [slots, heads, SC]
    char *states, *u;         // saved: [slots, heads, vdim, KD], [slots, heads, C, vdim] of Path::Kept
    char *dstates, *dr;       // gradients' workspace: the same forms
};

struct Span {
    long long start;          // first row (packed)
    int len;
    long long chunk;          // first chunk
};
__device__ __forceinline__ Span span_of(const DeltaArgs& A, long long s) {
    if (!A.off) return {0, A.n_steps, s * ((A.n_steps + C - 1) / C)};
    const long long n = A.n_steps, b = min(max((long long)A.off[s], 0ll), n), e = min(max((long long)A.off[s + 1], b), n);
    return {b, (int)(e - b), b / C + s};
}
__device__ __forceinline__ long long row_at(const DeltaArgs& A, const Heads& h, long long s, const Span& sp, int t) {
    return A.off ? (sp.start + t) * h.st : s * h.ss + t * h.st;
}

// decay's logarithm and rate of a step
template <typename T>
__device__ __forceinline__ float log_decay(const DeltaArgs& A, T g) {
    const float z = to_f32(g);
    if (!A.logit) return z;
    return z > 0.0f ? -log1pf(expf(-z)) : z - log1pf(expf(z));
}
template <typename T>
__device__ __forceinline__ float rate_of(const DeltaArgs& A, T b) {
    const float z = to_f32(b);
    return A.logit ? 1.0f / (1.0f + expf(-z)) : z;
}

// ---- copies to shared memory --------------------------------------------------
__device__ __forceinline__ void copy16(void* to, const void* from, bool there) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(to);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(a), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int B>
__device__ __forceinline__ void copy_word(void* to, const void* from, bool there) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(to);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(a), "l"(from), "n"(B), "r"(there ? B : 0) : "memory");
}
// R rows of W columns, r and w of them there, zeros in the others; rows `to` of stride W + PAD
template <typename T, int R, int W, int B>
__device__ __forceinline__ void load_by(T* to, const T* from, long long st, int r, int w, int tid, int threads) {
    constexpr int V = B / (int)sizeof(T), N = W / V;
#pragma unroll 4
    for (int i = tid; i < R * N; i += threads) {
        const int a = i / N, c = (i - a * N) * V;
        const bool there = a < r && c < w;
        if (B == 16) copy16(to + a * (W + PAD) + c, there ? from + a * st + c : from, there);
        else copy_word<B>(to + a * (W + PAD) + c, there ? from + a * st + c : from, there);
    }
}
template <typename T, int R, int W>
__device__ __forceinline__ void load_rows(T* to, const T* from, long long st, int r, int w, int word, int tid, int threads) {
    if (word == 16) return load_by<T, R, W, 16>(to, from, st, r, w, tid, threads);
    if (word == 8) return load_by<T, R, W, 8>(to, from, st, r, w, tid, threads);
    if (word == 4) return load_by<T, R, W, 4>(to, from, st, r, w, tid, threads);
    for (int i = tid; i < R * W; i += threads) {
        const int a = i / W, c = i - a * W;
        to[a * (W + PAD) + c] = a < r && c < w ? from[a * st + c] : from_f32<T>(0.0f);
    }
}
// words of 16 bytes as they are
__device__ __forceinline__ void load_words(void* to, const void* from, int bytes, int tid, int threads) {
    for (int i = tid * 16; i < bytes; i += threads * 16) copy16((char*)to + i, (const char*)from + i, true);
}
// one plane [C, C] of a lower triangular matrix: the blocks of 16 on and below the diagonal
template <typename T>
__device__ __forceinline__ void load_lower(T* to, const T* from, int tid, int threads) {
    constexpr int V = 16 / (int)sizeof(T), N = 16 / V;  // words of a block's row
    for (int i = tid; i < 160 * N; i += threads) {
        const int q = i / (16 * N), b = q < 1 ? 0 : q < 3 ? 1 : q < 6 ? 2 : 3;
        const int k = i - 16 * N * (b * (b + 1) / 2), w = N * (b + 1), r = k / w, c = (k - r * w) * V;
        copy16(to + (16 * b + r) * MS + c, from + (16 * b + r) * C + c, true);
    }
}

// ---- products -------------------------------------------------------------------
// A fragment of the first operand [16, 16] comes from two accumulator tiles [16, 8].
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], const void* p) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], const void* p) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma8(float (&d)[4], const unsigned* a, const unsigned* b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// two f32 as a pair of 16-bit values (the first one low), and what that leaves of them
template <typename T>
__device__ __forceinline__ unsigned pair_of(float x, float y) {
    unsigned w;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
    return w;
}
template <typename T>
__device__ __forceinline__ float2 of_pair(unsigned w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
        __half2 h;
        memcpy(&h, &w, 4);
        return __half22float2(h);
    }
}
template <typename T>
__device__ __forceinline__ unsigned piece(float& x, float& y) {
    const unsigned w = pair_of<T>(x, y);
    const float2 f = of_pair<T>(w);
    x -= f.x;
    y -= f.y;
    return w;
}

// 16-bit elements T
template <typename T_>
struct Path16 {
    using T = T_;
    using KE = __half;        // keys, queries and the planes of T and P
    static constexpr bool SCALED = true;
    static constexpr int PLANES = 2, OUT = std::is_same<T, __half>::value ? 2 : 1;  // pieces; of what reaches Y
    static constexpr int PLANE = C * MS, SQUARES = 2 * PLANES * C * C * 2;
    struct A {
        unsigned v[2][4];
    };
    struct B {
        unsigned v[2];
    };
    static __device__ __forceinline__ A split(const float (&x)[4], const float (&y)[4], float s) {
        A a;
        float c[8] = {x[0] * s, x[1] * s, x[2] * s, x[3] * s, y[0] * s, y[1] * s, y[2] * s, y[3] * s};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a.v[0][i] = piece<KE>(c[2 * i], c[2 * i + 1]);
            a.v[1][i] = pair_of<KE>(c[2 * i], c[2 * i + 1]);
        }
        return a;
    }
    // B [16, 2 x 8] with B[k][n] = m[n][k] (rows of m are n), or m[k][n]
    static __device__ __forceinline__ void by_rows(B (&b)[2], const KE* m, int st) {
        const int l = threadIdx.x & 31;
        unsigned r[4];
        ldsm4(r, m + ((l & 7) + (l >> 4) * 8) * st + ((l >> 3) & 1) * 8);
        b[0] = {{r[0], r[1]}};
        b[1] = {{r[2], r[3]}};
    }
    static __device__ __forceinline__ void by_columns(B (&b)[2], const KE* m, int st) {
        const int l = threadIdx.x & 31;
        unsigned r[4];
        ldsm4t(r, m + ((l & 7) + ((l >> 3) & 1) * 8) * st + (l >> 4) * 8);
        b[0] = {{r[0], r[1]}};
        b[1] = {{r[2], r[3]}};
    }
    // d += a b in N pieces of a
    template <int N>
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) {
#pragma unroll
        for (int p = N - 1; p >= 0; --p) {
            mma16<KE>(d0, a.v[p], b[0].v);
            mma16<KE>(d1, a.v[p], b[1].v);
        }
    }
    // the same with a matrix in N planes: the products of pieces i, j with i + j < N
    template <int N, bool ROWS>
    static __device__ __forceinline__ void square(float (&d0)[4], float (&d1)[4], const A& a, const KE* m) {
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            B b[2];
            if (ROWS) by_rows(b, m + j * PLANE, MS);
            else by_columns(b, m + j * PLANE, MS);
#pragma unroll
            for (int p = N - 1 - j; p >= 0; --p) {
                mma16<KE>(d0, a.v[p], b[0].v);
                mma16<KE>(d1, a.v[p], b[1].v);
            }
        }
    }
    // elements (i, j), (i, j + 1) of a matrix into its planes [C, C]
    static __device__ __forceinline__ void put(KE* m, int i, int j, float x, float y, float s) {
        x *= s;
        y *= s;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) *reinterpret_cast<unsigned*>(m + p * C * C + i * C + j) = piece<KE>(x, y);
    }
    // d0, d1 += x y^T for rows in shared memory: 16 rows of x, 2 x 8 of y, 16 columns
    static __device__ __forceinline__ void gram(float (&d0)[4], float (&d1)[4], const KE* x, const KE* y, int st) {
        const int l = threadIdx.x & 31;
        unsigned a[4];
        ldsm4(a, x + (l & 15) * st + (l >> 4) * 8);
        B b[2];
        by_rows(b, y, st);
        mma16<KE>(d0, a, b[0].v);
        mma16<KE>(d1, a, b[1].v);
    }
};

__device__ __forceinline__ unsigned tf32_of(float x) {
    unsigned w;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w) : "f"(x));
    return w;
}
__device__ __forceinline__ void tf32_split(float x, unsigned& h, unsigned& l) {
    h = tf32_of(x);
    l = tf32_of(x - __uint_as_float(h));
}
// f32 elements: two tf32 pieces on both sides.  The k index of an 8-deep product is
// permuted (0, 2, 4, 6, 1, 3, 5, 7), which makes accumulators its first operand.
struct Path32 {
    using T = float;
    using KE = float;
    static constexpr bool SCALED = false;
    static constexpr int PLANES = 1, OUT = 1;
    static constexpr int PLANE = C * MS, SQUARES = 2 * C * C * 4;
    struct A {
        unsigned h[8], l[8];
    };
    struct B {
        unsigned h[4], l[4];
    };
    static __device__ __forceinline__ A split(const float (&x)[4], const float (&y)[4], float) {
        A a;
        const float c[8] = {x[0], x[2], x[1], x[3], y[0], y[2], y[1], y[3]};
#pragma unroll
        for (int i = 0; i < 8; ++i) tf32_split(c[i], a.h[i], a.l[i]);
        return a;
    }
    static __device__ __forceinline__ void by_rows(B (&b)[2], const float* m, int st) {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 v = *reinterpret_cast<const float2*>(m + (n * 8 + g) * st + k * 8 + 2 * t);
                tf32_split(v.x, b[n].h[2 * k], b[n].l[2 * k]);
                tf32_split(v.y, b[n].h[2 * k + 1], b[n].l[2 * k + 1]);
            }
    }
    static __device__ __forceinline__ void by_columns(B (&b)[2], const float* m, int st) {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    tf32_split(m[(k * 8 + 2 * t + i) * st + n * 8 + g], b[n].h[2 * k + i], b[n].l[2 * k + i]);
    }
    static __device__ __forceinline__ void full(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mma8(d0, a.l + 4 * k, b[0].h + 2 * k);
            mma8(d1, a.l + 4 * k, b[1].h + 2 * k);
            mma8(d0, a.h + 4 * k, b[0].l + 2 * k);
            mma8(d1, a.h + 4 * k, b[1].l + 2 * k);
            mma8(d0, a.h + 4 * k, b[0].h + 2 * k);
            mma8(d1, a.h + 4 * k, b[1].h + 2 * k);
        }
    }
    template <int N>
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) { full(d0, d1, a, b); }
    template <int N, bool ROWS>
    static __device__ __forceinline__ void square(float (&d0)[4], float (&d1)[4], const A& a, const float* m) {
        B b[2];
        if (ROWS) by_rows(b, m, MS);
        else by_columns(b, m, MS);
        full(d0, d1, a, b);
    }
    static __device__ __forceinline__ void put(float* m, int i, int j, float x, float y, float) {
        *reinterpret_cast<float2*>(m + i * C + j) = make_float2(x, y);
    }
    // the first operand from shared memory: A[m][k] = x[m][k], or x[k][m]
    static __device__ __forceinline__ A rows_of(const float* x, int st) {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
        A a;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 v = *reinterpret_cast<const float2*>(x + (i * 8 + g) * st + k * 8 + 2 * t);
                tf32_split(v.x, a.h[4 * k + i], a.l[4 * k + i]);
                tf32_split(v.y, a.h[4 * k + 2 + i], a.l[4 * k + 2 + i]);
            }
        return a;
    }
    static __device__ __forceinline__ A columns_of(const float* x, int st) {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
        A a;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    tf32_split(x[(k * 8 + 2 * t + j) * st + i * 8 + g], a.h[4 * k + 2 * j + i], a.l[4 * k + 2 * j + i]);
        return a;
    }
    static __device__ __forceinline__ void gram(float (&d0)[4], float (&d1)[4], const float* x, const float* y, int st) {
        B b[2];
        by_rows(b, y, st);
        full(d0, d1, rows_of(x, st), b);
    }
};
template <typename T> struct PathOf;
template <> struct PathOf<__nv_bfloat16> { using P = Path16<__nv_bfloat16>; };
template <> struct PathOf<__half> { using P = Path16<__half>; };
template <> struct PathOf<float> { using P = Path32; };

// A power of two that brings the largest magnitude to 2^13 .. 2^14, near f16's largest
// values, so that smaller ones keep 24 bits down to 2^-17 of it; held to 2^-40 .. 2^40,
// so that what it multiplies stays finite
__device__ __forceinline__ float scale_for(float top) {
    const int e = min(max(140 + 127 - (int)(__float_as_uint(top) >> 23) , 127 - 40), 127 + 40);
    return __uint_as_float((unsigned)e << 23);
}
__device__ __forceinline__ float inverse_of(float s) {  // of a power of two
    return __uint_as_float((254u << 23) - __float_as_uint(s));
}
template <int N>
__device__ __forceinline__ float warp_scale(const float (&x)[N][4]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[i][j]));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    return scale_for(top);
}

// By one warp: sums of the logarithms of a chunk's decays (64 bits: differences of them
// are what counts) but for those of decays of 0, which are counted apart, and the rates
template <typename T>
__device__ __forceinline__ void chunk_decays(const DeltaArgs& A, long long s, const Span& sp, int t0, int n, int head, int lane,
                                             double* up, int* cut, float* rate) {
    double l[2];
    int z[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        float lg = 0.0f, r = 0.0f;
        if (t < n) {
            lg = log_decay(A, ((const T*)A.gate.p)[row_at(A, A.gate, s, sp, t0 + t) + head * A.gate.hs]);
            r = rate_of(A, ((const T*)A.beta.p)[row_at(A, A.beta, s, sp, t0 + t) + head * A.beta.hs]);
        }
        z[i] = lg == -INFINITY;
        l[i] = z[i] ? 0.0 : (double)lg;
        rate[t] = r;
    }
    double sum = l[0] + l[1];
    int cuts = z[0] + z[1];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double d = __shfl_up_sync(~0u, sum, o);
        const int c = __shfl_up_sync(~0u, cuts, o);
        if (lane >= o) {
            sum += d;
            cuts += c;
        }
    }
    up[2 * lane] = sum - l[1];
    up[2 * lane + 1] = sum;
    cut[2 * lane] = cuts - z[1];
    cut[2 * lane + 1] = cuts;
}
__device__ __forceinline__ float decay_between(const double* up, const int* cut, int i, int j) {
    return cut[i] == cut[j] ? expf((float)(up[i] - up[j])) : 0.0f;
}
// the sequence that chunk `slot` belongs to, the last that does not begin behind it
__device__ __forceinline__ long long sequence_of(const DeltaArgs& A, long long slot) {
    if (!A.off) return slot / ((A.n_steps + C - 1) / C);
    long long lo = 0, hi = A.n_seq - 1;
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (span_of(A, mid).chunk <= slot) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- keys, T, P and the factors of every chunk -----------------------------------
// A CTA of four warps for a chunk and head, 16 rows to a warp.  T by blocks of 16: a
// warp inverts its block on the diagonal by substitution, a column to a lane, then
// with N = -T_ii A_im:  T_ij = sum of N_im T_mj, one row of blocks after the other, in f32
// by two tf32 pieces.
constexpr int PREP = 128, XS = C + 8;
template <class P, int KD>
constexpr int prep_smem() {
    const int keys = 2 * C * (KD + PAD) * (int)sizeof(typename P::KE), m = C * XS * 4;
    return keys > m ? keys : m;  // A and T take the place of K and Q
}
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
// the same times s as KE, to shared memory (stride KD + PAD) and, unless null, to memory (stride KD)
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
        if (copy) *reinterpret_cast<uint4*>(copy + r * KD + c) = o;
    }
}
template <class P, int KD>
__global__ void __launch_bounds__(PREP) k_delta_prep(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using KE = typename P::KE;
    constexpr int KS = KD + PAD, WORDS = C * KD * (int)sizeof(T) / 16 / PREP;
    extern __shared__ __align__(16) char smem[];
    KE *K = reinterpret_cast<KE*>(smem), *Q = K + C * KS;
    float* M = reinterpret_cast<float*>(smem);  // [C][XS]
    __shared__ double up[C];
    __shared__ int cut[C];
    __shared__ float rate[C], top[4][4];
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
        if (warp == 3) chunk_decays<T>(A, s, sp, t0, n, head, lane, up, cut, rate);
        if constexpr (P::SCALED) {
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                a = fmaxf(a, __shfl_xor_sync(~0u, a, o));
                b = fmaxf(b, __shfl_xor_sync(~0u, b, o));
            }
            if (lane == 0) {
                top[0][warp] = a;
                top[1][warp] = b;
            }
            __syncthreads();
            ks = scale_for(fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3])));
            qs = scale_for(fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3])));
        }
        KE* copy = head % A.group == 0 ? (KE*)A.keys + (slot * A.hk + kh) * 2 * C * KD : nullptr;
        write_keys<T, KE, KD>(wk, K, copy, ks);
        write_keys<T, KE, KD>(wq, Q, copy ? copy + C * KD : nullptr, qs);
    }
    __syncthreads();
    const long long unit = slot * A.heads + head;
    float* F = A.factors + unit * SC;
    KE *Tm = reinterpret_cast<KE*>(A.squares + unit * P::SQUARES), *Pm = Tm + P::PLANES * C * C;
    if (tid < C) {
        F[tid] = cut[tid] ? 0.0f : expf((float)up[tid]);
        F[C + tid] = decay_between(up, cut, C - 1, tid);
        F[2 * C + tid] = rate[tid];
        reinterpret_cast<double*>(F + UP)[tid] = up[tid];
        reinterpret_cast<int*>(F + CUT)[tid] = cut[tid];
        if (tid == 0) F[LOST] = cut[C - 1] ? 1.0f : -expm1f((float)up[C - 1]);
    }
    // this warp's rows of the products of keys, and of queries with keys
    float kk[8][4] = {}, qk[8][4] = {};
#pragma unroll
    for (int np = 0; np < 4; ++np) {
        if (np > warp) break;  // above the diagonal
#pragma unroll 4
        for (int d = 0; d < KD; d += 16) {
            P::gram(kk[2 * np], kk[2 * np + 1], K + warp * 16 * KS + d, K + np * 16 * KS + d, KS);
            P::gram(qk[2 * np], qk[2 * np + 1], Q + warp * 16 * KS + d, K + np * 16 * KS + d, KS);
        }
    }
    const float kks = inverse_of(ks) * inverse_of(ks), qks = inverse_of(ks) * inverse_of(qs);
    __syncthreads();
    float most = 0.0f;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = warp * 16 + g + (e >> 1) * 8, j = nt * 8 + 2 * t4 + (e & 1);
            const float G = j <= i ? decay_between(up, cut, i, j) : 0.0f;
            // (a factor of 0 takes all: what lies above the diagonal may be anything)
            qk[nt][e] = G != 0.0f ? G * (qk[nt][e] * qks) : 0.0f;
            const float a = rate[i] * G;
            M[i * XS + j] = j < i && a != 0.0f ? a * (kk[nt][e] * kks) : 0.0f;
            most = fmaxf(most, fabsf(qk[nt][e]));
        }
    }
    __syncwarp();
    // the block on the diagonal
    float* own = M + warp * 16 * (XS + 1);
    {
        const int c = lane & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
            for (int m = 0; m < i; m += 2) {
                const float2 r = *reinterpret_cast<const float2*>(own + i * XS + m);
                a0 = fmaf(r.x, x[m], a0);
                if (m + 1 < i) a1 = fmaf(r.y, x[m + 1], a1);
            }
            x[i] = i < c ? 0.0f : (i == c ? 1.0f : 0.0f) - (a0 + a1);
        }
        __syncwarp();
        if (lane < 16)
#pragma unroll
            for (int i = 0; i < 16; ++i) own[i * XS + c] = x[i];
    }
    __syncwarp();
    float N[3][2][4] = {};
    {
        const Path32::A a = Path32::rows_of(own, XS);
#pragma unroll
        for (int m = 0; m < 3; ++m)
            if (m < warp) {
                Path32::B b[2];
                Path32::by_columns(b, M + warp * 16 * XS + m * 16, XS);
                Path32::full(N[m][0], N[m][1], a, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    N[m][0][e] = -N[m][0][e];
                    N[m][1][e] = -N[m][1][e];
                }
            }
    }
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        __syncthreads();  // the rows of blocks above are there
        if (warp != i) continue;
        float t[3][2][4] = {};
#pragma unroll
        for (int m = 0; m < i; ++m) {
            const Path32::A a = Path32::split(N[m][0], N[m][1], 1.0f);
#pragma unroll
            for (int j = 0; j <= m; ++j) {
                Path32::B b[2];
                Path32::by_columns(b, M + m * 16 * XS + j * 16, XS);
                Path32::full(t[j][0], t[j][1], a, b);
            }
        }
#pragma unroll
        for (int j = 0; j < i; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) M[(i * 16 + g + (e >> 1) * 8) * XS + j * 16 + h * 8 + 2 * t4 + (e & 1)] = t[j][h][e];
        __syncwarp();
    }
    // out, this warp's rows
    float ps = 1.0f, ts = 1.0f;
    const int pairs = 8 * (warp + 1);
    if constexpr (P::SCALED) {
        float big = 0.0f;
        for (int i = lane; i < 16 * pairs; i += 32) {
            const float2 v = *reinterpret_cast<const float2*>(M + (warp * 16 + i / pairs) * XS + 2 * (i % pairs));
            big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
            big = fmaxf(big, __shfl_xor_sync(~0u, big, o));
        }
        if (lane == 0) {
            top[2][warp] = most;
            top[3][warp] = big;
        }
        __syncthreads();
        ps = scale_for(fmaxf(fmaxf(top[2][0], top[2][1]), fmaxf(top[2][2], top[2][3])));
        ts = scale_for(fmaxf(fmaxf(top[3][0], top[3][1]), fmaxf(top[3][2], top[3][3])));
    }
    for (int i = lane; i < 16 * pairs; i += 32) {
        const int r = warp * 16 + i / pairs, c = 2 * (i % pairs);
        const float2 v = *reinterpret_cast<const float2*>(M + r * XS + c);
        P::put(Tm, r, c, v.x, v.y, ts);
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
        if (nt / 2 > warp) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) P::put(Pm, warp * 16 + g + h * 8, nt * 8 + 2 * t4, qk[nt][2 * h], qk[nt][2 * h + 1], ps);
    }
    if (tid == 0) {
        F[T_SCALE] = ts;
        F[P_SCALE] = ps;
        F[K_SCALE] = ks;
        F[Q_SCALE] = qs;
    }
}

// ---- along the sequences ------------------------------------------------------------
template <class P, int KD, int NW, int PP>  // PP: planes of P
struct Stage {
    using T = typename P::T;
    using KE = typename P::KE;
    static constexpr int VW = 16 * NW;
    static constexpr int KEYS = C * (KD + PAD) * (int)sizeof(KE), VALUES = C * (VW + PAD) * (int)sizeof(T);
    static constexpr int SQUARES = (P::PLANES + PP) * P::PLANE * (int)sizeof(KE);
    static constexpr int BYTES = 2 * KEYS + VALUES + SQUARES + SCAN_FACTORS * 4;
    static constexpr int STAGES = 2 * BYTES <= 227 * 1024 - 1024 ? 2 : 1;
    KE *k, *q, *t, *p;
    T* v;
    float* f;
    __device__ __forceinline__ explicit Stage(char* m) {
        k = reinterpret_cast<KE*>(m);
        q = reinterpret_cast<KE*>(m + KEYS);
        v = reinterpret_cast<T*>(m + 2 * KEYS);
        t = reinterpret_cast<KE*>(m + 2 * KEYS + VALUES);
        p = t + P::PLANES * P::PLANE;
        f = reinterpret_cast<float*>(m + 2 * KEYS + VALUES + SQUARES);
    }
    // chunk c of sequence s; vals: the values' rows or, backward, those of dy (or none)
    __device__ __forceinline__ void load(const DeltaArgs& A, const Heads& vals, long long s, const Span& sp, int c, int head,
                                         int col0, int tid) {
        const int n = min(C, sp.len - c * C);
        const long long slot = sp.chunk + c, unit = slot * A.heads + head;
        const KE* keys = (const KE*)A.keys + (slot * A.hk + head / A.group) * 2 * C * KD;
        load_rows<KE, C, KD>(k, keys, KD, C, KD, 16, tid, NW * 32);
        load_rows<KE, C, KD>(q, keys + C * KD, KD, C, KD, 16, tid, NW * 32);
        load_rows<T, C, VW>(v, (const T*)vals.p + row_at(A, vals, s, sp, c * C) + head * vals.hs + col0, vals.st,
                            vals.p ? n : 0, A.vdim - col0, vals.word, tid, NW * 32);
        const KE* sq = reinterpret_cast<const KE*>(A.squares + unit * P::SQUARES);
#pragma unroll
        for (int i = 0; i < P::PLANES; ++i) load_lower(t + i * P::PLANE, sq + i * C * C, tid, NW * 32);
#pragma unroll
        for (int i = 0; i < PP; ++i) load_lower(p + i * P::PLANE, sq + (P::PLANES + i) * C * C, tid, NW * 32);
        load_words(f, A.factors + unit * SC, SCAN_FACTORS * 4, tid, NW * 32);
    }
};

// a warp's tile [16 columns, C steps] (accumulators) as rows of T: into its columns of
// `stage` [C][VW + PAD], from there to memory
template <typename T, int ST>
__device__ __forceinline__ void store_tile(const float (&o)[8][4], T* stage, T* to, long long st, int n, int w, int word) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) stage[(i * 8 + 2 * t4 + (e & 1)) * ST + g + (e >> 1) * 8] = from_f32<T>(o[i][e]);
    __syncwarp();
    auto words = [&](auto z) {
        using W = decltype(z);
        constexpr int V = (int)(sizeof(W) / sizeof(T)), N = 16 / V;
        for (int i = lane; i < n * N; i += 32) {
            const int r = i / N, c = i % N * V;
            if (c < w) *reinterpret_cast<W*>(to + r * st + c) = *reinterpret_cast<const W*>(stage + r * ST + c);
        }
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

// S^T [16 columns, KD] of a warp as it is kept for the gradient: rows of KD elements
template <typename T, int NT>
__device__ __forceinline__ void keep_state(const float (&S)[NT][4], T* to, int w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    constexpr int KD = NT * 8;
#pragma unroll
    for (int i = 0; i < NT; i += 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // lanes of even t take four elements of tile i, of odd t of tile i + 1: 16 elements of a row in a store
            const bool odd = t4 & 1;
            const float x = odd ? S[i][2 * h] : S[i + 1][2 * h], y = odd ? S[i][2 * h + 1] : S[i + 1][2 * h + 1];
            const float px = __shfl_xor_sync(~0u, x, 1), py = __shfl_xor_sync(~0u, y, 1);
            const float mx = odd ? S[i + 1][2 * h] : S[i][2 * h], my = odd ? S[i + 1][2 * h + 1] : S[i][2 * h + 1];
            const int row = g + 8 * h, col = (i + odd) * 8 + (t4 >> 1) * 4;
            if (row < w) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(to + row * KD + col) = odd ? make_float4(px, py, mx, my) : make_float4(mx, my, px, py);
                } else {
                    const unsigned a = pair_of<T>(mx, my), b = pair_of<T>(px, py);
                    *reinterpret_cast<uint2*>(to + row * KD + col) = odd ? make_uint2(b, a) : make_uint2(a, b);
                }
            }
        }
}
// f32 states [kdim, vdim] from and to a warp's columns
template <int NT>
__device__ __forceinline__ void read_state(float (&S)[NT][4], const float* h, const DeltaArgs& A, int col) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = col + g + (e >> 1) * 8, d = i * 8 + 2 * t4 + (e & 1);
            S[i][e] = h && c < A.vdim && d < A.kdim ? h[(long long)d * A.vdim + c] : 0.0f;
        }
}
template <int NT>
__device__ __forceinline__ void write_state(const float (&S)[NT][4], float* h, const DeltaArgs& A, int col) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = col + g + (e >> 1) * 8, d = i * 8 + 2 * t4 + (e & 1);
            if (c < A.vdim && d < A.kdim) h[(long long)d * A.vdim + c] = S[i][e];
        }
}

// what the gradient needs of states and U in which type: bf16 gradients are rounded to
// 8 bits themselves
template <typename T> struct Kept { using K = float; };
template <> struct Kept<__nv_bfloat16> { using K = __nv_bfloat16; };

// rows of no sequence become zero in y-like tensors
template <typename T>
__device__ void zero_rest(const DeltaArgs& A, const Heads& r, int heads, int width, long long cta, long long ctas) {
    if (!r.p) return;
    const long long n = A.n_steps;
    const long long first = A.n_seq ? min(max((long long)A.off[0], 0ll), n) : n, last = A.n_seq ? min(max((long long)A.off[A.n_seq], first), n) : n;
    const long long rows = first + (n - last), per = (long long)heads * width;
    for (long long i = cta * blockDim.x + threadIdx.x; i < rows * per; i += ctas * blockDim.x) {
        const long long k = i / per, e = i - k * per, row = k < first ? k : last + (k - first);
        ((T*)r.p)[row * r.st + e / width * r.hs + e % width] = from_f32<T>(0.0f);
    }
}

template <class P, int KD, int NW>
__global__ void __launch_bounds__(NW * 32, 1) k_delta_scan(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using St = Stage<P, KD, NW, P::OUT>;
    using K = typename Kept<T>::K;
    constexpr int NT = KD / 8, KS = KD + PAD, VS = St::VW + PAD;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int head = blockIdx.y, col0 = (int)blockIdx.z * St::VW, col = col0 + warp * 16;
    const int w = A.vdim - col;  // this warp's columns (16 and more: all; none: it only loads)
    for (long long s = blockIdx.x; s < A.n_seq; s += gridDim.x) {
        const Span sp = span_of(A, s);
        const int chunks = (sp.len + C - 1) / C;
        float S[NT][4];
        read_state<NT>(S, A.h0 ? A.h0 + (s * A.heads + head) * A.kdim * A.vdim : nullptr, A, col);
        if (St::STAGES == 2 && chunks) St(smem).load(A, A.v, s, sp, 0, head, col0, tid);
        copies_end();
        for (int c = 0; c < chunks; ++c) {
            const St st(smem + (St::STAGES == 2 ? (c & 1) * St::BYTES : 0));
            if (St::STAGES == 1) St(smem).load(A, A.v, s, sp, c, head, col0, tid);
            else if (c + 1 < chunks) St(smem + ((c + 1) & 1) * St::BYTES).load(A, A.v, s, sp, c + 1, head, col0, tid);
            copies_end();
            copies_wait<St::STAGES - 1>();
            __syncthreads();
            if (w > 0) {
                const int n = min(C, sp.len - c * C);
                const long long unit = (sp.chunk + c) * A.heads + head;
                if (A.states) keep_state<K, NT>(S, (K*)A.states + (unit * A.vdim + col) * KD, w);
                float r[8][4] = {}, o[8][4] = {};
                float ss = 1.0f, back = 1.0f;
                if constexpr (P::SCALED) {
                    ss = warp_scale(S);
                    back = inverse_of(ss);
                }
#pragma unroll
                for (int d = 0; d < KD / 16; ++d) {
                    const typename P::A a = P::split(S[2 * d], S[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np) {
                        typename P::B b[2], e[2];
                        P::by_rows(b, st.k + np * 16 * KS + d * 16, KS);
                        P::by_rows(e, st.q + np * 16 * KS + d * 16, KS);
                        P::template mma<2>(r[2 * np], r[2 * np + 1], a, b);
                        P::template mma<P::OUT>(o[2 * np], o[2 * np + 1], a, e);
                    }
                }
                // r = b (v - since r), o = since o
                const float fk = P::SCALED ? back * inverse_of(st.f[K_SCALE]) : 1.0f, fq = P::SCALED ? back * inverse_of(st.f[Q_SCALE]) : 1.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 since = *reinterpret_cast<const float2*>(st.f + i * 8 + 2 * t4);
                    const float2 rate = *reinterpret_cast<const float2*>(st.f + 2 * C + i * 8 + 2 * t4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float f = e & 1 ? since.y : since.x;
                        const float v = to_f32(st.v[(i * 8 + 2 * t4 + (e & 1)) * VS + warp * 16 + g + (e >> 1) * 8]);
                        r[i][e] = (e & 1 ? rate.y : rate.x) * fmaf(-f * fk, r[i][e], v);
                        o[i][e] *= f * fq;
                    }
                }
                // U = T r
                float u[8][4] = {};
                if constexpr (P::SCALED) ss = warp_scale(r);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(r[2 * d], r[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np)
                        if (np >= d)
                            P::template square<P::PLANES, true>(u[2 * np], u[2 * np + 1], a, st.t + np * 16 * MS + d * 16);
                }
                if constexpr (P::SCALED) {
                    const float f = inverse_of(ss) * inverse_of(st.f[T_SCALE]);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[i][e] *= f;
                    ss = warp_scale(u);
                    const float up = ss * st.f[P_SCALE];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][e] *= up;
                    back = inverse_of(ss) * inverse_of(st.f[P_SCALE]);
                }
                // o += P U
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(u[2 * d], u[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np)
                        if (np >= d)
                            P::template square<P::OUT, true>(o[2 * np], o[2 * np + 1], a, st.p + np * 16 * MS + d * 16);
                }
                const float f = P::SCALED ? A.scale * back : A.scale;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] *= f;
                store_tile<T, VS>(o, st.v + warp * 16, (T*)A.y.p + row_at(A, A.y, s, sp, c * C) + head * A.y.hs + col, A.y.st, n, w, A.y.word);
                if (A.u) {
                    K* to = (K*)A.u + unit * C * A.vdim + col;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int t = i * 8 + 2 * t4 + (e & 1), cc = g + (e >> 1) * 8;
                            if (cc < w) to[(long long)t * A.vdim + cc] = from_f32<K>(u[i][e]);
                        }
                }
                // S = since_64 S + (until U)^T K; 1 - since_64 keeps its bits where decays are near 1
                const float lost = st.f[LOST];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 until = *reinterpret_cast<const float2*>(st.f + C + i * 8 + 2 * t4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[i][e] *= e & 1 ? until.y : until.x;
                }
                float both = 1.0f;
                if constexpr (P::SCALED) {
                    ss = warp_scale(u);
                    both = ss * st.f[K_SCALE];
                    back = inverse_of(ss) * inverse_of(st.f[K_SCALE]);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        S[i][e] = fmaf(-lost, S[i][e], S[i][e]);
                        if constexpr (P::SCALED) S[i][e] *= both;
                    }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(u[2 * d], u[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < KD / 16; ++np) {
                        typename P::B b[2];
                        P::by_columns(b, st.k + d * 16 * KS + np * 16, KS);
                        P::template mma<2>(S[2 * np], S[2 * np + 1], a, b);
                    }
                }
                if constexpr (P::SCALED)
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) S[i][e] *= back;
            }
            __syncthreads();
        }
        if (A.h && w > 0) write_state<NT>(S, A.h + (s * A.heads + head) * A.kdim * A.vdim, A, col);
        copies_wait<0>();
        __syncthreads();
    }
    if (A.zero) zero_rest<T>(A, A.y, A.heads, A.vdim, ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x,
                             (long long)gridDim.x * gridDim.y * gridDim.z);
}

// ---- gradients: the states' along the sequences, from the last chunk ------------------
// With D the gradient of the state behind a chunk, Z = scale dy:
//   dU = P^T Z + until K D,   R = T^T dU,   dV = b R,
//   D <- since_64 D + (since Z)^T Q - (since b R)^T K   (the transposed scan, in the same layout)
template <class P, int KD, int NW>
__global__ void __launch_bounds__(NW * 32, 1) k_delta_back(const __grid_constant__ DeltaArgs A) {
    using T = typename P::T;
    using St = Stage<P, KD, NW, P::PLANES>;
    using K = typename Kept<T>::K;
    constexpr int NT = KD / 8, KS = KD + PAD, VS = St::VW + PAD;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int head = blockIdx.y, col0 = (int)blockIdx.z * St::VW, col = col0 + warp * 16;
    const int w = A.vdim - col;
    for (long long s = blockIdx.x; s < A.n_seq; s += gridDim.x) {
        const Span sp = span_of(A, s);
        const int chunks = (sp.len + C - 1) / C;
        float D[NT][4];
        read_state<NT>(D, A.dh ? A.dh + (s * A.heads + head) * A.kdim * A.vdim : nullptr, A, col);
        if (St::STAGES == 2 && chunks) St(smem).load(A, A.dy, s, sp, chunks - 1, head, col0, tid);
        copies_end();
        for (int i = 0; i < chunks; ++i) {
            const int c = chunks - 1 - i;
            const St st(smem + (St::STAGES == 2 ? (i & 1) * St::BYTES : 0));
            if (St::STAGES == 1) St(smem).load(A, A.dy, s, sp, c, head, col0, tid);
            else if (c > 0) St(smem + ((i + 1) & 1) * St::BYTES).load(A, A.dy, s, sp, c - 1, head, col0, tid);
            copies_end();
            copies_wait<St::STAGES - 1>();
            __syncthreads();
            if (w > 0) {
                const int n = min(C, sp.len - c * C);
                const long long unit = (sp.chunk + c) * A.heads + head;
                keep_state<K, NT>(D, (K*)A.dstates + (unit * A.vdim + col) * KD, w);
                float u[8][4] = {}, r[8][4] = {}, z[8][4];
                float ss = 1.0f, back = 1.0f;
                if constexpr (P::SCALED) {
                    ss = warp_scale(D);
                    back = inverse_of(ss);
                }
#pragma unroll
                for (int d = 0; d < KD / 16; ++d) {
                    const typename P::A a = P::split(D[2 * d], D[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np) {
                        typename P::B b[2];
                        P::by_rows(b, st.k + np * 16 * KS + d * 16, KS);
                        P::template mma<2>(u[2 * np], u[2 * np + 1], a, b);
                    }
                }
                if constexpr (P::SCALED) back *= inverse_of(st.f[K_SCALE]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 until = *reinterpret_cast<const float2*>(st.f + C + j * 8 + 2 * t4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[j][e] *= (e & 1 ? until.y : until.x) * back;
                        z[j][e] = A.scale * to_f32(st.v[(j * 8 + 2 * t4 + (e & 1)) * VS + warp * 16 + g + (e >> 1) * 8]);
                    }
                }
                if constexpr (P::SCALED) {
                    ss = warp_scale(z);
                    const float f = ss * st.f[P_SCALE];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[j][e] *= f;
                }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(z[2 * d], z[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np)
                        if (np <= d)
                            P::template square<P::PLANES, false>(u[2 * np], u[2 * np + 1], a, st.p + d * 16 * MS + np * 16);
                }
                if constexpr (P::SCALED) {
                    back = inverse_of(ss) * inverse_of(st.f[P_SCALE]);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[j][e] *= back;
                    ss = warp_scale(u);
                }
                // R = T^T dU
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(u[2 * d], u[2 * d + 1], ss);
#pragma unroll
                    for (int np = 0; np < 4; ++np)
                        if (np <= d)
                            P::template square<P::PLANES, false>(r[2 * np], r[2 * np + 1], a, st.t + d * 16 * MS + np * 16);
                }
                const float f = P::SCALED ? inverse_of(ss) * inverse_of(st.f[T_SCALE]) : 1.0f;
                K* to = (K*)A.dr + unit * C * A.vdim + col;
                // u <- -since b R, z <- since Z
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 since = *reinterpret_cast<const float2*>(st.f + j * 8 + 2 * t4);
                    const float2 rate = *reinterpret_cast<const float2*>(st.f + 2 * C + j * 8 + 2 * t4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = j * 8 + 2 * t4 + (e & 1), cc = g + (e >> 1) * 8;
                        if constexpr (P::SCALED) r[j][e] *= f;
                        if (cc < w) to[(long long)t * A.vdim + cc] = from_f32<K>(r[j][e]);
                        const float si = e & 1 ? since.y : since.x;
                        r[j][e] *= e & 1 ? rate.y : rate.x;
                        u[j][e] = -si * r[j][e];
                        z[j][e] *= si;
                    }
                }
                const float lost = st.f[LOST];
                float su = 1.0f, sz = 1.0f, both = 1.0f;
                if constexpr (P::SCALED) {
                    both = fminf(warp_scale(u) * st.f[K_SCALE], warp_scale(z) * st.f[Q_SCALE]);
                    su = both * inverse_of(st.f[K_SCALE]);
                    sz = both * inverse_of(st.f[Q_SCALE]);
                    back = inverse_of(both);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        D[j][e] = fmaf(-lost, D[j][e], D[j][e]);
                        if constexpr (P::SCALED) D[j][e] *= both;
                    }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const typename P::A a = P::split(z[2 * d], z[2 * d + 1], sz), m = P::split(u[2 * d], u[2 * d + 1], su);
#pragma unroll
                    for (int np = 0; np < KD / 16; ++np) {
                        typename P::B b[2];
                        P::by_columns(b, st.q + d * 16 * KS + np * 16, KS);
                        P::template mma<2>(D[2 * np], D[2 * np + 1], a, b);
                        P::by_columns(b, st.k + d * 16 * KS + np * 16, KS);
                        P::template mma<2>(D[2 * np], D[2 * np + 1], m, b);
                    }
                }
                if constexpr (P::SCALED)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) D[j][e] *= back;
                store_tile<T, VS>(r, st.v + warp * 16, (T*)A.dv.p + row_at(A, A.dv, s, sp, c * C) + head * A.dv.hs + col, A.dv.st, n, w, A.dv.word);
            }
            __syncthreads();
        }
        if (A.dh0 && w > 0) write_state<NT>(D, A.dh0 + (s * A.heads + head) * A.kdim * A.vdim, A, col);
        copies_wait<0>();
        __syncthreads();
    }
}

// ---- gradients: what is left, for all chunks at once -------------------------------------
// With S before a chunk, D behind it, U and R as above, G the decays between steps:
//   p = G (Z U^T) (j <= i),   x = -b G (R U^T) (j < i)
//   dQ = since Z S^T + p K,   dK = -since b R S^T + until U D^T + x K + x^T K + p^T Q
//   db_i = R_i.V_i - since_i k_i.(S R_i) + sum_j x_ij k_i.k_j / b_i
// and for the logarithm of a decay all terms that it is a factor of: their sum over
// i >= t > j, as sums over rows less sums over columns from t on.
// Products over the values' columns have bf16 operands for bf16 tensors (as the results
// are rounded), otherwise f32 in two tf32 pieces; those over steps the keys' type, p and x in
// one piece of f16 for bf16 tensors, two for f16.  16 warps: 16 rows and a quarter
// of the columns each; half of the registers are accumulators.
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

// as load_rows, of another type F
template <typename E, int R, int W, typename F>
__device__ __forceinline__ void load_as(E* to, const F* from, long long st, int r, int w, int word, int tid, int threads) {
    if constexpr (std::is_same<E, F>::value) {
        load_rows<E, R, W>(to, from, st, r, w, word, tid, threads);
    } else {
        for (int i = tid; i < R * W; i += threads) {
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

constexpr int GRADS = 512;
template <typename T, int KD>
struct GradTile {
    using E = typename Kept<T>::K;             // of the blocks
    using KE = typename PathOf<T>::P::KE;      // of keys, p and x
    static constexpr int GW = sizeof(E) == 2 ? 64 : 32;  // columns of the values taken at a time
    static constexpr int STAGES = sizeof(E) == 2 ? 2 : 1, PIECES = sizeof(E) == 4 && sizeof(KE) == 2 ? 2 : 1;
    static constexpr int KEYS = C * (KD + PAD), ROWS = C * (GW + PAD), STATE = GW * (KD + PAD);
    static constexpr int BLOCK = 4 * ROWS + 2 * STATE, SQ = PIECES * C * MS;
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
    __shared__ float rows[4][4][C], cols[4][C], more[GRADS / 32], dots[C], top[2][GRADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int wr = warp & 3, wc = warp >> 2, kh = blockIdx.y;
    const long long slot = blockIdx.x, s = sequence_of(A, slot);
    const Span sp = span_of(A, s);
    const long long first = (slot - sp.chunk) * C;
    if (first < 0 || first >= sp.len) return;
    const int t0 = (int)first, n = min(C, sp.len - t0);
    const KE* keys = (const KE*)A.keys + (slot * A.hk + kh) * 2 * C * KD;
    float tq[NQ][4] = {}, tk[NQ][4] = {};
    const int n_blocks = (A.vdim + GW - 1) / GW;
    const int kept = (A.vdim * (int)sizeof(E)) % 16 == 0 ? 16 : (A.vdim * (int)sizeof(E)) % 8 == 0 ? 8 : (A.vdim * (int)sizeof(E)) % 4 == 0 ? 4 : 2;
#pragma unroll 1
    for (int gi = 0; gi < A.group; ++gi) {
        const int head = kh * A.group + gi;
        const long long unit = slot * A.heads + head;
        auto load = [&](int b) {
            E* m = blocks + (G::STAGES == 2 ? (b & 1) * G::BLOCK : 0);
            const int c0 = b * GW, w = A.vdim - c0;
            load_as<E, C, GW>(m, (const T*)A.dy.p + row_at(A, A.dy, s, sp, t0) + head * A.dy.hs + c0, A.dy.st, A.dy.p ? n : 0, w, A.dy.word, tid, GRADS);
            load_as<E, C, GW>(m + G::ROWS, (const E*)A.u + unit * C * A.vdim + c0, A.vdim, C, w, kept, tid, GRADS);
            load_as<E, C, GW>(m + 2 * G::ROWS, (const E*)A.dr + unit * C * A.vdim + c0, A.vdim, C, w, kept, tid, GRADS);
            load_as<E, C, GW>(m + 3 * G::ROWS, (const T*)A.v.p + row_at(A, A.v, s, sp, t0) + head * A.v.hs + c0, A.v.st, n, w, A.v.word, tid, GRADS);
            load_rows<E, GW, KD>(m + 4 * G::ROWS, (const E*)A.states + (unit * A.vdim + c0) * KD, KD, w, KD, 16, tid, GRADS);
            load_rows<E, GW, KD>(m + 4 * G::ROWS + G::STATE, (const E*)A.dstates + (unit * A.vdim + c0) * KD, KD, w, KD, 16, tid, GRADS);
        };
        if (gi == 0) {
            load_rows<KE, C, KD>(Ks, keys, KD, C, KD, 16, tid, GRADS);
            load_rows<KE, C, KD>(Qs, keys + C * KD, KD, C, KD, 16, tid, GRADS);
        }
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
#pragma unroll
            for (int k = 0; k < GW; k += 16) {
                const typename Op::A az = Op::rows_of(Z + wr * 16 * RS + k, RS), ar = Op::rows_of(R + wr * 16 * RS + k, RS);
                const typename Op::A au = Op::rows_of(U + wr * 16 * RS + k, RS);
                typename Op::B bb[2];
#pragma unroll
                for (int j = 0; j < NQ; j += 2) {
                    Op::by_columns(bb, S + k * KS + wc * (KD / 4) + j * 8, KS);
                    Op::mma(zq[j], zq[j + 1], az, bb);
                    Op::mma(zk[j], zk[j + 1], ar, bb);
                    Op::by_columns(bb, D + k * KS + wc * (KD / 4) + j * 8, KS);
                    Op::mma(zm[j], zm[j + 1], au, bb);
                }
                if (wc <= wr) {
                    Op::by_rows(bb, U + wc * 16 * RS + k, RS);
                    Op::mma(p[0], p[1], az, bb);
                    Op::mma(x[0], x[1], ar, bb);
                }
            }
            constexpr int V4 = 16 / (int)sizeof(E);
            static_assert(C * GW / V4 == GRADS, "a word of R and V to a thread");
            const int at = (tid >> 3) * RS + (tid & 7) * V4;
            rv = word_dot(R + at, V + at, rv);
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
        const double* up = reinterpret_cast<const double*>(F + UP);
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
        float tp = 0.0f, tx = 0.0f;
        if (wc <= wr)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = wr * 16 + g + (e >> 1) * 8, jj = wc * 16 + j * 8 + 2 * t4 + (e & 1);
                    const float d = jj <= i ? decay_between(up, cut, i, jj) : 0.0f;
                    const float pv = d != 0.0f ? A.scale * d * p[j][e] : 0.0f, xv = d != 0.0f && jj < i ? -d * x[j][e] : 0.0f;
                    const float xr = xv * (kk[j][e] * ik * ik), mp = pv * (qk[j][e] * ik * iq), both = fmaf(rate[i], xr, mp);
                    by_row[0][e >> 1] += both;
                    by_row[3][e >> 1] += xr;
                    by_col[j][e & 1] += both;
                    p[j][e] = pv;
                    x[j][e] = rate[i] * xv;
                    tp = fmaxf(tp, fabsf(p[j][e]));
                    tx = fmaxf(tx, fabsf(x[j][e]));
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
                const float si = since[i], un = until[i], ra = rate[i];
                float *q2 = zq[j] + 2 * h, *k2 = zk[j] + 2 * h, *m2 = zm[j] + 2 * h;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    q2[e] *= A.scale * si;
                    k2[e] *= -si;
                    m2[e] *= un;
                }
                by_row[0][h] = fmaf(iq, fmaf(qv.x, q2[0], qv.y * q2[1]), by_row[0][h]);
                by_row[2][h] = fmaf(ik, fmaf(kv.x, k2[0], kv.y * k2[1]), by_row[2][h]);
                by_row[1][h] = fmaf(ik, fmaf(kv.x, m2[0], kv.y * m2[1]), by_row[1][h]);
                k2[0] = fmaf(ra, k2[0], m2[0]);
                k2[1] = fmaf(ra, k2[1], m2[1]);
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
        for (int o = 16; o; o >>= 1) {
            inner += __shfl_xor_sync(~0u, inner, o);
            if constexpr (SCALED) {
                tp = fmaxf(tp, __shfl_xor_sync(~0u, tp, o));
                tx = fmaxf(tx, __shfl_xor_sync(~0u, tx, o));
            }
        }
        if (lane == 0) {
            more[warp] = inner;
            top[0][warp] = tp;
            top[1][warp] = tx;
        }
        float ps = 1.0f, xs = 1.0f, fq = 1.0f, fk = 1.0f;  // scales of p, x and of what they are added to
        if constexpr (SCALED) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < GRADS / 32; ++i) {
                tp = fmaxf(tp, top[0][i]);
                tx = fmaxf(tx, top[1][i]);
            }
            fk = fminf(scale_for(tx) * ks, scale_for(tp) * qs);  // x K and p^T Q meet in dK
            xs = fk * ik;
            ps = fk * iq;
            fq = ps * ks;
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    zq[j][e] *= fq;
                    zk[j][e] *= fk;
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
        // dQ += p K, dK += x K + x^T K + p^T Q
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            typename KOp::B bk[NQ], bq[NQ];
#pragma unroll
            for (int j = 0; j < NQ; j += 2) {
                KOp::by_columns(reinterpret_cast<typename KOp::B(&)[2]>(bk[j]), Ks + d * 16 * KS + wc * (KD / 4) + j * 8, KS);
                KOp::by_columns(reinterpret_cast<typename KOp::B(&)[2]>(bq[j]), Qs + d * 16 * KS + wc * (KD / 4) + j * 8, KS);
            }
#pragma unroll
            for (int i = PIECES - 1; i >= 0; --i) {
                if (d <= wr) {
                    const typename KOp::A ap = KOp::rows_of(Ps + i * C * MS + wr * 16 * MS + d * 16, MS);
                    const typename KOp::A ax = KOp::rows_of(Xs + i * C * MS + wr * 16 * MS + d * 16, MS);
#pragma unroll
                    for (int j = 0; j < NQ; j += 2) {
                        KOp::mma(zq[j], zq[j + 1], ap, reinterpret_cast<typename KOp::B(&)[2]>(bk[j]));
                        KOp::mma(zk[j], zk[j + 1], ax, reinterpret_cast<typename KOp::B(&)[2]>(bk[j]));
                    }
                }
                if (d >= wr) {
                    const typename KOp::A pt = KOp::columns_of(Ps + i * C * MS + d * 16 * MS + wr * 16, MS);
                    const typename KOp::A xt = KOp::columns_of(Xs + i * C * MS + d * 16 * MS + wr * 16, MS);
#pragma unroll
                    for (int j = 0; j < NQ; j += 2) {
                        KOp::mma(zk[j], zk[j + 1], xt, reinterpret_cast<typename KOp::B(&)[2]>(bk[j]));
                        KOp::mma(zk[j], zk[j + 1], pt, reinterpret_cast<typename KOp::B(&)[2]>(bq[j]));
                    }
                }
            }
        }
        const float bq1 = inverse_of(fq), bk1 = inverse_of(fk);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tq[j][e] = fmaf(zq[j][e], bq1, tq[j][e]);
                tk[j][e] = fmaf(zk[j][e], bk1, tk[j][e]);
            }
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
                    else if (to_f32(gate) == -INFINITY) dg = 0.0f;
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

// ---- launches, one file per type -----------------------------------------------------
struct DeltaSizes {
    int squares, key, kept;   // bytes of T and P of a chunk, of an element of keys, of one kept for the gradient
};
template <typename T> DeltaSizes delta_sizes();
template <typename T> void launch_prep(const DeltaArgs& A, cudaStream_t st);
template <typename T> void launch_scan(const DeltaArgs& A, int warps, cudaStream_t st);
template <typename T> void launch_grads(const DeltaArgs& A, int warps, cudaStream_t st);

template <typename F>
void set_smem(F* kernel, int bytes) {
    SNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}
}  // namespace snnb_delta
