// delta_tile.h - the delta-rule scan (snn_delta_scan) over chunks of 64 steps: what its
// kernels (delta_prep.h, delta_scan.h, delta_grads.h) share.
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
constexpr int MS = C + 8;     // row stride of [C, C] matrices in shared memory
constexpr int PAD = 8;        // elements behind a row in shared memory: eight rows lie in different banks
// T and P are lower triangular: row block b of 16 keeps its 16 (b + 1) columns and PAD
constexpr int LOW = C * (C + 16) / 2 + C * PAD;  // elements of such a matrix
__host__ __device__ constexpr int low_at(int b) { return 128 * b * (b + 2); }
__host__ __device__ constexpr int low_stride(int b) { return 16 * b + 16 + PAD; }
static_assert(low_at(4) == LOW, "row blocks fill it");
// floats of a chunk's factors: since, until, rate, those of Factor (scales of T and P by row
// blocks); for the gradients the logarithms' sums in two parts and the counts of decays of 0
enum Factor { LOST = 3 * C, K_SCALE, Q_SCALE, T_SCALE = LOST + 4, P_SCALE = LOST + 8, SCAN_FACTORS = LOST + 12,
              UP = SCAN_FACTORS, UP_LOW = UP + C, CUT = UP_LOW + C, SC = CUT + C };
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
    int n_steps, hk, heads, group, kdim, vdim, vpad;  // vpad: vdim in whole words of 16 bytes
    int logit, zero;
    float scale;
    char* keys;               // [slots, hk, 2, C, KD + PAD] of Path::KE: K and Q times their scales
    char* squares;            // [slots, heads] of Path::SQUARES bytes: planes of T, of P
    float* factors;           // [slots, heads, SC]
    char *states, *u;         // saved: [slots, heads, vdim, KD + PAD], [slots, heads, PLANES, C, vpad] of Kept
    char *dstates, *dr;       // gradients' workspace: the same forms
    // sequences cut into segments of `seg` chunks (0: whole), `items` in all (packed: at most): where each starts from
    // [items, heads, kdim, vdim] (`only`: the run that makes them, and of those between the products of their steps [..,
    // kdim, kdim])
    int seg, only, tiles;     // tiles: CTAs along the values' columns
    long long items;
    float *starts, *maps;
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
// the first item of sequence s, which has one at least
__device__ __forceinline__ long long item_at(const DeltaArgs& A, long long s, const Span& sp) {
    if (!A.seg) return s;
    return A.off ? sp.start / (A.seg * (long long)C) + s : s * (((A.n_steps + C - 1) / C + A.seg - 1) / A.seg);
}
// the sequence that an item belongs to: the last one whose first item is not behind it (by a whole warp)
__device__ __forceinline__ long long sequence_of_item(const DeltaArgs& A, long long item) {
    if (!A.seg) return item;
    if (!A.off) return item / (((A.n_steps + C - 1) / C + A.seg - 1) / A.seg);
    long long before = 0;
    for (long long base = 0; base < A.n_seq; base += 32) {
        const long long s = base + (threadIdx.x & 31);
        before += __popc(__ballot_sync(~0u, s < A.n_seq && item_at(A, s, span_of(A, s)) <= item));
    }
    return max(before - 1, 0ll);
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
__device__ __forceinline__ void stsm4(void* p, unsigned a, unsigned b, unsigned c, unsigned d) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// bytes (a multiple of 16, as the addresses) of shared memory to memory, by one thread, behind a fence of
// those that wrote them; the shared memory is read when store_read returns, all is done when store_done does
__device__ __forceinline__ void store_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void store_bulk(void* to, const void* from, int bytes) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(from);
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(at), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void stsm4t(void* p, unsigned a, unsigned b, unsigned c, unsigned d) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
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
    static constexpr int PIECES = 2, OUT = std::is_same<T, __half>::value ? 2 : 1;  // pieces; of what reaches Y
    static constexpr int SQUARES = 2 * PIECES * LOW * 2;
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
    // d += piece p of a, times b
    template <int p>
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) {
        mma16<KE>(d0, a.v[p], b[0].v);
        mma16<KE>(d1, a.v[p], b[1].v);
    }
    // two elements side by side of a matrix, into its planes
    static __device__ __forceinline__ void put(KE* m, float x, float y, float s) {
        x *= s;
        y *= s;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) *reinterpret_cast<unsigned*>(m + p * LOW) = piece<KE>(x, y);
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
    static constexpr int PIECES = 1, OUT = 1;  // (the two tf32 pieces go together)
    static constexpr int SQUARES = 2 * LOW * 4;
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
    // (The instruction cuts the bits that its sum has no room for, always towards zero, which adds
    // up over a long sum: it sums a depth of 16, and rounded additions those sums.)
    static __device__ __forceinline__ void full(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) {
        float t0[4] = {}, t1[4] = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mma8(t0, a.l + 4 * k, b[0].h + 2 * k);
            mma8(t1, a.l + 4 * k, b[1].h + 2 * k);
            mma8(t0, a.h + 4 * k, b[0].l + 2 * k);
            mma8(t1, a.h + 4 * k, b[1].l + 2 * k);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mma8(t0, a.h + 4 * k, b[0].h + 2 * k);
            mma8(t1, a.h + 4 * k, b[1].h + 2 * k);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            d0[e] += t0[e];
            d1[e] += t1[e];
        }
    }
    template <int p>
    static __device__ __forceinline__ void mma(float (&d0)[4], float (&d1)[4], const A& a, const B (&b)[2]) { full(d0, d1, a, b); }
    static __device__ __forceinline__ void put(float* m, float x, float y, float) { *reinterpret_cast<float2*>(m) = make_float2(x, y); }
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
// values, so that smaller ones keep 22 bits down to 2^-16 of it; 2^-113 at least (f32's largest values
// then lie below 2^15) and 2^80 at most (of a top below 2^-67 fewer bits are kept; those of keys, queries
// and P are held to 2^40, so that products with these have an inverse).  1 where all is zero.
constexpr float MOST_SCALE = 0x1p80f;
__device__ __forceinline__ float scale_for(float top) {
    const int b = (int)(__float_as_uint(top) >> 23), e = min(max(13 + 127 + 127 - b, 127 - 113), 127 + 80);
    return __uint_as_float((unsigned)(b ? e : 127) << 23);
}
__device__ __forceinline__ float inverse_of(float s) {  // of a power of two
    return __uint_as_float((254u << 23) - __float_as_uint(s));
}
// The product of two scales.  Where it is below 2^-126 it has no inverse, and what they scale has a product beyond
// f32, which is not to pass for a number.
__device__ __forceinline__ float scale_of_both(float a, float b) { return a * b < 0x1p-126f ? NAN : a * b; }
// The least of three powers of two, 2^-113 at least: a scale for what has a scale of its own and meets sums of other
// sizes, which must stay finite times it
__device__ __forceinline__ float scale_within(float own, float a, float b = INFINITY) { return fmaxf(fminf(own, fminf(a, b)), 0x1p-113f); }
__device__ __forceinline__ float finite_size(float x) { return fabsf(x) <= FLT_MAX ? fabsf(x) : 0.0f; }
template <int N>
__device__ __forceinline__ float warp_top(const float (&x)[N][4]) {
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a = fmaxf(a, fmaxf(fabsf(x[i][0]), fabsf(x[i][1])));
        b = fmaxf(b, fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
    }
    // (magnitudes order as their bits; fmaxf passes NaN over.  A column with an infinity is lost
    // and does not set the scale of its neighbours.)
    return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(fmaxf(finite_size(a), finite_size(b)))));
}
template <int N>
__device__ __forceinline__ float warp_scale(const float (&x)[N][4]) { return scale_for(warp_top(x)); }

// A decay whose logarithm lies below this is 0 in f32 (half of the smallest f32 is exp(-103.97)): the
// step forgets everything.  Such logarithms may be as low as the type goes and stay out of all sums.
constexpr float FORGETS = -104.0f;

// By one warp: sums of the logarithms of a chunk's decays (64 bits, kept as two f32 of
// their binary logarithms: differences of them are what counts) but for those of decays of
// 0, which are counted apart, and the rates.  In the last lane's `lost` 1 - the chunk's decay.
template <typename T>
__device__ __forceinline__ void chunk_decays(const DeltaArgs& A, long long s, const Span& sp, int t0, int n, int head, int lane,
                                             float* up, float* low, int* cut, float* rate, float& lost) {
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
        z[i] = lg < FORGETS;
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double v = (i ? sum : sum - l[1]) * 1.4426950408889634074;
        up[2 * lane + i] = (float)v;
        low[2 * lane + i] = (float)(v - (double)(float)v);
        cut[2 * lane + i] = cuts - (i ? 0 : z[1]);
    }
    const float whole = (float)sum, rest = (float)(sum - (double)whole);
    lost = cuts ? 1.0f : fmaf(-rest, expf(whole), -expm1f(whole));
}
// 2^x by the exponential unit: off by 2^-22 of the value, as expf
__device__ __forceinline__ float power_of_2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float decay_between(const float* up, const float* low, const int* cut, int i, int j) {
    return cut[i] == cut[j] ? power_of_2((up[i] - up[j]) + (low[i] - low[j])) : 0.0f;
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

// what the gradient needs of states and U in which type: bf16 gradients are rounded to
// 8 bits themselves
// (U and R in two pieces there: they meet states that are rounded)
template <typename T> struct Kept {
    using K = float;
    static constexpr int PLANES = 1;
};
template <> struct Kept<__nv_bfloat16> {
    using K = __nv_bfloat16;
    static constexpr int PLANES = 2;
};

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

// ---- launches, one file per type -----------------------------------------------------
struct DeltaSizes {
    int squares, key, kept, planes;  // bytes of T and P of a chunk, of an element of keys, of one kept for the gradient; planes of U
};
template <typename T> DeltaSizes delta_sizes();
template <typename T> void launch_prep(const DeltaArgs& A, cudaStream_t st);
template <typename T> void launch_scan(const DeltaArgs& A, int warps, cudaStream_t st);
template <typename T> void launch_grads(const DeltaArgs& A, int warps, cudaStream_t st);

// a kernel's dynamic shared memory, set once for a device
template <auto* KERNEL>
void set_smem(int bytes) {
    static std::atomic<unsigned long long> done;
    int dev = 0;
    SNN_CUDA(cudaGetDevice(&dev));
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done & bit)) return;
    SNN_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done |= bit;
}
}  // namespace snnb_delta
