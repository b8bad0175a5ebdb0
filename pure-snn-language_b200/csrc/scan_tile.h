// scan_tile.h - the leaky scan's kernels over tiles of steps and channels
// (k_scan_tile, k_scan_grad_tile) and what they share with scan.cu.  Each
// element type and direction is compiled by a file of its own (scan_*.cu).
#pragma once
#include <algorithm>
#include <cfloat>
#include "elem.h"

namespace snnb_scan {
using snnb::from_f32;
using snnb::to_f32;

// Steps between two states that the forward pass keeps for the backward pass.
// The backward pass recomputes the states inside a block from the inputs that
// it reads anyway: 4 bytes per 16 steps and channel instead of a second read
// of y, and the states stay f32.
constexpr int BLOCK = 16;

// how the decays are given: per step, as they are or as logits; per channel
enum { GATE_VALUE = 0, GATE_LOGIT = 1, GATE_CHANNEL = 2, GATE_CHANNEL_LOGIT = 3 };
template <int GM> constexpr bool per_channel = GM >= GATE_CHANNEL;
template <int GM> constexpr bool is_logit = (GM & 1) != 0;

struct Rows {
    void* p;
    long long ss, st;
};

struct ScanArgs {
    const int64_t* off;
    long long n_seq;
    int n_steps, D, logit, leaky;
    int zero;  // rows of no sequence become zero in what is written
    Rows gate, x, y, dgate, dx;
    const float* h0;
    float* h;
    float* saved;
    const float* dh;
    float* dh0;
    float* part;   // per-CTA sums of a channel gate's gradient
    int ctiles, workers, cluster;
    // sequences cut into chunks of `chunk` steps (0: whole): the chunks' maps,
    // then in map_h the states (gradient: r) that they start from
    int chunk;
    long long n_chunks;
    float *map_a, *map_l, *map_h;  // product of decays, what it lost, end state
};

// rows of sequence s: [begin, begin + len) of the flat row index (packed), or
// of the sequence itself (dense)
struct Span {
    long long begin, block0;
    int len;
};
__device__ __forceinline__ Span span_of(const ScanArgs& A, long long s) {
    Span r;
    long long flat;
    if (A.off) {
        const long long b = min(max((long long)A.off[s], 0ll), (long long)A.n_steps);
        const long long e = min(max((long long)A.off[s + 1], b), (long long)A.n_steps);
        r.begin = flat = b;
        r.len = (int)(e - b);
    } else {
        flat = s * A.n_steps;
        r.begin = 0;
        r.len = A.n_steps;
    }
    // first block of the sequence among the saved states: floor(flat / BLOCK) + s
    // leaves room for ceil(len / BLOCK) blocks in every sequence, whatever the lengths
    r.block0 = flat / BLOCK + s;
    return r;
}
// The k-th longest of up to 64 packed sequences: they are taken in that order, so
// that the longest do not start last.  All lanes of a warp call it.
constexpr int MAX_SORTED = 64;
__device__ __forceinline__ int by_length(const ScanArgs& A, int k) {
    const int lane = threadIdx.x & 31, n = (int)A.n_seq;
    const int a = lane < n ? span_of(A, lane).len : -1, b = lane + 32 < n ? span_of(A, lane + 32).len : -1;
    int ra = 0, rb = 0;
#pragma unroll 8
    for (int q = 0; q < 32; ++q) {
        const int x = __shfl_sync(~0u, a, q), y = __shfl_sync(~0u, b, q);
        ra += (x > a || (x == a && q < lane)) + (y > a);
        rb += (x >= b) + (y > b || (y == b && q < lane));
    }
    const unsigned ma = __ballot_sync(~0u, a >= 0 && ra == k), mb = __ballot_sync(~0u, b >= 0 && rb == k);
    return ma ? __ffs(ma) - 1 : 31 + __ffs(mb);
}
// Chunk j of the launch: steps [from, to) of sequence s.  Sequence s has the
// chunks from floor(flat / chunk) + s on, as with the blocks; the others hold
// nothing (from = to = 1).  An empty sequence has one chunk (from = to = 0).
__device__ __forceinline__ long long chunk0_of(const ScanArgs& A, long long s) {
    const long long flat = A.off ? min(max((long long)A.off[s], 0ll), (long long)A.n_steps) : s * A.n_steps;
    return flat / A.chunk + s;
}
__device__ __forceinline__ Span chunk_at(const ScanArgs& A, long long j, long long& s, int& from, int& to) {
    long long lo = 0, hi = A.n_seq;
    while (hi - lo > 1) {
        const long long mid = (lo + hi) >> 1;
        if (chunk0_of(A, mid) <= j) lo = mid;
        else hi = mid;
    }
    s = lo;
    const Span sp = span_of(A, s);
    const long long at = (j - chunk0_of(A, s)) * A.chunk;
    if (at < 0 || (at > 0 && at >= sp.len)) {
        from = to = 1;  // nothing
    } else {
        from = (int)at;
        to = (int)min(at + A.chunk, (long long)sp.len);
    }
    return sp;
}
__device__ __forceinline__ long long row_at(const ScanArgs& A, const Rows& r, long long s, const Span& sp, long long t) {
    return A.off ? (sp.begin + t) * r.st : s * r.ss + t * r.st;
}

// Rows of no sequence (before the first one, behind the last) of what a call
// writes, one CTA of n a row: zero.  The kernels do it behind their steps, where
// without such rows it costs two loads (a launch of its own 2 us).
template <typename T>
__device__ __forceinline__ void zero_rest(const ScanArgs& A, const Rows& r, long long cta, long long n) {
    const long long b = min(max((long long)A.off[0], 0ll), (long long)A.n_steps);
    const long long e = min(max((long long)A.off[A.n_seq], b), (long long)A.n_steps);
    for (long long i = cta; i < b + A.n_steps - e; i += n) {
        T* p = reinterpret_cast<T*>(r.p) + (i < b ? i : e + i - b) * r.st;
        for (int c = threadIdx.x; c < A.D; c += blockDim.x) p[c] = from_f32<T>(0.0f);
    }
}

// V values side by side; pairs go through the packed f32 instructions
template <int V>
struct Vec {
    float v[V];
};
template <int V>
__device__ __forceinline__ Vec<V> splat(float x) {
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = x;
    return r;
}
__device__ __forceinline__ Vec<1> vfma(Vec<1> a, Vec<1> b, Vec<1> c) { return {fmaf(a.v[0], b.v[0], c.v[0])}; }
__device__ __forceinline__ Vec<1> vmul(Vec<1> a, Vec<1> b) { return {a.v[0] * b.v[0]}; }
__device__ __forceinline__ Vec<1> vadd(Vec<1> a, Vec<1> b) { return {a.v[0] + b.v[0]}; }
__device__ __forceinline__ Vec<2> vfma(Vec<2> a, Vec<2> b, Vec<2> c) {
    Vec<2> d;
    asm("{.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(d.v[0]), "=f"(d.v[1])
        : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]), "f"(c.v[0]), "f"(c.v[1]));
    return d;
}
__device__ __forceinline__ Vec<2> vmul(Vec<2> a, Vec<2> b) {
    Vec<2> d;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(d.v[0]), "=f"(d.v[1])
        : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
    return d;
}
__device__ __forceinline__ Vec<2> vadd(Vec<2> a, Vec<2> b) {
    Vec<2> d;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;}"
        : "=f"(d.v[0]), "=f"(d.v[1])
        : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
    return d;
}

// The decays of V channels.  A logistic decay near 1 is 1 - s with a small s.
// Rounded to f32 it is off by up to 2^-25, which a memory of 1 / s steps adds
// up to 2^-25 / s of the state where the gate stays the same.  What the rounding
// lost is therefore kept wherever a state is carried on:
//  - as `lo` of the step (one more FMA) by per-channel and f32 gates, and by
//    16-bit ones in single steps;
//  - with 16-bit gates tiles do without inside a warp's 16 (gradient 8) steps:
//    the state goes on by the map of these steps, whose product keeps it (span_lo).
// (An infinite state times lo, or times what a product keeps, may be NaN:
// infinities do not survive, they end as infinities or NaN.)
template <int V, bool LO>
struct Decay {
    Vec<V> a;
    __device__ __forceinline__ Vec<V> step(Vec<V> h, Vec<V> u) const { return vfma(a, h, u); }
    __device__ __forceinline__ Vec<V> times(Vec<V> h) const { return vmul(a, h); }
    __device__ __forceinline__ void set_lo(int, float) {}
};
template <int V>
struct Decay<V, true> {
    Vec<V> a, lo;
    __device__ __forceinline__ Vec<V> step(Vec<V> h, Vec<V> u) const { return vfma(a, h, vfma(lo, h, u)); }
    __device__ __forceinline__ Vec<V> times(Vec<V> h) const { return vfma(a, h, vmul(lo, h)); }
    __device__ __forceinline__ void set_lo(int k, float x) { lo.v[k] = x; }
};
template <typename T, int GM>
constexpr bool keeps_lo = GM == GATE_CHANNEL_LOGIT || (GM == GATE_LOGIT && sizeof(T) == 4);
// The maps of spans keep what the product of their decays is off by (span_lo),
// but for given decays of 16 bits: those are 1 - 2^-11 at most, whose memory of
// 2,048 steps adds less than 2^-16 up.
template <typename T, int GM>
constexpr bool keeps_span = is_logit<GM> || per_channel<GM> || sizeof(T) == 4;
// 16-bit logits
template <typename T, int GM>
constexpr bool short_logit = GM == GATE_LOGIT && sizeof(T) == 2;

// The map of a span of steps, h -> (a + l) h + b: a the rounded product of its
// decays, l what that product is off by.  Where states come a long way a is near
// 1, and 1 - a is known better than a: as r = the sum over the steps of (1 -
// decay) times the product before it, each 1 - decay with its own relative
// precision.  So l = (1 - a) - r where 1 - a is exact; where a span halves the
// state, roundings of its own add up over few spans only, and l is 0.  (OVER:
// decays may be beyond 1.)
template <bool OVER, int V>
__device__ __forceinline__ Vec<V> span_lo(const Vec<V>& a, const Vec<V>& r) {
    Vec<V> l;
#pragma unroll
    for (int k = 0; k < V; ++k)
        l.v[k] = a.v[k] >= 0.5f && (!OVER || a.v[k] <= 2.0f) ? (1.0f - a.v[k]) - r.v[k] : 0.0f;
    return l;
}
// decay a = 1 / (1 + exp(-z)) and its rest 1 - a, each with its own relative
// precision: from e = exp(-|z|) the larger is 1 / (1 + e), the smaller e times
// that.  exp(-|z|) = 2^p (1 + q ln 2) with p the rounded product -|z| log2(e)
// and q what its rounding and log2(e)'s own lost: within 2 ulp, as the
// exponential instruction is, where the product alone would be off by |z|
// 2^-24.  Beyond |z| = 150 e is 0.
__device__ __forceinline__ void logistic(float z, float& a, float& lo, float& rest) {
    float m;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(z)), "f"(150.0f));
    const float p = m * -1.44269502f;  // log2(e) = 1.44269502 + 1.9259630e-8
    const float q = fmaf(m, -1.92596303e-8f, fmaf(m, -1.44269502f, -p));
    float e, big;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(p));
    e = fmaf(e, q * 0.693147182f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(big) : "f"(1.0f + e));
    const float s = e * big;
    const bool up = z >= 0.0f;
    const float near1 = 1.0f - s;
    a = up ? near1 : s;
    lo = up ? (1.0f - near1) - s : 0.0f;
    rest = up ? s : big;
}
// The same of V logits by the short instructions (2 ulp each, the argument
// rounded once): a = 1 / (1 + t) and rest = t a with t = exp(-z), each with its
// own relative precision on both sides of 0, so that nothing is selected.  t ends
// at 2^126, where the subtraction leaves a = 0.
template <int V>
__device__ __forceinline__ void logistic_fast(const Vec<V>& z, Vec<V>& a, Vec<V>& rest) {
    Vec<V> t = vmul(z, splat<V>(-1.4426950408889634f));
#pragma unroll
    for (int k = 0; k < V; ++k) {
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(t.v[k]) : "f"(126.0f));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t.v[k]));
    }
    a = vadd(t, splat<V>(1.0f));
#pragma unroll
    for (int k = 0; k < V; ++k) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a.v[k]));
    rest = vmul(t, a);
    a = vadd(a, splat<V>(-1.17549435e-38f));
}

// decay and rest of V gates
template <typename T, int GM, int V, bool LO>
__device__ __forceinline__ void decays(const Vec<V>& z, Decay<V, LO>& d, Vec<V>& rest) {
    if constexpr (short_logit<T, GM>) {
        logistic_fast(z, d.a, rest);
        const Vec<V> lo = span_lo<false>(d.a, rest);
#pragma unroll
        for (int k = 0; k < V; ++k) d.set_lo(k, lo.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float v = z.v[k];
            float a = v, lo = 0.0f, r = 1.0f - v;
            if (GM == GATE_LOGIT) logistic(v, a, lo, r);
            d.a.v[k] = a;
            d.set_lo(k, lo);
            rest.v[k] = r;
        }
    }
}
// those of the per-channel gates c .. c + V
template <int GM, int V, bool LO>
__device__ __forceinline__ void channel_decays(const ScanArgs& A, int c, int nl, Decay<V, LO>& d, Vec<V>& rest) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float v = k < nl ? reinterpret_cast<const float*>(A.gate.p)[c + k] : 0.0f;
        float a = v, lo = 0.0f, r = 1.0f - v;
        if (is_logit<GM>) logistic(v, a, lo, r);
        d.a.v[k] = a;
        d.set_lo(k, lo);
        rest.v[k] = r;
    }
}

// V elements of type T as the one register (or pair) that a load fills: they
// are unpacked where they are used, not where they are loaded, so that loads
// stay in flight
template <int BYTES>
struct Raw;
template <>
struct Raw<2> {
    using type = unsigned short;
};
template <>
struct Raw<4> {
    using type = unsigned;
};
template <>
struct Raw<8> {
    using type = uint2;
};
template <typename T, int V>
using Word = typename Raw<sizeof(T) * V>::type;
// what a lane reads of an input row: V elements, or the raster word they lie in
template <typename T, int V, bool RASTER>
using InWord = std::conditional_t<RASTER, unsigned, Word<T, V>>;

template <typename T>
struct Unpack;
template <>
struct Unpack<float> {
    static __device__ __forceinline__ Vec<1> get(unsigned w) { return {__uint_as_float(w)}; }
    static __device__ __forceinline__ Vec<2> get(uint2 w) { return {__uint_as_float(w.x), __uint_as_float(w.y)}; }
    static __device__ __forceinline__ unsigned put(Vec<1> x) { return __float_as_uint(x.v[0]); }
    static __device__ __forceinline__ uint2 put(Vec<2> x) { return {__float_as_uint(x.v[0]), __float_as_uint(x.v[1])}; }
};
template <>
struct Unpack<__nv_bfloat16> {
    static __device__ __forceinline__ Vec<1> get(unsigned short w) { return {__uint_as_float((unsigned)w << 16)}; }
    static __device__ __forceinline__ Vec<2> get(unsigned w) {
        return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    }
    static __device__ __forceinline__ unsigned short put(Vec<1> x) {
        return __bfloat16_as_ushort(__float2bfloat16_rn(x.v[0]));
    }
    static __device__ __forceinline__ unsigned put(Vec<2> x) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x.v[0], x.v[1]);
        unsigned r;
        memcpy(&r, &p, 4);
        return r;
    }
};
template <>
struct Unpack<__half> {
    static __device__ __forceinline__ Vec<1> get(unsigned short w) { return {__half2float(__ushort_as_half(w))}; }
    static __device__ __forceinline__ Vec<2> get(unsigned w) {
        __half2 p;
        memcpy(&p, &w, 4);
        const float2 f = __half22float2(p);
        return {f.x, f.y};
    }
    static __device__ __forceinline__ unsigned short put(Vec<1> x) { return __half_as_ushort(__float2half_rn(x.v[0])); }
    static __device__ __forceinline__ unsigned put(Vec<2> x) {
        const __half2 p = __floats2half2_rn(x.v[0], x.v[1]);
        unsigned r;
        memcpy(&r, &p, 4);
        return r;
    }
};
template <typename T, int V, bool RASTER>
__device__ __forceinline__ Vec<V> in_values(InWord<T, V, RASTER> w, int c) {
    if constexpr (RASTER) {
        Vec<V> r;
#pragma unroll
        for (int k = 0; k < V; ++k) r.v[k] = (w >> ((c + k) & 31)) & 1u ? 1.0f : 0.0f;
        return r;
    } else {
        return Unpack<T>::get(w);
    }
}
template <int V>
__device__ __forceinline__ Vec<V> load_f32(const float* p, bool live) {
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = live ? p[k] : 0.0f;
    return r;
}
template <int V>
__device__ __forceinline__ void store_f32(float* p, const Vec<V>& x) {
#pragma unroll
    for (int k = 0; k < V; ++k) p[k] = x.v[k];
}

// ---- tiles ---------------------------------------------------------------------
// A CTA of W warps takes W * L consecutive steps of 32 * V channels at a time:
// a warp L steps, a lane V channels (one 4-byte word of a row).  Over its L
// steps a warp's map of the state is h -> A h + H (A the product of the
// decays, H the end state from zero); the CTA joins its warps' maps in shared
// memory, so each warp learns the state it starts from and runs its steps once
// more with it, from registers.  With few channels a cluster of CTAs takes
// consecutive tiles and joins their maps through distributed shared memory;
// the state after the cluster's tiles is carried in registers to its next round.
template <int W_, int L_, int S_, int CTAS_>
struct Shape {
    static constexpr int W = W_, L = L_, TT = W_ * L_, threads = 32 * W_;
    static constexpr int S = S_;        // stages of rows in flight per warp
    static constexpr int CTAS = CTAS_;  // CTAs an SM is to hold
    static constexpr bool clusters = W_ == 8;
};
using Fwd = Shape<8, 16, 2, 2>;
using Bwd = Shape<8, 8, 3, 2>;
// Decays per channel leave the forward pass registers for a third CTA: 80 a
// thread, of which 16-bit forms spill 8 - 32 bytes (the gradient spills more and
// loses by one: documents 171 -> 187 us).
using FwdChannel = Shape<8, 16, 2, 3>;
// Without clusters the gradient takes smaller CTAs, twice as many on an SM.
using BwdMany = Shape<4, 8, 3, 4>;
// Where channels and sequences alone fill the SMs with warps: a warp by itself,
// which has its state at hand and needs no maps.
using FwdSeq = Shape<1, 16, 4, 12>;
using BwdSeq = Shape<1, 16, 3, 8>;
using FwdSeqChannel = Shape<1, 16, 4, 24>;
using BwdSeqChannel = Shape<1, 16, 3, 16>;
constexpr int MAX_CLUSTER = 8;
static_assert(Bwd::TT % BLOCK == 0 && BwdMany::TT % BLOCK == 0 && BwdSeq::TT % BLOCK == 0 && FwdSeq::L % BLOCK == 0 && Fwd::L % BLOCK == 0,
              "a gradient tile and a warp's forward steps begin with a saved state");
template <typename T>
constexpr int lane_channels = 4 / (int)sizeof(T);

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// store to the same shared-memory variable of CTA `rank` of the cluster
template <typename T>
__device__ __forceinline__ void store_peer(T* p, int rank, const T& x) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    float f[sizeof(T) / 4];
    memcpy(f, &x, sizeof(T));
    if constexpr (sizeof(T) == 16)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(r), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
    else if constexpr (sizeof(T) == 8)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(r), "f"(f[0]), "f"(f[1]) : "memory");
    else
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(r), "f"(f[0]) : "memory");
}

// the product (a, l) of spans times one more, each with what it is off by
template <int V>
__device__ __forceinline__ void span_times(const Vec<V>& sa, const Vec<V>& sl, Vec<V>& a, Vec<V>& l) {
    const Vec<V> n = vmul(sa, a);
    l = vfma(sa, l, vfma(sl, a, vfma(sa, a, vmul(splat<V>(-1.0f), n))));
    a = n;
}
template <int V>
struct alignas(8 * V) Pair {  // one word of shared memory
    Vec<V> a, b;
};
// A map applied to a state.  The product of decays beyond 1 (given ones, not
// logits') may overflow over a span in which the state is 0: then a h is NaN
// where the states stay 0.  The warps of a tile learn at their barrier whether a
// product among them did, and take the spans by join_spans then.  This is
// compiled for given decays alone: in the gradient of 16 x 4,096 x 2,048 bf16
// logits it would take 20 of 315 us (a test for NaN behind the joins 26).
template <bool KEEP, int V>
__device__ __forceinline__ Vec<V> plain(const Vec<V>& a, const Vec<V>& l, const Vec<V>& h, const Vec<V>& b) {
    return vfma(a, h, KEEP ? vfma(l, h, b) : b);
}
// the same with 0 as it is: equal wherever the plain form gives a number
template <bool KEEP, int V>
__device__ __forceinline__ Vec<V> mapped(const Vec<V>& a, const Vec<V>& l, const Vec<V>& h, const Vec<V>& b) {
    const Vec<V> r = plain<KEEP>(a, l, h, b);
    Vec<V> q;
#pragma unroll
    for (int k = 0; k < V; ++k) q.v[k] = h.v[k] == 0.0f ? b.v[k] : r.v[k];
    return q;
}
template <int V>
__device__ __forceinline__ bool overflowed(const Vec<V>& x) {  // infinite or NaN
    bool r = false;
#pragma unroll
    for (int k = 0; k < V; ++k) r |= !(fabsf(x.v[k]) <= FLT_MAX);
    return r;
}
template <int V>
__device__ __forceinline__ bool any_nan(const Vec<V>& x) {
    bool r = false;
#pragma unroll
    for (int k = 0; k < V; ++k) r |= x.v[k] != x.v[k];
    return r;
}
// n spans from state x: x the state behind them, own the one before span `at`;
// map(j, a, l, b) gives the j-th span's map.  Not unrolled: it keeps few registers.
template <bool KEEP, int V, typename F>
__device__ __forceinline__ void join_spans(int n, int at, Vec<V>& x, Vec<V>& own, F map) {
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        if (j == at) own = x;
        Vec<V> a, l, b;
        map(j, a, l, b);
        x = mapped<KEEP>(a, l, x, b);
    }
}
// Decays per channel: every warp's product is the same.  In shared memory, by
// lane: the products of 0 .. W warps.  Says whether one warp's overflows.
template <int V, int W>
struct Powers {
    Pair<V> p[W + 1][32];
};
template <int V, int W, bool LO>
__device__ __forceinline__ bool powers(Powers<V, W>& P, const Decay<V, LO>& d, const Vec<V>& rest, int steps, int w, int lane) {
    Vec<V> a = splat<V>(1.0f), r = splat<V>(0.0f), pa = a, pl = r;
    for (int i = 0; i < steps; ++i) {
        r = vfma(rest, a, r);
        a = vmul(d.a, a);
    }
    const Vec<V> l = span_lo<!LO>(a, r);
    if (w == 0) P.p[0][lane] = {pa, pl};
    for (int j = 0; j <= w; ++j) span_times(a, l, pa, pl);
    P.p[w + 1][lane] = {pa, pl};
    return __syncthreads_or(!LO && overflowed(a));
}
template <int V>
struct ClusterMaps {  // the tiles' maps of a round, by rank: (a, l) and the end state; two rounds
    Pair<V> p[2][MAX_CLUSTER][32];
    alignas(4 * V) Vec<V> h[2][MAX_CLUSTER][32];
};

// Rows are staged in shared memory by asynchronous copies, each warp its own
// rows, so that they need no barrier and no registers while in flight.  COPY is
// the words that all rows allow: 16 bytes, 4 bytes, or (16-bit types, odd row
// strides or offsets) the aligned 4-byte words that cover a row, 33 for 32.
// Of a word at a row's end that reaches past the tile only the lower half is
// read; one at a row's begin may hold the element before, which lies in the
// same allocation (allocations begin aligned).
template <int COPY>
constexpr int row_bytes = COPY == 2 ? 132 : 128;

template <int WORD>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src, int bytes) {
    if constexpr (WORD == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A stream of rows: where the warp's next rows begin and how they are staged
template <typename T, int COPY, int L>
struct Rower {
    const char* p;       // element 0 of the tile in the warp's next first row
    long long st, jump;  // bytes between rows, between a warp's first rows
    __device__ __forceinline__ void start(const T* first, long long stride, long long steps) {
        p = reinterpret_cast<const char*>(first);
        st = stride * (int)sizeof(T);
        jump = st * steps;
    }
    // rows 0 .. n (<= L) of nc channels to dst; zeros for the rest
    __device__ __forceinline__ void fetch(unsigned dst, int n, int nc, int lane) const {
        constexpr int E = (int)sizeof(T), FULL = 128 / E;
        if constexpr (COPY == 16) {
            const int ch = lane & 7, r0 = lane >> 3;
            const int most = ch * 16 < nc * E ? n : 0;
            const char* q = p + r0 * st + ch * 16;
            dst += r0 * 128 + ch * 16;
#pragma unroll
            for (int i = 0; i < L; i += 4) {
                copy_async<16>(dst + i * 128, r0 + i < most ? q : p, r0 + i < most ? 16 : 0);
                q += 4 * st;
            }
        } else if constexpr (COPY == 4) {
            const int most = lane * 4 < nc * E ? n : 0;
            const char* q = p + lane * 4;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                copy_async<4>(dst + i * 128 + lane * 4, i < most ? q : p, i < most ? 4 : 0);
                q += st;
            }
        } else {
            const char* q = p + lane * 4;
            if (n == L && nc == FULL) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    copy_async<4>(dst + i * 132 + lane * 4, (const void*)((uintptr_t)q & ~(uintptr_t)3), 4);
                    q += st;
                }
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const int e = 2 * lane - (int)(((uintptr_t)q >> 1) & 1);  // the word's lower element
                    const int b = i >= n ? 0 : e + 1 < nc ? 4 : e >= 0 && e < nc ? 2 : 0;
                    copy_async<4>(dst + i * 132 + lane * 4, (const void*)((uintptr_t)(b ? q : p) & ~(uintptr_t)3), b);
                    q += st;
                }
            }
            if (lane < L) {  // the 33rd words of all rows
                q = p + lane * st + 128;
                const int b = lane < n && nc == FULL && (((uintptr_t)q >> 1) & 1) ? 2 : 0;
                copy_async<4>(dst + lane * 132 + 128, (const void*)((uintptr_t)(b ? q : p) & ~(uintptr_t)3), b);
            }
        }
    }
    // for rows at q: by how many bits row i begins in its first word, by i's parity
    __device__ __forceinline__ unsigned shift(const char* q, int i) const {
        return COPY == 2 ? (unsigned)(((uintptr_t)q + (i & 1 ? st : 0)) & 2) * 8 : 0u;
    }
};
// the lane's word of a staged row
template <int COPY>
__device__ __forceinline__ unsigned staged(const char* rows, int i, int lane, unsigned shift) {
    const unsigned* r = reinterpret_cast<const unsigned*>(rows + i * row_bytes<COPY>) + lane;
    if constexpr (COPY == 2) return __funnelshift_r(r[0], r[1], shift);
    return r[0];
}
// the lane's channels of a written row
template <typename T, int COPY>
__device__ __forceinline__ void write_row(T* p, const Vec<lane_channels<T>>& x, int nl) {
    const auto w = Unpack<T>::put(x);
    if constexpr (COPY == 2 && sizeof(T) == 2) {
        reinterpret_cast<unsigned short*>(p)[0] = (unsigned short)w;
        if (nl > 1) reinterpret_cast<unsigned short*>(p)[1] = (unsigned short)(w >> 16);
    } else {
        *reinterpret_cast<unsigned*>(p) = w;
    }
}
template <int V>
__device__ __forceinline__ Vec<V> load_n(const float* p, int nl) {
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = k < nl ? p[k] : 0.0f;
    return r;
}
template <int V>
__device__ __forceinline__ void store_n(float* p, const Vec<V>& x, int nl) {
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (k < nl) p[k] = x.v[k];
}

// rows 0 .. n (<= L) of a tile's raster words (V a row) to dst, a word a lane
template <int V, int L>
__device__ __forceinline__ void fetch_raster(unsigned dst, const unsigned* p, long long st, int n, int words, int lane) {
    const int r = lane / V, k = lane % V;
    const bool in = r < L && r < n && k < words;
    copy_async<4>(dst + lane * 4, in ? p + r * st + k : p, in ? 4 : 0);
}
template <int V>
__device__ __forceinline__ Vec<V> raster_values(const char* words, int i, int lane) {
    const unsigned w = reinterpret_cast<const unsigned*>(words)[i * V + lane * V / 32];
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = (w >> ((lane * V + k) & 31)) & 1u ? 1.0f : 0.0f;
    return r;
}

// a warp's stage of rows: gate, x (or raster words), dy and the block's first
// state, where they are staged
template <int GM, bool RASTER, int COPY, int L, int V, bool GRAD>
struct Stage {
    static constexpr int rows = L * row_bytes<COPY>;
    static constexpr int gate = 0, x = per_channel<GM> ? 0 : rows;
    static constexpr int dy = x + (RASTER ? 128 : rows), state = dy + (GRAD ? rows : 0);
    static constexpr int bytes = state + (GRAD ? 128 * V : 0);
};

template <typename SH, typename T, int GM, bool RASTER, bool LEAKY, int COPY>
__global__ void __launch_bounds__(SH::threads, SH::CTAS) k_scan_tile(const ScanArgs A) {
    constexpr int W = SH::W, L = SH::L, TT = SH::TT, S = SH::S, V = lane_channels<T>;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>, KEEP = keeps_span<T, GM>, OVER = !is_logit<GM>;
    using St = Stage<GM, RASTER, COPY, L, V, false>;
    static_assert(L * V <= 32, "a lane holds one raster word");
    extern __shared__ __align__(16) char rows[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c0 = item % A.ctiles * 32 * V, c = c0 + lane * V;
    const int nc = min(32 * V, A.D - c0), nl = min(V, A.D - c);  // channels of the tile, of the lane (<= 0: none)
    const int round = CL * TT;
    char* const mine = rows + w * S * St::bytes;
    const unsigned mine_s = (unsigned)__cvta_generic_to_shared(mine);
    const Vec<V> one = splat<V>(1.0f), zero = splat<V>(0.0f);
    Decay<V, LO> fixed;
    Vec<V> factor = one;
    if (PC) channel_decays<GM>(A, c, nl, fixed, factor);
    __shared__ std::conditional_t<PC && (W > 1), Powers<V, W>, char> pw_s;
    bool over = false;  // a product of a warp's decays overflows
    if constexpr (PC && W > 1) over = powers<V, W>(pw_s, fixed, factor, L, w, lane);
    int par = 0;
    // a peer's shared memory may be written once the peer runs
    if (W > 1 && CL > 1) cluster_sync();
    const bool split = W == 1 && A.chunk > 0;
    for (long long j = item / A.ctiles; j < (split ? A.n_chunks : A.n_seq); j += A.workers) {
        long long s = j;
        int from_t = 0, to_t;
        Span sp;
        if (split) {
            sp = chunk_at(A, j, s, from_t, to_t);
        } else {
            if (A.off && A.n_seq <= MAX_SORTED) s = by_length(A, (int)j);
            sp = span_of(A, s);
            to_t = sp.len;
        }
        Vec<V> carry = split ? load_n<V>(A.map_h + j * A.D + c, nl) : load_n<V>(A.h0 + s * A.D + c, A.h0 ? nl : 0);
        if (to_t == from_t) {
            if (A.h && to_t == 0 && rank == 0 && w == 0) store_n<V>(A.h + s * A.D + c, carry, nl);
            continue;
        }
        const int t1 = from_t + rank * TT + w * L;  // the warp's first step
        Rower<T, COPY, L> rg, rx;
        rg.start(reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, t1) + c0, A.gate.st, round);
        rx.start(reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, t1) + c0, A.x.st, round);
        const unsigned* pw = reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, t1) + (c0 >> 5);
        T* py = reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, t1) + c;
        const long long yjump = A.y.st * round;
        const unsigned g0 = rg.shift(rg.p, 0), g1 = rg.shift(rg.p, 1), x0 = rx.shift(rx.p, 0), x1 = rx.shift(rx.p, 1);
        auto fetch = [&](int t, int slot) {  // this warp's steps from t on
            const int n = min(L, to_t - t);
            const unsigned dst = mine_s + slot * St::bytes;
            if (n > 0) {
                if (!PC) rg.fetch(dst + St::gate, n, nc, lane);
                if (RASTER) fetch_raster<V, L>(dst + St::x, pw, A.x.st, n, (nc + 31) >> 5, lane);
                else rx.fetch(dst + St::x, n, nc, lane);
            }
            rg.p += rg.jump;
            rx.p += rx.jump;
            pw += A.x.st * round;
            copy_commit();
        };
#pragma unroll
        for (int k = 0; k < S; ++k) fetch(t1 + k * round, k);
        int slot = 0;
        for (int t0 = t1; t0 - t1 < to_t - from_t; t0 += round) {
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> u[L], a = one, ar = zero;  // the product of the decays and 1 - it
            copy_wait<S - 1>();
            __syncwarp();
            const char* from = mine + slot * St::bytes;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                Vec<V> f = factor;
                if constexpr (!PC) {
                    const Vec<V> z = Unpack<T>::get(staged<COPY>(from + St::gate, i, lane, i & 1 ? g1 : g0));
                    decays<T, GM>(z, d[i], f);
                    if (W > 1 || short_logit<T, GM>) {
                        if (KEEP) ar = vfma(f, a, ar);
                        a = vmul(d[i].a, a);
                    }
                }
                if constexpr (RASTER) u[i] = raster_values<V>(from + St::x, i, lane);
                else u[i] = Unpack<T>::get(staged<COPY>(from + St::x, i, lane, i & 1 ? x1 : x0));
                if (LEAKY) u[i] = vmul(f, u[i]);
            }
            if (PC) d[0] = fixed;
            __syncwarp();
            fetch(t0 + S * round, slot);
            slot = slot + 1 == S ? 0 : slot + 1;
            Vec<V> h = carry;
            if constexpr (W > 1) {
                // (a, h), l and 1 - a of the warps' maps; h alone where the products are fixed.  (Words of which
                // only a half is read would lie in half of the banks.)
                constexpr int P2 = PC ? 1 : 2, PW = PC ? 1 : W, K2 = KEEP ? P2 : 1, KW = KEEP ? PW : 1;
                __shared__ Pair<V> maps[P2][PW][32];
                __shared__ Vec<V> los[K2][KW][32], rests[K2][KW][32], ends[PC ? 2 : 1][PC ? W : 1][32];
                __shared__ ClusterMaps<V> cm;
                h = zero;
#pragma unroll
                for (int i = 0; i < L; ++i) h = d[PC ? 0 : i].step(h, u[i]);
                if (t0 >= to_t) {  // steps behind the end, whose rows were not read
                    a = one;
                    ar = h = zero;
                }
                if constexpr (PC) {
                    ends[par][w][lane] = h;
                    __syncthreads();
                } else {
                    maps[par][w][lane] = {a, h};
                    if constexpr (KEEP) {
                        los[par][w][lane] = span_lo<OVER>(a, ar);
                        rests[par][w][lane] = ar;
                    }
                    if (!OVER) __syncthreads();
                    else over = __syncthreads_or(overflowed(a));
                }
                auto map = [&](int j, Vec<V>& ja, Vec<V>& jl, Vec<V>& jh) {
                    if constexpr (PC) {
                        ja = pw_s.p[1][lane].a;
                        jl = pw_s.p[1][lane].b;
                        jh = ends[par][j][lane];
                    } else {
                        ja = maps[par][j][lane].a;
                        jh = maps[par][j][lane].b;
                        jl = zero;
                        if constexpr (KEEP) jl = los[par][j][lane];
                    }
                };
                if (CL > 1) {
                    // The warps before this one as one map: state from zero ht, product ta and 1 - it.  The last
                    // warp, whose own steps end the tile, sends the tile's map to all.
                    Vec<V> ht = zero, ta = one, tr = zero, tl = zero;
                    if (OVER && over) {
                        Vec<V> end = zero;
                        join_spans<KEEP>(W, w, end, ht, map);
                    }
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        if (j == w) break;
                        Vec<V> ja, jl, jh;
                        map(j, ja, jl, jh);
                        if (!OVER || !over) ht = plain<KEEP>(ja, jl, ht, jh);
                        if constexpr (!PC) {
                            if constexpr (KEEP) tr = vfma(rests[par][j][lane], ta, tr);
                            ta = vmul(ja, ta);
                        }
                    }
                    if constexpr (PC) {
                        ta = pw_s.p[w][lane].a;
                        tl = pw_s.p[w][lane].b;
                    } else {
                        if (KEEP) tl = span_lo<OVER>(ta, tr);
                    }
                    if (w == W - 1) {
                        Vec<V> ja, jl, jh;
                        map(w, ja, jl, jh);
                        jh = OVER ? mapped<KEEP>(ja, jl, ht, jh) : plain<KEEP>(ja, jl, ht, jh);
                        if constexpr (!PC) {
                            if (KEEP) tr = vfma(ar, ta, tr);
                            ja = vmul(a, ta);
                            jl = KEEP ? span_lo<OVER>(ja, tr) : zero;
                        }
                        for (int r = 0; r < CL; ++r) {
                            if (!PC) store_peer(&cm.p[par][rank][lane], r, Pair<V>{ja, jl});
                            store_peer(&cm.h[par][rank][lane], r, jh);
                        }
                    }
                    cluster_sync();
                    auto tile_map = [&](int r, Vec<V>& ra, Vec<V>& rl, Vec<V>& rh) {
                        Pair<V> p;
                        if constexpr (PC) p = pw_s.p[W][lane];
                        else p = cm.p[par][r][lane];
                        ra = p.a;
                        rl = p.b;
                        rh = cm.h[par][r][lane];
                    };
                    const Vec<V> was = carry;
                    Vec<V> in = carry;
                    for (int r = 0; r < CL; ++r) {
                        if (r == rank) in = carry;
                        Vec<V> ra, rl, rh;
                        tile_map(r, ra, rl, rh);
                        carry = plain<KEEP>(ra, rl, carry, rh);
                    }
                    if (OVER && __any_sync(~0u, any_nan(carry))) {
                        carry = was;
                        join_spans<KEEP>(CL, rank, carry, in, tile_map);
                    }
                    h = OVER ? mapped<KEEP>(ta, tl, in, ht) : plain<KEEP>(ta, tl, in, ht);
                } else if (OVER && over) {  // the state before this warp (h) and behind the tile (carry)
                    join_spans<KEEP>(W, w, carry, h, map);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        if (j == w) h = carry;
                        Vec<V> ja, jl, jh;
                        map(j, ja, jl, jh);
                        carry = plain<KEEP>(ja, jl, carry, jh);
                    }
                }
                par ^= 1;
            }
            if constexpr (W == 1 && short_logit<T, GM>) {
                Vec<V> end = zero;
#pragma unroll
                for (int i = 0; i < L; ++i) end = d[i].step(end, u[i]);
                carry = plain<KEEP>(a, span_lo<OVER>(a, ar), carry, end);
            }
            const int n = min(L, to_t - t0);
            if (nl > 0 && n > 0) {
                if (A.saved) store_n<V>(A.saved + (sp.block0 + t0 / BLOCK) * A.D + c, h, nl);
                T* qy = py;
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (i < n) {
                        h = d[PC ? 0 : i].step(h, u[i]);
                        write_row<T, COPY>(qy, h, nl);
                    }
                    qy += A.y.st;
                }
                if (A.h && t0 + n == sp.len) store_n<V>(A.h + s * A.D + c, h, nl);
                if (W == 1 && !short_logit<T, GM>) carry = h;
            }
            py += yjump;
        }
        copy_wait<0>();
        __syncwarp();
    }
    if (A.zero) zero_rest<T>(A, A.y, blockIdx.x, gridDim.x);
}

// The gradient runs from the last tile to the first.  With r the gradient that
// reaches a step from later ones, g = o + r and r' = a g: the map of a tile is
// r -> A r + R.  The states inside the tile come from its saved first state.
template <typename SH, typename T, int GM, bool RASTER, bool LEAKY, int COPY>
__global__ void __launch_bounds__(SH::threads, SH::CTAS) k_scan_grad_tile(const ScanArgs A) {
    constexpr int W = SH::W, L = SH::L, TT = SH::TT, S = SH::S, V = lane_channels<T>;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>, KEEP = keeps_span<T, GM>, OVER = !is_logit<GM>;
    using St = Stage<GM, RASTER, COPY, L, V, true>;
    extern __shared__ __align__(16) char rows[];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c0 = item % A.ctiles * 32 * V, c = c0 + lane * V;
    const int nc = min(32 * V, A.D - c0), nl = min(V, A.D - c);
    const int round = CL * TT;
    char* const mine = rows + w * S * St::bytes;
    const unsigned mine_s = (unsigned)__cvta_generic_to_shared(mine);
    const Vec<V> one = splat<V>(1.0f), zero = splat<V>(0.0f), minus = splat<V>(-1.0f);
    Decay<V, LO> fixed;
    Vec<V> factor = one, sum = zero;
    if (PC) channel_decays<GM>(A, c, nl, fixed, factor);
    __shared__ std::conditional_t<PC && (W > 1), Powers<V, W>, char> pw_s;
    bool over = false;  // a product of a warp's decays overflows
    if constexpr (PC && W > 1) over = powers<V, W>(pw_s, fixed, factor, L, w, lane);
    int par = 0;
    // a peer's shared memory may be written once the peer runs
    if (W > 1 && CL > 1) cluster_sync();
    const bool split = W == 1 && A.chunk > 0;
    for (long long j = item / A.ctiles; j < (split ? A.n_chunks : A.n_seq); j += A.workers) {
        long long s = j;
        int from_t = 0, to_t;
        Span sp;
        if (split) {
            sp = chunk_at(A, j, s, from_t, to_t);
        } else {
            if (A.off && A.n_seq <= MAX_SORTED) s = by_length(A, (int)j);
            sp = span_of(A, s);
            to_t = sp.len;
        }
        Vec<V> carry = load_n<V>(A.map_h + j * A.D + c, split ? nl : 0);
        if (to_t == from_t) {
            if (A.dh0 && to_t == 0 && rank == 0 && w == 0)
                store_n<V>(A.dh0 + s * A.D + c, load_n<V>(A.dh + s * A.D + c, A.dh ? nl : 0), nl);
            continue;
        }
        const int tiles = (to_t - from_t + TT - 1) / TT;
        // the warp's first (latest) steps; before from_t where the CTA has no tile
        const int t1 = from_t + (tiles - 1 - rank) * TT + w * L;
        Rower<T, COPY, L> rg, rx, rd;
        rg.start(reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, t1) + c0, A.gate.st, -round);
        rx.start(reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, t1) + c0, A.x.st, -round);
        rd.start(reinterpret_cast<const T*>(A.y.p) + row_at(A, A.y, s, sp, t1) + c0, A.y.st, -round);
        const unsigned* pw = reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, t1) + (c0 >> 5);
        T* pdg = reinterpret_cast<T*>(A.dgate.p) + (PC ? 0 : row_at(A, A.dgate, s, sp, t1 + L - 1) + c);
        T* pdx = reinterpret_cast<T*>(A.dx.p) + row_at(A, A.dx, s, sp, t1 + L - 1) + c;
        const long long gjump = A.dgate.st * round, xjump = A.dx.st * round;
        const unsigned g0 = rg.shift(rg.p, 0), g1 = rg.shift(rg.p, 1), x0 = rx.shift(rx.p, 0), x1 = rx.shift(rx.p, 1);
        const unsigned d0 = rd.shift(rd.p, 0), d1 = rd.shift(rd.p, 1);
        auto fetch = [&](int t, int slot) {
            if (t >= from_t && t < to_t) {
                const int n = min(L, to_t - t);
                const unsigned dst = mine_s + slot * St::bytes;
                if (!PC) rg.fetch(dst + St::gate, n, nc, lane);
                if (RASTER) fetch_raster<V, L>(dst + St::x, pw, A.x.st, n, (nc + 31) >> 5, lane);
                else rx.fetch(dst + St::x, n, nc, lane);
                if (A.y.p) rd.fetch(dst + St::dy, n, nc, lane);
            }
            if (t >= from_t) {  // the tile's first state, where t lies behind the end too
                const float* q = A.saved + (sp.block0 + (t - w * L) / BLOCK) * A.D + c;
#pragma unroll
                for (int k = 0; k < V; ++k)
                    copy_async<4>(mine_s + slot * St::bytes + St::state + (lane * V + k) * 4, k < nl ? q + k : A.saved,
                                  k < nl ? 4 : 0);
            }
            rg.p += rg.jump;
            rx.p += rx.jump;
            rd.p += rd.jump;
            pw -= A.x.st * round;
            copy_commit();
        };
#pragma unroll
        for (int k = 0; k < S; ++k) fetch(t1 - k * round, k);
        int slot = 0, t0 = t1;
        for (int b = 0; b < tiles; b += CL, t0 -= round) {  // t0 before from_t: no tile left for this CTA
            const bool some = t0 >= from_t && t0 < to_t;
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> rest[PC ? 1 : L], x[L], o[L], a = one, ar = zero;
            copy_wait<S - 1>();
            __syncwarp();
            const char* from = mine + slot * St::bytes;
            const Vec<V> h0 = reinterpret_cast<const Vec<V>*>(from + St::state)[lane];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if constexpr (!PC) {
                    const Vec<V> z = Unpack<T>::get(staged<COPY>(from + St::gate, i, lane, i & 1 ? g1 : g0));
                    decays<T, GM>(z, d[i], rest[i]);
                    if (W > 1 || short_logit<T, GM>) {
                        if (KEEP) ar = vfma(rest[i], a, ar);
                        a = vmul(d[i].a, a);
                    }
                }
                if constexpr (RASTER) x[i] = raster_values<V>(from + St::x, i, lane);
                else x[i] = Unpack<T>::get(staged<COPY>(from + St::x, i, lane, i & 1 ? x1 : x0));
                o[i] = splat<V>(0.0f);
                if (A.y.p) o[i] = Unpack<T>::get(staged<COPY>(from + St::dy, i, lane, i & 1 ? d1 : d0));
            }
            if (A.dh && some && t0 + L >= sp.len) {  // the last step
                const Vec<V> dh = load_n<V>(A.dh + s * A.D + c, nl);
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (t0 + i == sp.len - 1) o[i] = vadd(o[i], dh);
            }
            if (PC) d[0] = fixed;
            __syncwarp();
            fetch(t0 - S * round, slot);
            slot = slot + 1 == S ? 0 : slot + 1;
            Vec<V> h = h0, r = carry;
            if constexpr (W > 1) {
                // (a, h), (r, l) and 1 - a of the warps' maps; h and r where that is all
                constexpr bool PAIR = KEEP && !PC, RESTS = PAIR && SH::clusters;
                __shared__ Pair<V> maps[PC ? 1 : 2][PC ? 1 : W][32], back[PAIR ? 2 : 1][PAIR ? W : 1][32];
                __shared__ Vec<V> ends[PC ? 2 : 1][PC ? W : 1][32], rs[PAIR ? 1 : 2][PAIR ? 1 : W][32];
                __shared__ Vec<V> rests[RESTS ? 2 : 1][RESTS ? W : 1][32];
                h = r = zero;
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    h = d[PC ? 0 : i].step(h, LEAKY ? vmul(PC ? factor : rest[PC ? 0 : i], x[i]) : x[i]);
                    r = d[PC ? 0 : L - 1 - i].times(vadd(o[L - 1 - i], r));
                }
                if (!some) {  // steps behind the end, whose rows were not read: there r is 0 and stays so
                    a = one;
                    ar = r = zero;
                }
                if constexpr (PC) {
                    ends[par][w][lane] = h;
                    rs[par][w][lane] = r;
                    __syncthreads();
                } else {
                    maps[par][w][lane] = {a, h};
                    if constexpr (PAIR) back[par][w][lane] = {r, span_lo<OVER>(a, ar)};
                    else rs[par][w][lane] = r;
                    if constexpr (RESTS) rests[par][w][lane] = ar;
                    if (!OVER) __syncthreads();
                    else over = __syncthreads_or(overflowed(a));
                }
                // The states start anew in every tile: they do without l.
                auto map = [&](int j, Vec<V>& ja, Vec<V>& jl, Vec<V>& jh) {
                    jl = zero;
                    if constexpr (PC) {
                        ja = pw_s.p[1][lane].a;
                        jh = ends[par][j][lane];
                    } else {
                        ja = maps[par][j][lane].a;
                        jh = maps[par][j][lane].b;
                    }
                };
                auto map_back = [&](int j, Vec<V>& ja, Vec<V>& jl, Vec<V>& jr) {
                    const int k = W - 1 - j;
                    if constexpr (PC) {
                        ja = pw_s.p[1][lane].a;
                        jl = pw_s.p[1][lane].b;
                    } else {
                        ja = maps[par][k][lane].a;
                    }
                    if constexpr (PAIR) {
                        jr = back[par][k][lane].a;
                        jl = back[par][k][lane].b;
                    } else {
                        jr = rs[par][k][lane];
                        if (!PC) jl = zero;
                    }
                };
                if (OVER && over) {
                    Vec<V> end = h0;
                    join_spans<KEEP>(W, w, end, h, map);
                } else {
                    h = h0;
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        if (j == w) break;
                        Vec<V> ja, jl, jh;
                        map(j, ja, jl, jh);
                        h = vfma(ja, h, jh);
                    }
                }
                bool joined = false;
                if constexpr (SH::clusters) if (CL > 1) {
                    __shared__ ClusterMaps<V> cm;
                    // as in the forward pass, from the last warp to the first
                    Vec<V> rt = zero, ta = one, tr = zero, tl = zero;
                    if (OVER && over) {
                        Vec<V> end = zero;
                        join_spans<KEEP>(W, W - 1 - w, end, rt, map_back);
                    }
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        if (W - 1 - j == w) break;
                        Vec<V> ja, jl, jr;
                        map_back(j, ja, jl, jr);
                        if (!OVER || !over) rt = plain<KEEP>(ja, jl, rt, jr);
                        if constexpr (!PC) {
                            if constexpr (RESTS) tr = vfma(rests[par][W - 1 - j][lane], ta, tr);
                            ta = vmul(ja, ta);
                        }
                    }
                    if constexpr (PC) {
                        ta = pw_s.p[W - 1 - w][lane].a;
                        tl = pw_s.p[W - 1 - w][lane].b;
                    } else {
                        if (KEEP) tl = span_lo<OVER>(ta, tr);
                    }
                    if (w == 0) {
                        Vec<V> ja, jl, jr;
                        map_back(W - 1, ja, jl, jr);
                        jr = OVER ? mapped<KEEP>(ja, jl, rt, jr) : plain<KEEP>(ja, jl, rt, jr);
                        if constexpr (!PC) {
                            if (KEEP) tr = vfma(ar, ta, tr);
                            ja = vmul(a, ta);
                            jl = KEEP ? span_lo<OVER>(ja, tr) : zero;
                        }
                        for (int q = 0; q < CL; ++q) {
                            if (!PC) store_peer(&cm.p[par][rank][lane], q, Pair<V>{ja, jl});
                            store_peer(&cm.h[par][rank][lane], q, jr);
                        }
                    }
                    cluster_sync();
                    auto tile_map = [&](int q, Vec<V>& qa, Vec<V>& ql, Vec<V>& qr) {
                        Pair<V> p;
                        if constexpr (PC) p = pw_s.p[W][lane];
                        else p = cm.p[par][q][lane];
                        qa = p.a;
                        ql = p.b;
                        qr = cm.h[par][q][lane];
                    };
                    const Vec<V> was = carry;
                    Vec<V> in = carry;
                    for (int q = 0; q < CL; ++q) {
                        if (q == rank) in = carry;
                        Vec<V> qa, ql, qr;
                        tile_map(q, qa, ql, qr);
                        carry = plain<KEEP>(qa, ql, carry, qr);
                    }
                    if (OVER && __any_sync(~0u, any_nan(carry))) {
                        carry = was;
                        join_spans<KEEP>(CL, rank, carry, in, tile_map);
                    }
                    r = OVER ? mapped<KEEP>(ta, tl, in, rt) : plain<KEEP>(ta, tl, in, rt);
                    joined = true;
                }
                if (joined) {
                } else if (OVER && over) {  // r behind this warp's steps (r) and before the tile's (carry)
                    join_spans<KEEP>(W, W - 1 - w, carry, r, map_back);
                } else {
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        if (W - 1 - j == w) r = carry;
                        Vec<V> ja, jl, jr;
                        map_back(j, ja, jl, jr);
                        carry = plain<KEEP>(ja, jl, carry, jr);
                    }
                }
                par ^= 1;
            }
            if constexpr (W == 1 && short_logit<T, GM>) {
                Vec<V> end = zero;
#pragma unroll
                for (int i = L - 1; i >= 0; --i) end = d[i].times(vadd(o[i], end));
                carry = plain<KEEP>(a, span_lo<OVER>(a, ar), carry, end);
            }
            if (nl > 0 && some) {
                // x becomes the derivative of h_t in a_t: h_{t-1}, or h_{t-1} - x_t
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const Vec<V> before = h, xi = x[i];
                    h = d[PC ? 0 : i].step(h, LEAKY ? vmul(PC ? factor : rest[PC ? 0 : i], xi) : xi);
                    x[i] = LEAKY ? vfma(minus, xi, before) : before;
                }
                const int n = min(L, to_t - t0);
                T *qg = pdg, *qx = pdx;
#pragma unroll
                for (int i = L - 1; i >= 0; --i) {
                    if (i < n) {
                        const Decay<V, LO>& q = d[PC ? 0 : i];
                        const Vec<V> g = vadd(o[i], r);
                        if (PC) {
                            sum = vfma(g, x[i], sum);
                        } else if (A.dgate.p) {
                            Vec<V> da = vmul(g, x[i]);
                            if (GM == GATE_LOGIT) da = vmul(da, vmul(q.a, rest[PC ? 0 : i]));
                            write_row<T, COPY>(qg, da, nl);
                        }
                        if (A.dx.p) write_row<T, COPY>(qx, LEAKY ? vmul(PC ? factor : rest[PC ? 0 : i], g) : g, nl);
                        r = q.times(g);
                    }
                    qg -= A.dgate.st;
                    qx -= A.dx.st;
                }
                if (t0 == 0 && A.dh0) store_n<V>(A.dh0 + s * A.D + c, r, nl);
                if (W == 1 && !short_logit<T, GM>) carry = r;
            }
            pdg -= gjump;
            pdx -= xjump;
        }
        copy_wait<0>();
        __syncwarp();
    }
    if (A.zero) {
        if (A.dx.p) zero_rest<T>(A, A.dx, blockIdx.x, gridDim.x);
        if (!PC && A.dgate.p) zero_rest<T>(A, A.dgate, blockIdx.x, gridDim.x);
    }
    if (PC && A.part) {
        Vec<V> t = sum;
        if constexpr (W > 1) {
            __shared__ Vec<V> sums[W][32];
            sums[w][lane] = sum;
            __syncthreads();
            t = splat<V>(0.0f);
            for (int k = 0; k < W; ++k) t = vadd(t, sums[k][lane]);
        }
        if (w == 0) store_n<V>(A.part + ((long long)(item / A.ctiles) * CL + rank) * A.D + c, t, nl);
    }
}

// The map of a chunk of steps, a warp for each (chunk, tile of channels): the
// decays' product and the end state from zero (GRAD: r at its first step).
// The last chunk of a sequence (GRAD: the first) needs none.
template <typename SH, typename T, int GM, bool RASTER, bool LEAKY, int COPY, bool GRAD>
__global__ void __launch_bounds__(SH::threads, SH::CTAS) k_scan_map(const ScanArgs A) {
    constexpr int L = SH::L, S = SH::S, V = lane_channels<T>;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>, KEEP = keeps_span<T, GM>, OVER = !is_logit<GM>;
    using St = Stage<GM, RASTER, COPY, L, V, false>;  // its x is dy for the gradient
    static_assert(SH::W == 1, "a warp by itself");
    extern __shared__ __align__(16) char rows[];
    const int lane = threadIdx.x;
    const int item = blockIdx.x;
    const int c0 = item % A.ctiles * 32 * V, c = c0 + lane * V;
    const int nc = min(32 * V, A.D - c0), nl = min(V, A.D - c);
    const unsigned rows_s = (unsigned)__cvta_generic_to_shared(rows);
    for (long long j = item / A.ctiles; j < A.n_chunks; j += A.workers) {
        long long s;
        int from_t, to_t;
        const Span sp = chunk_at(A, j, s, from_t, to_t);
        if (from_t == to_t || (GRAD ? from_t == 0 : to_t == sp.len)) continue;
        const int tiles = (to_t - from_t + L - 1) / L;
        const int step = GRAD ? -L : L, t1 = GRAD ? from_t + (tiles - 1) * L : from_t;
        const Rows& in = GRAD ? A.y : A.x;
        Rower<T, COPY, L> rg, rx;
        rg.start(reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, t1) + c0, A.gate.st, step);
        rx.start(reinterpret_cast<const T*>(in.p) + row_at(A, in, s, sp, t1) + c0, in.st, step);
        const unsigned* pw = reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, t1) + (c0 >> 5);
        const unsigned g0 = rg.shift(rg.p, 0), g1 = rg.shift(rg.p, 1), x0 = rx.shift(rx.p, 0), x1 = rx.shift(rx.p, 1);
        auto fetch = [&](int t, int slot) {
            const int n = min(L, to_t - t);
            const unsigned dst = rows_s + slot * St::bytes;
            if (t >= from_t && n > 0) {
                if (!PC) rg.fetch(dst + St::gate, n, nc, lane);
                if (RASTER) fetch_raster<V, L>(dst + St::x, pw, A.x.st, n, (nc + 31) >> 5, lane);
                else if (in.p) rx.fetch(dst + St::x, n, nc, lane);
            }
            rg.p += rg.jump;
            rx.p += rx.jump;
            pw += A.x.st * step;
            copy_commit();
        };
#pragma unroll
        for (int k = 0; k < S; ++k) fetch(t1 + k * step, k);
        Decay<V, LO> fixed;
        Vec<V> factor = splat<V>(1.0f);
        if (PC) channel_decays<GM>(A, c, nl, fixed, factor);
        const Vec<V> one = splat<V>(1.0f), zero = splat<V>(0.0f);
        Vec<V> a = one, l = zero, h = zero;
        auto product = [&](int n, Vec<V>& pa, Vec<V>& pr) {  // of n decays per channel, and 1 - it
            pa = one;
            pr = zero;
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                if (KEEP) pr = vfma(factor, pa, pr);
                pa = vmul(fixed.a, pa);
            }
        };
        Vec<V> all_a, all_r;
        if (PC) product(L, all_a, all_r);
        int slot = 0, t0 = t1;
        for (int b = 0; b < tiles; ++b, t0 += step) {
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> u[L], f[PC ? 1 : L], ra = one, rr = zero;  // these steps' product of decays and 1 - it
            f[0] = factor;
            copy_wait<S - 1>();
            __syncwarp();
            const char* from = rows + slot * St::bytes;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if constexpr (!PC) {
                    const Vec<V> z = Unpack<T>::get(staged<COPY>(from + St::gate, i, lane, i & 1 ? g1 : g0));
                    decays<T, GM>(z, d[i], f[i]);
                }
                if constexpr (RASTER) u[i] = raster_values<V>(from + St::x, i, lane);
                else u[i] = Unpack<T>::get(staged<COPY>(from + St::x, i, lane, i & 1 ? x1 : x0));
                if (!in.p) u[i] = zero;
                if (LEAKY && !GRAD) u[i] = vmul(f[PC ? 0 : i], u[i]);
            }
            if (PC) d[0] = fixed;
            __syncwarp();
            fetch(t0 + S * step, slot);
            slot = slot + 1 == S ? 0 : slot + 1;
            const int n = min(L, to_t - t0);
            const Vec<V> before = h;
            if (short_logit<T, GM>) h = zero;
            if (GRAD && A.dh && t0 + n == sp.len) {
                const Vec<V> dh = load_n<V>(A.dh + s * A.D + c, nl);
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (i == n - 1) u[i] = vadd(u[i], dh);
            }
#pragma unroll
            for (int k = 0; k < L; ++k) {
                const int i = GRAD ? L - 1 - k : k;
                if (i < n) {
                    if (GRAD) h = d[PC ? 0 : i].times(vadd(u[i], h));
                    else h = d[PC ? 0 : i].step(h, u[i]);
                    if constexpr (!PC) {
                        if (KEEP) rr = vfma(f[i], ra, rr);
                        ra = vmul(d[i].a, ra);
                    }
                }
            }
            if (PC) {
                if (n == L) {
                    ra = all_a;
                    rr = all_r;
                } else {
                    product(n, ra, rr);
                }
            }
            if (KEEP) span_times(ra, span_lo<OVER>(ra, rr), a, l);
            else a = vmul(ra, a);
            if (short_logit<T, GM>) h = plain<KEEP>(ra, span_lo<OVER>(ra, rr), before, h);
        }
        copy_wait<0>();
        __syncwarp();
        store_n<V>(A.map_a + j * A.D + c, a, nl);
        if (KEEP) store_n<V>(A.map_l + j * A.D + c, l, nl);
        store_n<V>(A.map_h + j * A.D + c, h, nl);
    }
}

struct Plan {
    int ctiles, workers, cluster;
    int shape;  // 0 tiles, 1 smaller tiles (gradient), 2 a warp by itself
    int chunk;  // 2: the sequences are cut into chunks of so many steps (0: not)
    int64_t n_chunks;
};

// the forward (GRAD = false) or gradient kernel of element type T; map: that of
// the chunks' maps
template <bool GRAD, typename T>
void launch_tiles(int gate_mode, bool raster, int words, bool map, const Plan& p, ScanArgs& A, cudaStream_t st);

#ifdef SNN_SCAN_TILE_LAUNCH
inline void launch(const void* kernel, std::atomic<uint64_t>& ready, int threads, int smem, const Plan& p, ScanArgs& A,
                   cudaStream_t st) {
    A.ctiles = p.ctiles;
    A.workers = p.workers;
    A.cluster = p.cluster;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    SNN_REQUIRE((int64_t)p.ctiles * p.workers * p.cluster < (1ll << 31), SNN_ERR_ARG, "scan: too many tiles");
    cfg.gridDim = dim3((unsigned)(p.ctiles * p.workers * p.cluster));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    if (smem > 0) {  // more than the default needs asking, once on a device
        int dev = 0;
        SNN_CUDA(cudaGetDevice(&dev));
        SNN_REQUIRE(dev >= 0 && dev < 64, SNN_ERR_ARG, "device ordinal above 63");
        if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
            SNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            ready.fetch_or(1ull << dev, std::memory_order_relaxed);
        }
    }
    void* args[] = {&A};
    SNN_CUDA(cudaLaunchKernelExC(&cfg, kernel, args));
}

template <bool GRAD, typename SH, typename T, int GM, bool RASTER, int COPY>
void launch_shape(const Plan& p, ScanArgs& A, cudaStream_t st) {
    const int smem = SH::W * SH::S * Stage<GM, RASTER, COPY, SH::L, lane_channels<T>, GRAD>::bytes;
    const void* k;
    if constexpr (GRAD)
        k = A.leaky ? (const void*)k_scan_grad_tile<SH, T, GM, RASTER, true, COPY>
                    : (const void*)k_scan_grad_tile<SH, T, GM, RASTER, false, COPY>;
    else
        k = A.leaky ? (const void*)k_scan_tile<SH, T, GM, RASTER, true, COPY>
                    : (const void*)k_scan_tile<SH, T, GM, RASTER, false, COPY>;
    static std::atomic<uint64_t> ready[2];  // by device, of the two kernels
    launch(k, ready[A.leaky ? 1 : 0], SH::threads, smem, p, A, st);
}
template <bool GRAD, typename T, int GM, bool RASTER, int COPY>
void launch_map(const Plan& p, ScanArgs& A, cudaStream_t st) {
    // the gradient's maps read the gate and dy alone
    constexpr bool RA = RASTER && !GRAD;
    using SH = std::conditional_t<per_channel<GM>, FwdSeqChannel, FwdSeq>;
    const int smem = SH::S * Stage<GM, RA, COPY, SH::L, lane_channels<T>, false>::bytes;
    const bool leaky = A.leaky && !GRAD;
    const void* k;
    if constexpr (GRAD) k = (const void*)k_scan_map<SH, T, GM, false, false, COPY, true>;
    else
        k = leaky ? (const void*)k_scan_map<SH, T, GM, RASTER, true, COPY, false>
                  : (const void*)k_scan_map<SH, T, GM, RASTER, false, COPY, false>;
    static std::atomic<uint64_t> ready[2];
    launch(k, ready[leaky ? 1 : 0], 32, smem, p, A, st);
}
template <bool GRAD, typename T, int GM, bool RASTER, int COPY>
void launch_copy(bool map, const Plan& p, ScanArgs& A, cudaStream_t st) {
    if (map) return launch_map<GRAD, T, GM, RASTER, COPY>(p, A, st);
    using Seq = std::conditional_t<GRAD, std::conditional_t<per_channel<GM>, BwdSeqChannel, BwdSeq>,
                                   std::conditional_t<per_channel<GM>, FwdSeqChannel, FwdSeq>>;
    if (p.shape == 2) return launch_shape<GRAD, Seq, T, GM, RASTER, COPY>(p, A, st);
    if constexpr (GRAD) {
        if (p.shape == 1) return launch_shape<true, BwdMany, T, GM, RASTER, COPY>(p, A, st);
        launch_shape<true, Bwd, T, GM, RASTER, COPY>(p, A, st);
    } else {
        launch_shape<false, std::conditional_t<per_channel<GM>, FwdChannel, Fwd>, T, GM, RASTER, COPY>(p, A, st);
    }
}
template <bool GRAD, typename T, int GM>
void launch_gate(bool raster, int words, bool map, const Plan& p, ScanArgs& A, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (words == 2)
            return raster ? launch_copy<GRAD, T, GM, true, 2>(map, p, A, st) : launch_copy<GRAD, T, GM, false, 2>(map, p, A, st);
    if (raster) launch_copy<GRAD, T, GM, true, 4>(map, p, A, st);
    else if (words == 16) launch_copy<GRAD, T, GM, false, 16>(map, p, A, st);
    else launch_copy<GRAD, T, GM, false, 4>(map, p, A, st);
}
template <bool GRAD, typename T>
void launch_tiles(int gate_mode, bool raster, int words, bool map, const Plan& p, ScanArgs& A, cudaStream_t st) {
    if (gate_mode == GATE_VALUE) launch_gate<GRAD, T, GATE_VALUE>(raster, words, map, p, A, st);
    else if (gate_mode == GATE_LOGIT) launch_gate<GRAD, T, GATE_LOGIT>(raster, words, map, p, A, st);
    else if (gate_mode == GATE_CHANNEL) launch_gate<GRAD, T, GATE_CHANNEL>(raster, words, map, p, A, st);
    else launch_gate<GRAD, T, GATE_CHANNEL_LOGIT>(raster, words, map, p, A, st);
}
#endif

}  // namespace snnb_scan
