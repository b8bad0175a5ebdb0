// scan.cu - leaky scans (snn_leaky_scan, snn_leaky_scan_grad): the linear
// recurrence h_t = a_t h_{t-1} + u_t along sequences, and its gradients.
#include <algorithm>
#include "elem.h"

namespace {
using snnb::from_f32;
using snnb::to_f32;

// Steps between two states that the forward pass keeps for the backward pass.
// The backward pass recomputes the states inside a block from the inputs that
// it reads anyway: 4 bytes per 64 steps and channel instead of a second read
// of y, and the states stay f32.
constexpr int BLOCK = 64;

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
    long long n_seq, n_steps;
    int D, logit, leaky;
    Rows gate, x, y, dgate, dx;
    const float* h0;
    float* h;
    float* saved;
    const float* dh;
    float* dh0;
    float* part;   // per-CTA sums of a channel gate's gradient
    int ctiles, workers, cluster;
};

// rows of sequence s: [begin, begin + len) of the flat row index (packed), or
// of the sequence itself (dense)
struct Span {
    long long begin, len, block0;
};
__device__ __forceinline__ Span span_of(const ScanArgs& A, long long s) {
    Span r;
    long long flat;
    if (A.off) {
        const long long b = min(max((long long)A.off[s], 0ll), A.n_steps);
        const long long e = min(max((long long)A.off[s + 1], b), A.n_steps);
        r.begin = flat = b;
        r.len = e - b;
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
__device__ __forceinline__ long long row_at(const ScanArgs& A, const Rows& r, long long s, const Span& sp, long long t) {
    return A.off ? (sp.begin + t) * r.st : s * r.ss + t * r.st;
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
// up to 2^-25 / s of the state where the gate stays the same.  Per-channel
// gates and f32 gates therefore keep what the rounding lost as `lo` (one more
// FMA a step); 16-bit gates, whose own rounding is 2^-9 and up of the exponent
// and differs from step to step, do not.  (An infinite state times lo may be
// NaN: infinities do not survive, they end as infinities or NaN.)
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

// decay a = 1 / (1 + exp(-z)) and its rest 1 - a, each with its own relative
// precision: from e = exp(-|z|) the larger is 1 / (1 + e), the smaller e times
// that.  exp(-|z|) = 2^p (1 + q ln 2) with p the rounded product -|z| log2(e)
// and q what its rounding and log2(e)'s own lost: within 2 ulp, as the
// exponential instruction is, where the product alone would be off by |z|
// 2^-24.  Beyond |z| = 150 e is 0.
__device__ __forceinline__ void logistic(float z, float& a, float& lo, float& rest) {
    const float m = fminf(fabsf(z), 150.0f);
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
    if (z != z) a = rest = z;
}
// the same by the short instructions (2 ulp each, the argument rounded once)
__device__ __forceinline__ void logistic_fast(float z, float& a, float& rest) {
    float e, big;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(z) * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(big) : "f"(1.0f + e));
    const float s = e * big;
    const bool up = z >= 0.0f;
    a = up ? big : s;
    rest = up ? s : big;
}

// decay and rest of V gates
template <typename T, int GM, int V>
__device__ __forceinline__ void decays(const Vec<V>& z, Decay<V, keeps_lo<T, GM>>& d, Vec<V>& rest) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float v = z.v[k];
        float a = v, lo = 0.0f, r = 1.0f - v;
        if (GM == GATE_LOGIT) {
            if (sizeof(T) == 4) logistic(v, a, lo, r);
            else logistic_fast(v, a, r);
        }
        d.a.v[k] = a;
        d.set_lo(k, lo);
        rest.v[k] = r;
    }
}
// those of the per-channel gates c .. c + V
template <typename T, int GM, int V>
__device__ __forceinline__ void channel_decays(const ScanArgs& A, int c, int nl, Decay<V, keeps_lo<T, GM>>& d,
                                               Vec<V>& rest) {
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

// ---- short sequences: a thread per sequence and V channels, a step at a time ----
template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(128) k_scan_steps(const ScanArgs A) {
    using X = InWord<T, V, RASTER>;
    const int c = (int)(blockIdx.x * 128 + threadIdx.x) * V;
    if (c >= A.D) return;
    for (long long s = blockIdx.y; s < A.n_seq; s += gridDim.y) {
        const Span sp = span_of(A, s);
        Decay<V, keeps_lo<T, GM>> d;
        Vec<V> rest;
        if (per_channel<GM>) channel_decays<T, GM, V>(A, c, V, d, rest);
        Vec<V> h = load_f32<V>(A.h0 + s * A.D + c, A.h0 != nullptr);
        for (long long t = 0; t < sp.len; ++t) {
            if (A.saved && t % BLOCK == 0) store_f32<V>(A.saved + (sp.block0 + t / BLOCK) * A.D + c, h);
            if (!per_channel<GM>) {
                const Word<T, V> g = *reinterpret_cast<const Word<T, V>*>(
                    reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, t) + c);
                decays<T, GM, V>(Unpack<T>::get(g), d, rest);
            }
            const long long xr = row_at(A, A.x, s, sp, t);
            const X xw = RASTER ? *reinterpret_cast<const X*>(reinterpret_cast<const unsigned*>(A.x.p) + xr + (c >> 5))
                                : *reinterpret_cast<const X*>(reinterpret_cast<const T*>(A.x.p) + xr + c);
            Vec<V> u = in_values<T, V, RASTER>(xw, c);
            if (A.leaky) u = vmul(rest, u);
            h = d.step(h, u);
            *reinterpret_cast<Word<T, V>*>(reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, t) + c) = Unpack<T>::put(h);
        }
        if (A.h) store_f32<V>(A.h + s * A.D + c, h);
    }
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
constexpr int W = 8;
constexpr int TILE_THREADS = 32 * W;
constexpr int L_FWD = 16, L_BWD = 8;
constexpr int S_FWD = 2, S_BWD = 3;  // stages of rows in flight per warp
constexpr int MAX_CLUSTER = 8;
static_assert(W * L_BWD == BLOCK && BLOCK % L_FWD == 0, "blocks start at a warp's steps");
template <typename T>
constexpr int lane_channels = 4 / (int)sizeof(T);

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// store to the same shared-memory variable of CTA `rank` of the cluster
template <int V>
__device__ __forceinline__ void store_peer(Vec<V>* p, int rank, const Vec<V>& x) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(p);
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
#pragma unroll
    for (int k = 0; k < V; ++k)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(r + 4 * k), "f"(x.v[k]) : "memory");
}

template <int V>
struct ClusterMaps {  // the tiles' maps of a round, by rank; two rounds
    Vec<V> a[2][MAX_CLUSTER][32], h[2][MAX_CLUSTER][32];
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

__device__ __forceinline__ void copy_async(unsigned dst, const void* src, int bytes, int words16) {
    if (words16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// rows 0 .. n of L (the rest zero) of a tile of nc channels, row 0 at p, to dst
template <typename T, int COPY, int L>
__device__ __forceinline__ void stage_rows(unsigned dst, const T* p, long long st, int n, int nc, int lane) {
    constexpr int E = (int)sizeof(T);
    if constexpr (COPY == 16) {
        const int ch = lane & 7, r0 = lane >> 3;
        const int most = ch * 16 < nc * E ? n : 0;
        const char* q = reinterpret_cast<const char*>(p) + (r0 * st * E + ch * 16);
#pragma unroll
        for (int i = 0; i < L; i += 4)
            copy_async(dst + (r0 + i) * 128 + ch * 16, r0 + i < most ? q + (long long)i * E * st : (const char*)p,
                       r0 + i < most ? 16 : 0, 1);
    } else if constexpr (COPY == 4) {
        const int most = lane * 4 < nc * E ? n : 0;
        const char* q = reinterpret_cast<const char*>(p) + lane * 4;
#pragma unroll
        for (int i = 0; i < L; ++i)
            copy_async(dst + i * 128 + lane * 4, i < most ? q + (long long)i * E * st : (const char*)((uintptr_t)p & ~3ull),
                       i < most ? 4 : 0, 0);
    } else {
        const uintptr_t any = (uintptr_t)p & ~(uintptr_t)3;
        auto half = [&](int e) { return e + 1 < nc ? 4 : e >= 0 && e < nc ? 2 : 0; };  // bytes of the word at element e
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const uintptr_t q = (uintptr_t)(p + i * st);
            const int b = i < n ? half(2 * lane - (int)((q >> 1) & 1)) : 0;
            copy_async(dst + i * 132 + lane * 4, (const void*)(b ? (q & ~(uintptr_t)3) + lane * 4 : any), b, 0);
        }
        if (lane < L) {
            const uintptr_t q = (uintptr_t)(p + lane * st);
            const int b = lane < n && ((q >> 1) & 1) && 63 < nc ? 2 : 0;
            copy_async(dst + lane * 132 + 128, (const void*)(b ? (q & ~(uintptr_t)3) + 128 : any), b, 0);
        }
    }
}
// the lane's word of row i; odd: the row begins in the upper half of its first word
template <int COPY>
__device__ __forceinline__ unsigned staged(const char* rows, int i, int lane, unsigned odd) {
    const unsigned* r = reinterpret_cast<const unsigned*>(rows + i * row_bytes<COPY>) + lane;
    if constexpr (COPY == 2) return __funnelshift_r(r[0], r[1], odd * 16);
    return r[0];
}
template <int COPY, typename T>
__device__ __forceinline__ unsigned odd_row(const T* p, long long st, int i) {
    return COPY == 2 ? (unsigned)(((uintptr_t)p >> 1) + (uintptr_t)(i * st)) & 1u : 0u;
}
// the lane's channels of a written row
template <typename T, int COPY>
__device__ __forceinline__ void write_row(T* p, const Vec<lane_channels<T>>& x, int nl) {
    const unsigned w = Unpack<T>::put(x);
    if constexpr (COPY == 2) {
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

// A raster's words of L rows of a tile: lane (row, word) holds one (V words a row)
template <int V, int L>
__device__ __forceinline__ unsigned raster_word(const unsigned* p, long long st, int n, int words, int lane) {
    const int r = lane / V, k = lane % V;
    return r < L && r < n && k < words ? p[r * st + k] : 0u;
}
template <int V>
__device__ __forceinline__ Vec<V> raster_values(unsigned held, int i, int lane) {
    const unsigned w = __shfl_sync(~0u, held, i * V + lane * V / 32);
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = (w >> ((lane * V + k) & 31)) & 1u ? 1.0f : 0.0f;
    return r;
}

template <typename T, int GM, bool RASTER, int COPY>
struct FwdStage {  // a warp's staged rows
    static constexpr int gate = 0, x = per_channel<GM> ? 0 : L_FWD * row_bytes<COPY>;
    static constexpr int bytes = x + (RASTER ? 0 : L_FWD * row_bytes<COPY>);
};
template <typename T, int GM, bool RASTER, int COPY>
struct BwdStage {
    static constexpr int gate = 0, x = per_channel<GM> ? 0 : L_BWD * row_bytes<COPY>;
    static constexpr int dy = x + (RASTER ? 0 : L_BWD * row_bytes<COPY>), bytes = dy + L_BWD * row_bytes<COPY>;
};

template <typename T, int GM, bool RASTER, bool LEAKY, int COPY>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_tile(const ScanArgs A) {
    constexpr int L = L_FWD, TT = W * L, V = lane_channels<T>, S = S_FWD;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>;
    using Stage = FwdStage<T, GM, RASTER, COPY>;
    extern __shared__ __align__(16) char rows[];
    __shared__ Vec<V> sa[2][W][32], sh[2][W][32];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c0 = item % A.ctiles * 32 * V, c = c0 + lane * V;
    const int nc = min(32 * V, A.D - c0), nl = min(V, A.D - c);  // channels of the tile, of the lane (<= 0: none)
    char* const mine = rows + w * S * Stage::bytes;
    const unsigned mine_s = (unsigned)__cvta_generic_to_shared(mine);
    Decay<V, LO> fixed;
    Vec<V> factor = splat<V>(1.0f);
    if (PC) channel_decays<T, GM, V>(A, c, nl, fixed, factor);
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        Vec<V> carry = load_n<V>(A.h0 + s * A.D + c, A.h0 ? nl : 0);
        if (sp.len == 0) {
            if (A.h && rank == 0 && w == 0) store_n<V>(A.h + s * A.D + c, carry, nl);
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c0;
        const T* px = reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, 0) + c0;
        const unsigned* pw = reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (c0 >> 5);
        T* py = reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c;
        const long long round = (long long)CL * TT;
        unsigned words = 0;
        auto fetch = [&](long long t, int slot) {  // this warp's steps from t on
            const int n = (int)max(0ll, min((long long)L, sp.len - t));
            const unsigned dst = mine_s + slot * Stage::bytes;
            if (n > 0) {
                if (!PC) stage_rows<T, COPY, L>(dst + Stage::gate, pg + t * A.gate.st, A.gate.st, n, nc, lane);
                if (!RASTER) stage_rows<T, COPY, L>(dst + Stage::x, px + t * A.x.st, A.x.st, n, nc, lane);
            }
            copy_commit();
        };
        auto fetch_words = [&](long long t) {
            if (RASTER)
                words = t < sp.len ? raster_word<V, L>(pw + t * A.x.st, A.x.st, (int)min((long long)L, sp.len - t),
                                                       (nc + 31) >> 5, lane)
                                   : 0u;
        };
        const long long t1 = (long long)rank * TT + w * L;
        for (int k = 0; k < S; ++k) fetch(t1 + k * round, k);
        fetch_words(t1);
        int slot = 0;
        for (long long b = 0; b < sp.len; b += round) {
            const long long t0 = b + t1;
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> u[L];
            copy_wait<S - 1>();
            __syncwarp();
            const char* from = mine + slot * Stage::bytes;
            const unsigned held = words;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                Vec<V> f = factor;
                if (!PC)
                    decays<T, GM, V>(Unpack<T>::get(staged<COPY>(from + Stage::gate, i, lane,
                                                                 odd_row<COPY>(pg + t0 * A.gate.st, A.gate.st, i))),
                                     d[i], f);
                if constexpr (RASTER) u[i] = raster_values<V>(held, i, lane);
                else u[i] = Unpack<T>::get(staged<COPY>(from + Stage::x, i, lane, odd_row<COPY>(px + t0 * A.x.st, A.x.st, i)));
                if (LEAKY) u[i] = vmul(f, u[i]);
            }
            if (PC) d[0] = fixed;
            __syncwarp();
            fetch(t0 + S * round, slot);
            fetch_words(t0 + round);
            slot = slot + 1 == S ? 0 : slot + 1;
            Vec<V> a = splat<V>(1.0f), h = splat<V>(0.0f);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Decay<V, LO>& q = d[PC ? 0 : i];
                h = q.step(h, u[i]);
                a = q.times(a);
            }
            sa[par][w][lane] = a;
            sh[par][w][lane] = h;
            __syncthreads();
            // the maps of the warps before this one (a, h) and of the whole tile (ta, th)
            Vec<V> ta = splat<V>(1.0f), th = CL > 1 ? splat<V>(0.0f) : carry;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (j == w) {
                    a = ta;
                    h = th;
                }
                const Vec<V> ja = sa[par][j][lane];
                th = vfma(ja, th, sh[par][j][lane]);
                ta = vmul(ja, ta);
            }
            if (CL > 1) {
                for (int r = w; r < CL; r += W) {
                    store_peer<V>(&cm.a[par][rank][lane], r, ta);
                    store_peer<V>(&cm.h[par][rank][lane], r, th);
                }
                cluster_sync();
                Vec<V> in = carry;
                for (int r = 0; r < CL; ++r) {
                    if (r == rank) in = carry;
                    carry = vfma(cm.a[par][r][lane], carry, cm.h[par][r][lane]);
                }
                h = vfma(a, in, h);
            } else {
                carry = th;
            }
            par ^= 1;
            if (nl <= 0 || t0 >= sp.len) continue;
            if (A.saved && t0 % BLOCK == 0) store_n<V>(A.saved + (sp.block0 + t0 / BLOCK) * A.D + c, h, nl);
            T* qy = py + t0 * A.y.st;
            const int n = (int)min((long long)L, sp.len - t0);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (i < n) {
                    h = d[PC ? 0 : i].step(h, u[i]);
                    write_row<T, COPY>(qy, h, nl);
                }
                qy += A.y.st;
            }
            if (A.h && t0 + n == sp.len) store_n<V>(A.h + s * A.D + c, h, nl);
        }
        copy_wait<0>();
        __syncwarp();
    }
}

// The gradient runs from the last tile to the first.  With r the gradient that
// reaches a step from later ones, g = o + r and r' = a g: the map of a tile is
// r -> A r + R.  The states inside the tile come from its saved first state.
template <typename T, int GM, bool RASTER, bool LEAKY, int COPY>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_grad_tile(const ScanArgs A) {
    constexpr int L = L_BWD, TT = W * L, V = lane_channels<T>, S = S_BWD;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>;
    using Stage = BwdStage<T, GM, RASTER, COPY>;
    extern __shared__ __align__(16) char rows[];
    __shared__ Vec<V> sa[2][W][32], sh[2][W][32], sr[2][W][32];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c0 = item % A.ctiles * 32 * V, c = c0 + lane * V;
    const int nc = min(32 * V, A.D - c0), nl = min(V, A.D - c);
    char* const mine = rows + w * S * Stage::bytes;
    const unsigned mine_s = (unsigned)__cvta_generic_to_shared(mine);
    const Vec<V> one = splat<V>(1.0f), minus = splat<V>(-1.0f);
    Decay<V, LO> fixed;
    Vec<V> factor = one, sum = splat<V>(0.0f);
    if (PC) channel_decays<T, GM, V>(A, c, nl, fixed, factor);
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        Vec<V> carry = splat<V>(0.0f);
        if (sp.len == 0) {
            if (A.dh0 && rank == 0 && w == 0)
                store_n<V>(A.dh0 + s * A.D + c, load_n<V>(A.dh + s * A.D + c, A.dh ? nl : 0), nl);
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c0;
        const T* px = reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, 0) + c0;
        const unsigned* pw = reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (c0 >> 5);
        const T* pd = reinterpret_cast<const T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c0;
        T* pdg = reinterpret_cast<T*>(A.dgate.p) + (PC ? 0 : row_at(A, A.dgate, s, sp, 0) + c);
        T* pdx = reinterpret_cast<T*>(A.dx.p) + row_at(A, A.dx, s, sp, 0) + c;
        Vec<V> first = splat<V>(0.0f);
        unsigned words = 0;
        auto fetch = [&](long long t, int slot) {
            if (t >= 0 && t < sp.len) {
                const int n = (int)min((long long)L, sp.len - t);
                const unsigned dst = mine_s + slot * Stage::bytes;
                if (!PC) stage_rows<T, COPY, L>(dst + Stage::gate, pg + t * A.gate.st, A.gate.st, n, nc, lane);
                if (!RASTER) stage_rows<T, COPY, L>(dst + Stage::x, px + t * A.x.st, A.x.st, n, nc, lane);
                if (A.y.p) stage_rows<T, COPY, L>(dst + Stage::dy, pd + t * A.y.st, A.y.st, n, nc, lane);
            }
            copy_commit();
        };
        auto fetch_words = [&](long long t) {
            if (t >= 0) first = load_n<V>(A.saved + (sp.block0 + t / BLOCK) * A.D + c, nl);
            if (RASTER)
                words = t >= 0 && t < sp.len ? raster_word<V, L>(pw + t * A.x.st, A.x.st, (int)min((long long)L, sp.len - t),
                                                                 (nc + 31) >> 5, lane)
                                             : 0u;
        };
        const long long tiles = (sp.len + TT - 1) / TT, round = (long long)CL * TT;
        const long long t1 = (tiles - 1 - rank) * TT + w * L;
        for (int k = 0; k < S; ++k) fetch(t1 - k * round, k);
        fetch_words(t1);
        int slot = 0;
        for (long long b = 0; b < tiles; b += CL) {
            const long long t0 = t1 - b * TT;  // negative: no tile left for this CTA
            const bool some = t0 >= 0 && t0 < sp.len;
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> rest[PC ? 1 : L], x[L], o[L];
            copy_wait<S - 1>();
            __syncwarp();
            const char* from = mine + slot * Stage::bytes;
            const unsigned held = words;
            const Vec<V> h0 = first;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (!PC)
                    decays<T, GM, V>(Unpack<T>::get(staged<COPY>(from + Stage::gate, i, lane,
                                                                 odd_row<COPY>(pg + t0 * A.gate.st, A.gate.st, i))),
                                     d[i], rest[i]);
                if constexpr (RASTER) x[i] = raster_values<V>(held, i, lane);
                else x[i] = Unpack<T>::get(staged<COPY>(from + Stage::x, i, lane, odd_row<COPY>(px + t0 * A.x.st, A.x.st, i)));
                o[i] = splat<V>(0.0f);
                if (A.y.p && some)
                    o[i] = Unpack<T>::get(staged<COPY>(from + Stage::dy, i, lane, odd_row<COPY>(pd + t0 * A.y.st, A.y.st, i)));
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
            fetch_words(t0 - round);
            slot = slot + 1 == S ? 0 : slot + 1;
            Vec<V> a = one, h = splat<V>(0.0f), r = h;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Decay<V, LO>& q = d[PC ? 0 : i];
                h = q.step(h, LEAKY ? vmul(PC ? factor : rest[PC ? 0 : i], x[i]) : x[i]);
                a = q.times(a);
                r = d[PC ? 0 : L - 1 - i].times(vadd(o[L - 1 - i], r));
            }
            if (!some) {  // steps behind the end, whose rows were not read: r passes unchanged
                a = one;
                r = splat<V>(0.0f);
            }
            sa[par][w][lane] = a;
            sh[par][w][lane] = h;
            sr[par][w][lane] = r;
            __syncthreads();
            Vec<V> hw = h0;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (j == w) h = hw;
                if (j < W - 1) hw = vfma(sa[par][j][lane], hw, sh[par][j][lane]);
            }
            // the maps of the warps behind this one (a, r) and of the whole tile (ta, tr)
            Vec<V> ta = one, tr = CL > 1 ? splat<V>(0.0f) : carry;
#pragma unroll
            for (int j = W - 1; j >= 0; --j) {
                if (j == w) {
                    a = ta;
                    r = tr;
                }
                const Vec<V> ja = sa[par][j][lane];
                tr = vfma(ja, tr, sr[par][j][lane]);
                ta = vmul(ja, ta);
            }
            if (CL > 1) {
                for (int q = w; q < CL; q += W) {
                    store_peer<V>(&cm.a[par][rank][lane], q, ta);
                    store_peer<V>(&cm.h[par][rank][lane], q, tr);
                }
                cluster_sync();
                Vec<V> in = carry;
                for (int q = 0; q < CL; ++q) {
                    if (q == rank) in = carry;
                    carry = vfma(cm.a[par][q][lane], carry, cm.h[par][q][lane]);
                }
                r = vfma(a, in, r);
            } else {
                carry = tr;
            }
            par ^= 1;
            if (nl <= 0 || !some) continue;
            // x becomes the derivative of h_t in a_t: h_{t-1}, or h_{t-1} - x_t
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Vec<V> before = h, xi = x[i];
                h = d[PC ? 0 : i].step(h, LEAKY ? vmul(PC ? factor : rest[PC ? 0 : i], xi) : xi);
                x[i] = LEAKY ? vfma(minus, xi, before) : before;
            }
            const int n = (int)min((long long)L, sp.len - t0);
            T* qg = pdg + (t0 + L - 1) * A.dgate.st;
            T* qx = pdx + (t0 + L - 1) * A.dx.st;
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
        }
        copy_wait<0>();
        __syncwarp();
    }
    if (PC && A.part) {
        __syncthreads();
        sa[0][w][lane] = sum;
        __syncthreads();
        if (w == 0 && nl > 0) {
            Vec<V> t = splat<V>(0.0f);
            for (int j = 0; j < W; ++j) t = vadd(t, sa[0][j][lane]);
            store_n<V>(A.part + ((long long)(item / A.ctiles) * CL + rank) * A.D + c, t, nl);
        }
    }
}

// dgate of a channel gate: the CTAs' sums, every eighth by one warp
__global__ void __launch_bounds__(256) k_scan_gate_sum(const ScanArgs A, int rows) {
    __shared__ float s[8][32];
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = (int)blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (c < A.D)
        for (int w = grp; w < rows; w += 8) sum += A.part[(long long)w * A.D + c];
    s[grp][lane] = sum;
    __syncthreads();
    if (grp != 0 || c >= A.D) return;
    for (int g = 1; g < 8; ++g) sum += s[g][lane];
    if (A.logit) {
        float a, lo, rest;
        logistic(reinterpret_cast<const float*>(A.gate.p)[c], a, lo, rest);
        sum *= a * rest;
    }
    reinterpret_cast<float*>(A.dgate.p)[c] = sum;
}

void check_desc(const snn_scan* d) {
    SNN_REQUIRE(d, SNN_ERR_ARG, "null scan description");
    SNN_REQUIRE(snnb::elem_type_ok(d->type), SNN_ERR_ARG, "scan: type must be SNN_F32, SNN_BF16 or SNN_F16");
    SNN_REQUIRE((d->flags & ~(SNN_SCAN_LOGIT | SNN_SCAN_LEAKY | SNN_SCAN_CHANNEL | SNN_SCAN_RASTER)) == 0,
                SNN_ERR_ARG, "scan: unknown flags");
    SNN_REQUIRE(d->n_seq >= 0 && d->n_seq < (1ll << 31), SNN_ERR_ARG, "scan: n_seq must lie in [0, 2^31)");
    SNN_REQUIRE(d->n_channels >= 1 && d->n_channels < (1ll << 30), SNN_ERR_ARG,
                "scan: n_channels must lie in [1, 2^30)");
    SNN_REQUIRE(d->n_steps >= 0 && d->n_steps < (1ll << 40), SNN_ERR_ARG, "scan: n_steps must lie in [0, 2^40)");
    SNN_REQUIRE(d->n_seq == 0 || d->n_steps <= (1ll << 46) / d->n_seq, SNN_ERR_ARG, "scan: too many steps in all");
}

int64_t saved_floats(const snn_scan* d) {
    const int64_t rows = d->offsets ? d->n_steps : d->n_seq * d->n_steps;
    return (rows / BLOCK + d->n_seq) * d->n_channels;
}

// the tensor of rows r of a scan whose rows are `width` elements of `size`
// bytes.  Inputs may be broadcast over steps or sequences (stride 0); what is
// written must not overlap itself.
Rows rows_of(const snn_scan* d, const snn_rows* r, const char* name, int64_t width, int size, bool written = false) {
    SNN_REQUIRE(r && (r->data || d->n_steps == 0), SNN_ERR_ARG, std::string("scan: null ") + name);
    SNN_REQUIRE((uintptr_t)r->data % size == 0, SNN_ERR_ARG, std::string("scan: misaligned ") + name);
    const int64_t seqs = d->offsets ? 1 : d->n_seq, steps = d->n_steps;
    const int64_t ss = seqs > 1 ? r->seq_stride : 0, st = steps > 1 ? r->step_stride : 0, most = 1ll << 52;
    SNN_REQUIRE(ss >= 0 && st >= 0 && ss <= most / std::max<int64_t>(seqs, 1) && st <= most / std::max<int64_t>(steps, 1),
                SNN_ERR_ARG, std::string("scan: bad strides of ") + name);
    if (written && steps > 0) {
        const bool steps_inside = (steps == 1 || st >= width) && (seqs == 1 || ss >= st * (steps - 1) + width);
        const bool seqs_inside = (seqs == 1 || ss >= width) && (steps == 1 || st >= ss * (seqs - 1) + width);
        SNN_REQUIRE(steps_inside || seqs_inside, SNN_ERR_ARG, std::string("scan: rows overlap in ") + name);
    }
    return {r->data, ss, st};
}

ScanArgs base_args(const snn_scan* d, const snn_rows* gate, const snn_rows* x) {
    ScanArgs A;
    memset(&A, 0, sizeof(A));
    A.off = d->offsets;
    A.n_seq = d->n_seq;
    A.n_steps = d->n_steps;
    A.D = (int)d->n_channels;
    A.logit = (d->flags & SNN_SCAN_LOGIT) != 0;
    A.leaky = (d->flags & SNN_SCAN_LEAKY) != 0;
    const int size = snnb::elem_size(d->type);
    if (d->flags & SNN_SCAN_CHANNEL) {
        SNN_REQUIRE(gate && gate->data && (uintptr_t)gate->data % 4 == 0, SNN_ERR_ARG, "scan: null or misaligned gate");
        A.gate = {gate->data, 0, 0};
    } else {
        A.gate = rows_of(d, gate, "gate", d->n_channels, size);
    }
    if (d->flags & SNN_SCAN_RASTER) A.x = rows_of(d, x, "x", (d->n_channels + 31) / 32, 4);
    else A.x = rows_of(d, x, "x", d->n_channels, size);
    return A;
}

// f(T(), gate mode, raster) as compile-time constants
template <int V>
using Const = std::integral_constant<int, V>;
template <typename F>
void dispatch(const snn_scan* d, F&& f) {
    snnb::with_elem(d->type, [&](auto t) {
        auto with_gate = [&](auto gm) { d->flags & SNN_SCAN_RASTER ? f(t, gm, Const<1>()) : f(t, gm, Const<0>()); };
        if (d->flags & SNN_SCAN_CHANNEL)
            d->flags & SNN_SCAN_LOGIT ? with_gate(Const<GATE_CHANNEL_LOGIT>()) : with_gate(Const<GATE_CHANNEL>());
        else
            d->flags & SNN_SCAN_LOGIT ? with_gate(Const<GATE_LOGIT>()) : with_gate(Const<GATE_VALUE>());
    });
}

// Grid of the tile kernels.  The sizes alone decide (the sums of a channel
// gate's gradient follow the grid): a cluster per (tile of channels, worker), a
// worker for each sequence up to 32 CTAs an SM, the rest taken in turn; where
// that leaves SMs empty, a cluster of up to MAX_CLUSTER CTAs along the steps.
constexpr int SMS = 148;
struct Plan {
    int ctiles, workers, cluster;
};
int64_t mean_steps(const snn_scan* d) { return d->offsets ? d->n_steps / std::max<int64_t>(d->n_seq, 1) : d->n_steps; }
Plan plan_of(const snn_scan* d, int tile) {
    const int width = 128 / snnb::elem_size(d->type);
    Plan p;
    p.ctiles = (int)((d->n_channels + width - 1) / width);
    p.workers = (int)std::min<int64_t>(d->n_seq, std::max(32, 32 * SMS / p.ctiles));
    p.cluster = 1;
    while (p.cluster < MAX_CLUSTER && (int64_t)p.ctiles * p.workers * p.cluster < 2 * SMS &&
           (int64_t)tile * p.cluster < mean_steps(d))
        p.cluster *= 2;
    return p;
}

// whether r's rows are words of `bytes` from the first element on
bool fits(const Rows& r, int size, int bytes) {
    return (uintptr_t)r.p % bytes == 0 && r.ss * size % bytes == 0 && r.st * size % bytes == 0;
}
// The words that rows are staged in (see stage_rows); written rows go in 4-byte
// words, or in the third form an element at a time.
int copy_words(const snn_scan* d, std::initializer_list<Rows> in, std::initializer_list<Rows> out) {
    const int size = snnb::elem_size(d->type);
    auto all = [&](std::initializer_list<Rows> rows, int bytes) {
        return d->n_channels * size % bytes == 0 &&
               std::all_of(rows.begin(), rows.end(), [&](const Rows& r) { return !r.p || fits(r, size, bytes); });
    };
    if (!all(in, 4) || !all(out, 4)) return 2;
    return all(in, 16) ? 16 : 4;
}

void launch(const void* kernel, int smem, const Plan& p, ScanArgs& A, cudaStream_t st) {
    A.ctiles = p.ctiles;
    A.workers = p.workers;
    A.cluster = p.cluster;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    SNN_REQUIRE((int64_t)p.ctiles * p.workers * p.cluster < (1ll << 31), SNN_ERR_ARG, "scan: too many tiles");
    cfg.gridDim = dim3((unsigned)(p.ctiles * p.workers * p.cluster));
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    SNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    void* args[] = {&A};
    SNN_CUDA(cudaLaunchKernelExC(&cfg, kernel, args));
}

template <typename T, int GM, bool RASTER, int COPY>
void launch_fwd(const Plan& p, ScanArgs& A, cudaStream_t st) {
    const int smem = W * S_FWD * FwdStage<T, GM, RASTER, COPY>::bytes;
    launch(A.leaky ? (const void*)k_scan_tile<T, GM, RASTER, true, COPY> : (const void*)k_scan_tile<T, GM, RASTER, false, COPY>,
           smem, p, A, st);
}
template <typename T, int GM, bool RASTER, int COPY>
void launch_bwd(const Plan& p, ScanArgs& A, cudaStream_t st) {
    const int smem = W * S_BWD * BwdStage<T, GM, RASTER, COPY>::bytes;
    launch(A.leaky ? (const void*)k_scan_grad_tile<T, GM, RASTER, true, COPY>
                   : (const void*)k_scan_grad_tile<T, GM, RASTER, false, COPY>,
           smem, p, A, st);
}

}  // namespace

namespace snnb {

int64_t leaky_scan_saved(const snn_scan* d) {
    check_desc(d);
    return saved_floats(d);
}

int64_t leaky_scan_grad_workspace(const snn_scan* d) {
    check_desc(d);
    if (!(d->flags & SNN_SCAN_CHANNEL)) return 0;
    const Plan p = plan_of(d, W * L_BWD);
    return (int64_t)p.workers * p.cluster * d->n_channels * 4;
}

void leaky_scan(const snn_scan* d, const snn_rows* gate, const snn_rows* x, const float* h0,
                const snn_rows* y, float* h, float* saved, cudaStream_t st) {
    check_desc(d);
    if (d->n_seq == 0) return;
    ScanArgs A = base_args(d, gate, x);
    A.y = rows_of(d, y, "y", d->n_channels, elem_size(d->type), true);
    A.h0 = h0;
    A.h = h;
    A.saved = saved;
    const bool raster_x = (d->flags & SNN_SCAN_RASTER) != 0, channel = (d->flags & SNN_SCAN_CHANNEL) != 0;
    const Rows none = {nullptr, 0, 0};
    const int words = copy_words(d, {channel ? none : A.gate, raster_x ? none : A.x}, {A.y});
    if (mean_steps(d) <= 8) {
        const int vec = d->type != SNN_F32 && words > 2 ? 2 : 1;
        const dim3 grid((unsigned)((d->n_channels + 128 * vec - 1) / (128 * vec)),
                        (unsigned)std::min<int64_t>(d->n_seq, 65535));
        dispatch(d, [&](auto t, auto gm, auto raster) {
            using T = decltype(t);
            constexpr int GM = decltype(gm)::value;
            constexpr bool RA = decltype(raster)::value != 0;
            if (vec == 2) k_scan_steps<T, GM, RA, 2><<<grid, 128, 0, st>>>(A);
            else k_scan_steps<T, GM, RA, 1><<<grid, 128, 0, st>>>(A);
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const Plan p = plan_of(d, W * L_FWD);
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if (words == 16) return launch_fwd<T, GM, RA, 16>(p, A, st);
        if constexpr (sizeof(T) == 2)
            if (words == 2) return launch_fwd<T, GM, RA, 2>(p, A, st);
        launch_fwd<T, GM, RA, 4>(p, A, st);
    });
}

void leaky_scan_grad(const snn_scan* d, const snn_rows* gate, const snn_rows* x, const float* saved,
                     const snn_rows* dy, const float* dh, const snn_rows* dgate, const snn_rows* dx,
                     float* dh0, void* work, int64_t work_bytes, cudaStream_t st) {
    check_desc(d);
    SNN_REQUIRE(dy || dh, SNN_ERR_ARG, "scan: neither dy nor dh");
    SNN_REQUIRE(!(dx && (d->flags & SNN_SCAN_RASTER)), SNN_ERR_ARG, "scan: a raster has no gradient");
    const bool channel = (d->flags & SNN_SCAN_CHANNEL) != 0;
    if (d->n_seq == 0) {
        if (channel && dgate && dgate->data)
            SNN_CUDA(cudaMemsetAsync(dgate->data, 0, (size_t)d->n_channels * 4, st));
        return;
    }
    SNN_REQUIRE(saved, SNN_ERR_ARG, "scan: null saved");
    ScanArgs A = base_args(d, gate, x);
    const int size = elem_size(d->type);
    A.saved = const_cast<float*>(saved);
    A.dh = dh;
    A.dh0 = dh0;
    if (dy) A.y = rows_of(d, dy, "dy", d->n_channels, size);
    if (dx) A.dx = rows_of(d, dx, "dx", d->n_channels, size, true);
    if (dgate && channel) {
        SNN_REQUIRE(dgate->data && (uintptr_t)dgate->data % 4 == 0, SNN_ERR_ARG, "scan: null or misaligned dgate");
        SNN_REQUIRE(work && (uintptr_t)work % 256 == 0 && work_bytes >= leaky_scan_grad_workspace(d), SNN_ERR_ARG,
                    "scan: workspace null, misaligned or too small");
        A.dgate = {dgate->data, 0, 0};
        A.part = (float*)work;
    } else if (dgate) {
        A.dgate = rows_of(d, dgate, "dgate", d->n_channels, size, true);
    }
    const Rows none = {nullptr, 0, 0};
    const int words = copy_words(d, {channel ? none : A.gate, d->flags & SNN_SCAN_RASTER ? none : A.x, A.y},
                                 {channel ? none : A.dgate, A.dx});
    const Plan p = plan_of(d, W * L_BWD);
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if (words == 16) return launch_bwd<T, GM, RA, 16>(p, A, st);
        if constexpr (sizeof(T) == 2)
            if (words == 2) return launch_bwd<T, GM, RA, 2>(p, A, st);
        launch_bwd<T, GM, RA, 4>(p, A, st);
    });
    if (A.part) {
        k_scan_gate_sum<<<(unsigned)((d->n_channels + 31) / 32), 256, 0, st>>>(A, p.workers * p.cluster);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
