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
// precision: from e = exp(-|z|) the larger is 1 / (1 + e), the smaller e times that
__device__ __forceinline__ void logistic(float z, float& a, float& lo, float& rest) {
    const float e = expf(-fabsf(z));
    const float big = __frcp_rn(1.0f + e), s = e * big;
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
__device__ __forceinline__ void channel_decays(const ScanArgs& A, int c, bool live, Decay<V, keeps_lo<T, GM>>& d,
                                               Vec<V>& rest) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float v = live ? reinterpret_cast<const float*>(A.gate.p)[c + k] : 0.0f;
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
        if (per_channel<GM>) channel_decays<T, GM, V>(A, c, true, d, rest);
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
// a warp L steps, a lane V channels, all in registers.  Over its L steps a
// warp's map of the state is h -> A h + H (A the product of the decays, H the
// end state from zero); the CTA joins its warps' maps in shared memory, so
// each warp learns the state it starts from and runs its steps once more with
// it.  With few channels a cluster of CTAs takes consecutive tiles and joins
// their maps through distributed shared memory; the state after the cluster's
// tiles is carried in registers to its next round.
constexpr int W = 8;
constexpr int TILE_THREADS = 32 * W;
template <typename T>
constexpr int fwd_steps = sizeof(T) == 4 ? 8 : 16;
constexpr int L_BWD = 8;
constexpr int MAX_CLUSTER = 8;
static_assert(W * L_BWD == BLOCK && BLOCK % (2 * L_BWD) == 0, "blocks start at a warp's steps");

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

template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_tile(const ScanArgs A) {
    constexpr int L = fwd_steps<T>, TT = W * L;
    constexpr bool LO = keeps_lo<T, GM>;
    using G = Word<T, V>;
    using X = InWord<T, V, RASTER>;
    using XE = std::conditional_t<RASTER, unsigned, T>;
    __shared__ Vec<V> sa[2][W][32], sh[2][W][32];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c = (item % A.ctiles * 32 + lane) * V;
    const bool live = c < A.D;
    Decay<V, LO> fixed;
    Vec<V> factor = splat<V>(1.0f);
    if (per_channel<GM>) {
        channel_decays<T, GM, V>(A, c, live, fixed, factor);
        if (!A.leaky) factor = splat<V>(1.0f);
    }
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        Vec<V> carry = load_f32<V>(A.h0 + s * A.D + c, A.h0 && live);
        if (sp.len == 0) {
            if (A.h && live && rank == 0 && w == 0) store_f32<V>(A.h + s * A.D + c, carry);
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c;
        const XE* px = reinterpret_cast<const XE*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (RASTER ? c >> 5 : c);
        T* py = reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c;
        G rg[L];
        X rx[L];
        auto fetch = [&](long long t0) {
            const T* qg = pg + t0 * A.gate.st;
            const XE* qx = px + t0 * A.x.st;
            const int n = live ? (int)min((long long)L, sp.len - t0) : 0;
            if (n == L) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (!per_channel<GM>) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st);
                }
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (i >= n) continue;
                    if (!per_channel<GM>) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < L; ++i) {
            memset(&rg[i], 0, sizeof(G));
            memset(&rx[i], 0, sizeof(X));
        }
        const long long round = (long long)CL * TT;
        fetch((long long)rank * TT + w * L);
        for (long long b = 0; b < sp.len; b += round) {
            const long long t0 = b + (long long)rank * TT + w * L;
            Decay<V, LO> d[per_channel<GM> ? 1 : L];
            Vec<V> u[L];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                Vec<V> f = factor;
                if (!per_channel<GM>) {
                    decays<T, GM, V>(Unpack<T>::get(rg[i]), d[i], f);
                    if (!A.leaky) f = splat<V>(1.0f);
                }
                u[i] = vmul(f, in_values<T, V, RASTER>(rx[i], c));
            }
            if (per_channel<GM>) d[0] = fixed;
            if (b + round < sp.len) fetch(t0 + round);
            Vec<V> a = splat<V>(1.0f), h = splat<V>(0.0f);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Decay<V, LO>& q = d[per_channel<GM> ? 0 : i];
                h = q.step(h, u[i]);
                a = q.times(a);
            }
            sa[par][w][lane] = a;
            sh[par][w][lane] = h;
            __syncthreads();
            if (CL > 1) {
                if (w == 0) {
                    Vec<V> ta = splat<V>(1.0f), th = splat<V>(0.0f);
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        th = vfma(sa[par][j][lane], th, sh[par][j][lane]);
                        ta = vmul(sa[par][j][lane], ta);
                    }
                    for (int r = 0; r < CL; ++r) {
                        store_peer<V>(&cm.a[par][rank][lane], r, ta);
                        store_peer<V>(&cm.h[par][rank][lane], r, th);
                    }
                }
                cluster_sync();
            }
            h = carry;
            if (CL > 1) {
                for (int r = 0; r < rank; ++r) h = vfma(cm.a[par][r][lane], h, cm.h[par][r][lane]);
                carry = h;
                for (int r = rank; r < CL; ++r) carry = vfma(cm.a[par][r][lane], carry, cm.h[par][r][lane]);
            }
            for (int j = 0; j < w; ++j) h = vfma(sa[par][j][lane], h, sh[par][j][lane]);
            if (CL == 1) {
                carry = h;
                for (int j = w; j < W; ++j) carry = vfma(sa[par][j][lane], carry, sh[par][j][lane]);
            }
            par ^= 1;
            if (!live || t0 >= sp.len) continue;
            if (A.saved && t0 % BLOCK == 0) store_f32<V>(A.saved + (sp.block0 + t0 / BLOCK) * A.D + c, h);
            T* qy = py + t0 * A.y.st;
            const int n = (int)min((long long)L, sp.len - t0);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (i < n) {
                    h = d[per_channel<GM> ? 0 : i].step(h, u[i]);
                    *reinterpret_cast<G*>(qy) = Unpack<T>::put(h);
                }
                qy += A.y.st;
            }
            if (A.h && t0 + n == sp.len) store_f32<V>(A.h + s * A.D + c, h);
        }
    }
}

// The gradient runs from the last tile to the first.  With r the gradient that
// reaches a step from later ones, g = o + r and r' = a g: the map of a tile is
// r -> A r + R.  The states inside the tile come from its saved first state.
template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_grad_tile(const ScanArgs A) {
    constexpr int L = L_BWD, TT = W * L;
    constexpr bool LO = keeps_lo<T, GM>, PC = per_channel<GM>;
    using G = Word<T, V>;
    using X = InWord<T, V, RASTER>;
    using XE = std::conditional_t<RASTER, unsigned, T>;
    __shared__ Vec<V> sa[2][W][32], sh[2][W][32], sr[2][W][32];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c = (item % A.ctiles * 32 + lane) * V;
    const bool live = c < A.D;
    const Vec<V> one = splat<V>(1.0f), minus = splat<V>(A.leaky ? -1.0f : 0.0f);
    Decay<V, LO> fixed;
    Vec<V> factor = one, sum = splat<V>(0.0f);
    if (PC) {
        channel_decays<T, GM, V>(A, c, live, fixed, factor);
        if (!A.leaky) factor = one;
    }
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        Vec<V> carry = splat<V>(0.0f);
        if (sp.len == 0) {
            if (A.dh0 && live && rank == 0 && w == 0)
                store_f32<V>(A.dh0 + s * A.D + c, load_f32<V>(A.dh + s * A.D + c, A.dh != nullptr));
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c;
        const XE* px = reinterpret_cast<const XE*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (RASTER ? c >> 5 : c);
        const T* pd = reinterpret_cast<const T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c;
        T* pdg = reinterpret_cast<T*>(A.dgate.p) + (PC ? 0 : row_at(A, A.dgate, s, sp, 0) + c);
        T* pdx = reinterpret_cast<T*>(A.dx.p) + row_at(A, A.dx, s, sp, 0) + c;
        G rg[L], rd[L];
        X rx[L];
        Vec<V> rs = splat<V>(0.0f);
        auto fetch = [&](long long t0) {
            if (t0 < 0) return;
            const T* qg = pg + t0 * A.gate.st;
            const T* qd = pd + t0 * A.y.st;
            const XE* qx = px + t0 * A.x.st;
            const int n = live ? (int)min((long long)L, sp.len - t0) : 0;
            if (n == L && A.y.p) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (!PC) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st);
                    rd[i] = *reinterpret_cast<const G*>(qd + i * A.y.st);
                }
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (i >= n) continue;
                    if (!PC) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st);
                    if (A.y.p) rd[i] = *reinterpret_cast<const G*>(qd + i * A.y.st);
                }
            }
            rs = load_f32<V>(A.saved + (sp.block0 + t0 / BLOCK) * A.D + c, live);
        };
#pragma unroll
        for (int i = 0; i < L; ++i) {
            memset(&rg[i], 0, sizeof(G));
            memset(&rd[i], 0, sizeof(G));
            memset(&rx[i], 0, sizeof(X));
        }
        const long long tiles = (sp.len + TT - 1) / TT;
        fetch((tiles - 1 - rank) * TT + w * L);
        for (long long b = 0; b < tiles; b += CL) {
            const long long t0 = (tiles - 1 - b - rank) * TT + w * L;  // negative: no tile left for this CTA
            Decay<V, LO> d[PC ? 1 : L];
            Vec<V> rest[PC ? 1 : L], x[L], o[L];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (!PC) decays<T, GM, V>(Unpack<T>::get(rg[i]), d[i], rest[i]);
                x[i] = in_values<T, V, RASTER>(rx[i], c);
                o[i] = Unpack<T>::get(rd[i]);
                if (t0 + i == sp.len - 1) o[i] = vadd(o[i], load_f32<V>(A.dh + s * A.D + c, A.dh && live));
            }
            if (PC) d[0] = fixed;
            const Vec<V> h0 = rs;
            if (b + CL < tiles) fetch(t0 - (long long)CL * TT);
            Vec<V> a = one, h = splat<V>(0.0f), r = h;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Decay<V, LO>& q = d[PC ? 0 : i];
                const Vec<V> f = PC ? factor : A.leaky ? rest[PC ? 0 : i] : one;
                h = q.step(h, vmul(f, x[i]));
                a = q.times(a);
                r = d[PC ? 0 : L - 1 - i].times(vadd(o[L - 1 - i], r));
            }
            sa[par][w][lane] = a;
            sh[par][w][lane] = h;
            sr[par][w][lane] = r;
            __syncthreads();
            if (CL > 1) {
                if (w == 0) {
                    Vec<V> ta = one, tr = splat<V>(0.0f);
#pragma unroll
                    for (int j = W - 1; j >= 0; --j) {
                        tr = vfma(sa[par][j][lane], tr, sr[par][j][lane]);
                        ta = vmul(sa[par][j][lane], ta);
                    }
                    for (int q = 0; q < CL; ++q) {
                        store_peer<V>(&cm.a[par][rank][lane], q, ta);
                        store_peer<V>(&cm.h[par][rank][lane], q, tr);
                    }
                }
                cluster_sync();
            }
            h = h0;
            for (int j = 0; j < w; ++j) h = vfma(sa[par][j][lane], h, sh[par][j][lane]);
            r = carry;
            if (CL > 1) {
                for (int q = 0; q < rank; ++q) r = vfma(cm.a[par][q][lane], r, cm.h[par][q][lane]);
                carry = r;
                for (int q = rank; q < CL; ++q) carry = vfma(cm.a[par][q][lane], carry, cm.h[par][q][lane]);
            }
            for (int j = W - 1; j > w; --j) r = vfma(sa[par][j][lane], r, sr[par][j][lane]);
            if (CL == 1) {
                carry = r;
                for (int j = w; j >= 0; --j) carry = vfma(sa[par][j][lane], carry, sr[par][j][lane]);
            }
            par ^= 1;
            if (!live || t0 < 0 || t0 >= sp.len) continue;
            // x becomes the derivative of h_t in a_t: h_{t-1}, or h_{t-1} - x_t
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const Vec<V> f = PC ? factor : A.leaky ? rest[PC ? 0 : i] : one;
                const Vec<V> before = h, xi = x[i];
                h = d[PC ? 0 : i].step(h, vmul(f, xi));
                x[i] = A.leaky ? vfma(minus, xi, before) : before;
            }
            const int n = (int)min((long long)L, sp.len - t0);
            T* qg = pdg + (t0 + L - 1) * A.dgate.st;
            T* qx = pdx + (t0 + L - 1) * A.dx.st;
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
                if (i < n) {
                    const Decay<V, LO>& q = d[PC ? 0 : i];
                    const Vec<V> f = PC ? factor : A.leaky ? rest[PC ? 0 : i] : one;
                    const Vec<V> g = vadd(o[i], r);
                    if (PC) {
                        sum = vfma(g, x[i], sum);
                    } else if (A.dgate.p) {
                        Vec<V> da = vmul(g, x[i]);
                        if (GM == GATE_LOGIT) da = vmul(da, vmul(q.a, rest[PC ? 0 : i]));
                        *reinterpret_cast<G*>(qg) = Unpack<T>::put(da);
                    }
                    if (A.dx.p) *reinterpret_cast<G*>(qx) = Unpack<T>::put(vmul(f, g));
                    r = q.times(g);
                }
                qg -= A.dgate.st;
                qx -= A.dx.st;
            }
            if (t0 == 0 && A.dh0) store_f32<V>(A.dh0 + s * A.D + c, r);
        }
    }
    if (PC && A.part) {
        __syncthreads();
        sa[0][w][lane] = sum;
        __syncthreads();
        if (w == 0 && live) {
            Vec<V> t = splat<V>(0.0f);
            for (int j = 0; j < W; ++j) t = vadd(t, sa[0][j][lane]);
            store_f32<V>(A.part + ((long long)(item / A.ctiles) * CL + rank) * A.D + c, t);
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
    int vec, ctiles, workers, cluster;
};
bool fits_vec(const Rows& r, int size, int vec) {
    return (uintptr_t)r.p % (size * vec) == 0 && r.ss % vec == 0 && r.st % vec == 0;
}
int64_t mean_steps(const snn_scan* d) { return d->offsets ? d->n_steps / std::max<int64_t>(d->n_seq, 1) : d->n_steps; }
Plan plan_of(const snn_scan* d, int vec, int tile) {
    Plan p;
    p.vec = vec;
    p.ctiles = (int)((d->n_channels + 32 * vec - 1) / (32 * vec));
    p.workers = (int)std::min<int64_t>(d->n_seq, std::max(32, 32 * SMS / p.ctiles));
    p.cluster = 1;
    while (p.cluster < MAX_CLUSTER && (int64_t)p.ctiles * p.workers * p.cluster < 2 * SMS &&
           (int64_t)tile * p.cluster < mean_steps(d))
        p.cluster *= 2;
    return p;
}

void launch(const void* kernel, const Plan& p, ScanArgs& A, cudaStream_t st) {
    A.ctiles = p.ctiles;
    A.workers = p.workers;
    A.cluster = p.cluster;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    SNN_REQUIRE((int64_t)p.ctiles * p.workers * p.cluster < (1ll << 31), SNN_ERR_ARG, "scan: too many tiles");
    cfg.gridDim = dim3((unsigned)(p.ctiles * p.workers * p.cluster));
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    void* args[] = {&A};
    SNN_CUDA(cudaLaunchKernelExC(&cfg, kernel, args));
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
    int64_t most = 0;  // of the words that the alignment may choose
    for (int vec = 1; vec <= 2; ++vec) {
        const Plan p = plan_of(d, vec, W * L_BWD);
        most = std::max(most, (int64_t)p.workers * p.cluster * d->n_channels * 4);
    }
    return most;
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
    const int size = elem_size(d->type);
    const bool raster_x = (d->flags & SNN_SCAN_RASTER) != 0, channel = (d->flags & SNN_SCAN_CHANNEL) != 0;
    const bool two = d->n_channels % 2 == 0 && (channel || fits_vec(A.gate, size, 2)) &&
                     (raster_x || fits_vec(A.x, size, 2)) && fits_vec(A.y, size, 2);
    if (mean_steps(d) <= 8) {
        const int vec = two ? 2 : 1;
        const dim3 grid((unsigned)((d->n_channels + 128 * vec - 1) / (128 * vec)),
                        (unsigned)std::min<int64_t>(d->n_seq, 65535));
        dispatch(d, [&](auto t, auto gm, auto raster) {
            using T = decltype(t);
            constexpr int GM = decltype(gm)::value;
            constexpr bool RA = decltype(raster)::value != 0;
            if (two) k_scan_steps<T, GM, RA, 2><<<grid, 128, 0, st>>>(A);
            else k_scan_steps<T, GM, RA, 1><<<grid, 128, 0, st>>>(A);
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const Plan p = plan_of(d, two ? 2 : 1, W * (size == 4 ? fwd_steps<float> : fwd_steps<__half>));
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if (two) return launch((const void*)k_scan_tile<T, GM, RA, 2>, p, A, st);
        launch((const void*)k_scan_tile<T, GM, RA, 1>, p, A, st);
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
    const bool two = d->n_channels % 2 == 0 && (channel || fits_vec(A.gate, size, 2)) &&
                     ((d->flags & SNN_SCAN_RASTER) || fits_vec(A.x, size, 2)) && fits_vec(A.y, size, 2) &&
                     fits_vec(A.dx, size, 2) && (channel || fits_vec(A.dgate, size, 2));
    const Plan p = plan_of(d, two ? 2 : 1, W * L_BWD);
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if (two) return launch((const void*)k_scan_grad_tile<T, GM, RA, 2>, p, A, st);
        launch((const void*)k_scan_grad_tile<T, GM, RA, 1>, p, A, st);
    });
    if (A.part) {
        k_scan_gate_sum<<<(unsigned)((d->n_channels + 31) / 32), 256, 0, st>>>(A, p.workers * p.cluster);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
