// adamw.cu - one AdamW step over many tensors (snn_adamw), first and second
// moments in f32 or in 8 bits.
//
// Bound by memory: 28 bytes an element with f32 moments and f32 gradients (p, m, v
// read and written, g read), 16 with 8-bit ones.  Descriptions of the tensors travel
// as kernel parameters, so a step over up to 400 tensors is one launch and needs
// no table on the device.  69 M parameters, 16-bit gradients and copies: a step 353 us, 297 at the
// copy rate; 8-bit moments 307 of 169, bound by the instructions (120 an element).  Roundings are those of the formula taken one operation
// at a time (this file is compiled without contraction).
//
// 8-bit moments: e4m3 values (half a step is 2^-4 of a value) with an f32 scale for
// every 256 elements, the largest magnitude times 1 / 448.  Of the second moment the
// root is held, which halves its range, and a root above zero as 2^-9 (the smallest
// e4m3 value) at least: a second moment that is lost to zero beside a first one that
// is not would make a step of m / eps.
#include <algorithm>
#include <cmath>
#include <cuda_fp8.h>
#include "elem.h"

namespace {
using snnb::from_f32;
using snnb::to_f32;
constexpr int THREADS = 256, BLOCK = 256;
constexpr int CHUNK = 2048;    // elements of a CTA: a block for each warp, or two rounds of 4 elements a thread
constexpr int FEW = 48, MANY = 400;  // tensors of a launch: 3.5 or 29 kB of parameters (at most 32,764 bytes)

struct Tensor {
    float* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    void* copy;
    int64_t n;
    int32_t first;             // the first CTA of this tensor
    uint8_t g_type, copy_type, wide;
};
struct Rule {
    float b1, c1, b2, c2, decay, eps, grad_scale, size, root;
    const int64_t* step;       // device: size and root are made from lr, beta1, beta2 there
    double lr, beta1, beta2;
};
template <int N>
struct StepArgs {
    Rule r;
    int n;
    Tensor t[N];
};

struct Moments {
    float m, v;
};
__device__ __forceinline__ Moments moments(const Rule& r, float g, float m, float v) {
    g = g * r.grad_scale;
    return {m * r.b1 + g * r.c1, v * r.b2 + g * g * r.c2};
}
__device__ __forceinline__ float updated(const Rule& r, float size, float root, float p, Moments x) {
    return p * r.decay - x.m / (sqrtf(x.v) * root + r.eps) * size;
}
// Four e4m3 values in a word
__device__ __forceinline__ void from_e4m3(unsigned w, float* o) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3));
        const float2 f = __half22float2(h);
        o[2 * i] = f.x;
        o[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ unsigned to_e4m3(const float* v) {
    return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3) |
           (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}
// Quotients by one divisor, rounded as a division is: from the rounded reciprocal, a product and
// one correction by the remainder, which a fused product has exactly (Markstein 1990).  The remainder
// must not be lost below the smallest numbers: divisors outside 2^-80 .. 2^80 are divided by.
struct Divisor {
    float d, inv;
    bool plain;
    __device__ __forceinline__ explicit Divisor(float v) : d(v), inv(1.0f / v), plain(!(v > 0x1p-80f && v < 0x1p80f)) {}
    __device__ __forceinline__ float under(float a) const {
        if (plain) return a / d;
        const float q = a * inv;
        return fmaf(fmaf(-q, d, a), inv, q);
    }
};

template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Word {
    T v[V];
};
// n <= V elements (all, or fewer at a tensor's end)
template <int V, typename T>
__device__ __forceinline__ void load(const T* p, int n, bool wide, T (&o)[V]) {
    if (wide && n == V) {
        const Word<T, V> w = *reinterpret_cast<const Word<T, V>*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = w.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = i < n ? p[i] : T();
    }
}
template <int V, typename T>
__device__ __forceinline__ void store(T* p, int n, bool wide, const T (&o)[V]) {
    if (wide && n == V) {
        Word<T, V> w;
#pragma unroll
        for (int i = 0; i < V; ++i) w.v[i] = o[i];
        *reinterpret_cast<Word<T, V>*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = o[i];
    }
}
// eight bytes
__device__ __forceinline__ void load8(const unsigned char* p, int n, bool wide, unsigned (&o)[2]) {
    if (wide && n == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        o[0] = w.x;
        o[1] = w.y;
    } else {
        o[0] = o[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) o[i / 4] |= (unsigned)p[i] << (8 * (i % 4));
    }
}
__device__ __forceinline__ void store8(unsigned char* p, int n, bool wide, const unsigned (&o)[2]) {
    if (wide && n == 8) {
        *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (unsigned char)(o[i / 4] >> (8 * (i % 4)));
    }
}
template <int V>
__device__ __forceinline__ void store_copy(const Tensor& t, int64_t at, int n, const float (&p)[V]) {
    auto put = [&](auto z) {
        using T = decltype(z);
        T o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = from_f32<T>(p[i]);
        store<V>(reinterpret_cast<T*>(t.copy) + at, n, t.wide, o);
    };
    if (t.copy_type == SNN_BF16) put(__nv_bfloat16());
    else put(__half());
}

template <typename G, bool BITS8>
__device__ __forceinline__ void chunk(const Rule& r, const Tensor& t, int64_t begin, float size, float root) {
    if constexpr (!BITS8) {
        constexpr int V = 4;
        const int64_t end = min(t.n, begin + CHUNK);
#pragma unroll 2
        for (int64_t at = begin + threadIdx.x * V; at < end; at += THREADS * V) {
            const int n = (int)min((int64_t)V, end - at);
            G g[V];
            float p[V], m[V], v[V];
            load<V>(reinterpret_cast<const G*>(t.g) + at, n, t.wide, g);
            load<V>(t.p + at, n, t.wide, p);
            load<V>(reinterpret_cast<const float*>(t.m) + at, n, t.wide, m);
            load<V>(reinterpret_cast<const float*>(t.v) + at, n, t.wide, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const Moments x = moments(r, to_f32(g[i]), m[i], v[i]);
                p[i] = updated(r, size, root, p[i], x);
                m[i] = x.m;
                v[i] = x.v;
            }
            store<V>(t.p + at, n, t.wide, p);
            store<V>(reinterpret_cast<float*>(t.m) + at, n, t.wide, m);
            store<V>(reinterpret_cast<float*>(t.v) + at, n, t.wide, v);
            if (t.copy) store_copy<V>(t, at, n, p);
        }
    } else {  // a warp per block of 256 elements, 8 a lane
        constexpr int V = 8;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int64_t end = min(t.n, begin + CHUNK);
#pragma unroll 2
        for (int64_t b = begin + warp * BLOCK; b < end; b += THREADS / 32 * BLOCK) {
            const int64_t at = b + lane * V;
            const int n = (int)max((int64_t)0, min((int64_t)V, end - at));
            G g[V];
            float p[V], m[V], v[V];
            unsigned m8[2], v8[2];
            load<V>(reinterpret_cast<const G*>(t.g) + at, n, t.wide, g);
            load<V>(t.p + at, n, t.wide, p);
            load8(reinterpret_cast<const unsigned char*>(t.m) + at, n, t.wide, m8);
            load8(reinterpret_cast<const unsigned char*>(t.v) + at, n, t.wide, v8);
            float om[V], ov[V];
            from_e4m3(m8[0], om);
            from_e4m3(m8[1], om + 4);
            from_e4m3(v8[0], ov);
            from_e4m3(v8[1], ov + 4);
            float ms = t.ms[b / BLOCK], vs = t.vs[b / BLOCK], top_m = 0.0f, top_v = 0.0f;
            bool nan_m = false, nan_v = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float root_v = ov[i] * vs;
                const Moments x = moments(r, to_f32(g[i]), om[i] * ms, root_v * root_v);
                v[i] = sqrtf(x.v);
                p[i] = p[i] * r.decay - x.m / (v[i] * root + r.eps) * size;
                m[i] = x.m;
                if (i < n) {
                    top_m = fmaxf(top_m, fabsf(m[i]));
                    top_v = fmaxf(top_v, v[i]);
                    nan_m |= isnan(m[i]);
                    nan_v |= isnan(v[i]);
                }
            }
            store<V>(t.p + at, n, t.wide, p);
            if (t.copy) store_copy<V>(t, at, n, p);
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                top_m = fmaxf(top_m, __shfl_xor_sync(~0u, top_m, o));
                top_v = fmaxf(top_v, __shfl_xor_sync(~0u, top_v, o));
            }
            // a block that holds a NaN becomes NaN as a whole, and says so
            ms = __any_sync(~0u, nan_m) ? NAN : top_m * (1.0f / 448.0f);
            vs = __any_sync(~0u, nan_v) ? NAN : top_v * (1.0f / 448.0f);
            const Divisor dm(ms), dv(vs);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                m[i] = ms > 0.0f ? dm.under(m[i]) : ms;
                const float z = vs > 0.0f ? dv.under(v[i]) : vs;
                v[i] = v[i] > 0.0f ? fmaxf(z, 0x1p-9f) : z;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m8[i] = to_e4m3(m + 4 * i);
                v8[i] = to_e4m3(v + 4 * i);
            }
            store8(reinterpret_cast<unsigned char*>(t.m) + at, n, t.wide, m8);
            store8(reinterpret_cast<unsigned char*>(t.v) + at, n, t.wide, v8);
            if (lane == 0) {
                t.ms[b / BLOCK] = ms;
                t.vs[b / BLOCK] = vs;
            }
        }
    }
}

template <int N, bool BITS8>
__global__ void __launch_bounds__(THREADS) k_adamw(const __grid_constant__ StepArgs<N> A) {
    int lo = 0, hi = A.n - 1;  // the last tensor whose first CTA is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (A.t[mid].first <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const Tensor& t = A.t[lo];
    float size = A.r.size, root = A.r.root;
    if (A.r.step) {
        __shared__ float s[2];
        if (threadIdx.x == 0) {
            const double n = (double)*A.r.step;
            s[0] = (float)(A.r.lr / (1.0 - pow(A.r.beta1, n)));
            s[1] = (float)(1.0 / sqrt(1.0 - pow(A.r.beta2, n)));
        }
        __syncthreads();
        size = s[0];
        root = s[1];
    }
    const int64_t begin = (int64_t)((int)blockIdx.x - t.first) * CHUNK;
    if (t.g_type == SNN_F32) chunk<float, BITS8>(A.r, t, begin, size, root);
    else if (t.g_type == SNN_BF16) chunk<__nv_bfloat16, BITS8>(A.r, t, begin, size, root);
    else chunk<__half, BITS8>(A.r, t, begin, size, root);
}

template <int N>
void launch(const Rule& r, const Tensor* t, int n, int ctas, bool bits8, cudaStream_t st) {
    static_assert(sizeof(StepArgs<N>) <= 32764, "kernel parameters");
    StepArgs<N> A;
    A.r = r;
    A.n = n;
    std::copy(t, t + n, A.t);
    if (bits8) k_adamw<N, true><<<ctas, THREADS, 0, st>>>(A);
    else k_adamw<N, false><<<ctas, THREADS, 0, st>>>(A);
    SNN_CUDA(cudaGetLastError());
}

}  // namespace

namespace snnb {

void adamw(const snn_adamw_tensor* tensors, int64_t count, int32_t bits, const snn_adamw_rule* rule, cudaStream_t st) {
    SNN_REQUIRE(count >= 0 && count <= (1 << 20) && (tensors || count == 0), SNN_ERR_ARG,
                "adamw: count must lie in [0, 2^20], with tensors");
    SNN_REQUIRE(bits == 32 || bits == 8, SNN_ERR_ARG, "adamw: moments have 32 or 8 bits");
    SNN_REQUIRE(rule, SNN_ERR_ARG, "adamw: null rule");
    SNN_REQUIRE(rule->beta1 >= 0 && rule->beta1 < 1 && rule->beta2 >= 0 && rule->beta2 < 1, SNN_ERR_ARG,
                "adamw: betas must lie in [0, 1)");
    SNN_REQUIRE(rule->eps >= 0, SNN_ERR_ARG, "adamw: eps must not be negative");
    SNN_REQUIRE(rule->step_device || rule->step >= 1, SNN_ERR_ARG, "adamw: steps are counted from 1");
    SNN_REQUIRE((uintptr_t)rule->step_device % 8 == 0, SNN_ERR_ARG, "adamw: misaligned step");
    Rule r;
    r.b1 = (float)rule->beta1;
    r.c1 = (float)(1.0 - rule->beta1);
    r.b2 = (float)rule->beta2;
    r.c2 = (float)(1.0 - rule->beta2);
    r.decay = (float)(1.0 - rule->lr * rule->weight_decay);
    r.eps = (float)rule->eps;
    r.grad_scale = (float)rule->grad_scale;
    r.step = rule->step_device;
    r.lr = rule->lr;
    r.beta1 = rule->beta1;
    r.beta2 = rule->beta2;
    r.size = r.root = 0.0f;
    if (!r.step) {
        r.size = (float)(rule->lr / (1.0 - std::pow(rule->beta1, (double)rule->step)));
        r.root = (float)(1.0 / std::sqrt(1.0 - std::pow(rule->beta2, (double)rule->step)));
    }
    std::vector<Tensor> all;
    all.reserve((size_t)count);
    for (int64_t i = 0; i < count; ++i) {  // all are looked at before the first launch
        const snn_adamw_tensor& s = tensors[i];
        if (!s.g || s.n == 0) continue;
        const int gs = s.g_type == SNN_F32 ? 4 : 2;
        SNN_REQUIRE(s.n > 0 && s.n <= (1ll << 40), SNN_ERR_ARG, "adamw: n must lie in [0, 2^40]");
        SNN_REQUIRE(elem_type_ok(s.g_type), SNN_ERR_ARG, "adamw: gradients are SNN_F32, SNN_BF16 or SNN_F16");
        SNN_REQUIRE(!s.copy || s.copy_type == SNN_BF16 || s.copy_type == SNN_F16, SNN_ERR_ARG,
                    "adamw: copies are SNN_BF16 or SNN_F16");
        SNN_REQUIRE(s.p && s.m && s.v && (bits == 32 || (s.m_scale && s.v_scale)), SNN_ERR_ARG,
                    "adamw: null parameters, moments or scales");
        const uintptr_t own = (uintptr_t)s.p | (bits == 32 ? (uintptr_t)s.m | (uintptr_t)s.v
                                                            : (uintptr_t)s.m_scale | (uintptr_t)s.v_scale);
        SNN_REQUIRE(own % 4 == 0 && (uintptr_t)s.g % gs == 0 && (uintptr_t)s.copy % 2 == 0, SNN_ERR_ARG,
                    "adamw: misaligned tensor");
        Tensor t;
        t.p = s.p;
        t.g = s.g;
        t.m = s.m;
        t.v = s.v;
        t.ms = s.m_scale;
        t.vs = s.v_scale;
        t.copy = s.copy;
        t.n = s.n;
        t.first = 0;
        t.g_type = (uint8_t)s.g_type;
        t.copy_type = (uint8_t)s.copy_type;
        // words: 4 elements with f32 moments, 8 with 8-bit ones
        const uintptr_t mom = (uintptr_t)s.m | (uintptr_t)s.v, x = (uintptr_t)s.p;
        t.wide = bits == 32 ? (x | mom) % 16 == 0 && (uintptr_t)s.g % (4 * gs) == 0 && (uintptr_t)s.copy % 8 == 0
                            : x % 16 == 0 && mom % 8 == 0 && (uintptr_t)s.g % 16 == 0 && (uintptr_t)s.copy % 16 == 0;
        all.push_back(t);
    }
    size_t i = 0;
    while (i < all.size()) {  // launches of up to MANY tensors and 2^30 CTAs
        int n = 0;
        int64_t ctas = 0;
        const size_t from = i;
        while (i < all.size() && n < MANY) {
            const int64_t more = (all[i].n + CHUNK - 1) / CHUNK;
            if (n && ctas + more > (1ll << 30)) break;
            all[i].first = (int32_t)ctas;
            ctas += more;
            ++n;
            ++i;
        }
        if (n <= FEW) launch<FEW>(r, &all[from], n, (int)ctas, bits == 8, st);
        else launch<MANY>(r, &all[from], n, (int)ctas, bits == 8, st);
    }
}

}  // namespace snnb
