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

enum { GATE_VALUE = 0, GATE_LOGIT = 1, GATE_CHANNEL = 2 };

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

// A decay in the form the recurrence needs it: a = m, or a = 1 + m where
// `keep` is all ones.  The logistic decay of a large gate is 1 - s with a
// small s; kept as -s it has s's relative precision, which is what a state
// with a long memory (1/s steps) is proportional to, while 1 - s rounded to
// f32 is off by 2^-25 / s of it.
struct Decay {
    float m;
    unsigned keep;
    __device__ __forceinline__ float step(float h, float u) const {
        return fmaf(m, h, __uint_as_float(__float_as_uint(h) & keep) + u);
    }
    __device__ __forceinline__ float times(float h) const {
        return fmaf(m, h, __uint_as_float(__float_as_uint(h) & keep));
    }
    __device__ __forceinline__ float rest() const { return keep ? -m : 1.0f - m; }  // 1 - a
    __device__ __forceinline__ float slope() const {                                // a (1 - a) of a logistic decay
        const float s = fabsf(m);
        return s * (1.0f - s);
    }
};
__device__ __forceinline__ Decay decay_value(float a) { return {a, 0u}; }
__device__ __forceinline__ Decay decay_logit(float z) {
    const float e = expf(-fabsf(z));
    const float s = __fdiv_rn(e, 1.0f + e);
    Decay d;
    d.keep = (__float_as_uint(z) >> 31) - 1u;  // z >= 0: all ones
    d.m = d.keep ? -s : s;
    return d;
}

template <typename T, int GM>
__device__ __forceinline__ Decay decay_at(const ScanArgs& A, long long row, int c, const Decay& fixed) {
    if (GM == GATE_CHANNEL) return fixed;
    const float v = to_f32(reinterpret_cast<const T*>(A.gate.p)[row + c]);
    return GM == GATE_LOGIT ? decay_logit(v) : decay_value(v);
}
__device__ __forceinline__ Decay decay_channel(const ScanArgs& A, int c) {
    const float v = reinterpret_cast<const float*>(A.gate.p)[c];
    return A.logit ? decay_logit(v) : decay_value(v);
}
template <typename T, bool RASTER>
__device__ __forceinline__ float input_at(const ScanArgs& A, long long row, int c) {
    if (RASTER) return (float)((reinterpret_cast<const unsigned*>(A.x.p)[row + (c >> 5)] >> (c & 31)) & 1u);
    return to_f32(reinterpret_cast<const T*>(A.x.p)[row + c]);
}

// One thread per sequence and channel, a step at a time.
template <typename T, int GM, bool RASTER>
__global__ void __launch_bounds__(128) k_scan_seq(const ScanArgs A) {
    const int c = (int)(blockIdx.x * 128 + threadIdx.x);
    if (c >= A.D) return;
    for (long long s = blockIdx.y; s < A.n_seq; s += gridDim.y) {
        const Span sp = span_of(A, s);
        const Decay fixed = GM == GATE_CHANNEL ? decay_channel(A, c) : Decay();
        float h = A.h0 ? A.h0[s * A.D + c] : 0.0f;
        for (long long t = 0; t < sp.len; ++t) {
            if (A.saved && t % BLOCK == 0) A.saved[(sp.block0 + t / BLOCK) * A.D + c] = h;
            const Decay d = decay_at<T, GM>(A, row_at(A, A.gate, s, sp, t), c, fixed);
            float u = input_at<T, RASTER>(A, row_at(A, A.x, s, sp, t), c);
            if (A.leaky) u = d.rest() * u;
            h = d.step(h, u);
            reinterpret_cast<T*>(A.y.p)[row_at(A, A.y, s, sp, t) + c] = from_f32<T>(h);
        }
        if (A.h) A.h[s * A.D + c] = h;
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
constexpr int L_FWD = 16, L_BWD = 8;
constexpr int MAX_CLUSTER = 8;
static_assert((W * L_BWD) == BLOCK && (W * L_FWD) % BLOCK == 0 && BLOCK % L_FWD == 0, "blocks start at a warp's steps");

template <typename T, int V>
struct alignas(sizeof(T) * V) Word {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Word<T, V> zero_word() {
    Word<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = from_f32<T>(0.0f);
    return r;
}
// what a lane reads of an input row: V elements, or the raster word they lie in
template <typename T, int V, bool RASTER>
struct InWord {
    using type = Word<T, V>;
};
template <typename T, int V>
struct InWord<T, V, true> {
    using type = unsigned;
};
template <int V, typename T>
__device__ __forceinline__ float in_value(const Word<T, V>& w, int k, int) {
    return to_f32(w.v[k]);
}
template <int V>
__device__ __forceinline__ float in_value(unsigned w, int k, int c) {
    return (float)((w >> ((c + k) & 31)) & 1u);
}

// The decay of a gate as one float.  GATE_LOGIT: the sign says the form (m, or
// 1 + m for a set sign, -0 included).  16-bit gates use the short exponential
// and reciprocal: off by some 2^-20 relative, their own rounding by 2^-9.
template <typename T, int GM>
__device__ __forceinline__ float gate_m(float z) {
    if (GM != GATE_LOGIT) return z;
    float s;
    if (sizeof(T) == 4) {
        const float e = expf(-fabsf(z));
        s = __fdiv_rn(e, 1.0f + e);
    } else {
        const float e = __expf(-fabsf(z));
        s = __fdividef(e, 1.0f + e);
    }
    return __uint_as_float((__float_as_uint(s) & 0x7fffffffu) | (~__float_as_uint(z) & 0x80000000u));
}
template <int GM>
__device__ __forceinline__ Decay decay_m(float m, unsigned keep) {
    Decay d;
    d.m = m;
    d.keep = GM == GATE_VALUE ? 0u : GM == GATE_LOGIT ? (unsigned)(__float_as_int(m) >> 31) : keep;
    return d;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// store to the same shared-memory variable of CTA `rank` of the cluster
__device__ __forceinline__ void store_peer(float* p, int rank, float v) {
    unsigned a = (unsigned)__cvta_generic_to_shared(p), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(r), "f"(v) : "memory");
}

template <int V>
struct ClusterMaps {  // the tiles' maps of a round, by rank; two rounds
    float a[2][MAX_CLUSTER][32 * V], h[2][MAX_CLUSTER][32 * V];
};

template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_tile(const ScanArgs A) {
    constexpr int L = L_FWD, TT = W * L;
    using G = Word<T, V>;
    using X = typename InWord<T, V, RASTER>::type;
    __shared__ float sa[2][W][32 * V], sh[2][W][32 * V];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c = (item % A.ctiles * 32 + lane) * V;
    const bool live = c < A.D;
    float fm[V];
    unsigned fk[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        fm[k] = 0.0f;
        fk[k] = 0u;
        if (GM == GATE_CHANNEL && live) {
            const Decay d = decay_channel(A, c + k);
            fm[k] = d.m;
            fk[k] = d.keep;
        }
    }
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        float carry[V];
#pragma unroll
        for (int k = 0; k < V; ++k) carry[k] = A.h0 && live ? A.h0[s * A.D + c + k] : 0.0f;
        if (sp.len == 0) {
            if (A.h && live && rank == 0 && w == 0)
#pragma unroll
                for (int k = 0; k < V; ++k) A.h[s * A.D + c + k] = carry[k];
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c;
        const char* px = RASTER ? (const char*)(reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (c >> 5))
                                : (const char*)(reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, 0) + c);
        T* py = reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c;
        constexpr int XS = RASTER ? 4 : sizeof(T);
        G rg[L];
        X rx[L];
        auto fetch = [&](long long t0) {
            const T* qg = pg + t0 * A.gate.st;
            const char* qx = px + t0 * A.x.st * XS;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (live && t0 + i < sp.len) {
                    if (GM != GATE_CHANNEL) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st * XS);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < L; ++i) {
            rg[i] = zero_word<T, V>();
            memset(&rx[i], 0, sizeof(X));
        }
        const long long round = (long long)CL * TT;
        fetch((long long)rank * TT + w * L);
        for (long long b = 0; b < sp.len; b += round) {
            const long long t0 = b + (long long)rank * TT + w * L;
            float m[L][V], u[L][V], a[V], h[V];
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    m[i][k] = GM == GATE_CHANNEL ? fm[k] : gate_m<T, GM>(to_f32(rg[i].v[k]));
                    u[i][k] = in_value<V>(rx[i], k, c);
                    if (A.leaky) u[i][k] *= decay_m<GM>(m[i][k], fk[k]).rest();
                }
            if (b + round < sp.len) fetch(t0 + round);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                a[k] = 1.0f;
                h[k] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Decay d = decay_m<GM>(m[i][k], fk[k]);
                    h[k] = d.step(h[k], u[i][k]);
                    a[k] = d.times(a[k]);
                }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                sa[par][w][lane * V + k] = a[k];
                sh[par][w][lane * V + k] = h[k];
            }
            __syncthreads();
            if (CL > 1) {
                if (w == 0) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float ta = 1.0f, th = 0.0f;
                        for (int j = 0; j < W; ++j) {
                            th = fmaf(sa[par][j][lane * V + k], th, sh[par][j][lane * V + k]);
                            ta *= sa[par][j][lane * V + k];
                        }
                        for (int r = 0; r < CL; ++r) {
                            store_peer(&cm.a[par][rank][lane * V + k], r, ta);
                            store_peer(&cm.h[par][rank][lane * V + k], r, th);
                        }
                    }
                }
                cluster_sync();
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float hk = carry[k];
                if (CL > 1) {
                    for (int r = 0; r < rank; ++r) hk = fmaf(cm.a[par][r][lane * V + k], hk, cm.h[par][r][lane * V + k]);
                    float next = hk;
                    for (int r = rank; r < CL; ++r) next = fmaf(cm.a[par][r][lane * V + k], next, cm.h[par][r][lane * V + k]);
                    carry[k] = next;
                }
                for (int j = 0; j < w; ++j) hk = fmaf(sa[par][j][lane * V + k], hk, sh[par][j][lane * V + k]);
                h[k] = hk;
                if (CL == 1) {
                    for (int j = w; j < W; ++j) hk = fmaf(sa[par][j][lane * V + k], hk, sh[par][j][lane * V + k]);
                    carry[k] = hk;
                }
            }
            par ^= 1;
            if (A.saved && live && t0 % BLOCK == 0 && t0 < sp.len)
#pragma unroll
                for (int k = 0; k < V; ++k) A.saved[(sp.block0 + t0 / BLOCK) * A.D + c + k] = h[k];
            T* qy = py + t0 * A.y.st;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (t0 + i >= sp.len) break;
                G o;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    h[k] = decay_m<GM>(m[i][k], fk[k]).step(h[k], u[i][k]);
                    o.v[k] = from_f32<T>(h[k]);
                }
                if (live) *reinterpret_cast<G*>(qy + i * A.y.st) = o;
                if (t0 + i == sp.len - 1 && A.h && live)
#pragma unroll
                    for (int k = 0; k < V; ++k) A.h[s * A.D + c + k] = h[k];
            }
        }
    }
}

// The gradient runs from the last tile to the first.  With r the gradient that
// reaches a step from later ones, g = o + r and r' = a g: the map of a tile is
// r -> A r + R.  The states inside the tile come from its saved first state.
template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(TILE_THREADS, 2) k_scan_grad_tile(const ScanArgs A) {
    constexpr int L = L_BWD, TT = W * L;
    using G = Word<T, V>;
    using X = typename InWord<T, V, RASTER>::type;
    __shared__ float sa[2][W][32 * V], sh[2][W][32 * V], sr[2][W][32 * V];
    __shared__ ClusterMaps<V> cm;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int CL = A.cluster, rank = blockIdx.x % CL, item = blockIdx.x / CL;
    const int c = (item % A.ctiles * 32 + lane) * V;
    const bool live = c < A.D;
    float fm[V], sum[V];
    unsigned fk[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        fm[k] = sum[k] = 0.0f;
        fk[k] = 0u;
        if (GM == GATE_CHANNEL && live) {
            const Decay d = decay_channel(A, c + k);
            fm[k] = d.m;
            fk[k] = d.keep;
        }
    }
    int par = 0;
    for (long long s = item / A.ctiles; s < A.n_seq; s += A.workers) {
        const Span sp = span_of(A, s);
        float carry[V];
#pragma unroll
        for (int k = 0; k < V; ++k) carry[k] = 0.0f;
        if (sp.len == 0) {
            if (A.dh0 && live && rank == 0 && w == 0)
#pragma unroll
                for (int k = 0; k < V; ++k) A.dh0[s * A.D + c + k] = A.dh ? A.dh[s * A.D + c + k] : 0.0f;
            continue;
        }
        const T* pg = reinterpret_cast<const T*>(A.gate.p) + row_at(A, A.gate, s, sp, 0) + c;
        const char* px = RASTER ? (const char*)(reinterpret_cast<const unsigned*>(A.x.p) + row_at(A, A.x, s, sp, 0) + (c >> 5))
                                : (const char*)(reinterpret_cast<const T*>(A.x.p) + row_at(A, A.x, s, sp, 0) + c);
        const T* pd = A.y.p ? reinterpret_cast<const T*>(A.y.p) + row_at(A, A.y, s, sp, 0) + c : nullptr;
        T* pdg = GM != GATE_CHANNEL && A.dgate.p ? reinterpret_cast<T*>(A.dgate.p) + row_at(A, A.dgate, s, sp, 0) + c : nullptr;
        T* pdx = A.dx.p ? reinterpret_cast<T*>(A.dx.p) + row_at(A, A.dx, s, sp, 0) + c : nullptr;
        constexpr int XS = RASTER ? 4 : sizeof(T);
        G rg[L], rd[L];
        X rx[L];
        float rs[V];
        auto fetch = [&](long long t0) {
            if (!live || t0 < 0) return;
            const T* qg = pg + t0 * A.gate.st;
            const T* qd = pd + t0 * A.y.st;
            const char* qx = px + t0 * A.x.st * XS;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (t0 + i < sp.len) {
                    if (GM != GATE_CHANNEL) rg[i] = *reinterpret_cast<const G*>(qg + i * A.gate.st);
                    rx[i] = *reinterpret_cast<const X*>(qx + i * A.x.st * XS);
                    if (pd) rd[i] = *reinterpret_cast<const G*>(qd + i * A.y.st);
                } else {
                    rd[i] = zero_word<T, V>();
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) rs[k] = A.saved[(sp.block0 + t0 / BLOCK) * A.D + c + k];
        };
#pragma unroll
        for (int i = 0; i < L; ++i) {
            rg[i] = rd[i] = zero_word<T, V>();
            memset(&rx[i], 0, sizeof(X));
        }
#pragma unroll
        for (int k = 0; k < V; ++k) rs[k] = 0.0f;
        const long long tiles = (sp.len + TT - 1) / TT;
        fetch((tiles - 1 - rank) * TT + w * L);
        for (long long b = 0; b < tiles; b += CL) {
            const long long t0 = (tiles - 1 - b - rank) * TT + w * L;  // negative: no tile left for this CTA
            float m[L][V], xv[L][V], o[L][V], a[V], h[V], r[V], h0[V];
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    m[i][k] = GM == GATE_CHANNEL ? fm[k] : gate_m<T, GM>(to_f32(rg[i].v[k]));
                    xv[i][k] = in_value<V>(rx[i], k, c);
                    o[i][k] = to_f32(rd[i].v[k]);
                    if (t0 + i == sp.len - 1 && A.dh && live) o[i][k] += A.dh[s * A.D + c + k];
                }
#pragma unroll
            for (int k = 0; k < V; ++k) h0[k] = rs[k];
            if (b + CL < tiles) fetch(t0 - (long long)CL * TT);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                a[k] = 1.0f;
                h[k] = r[k] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Decay d = decay_m<GM>(m[i][k], fk[k]);
                    h[k] = d.step(h[k], A.leaky ? d.rest() * xv[i][k] : xv[i][k]);
                    a[k] = d.times(a[k]);
                    const Decay e = decay_m<GM>(m[L - 1 - i][k], fk[k]);
                    r[k] = e.times(o[L - 1 - i][k] + r[k]);
                }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                sa[par][w][lane * V + k] = a[k];
                sh[par][w][lane * V + k] = h[k];
                sr[par][w][lane * V + k] = r[k];
            }
            __syncthreads();
            if (CL > 1) {
                if (w == 0) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float ta = 1.0f, tr = 0.0f;
                        for (int j = W - 1; j >= 0; --j) {
                            tr = fmaf(sa[par][j][lane * V + k], tr, sr[par][j][lane * V + k]);
                            ta *= sa[par][j][lane * V + k];
                        }
                        for (int q = 0; q < CL; ++q) {
                            store_peer(&cm.a[par][rank][lane * V + k], q, ta);
                            store_peer(&cm.h[par][rank][lane * V + k], q, tr);
                        }
                    }
                }
                cluster_sync();
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float hk = h0[k];
                for (int j = 0; j < w; ++j) hk = fmaf(sa[par][j][lane * V + k], hk, sh[par][j][lane * V + k]);
                h[k] = hk;
                float rk = carry[k];
                if (CL > 1) {
                    for (int q = 0; q < rank; ++q) rk = fmaf(cm.a[par][q][lane * V + k], rk, cm.h[par][q][lane * V + k]);
                    float next = rk;
                    for (int q = rank; q < CL; ++q) next = fmaf(cm.a[par][q][lane * V + k], next, cm.h[par][q][lane * V + k]);
                    carry[k] = next;
                }
                for (int j = W - 1; j > w; --j) rk = fmaf(sa[par][j][lane * V + k], rk, sr[par][j][lane * V + k]);
                r[k] = rk;
                if (CL == 1) {
                    for (int j = w; j >= 0; --j) rk = fmaf(sa[par][j][lane * V + k], rk, sr[par][j][lane * V + k]);
                    carry[k] = rk;
                }
            }
            par ^= 1;
            if (t0 < 0) continue;
            // xv becomes the derivative of h_t in a_t: h_{t-1}, or h_{t-1} - x_t
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Decay d = decay_m<GM>(m[i][k], fk[k]);
                    const float before = h[k], x = xv[i][k];
                    h[k] = d.step(before, A.leaky ? d.rest() * x : x);
                    xv[i][k] = A.leaky ? before - x : before;
                }
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
                if (t0 + i >= sp.len) continue;
                G og, ox;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const Decay d = decay_m<GM>(m[i][k], fk[k]);
                    const float g = o[i][k] + r[k], da = g * xv[i][k];
                    if (GM == GATE_CHANNEL) sum[k] += da;
                    og.v[k] = from_f32<T>(GM == GATE_LOGIT ? da * d.slope() : da);
                    ox.v[k] = from_f32<T>(A.leaky ? d.rest() * g : g);
                    r[k] = d.times(g);
                }
                if (live && pdg) *reinterpret_cast<G*>(pdg + (t0 + i) * A.dgate.st) = og;
                if (live && pdx) *reinterpret_cast<G*>(pdx + (t0 + i) * A.dx.st) = ox;
            }
            if (t0 == 0 && A.dh0 && live)
#pragma unroll
                for (int k = 0; k < V; ++k) A.dh0[s * A.D + c + k] = r[k];
        }
    }
    if (GM == GATE_CHANNEL && A.part) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) sa[0][w][lane * V + k] = sum[k];
        __syncthreads();
        if (w == 0 && live)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float t = 0.0f;
                for (int j = 0; j < W; ++j) t += sa[0][j][lane * V + k];
                A.part[((long long)(item / A.ctiles) * CL + rank) * A.D + c + k] = t;
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
    if (A.logit) sum *= decay_channel(A, c).slope();
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
        const bool raster = (d->flags & SNN_SCAN_RASTER) != 0;
        const int gm = d->flags & SNN_SCAN_CHANNEL ? GATE_CHANNEL : d->flags & SNN_SCAN_LOGIT ? GATE_LOGIT : GATE_VALUE;
        if (gm == GATE_CHANNEL) raster ? f(t, Const<GATE_CHANNEL>(), Const<1>()) : f(t, Const<GATE_CHANNEL>(), Const<0>());
        else if (gm == GATE_LOGIT) raster ? f(t, Const<GATE_LOGIT>(), Const<1>()) : f(t, Const<GATE_LOGIT>(), Const<0>());
        else raster ? f(t, Const<GATE_VALUE>(), Const<1>()) : f(t, Const<GATE_VALUE>(), Const<0>());
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
    if (mean_steps(d) <= 8) {
        const dim3 grid((unsigned)((d->n_channels + 127) / 128), (unsigned)std::min<int64_t>(d->n_seq, 65535));
        dispatch(d, [&](auto t, auto gm, auto raster) {
            k_scan_seq<decltype(t), decltype(gm)::value, decltype(raster)::value != 0><<<grid, 128, 0, st>>>(A);
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const int size = elem_size(d->type);
    const bool raster_x = (d->flags & SNN_SCAN_RASTER) != 0, channel = (d->flags & SNN_SCAN_CHANNEL) != 0;
    const bool two = size == 2 && d->n_channels % 2 == 0 && (channel || fits_vec(A.gate, size, 2)) &&
                     (raster_x || fits_vec(A.x, size, 2)) && fits_vec(A.y, size, 2);
    const Plan p = plan_of(d, two ? 2 : 1, W * L_FWD);
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if constexpr (sizeof(T) == 2)
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
    const bool two = size == 2 && d->n_channels % 2 == 0 && (channel || fits_vec(A.gate, size, 2)) &&
                     ((d->flags & SNN_SCAN_RASTER) || fits_vec(A.x, size, 2)) && fits_vec(A.y, size, 2) &&
                     fits_vec(A.dx, size, 2) && (channel || fits_vec(A.dgate, size, 2));
    const Plan p = plan_of(d, two ? 2 : 1, W * L_BWD);
    dispatch(d, [&](auto t, auto gm, auto raster) {
        using T = decltype(t);
        constexpr int GM = decltype(gm)::value;
        constexpr bool RA = decltype(raster)::value != 0;
        if constexpr (sizeof(T) == 2)
            if (two) return launch((const void*)k_scan_grad_tile<T, GM, RA, 2>, p, A, st);
        launch((const void*)k_scan_grad_tile<T, GM, RA, 1>, p, A, st);
    });
    if (A.part) {
        k_scan_gate_sum<<<(unsigned)((d->n_channels + 31) / 32), 256, 0, st>>>(A, p.workers * p.cluster);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
