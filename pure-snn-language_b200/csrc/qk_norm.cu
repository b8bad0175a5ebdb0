// qk_norm.cu - norms of queries and keys for each head with the position
// rotation in the same pass (snn_qk_norm), and their gradients.
//
//   n = x r,  r = 1 / sqrt(sum x^2 / count + eps),  y = turn(n w)
//   z = turn^-1(dy),  dw = sum z n,  dx = r (z w - n sum(z w n) / count)
// Bound by memory: every element is read once and written once.  A group of G
// lanes takes a head, a lane whole words of up to 16 bytes of it such that both
// elements of a rotated pair are its own, so that nothing but the sum of squares
// crosses lanes.  Cosines and sines of a row are made once for all of its heads,
// in shared memory; angles are products in 64 bits (a position of 1e5 has an angle
// whose f32 would be off by 4e-3), reduced to a turn before the f32 sine.
#include <algorithm>
#include "elem.h"

namespace {
using snnb::from_f32;
using snnb::to_f32;
constexpr int SMS = 148, THREADS = 256, MAX_DIM = 512, MAX_ROWS = 8;

struct Heads {
    void* p;
    long long ss, st, hs;  // strides of sequences, steps, heads
};
struct Side {              // queries or keys
    Heads x, y, dx;        // GRAD: y holds dy
    const float* w;
    float *part, *dw;      // sums of the CTAs, their sum
    int heads;
};
struct NormArgs {
    Side side[2];
    const void* pos;
    const float* freqs;
    long long rows, steps;
    int dim, rot, per_tile, pos64, adjacent;
    float eps, inv_count;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Word {
    T v[V];
};
__device__ __forceinline__ long long row_at(const Heads& h, const NormArgs& A, long long row) {
    const long long s = row / A.steps;
    return s * h.ss + (row - s * A.steps) * h.st;
}

// Words a, b of slot s.  Pairs of the first and second half: words s and s + P of the
// P that each half has, then the rest two by two; else neighbours.
template <int V, bool IN>
__device__ __forceinline__ void words_of(const NormArgs& A, int s, int& a, int& b) {
    a = 2 * s;
    b = 2 * s + 1;
    const int P = A.rot / (2 * V);
    if (!IN && !A.adjacent && s < P) {
        a = s;
        b = s + P;
    }
}
// The pairs of words a, b of slot s turned (BACK: the other way).  IN: pairs lie
// inside a word.
template <int V, bool IN, bool BACK>
__device__ __forceinline__ void turn(const NormArgs& A, const float2* cs, int s, float (&a)[V], float (&b)[V]) {
    auto pair = [&](float& u, float& v, int j) {
        const float2 c = cs[j];
        const float si = BACK ? -c.y : c.y, x = u, y = v;
        u = x * c.x - y * si;
        v = x * si + y * c.x;
    };
    const int half = A.rot / 2;
    if constexpr (IN) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const int j = s * V + i;
                if (j < half) pair(a[2 * i], a[2 * i + 1], j);
                if (j + V / 2 < half) pair(b[2 * i], b[2 * i + 1], j + V / 2);
            }
        }
    } else if (s * V < half) {
#pragma unroll
        for (int i = 0; i < V; ++i) pair(a[i], b[i], s * V + i);
    }
}

// V elements a word, SL slots of two words a lane, G lanes a head
template <typename T, int V, int SL, bool IN, bool GRAD>
__global__ void __launch_bounds__(THREADS) k_qk_norm(const __grid_constant__ NormArgs A, int G) {
    extern __shared__ float2 cs[];  // [rows of a tile][rot / 2]
    __shared__ float sum[GRAD ? MAX_DIM : 1];
    using W = Word<T, V>;
    const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G, groups = THREADS / G, half = A.rot / 2;
    const int words = A.dim / V;
    const unsigned mask = G == 32 ? ~0u : ((1u << G) - 1) << ((threadIdx.x & 31) & ~(G - 1));
    auto all = [&](float v) {
        for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
        return v;
    };
    int wa[SL], wb[SL];
#pragma unroll
    for (int i = 0; i < SL; ++i) words_of<V, IN>(A, lane + i * G, wa[i], wb[i]);
    auto load = [&](const T* p, int w, float (&o)[V]) {
        if (w < words) {
            const W x = *reinterpret_cast<const W*>(p + w * V);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = to_f32(x.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = 0.0f;
        }
    };
    auto store = [&](T* p, int w, const float (&o)[V]) {
        if (w >= words) return;
        W x;
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(o[i]);
        *reinterpret_cast<W*>(p + w * V) = x;
    };
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const Side& S = A.side[which];
        if (!S.x.p) continue;
        float ga[SL][V], gb[SL][V], da[GRAD ? SL : 1][V], db[GRAD ? SL : 1][V];
#pragma unroll
        for (int i = 0; i < SL; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ga[i][j] = S.w && wa[i] < words ? S.w[wa[i] * V + j] : 1.0f;
                gb[i][j] = S.w && wb[i] < words ? S.w[wb[i] * V + j] : 1.0f;
                if (GRAD) da[i][j] = db[i][j] = 0.0f;
            }
#pragma unroll 1
        for (long long tile = (long long)blockIdx.x * A.per_tile; tile < A.rows; tile += (long long)gridDim.x * A.per_tile) {
            const int n = (int)min((long long)A.per_tile, A.rows - tile);
            __syncthreads();
            for (int i = threadIdx.x; i < n * half; i += THREADS) {
                const int r = i / half;
                const long long at = tile + r;
                const double pos = A.pos64 ? (double)reinterpret_cast<const long long*>(A.pos)[at]
                                           : (double)reinterpret_cast<const int*>(A.pos)[at];
                const double turns = pos * (double)A.freqs[i - r * half] * 0.15915494309189533577;  // 1 / (2 pi)
                float s, c;
                sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
                cs[i] = make_float2(c, s);
            }
            __syncthreads();
            for (int e = group; e < n * S.heads; e += groups) {
                const int r = e / S.heads, head = e - r * S.heads;
                const long long row = tile + r;
                const float2* c = cs + r * half;
                const T* x = reinterpret_cast<const T*>(S.x.p) + row_at(S.x, A, row) + head * S.x.hs;
                T* y = reinterpret_cast<T*>(S.y.p) + row_at(S.y, A, row) + head * S.y.hs;
                float a[SL][V], b[SL][V], za[GRAD ? SL : 1][V], zb[GRAD ? SL : 1][V];
#pragma unroll
                for (int i = 0; i < SL; ++i) {
                    load(x, wa[i], a[i]);
                    load(x, wb[i], b[i]);
                    if constexpr (GRAD) {
                        load(y, wa[i], za[i]);
                        load(y, wb[i], zb[i]);
                    }
                }
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < SL; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) sq = fmaf(a[i][j], a[i][j], fmaf(b[i][j], b[i][j], sq));
                const float inv = 1.0f / sqrtf(fmaf(all(sq), A.inv_count, A.eps));
                if constexpr (!GRAD) {
#pragma unroll
                    for (int i = 0; i < SL; ++i) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            a[i][j] = a[i][j] * inv * ga[i][j];
                            b[i][j] = b[i][j] * inv * gb[i][j];
                        }
                        turn<V, IN, false>(A, c, lane + i * G, a[i], b[i]);
                        store(y, wa[i], a[i]);
                        store(y, wb[i], b[i]);
                    }
                } else {
                    float dot = 0.0f;
#pragma unroll
                    for (int i = 0; i < SL; ++i) {
                        turn<V, IN, true>(A, c, lane + i * G, za[i], zb[i]);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            a[i][j] *= inv;
                            b[i][j] *= inv;
                            da[i][j] = fmaf(za[i][j], a[i][j], da[i][j]);
                            db[i][j] = fmaf(zb[i][j], b[i][j], db[i][j]);
                            za[i][j] *= ga[i][j];
                            zb[i][j] *= gb[i][j];
                            dot = fmaf(za[i][j], a[i][j], fmaf(zb[i][j], b[i][j], dot));
                        }
                    }
                    dot = all(dot) * A.inv_count;
                    T* dx = reinterpret_cast<T*>(S.dx.p) + row_at(S.dx, A, row) + head * S.dx.hs;
#pragma unroll
                    for (int i = 0; i < SL; ++i) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            a[i][j] = inv * fmaf(-a[i][j], dot, za[i][j]);
                            b[i][j] = inv * fmaf(-b[i][j], dot, zb[i][j]);
                        }
                        store(dx, wa[i], a[i]);
                        store(dx, wb[i], b[i]);
                    }
                }
            }
        }
        if constexpr (GRAD) {  // the groups' sums, one group after the other
            if (!S.part) continue;
#pragma unroll 1
            for (int g = 0; g < groups; ++g) {
                __syncthreads();
                if (group == g)
#pragma unroll
                    for (int i = 0; i < SL; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const int ea = wa[i] * V + j, eb = wb[i] * V + j;
                            if (wa[i] < words) sum[ea] = g ? sum[ea] + da[i][j] : da[i][j];
                            if (wb[i] < words) sum[eb] = g ? sum[eb] + db[i][j] : db[i][j];
                        }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < A.dim; i += THREADS) S.part[(long long)blockIdx.x * A.dim + i] = sum[i];
        }
    }
}

// the CTAs' sums of one side's weights: every 32nd by one warp
__global__ void __launch_bounds__(1024) k_qk_norm_sum(const __grid_constant__ NormArgs A, int ctas) {
    __shared__ float s[32][33];
    const Side& S = A.side[blockIdx.y];
    if (!S.part) return;
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < A.dim)
        for (int i = g; i < ctas; i += 32) v += S.part[(long long)i * A.dim + c];
    s[g][lane] = v;
    __syncthreads();
    v = s[lane][g];  // warp g: column g of this tile
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (lane == 0 && blockIdx.x * 32 + g < A.dim) S.dw[blockIdx.x * 32 + g] = v;
}

void check_desc(const snn_qk* d) {
    SNN_REQUIRE(d, SNN_ERR_ARG, "qk_norm: null description");
    SNN_REQUIRE(snnb::elem_type_ok(d->type), SNN_ERR_ARG, "qk_norm: type must be SNN_F32, SNN_BF16 or SNN_F16");
    SNN_REQUIRE((d->flags & ~(SNN_QK_UNIT | SNN_QK_ADJACENT)) == 0, SNN_ERR_ARG, "qk_norm: unknown flags");
    SNN_REQUIRE(d->n_seq >= 0 && d->n_steps >= 0 && d->n_seq <= (1ll << 30) && d->n_steps <= (1ll << 30) &&
                    d->n_seq * d->n_steps <= (1ll << 32),
                SNN_ERR_ARG, "qk_norm: n_seq and n_steps must lie in [0, 2^30], their product in [0, 2^32]");
    SNN_REQUIRE(d->dim >= 1 && d->dim <= MAX_DIM, SNN_ERR_ARG, "qk_norm: dim must lie in [1, 512]");
    SNN_REQUIRE(d->rot >= 0 && d->rot <= d->dim && d->rot % 2 == 0, SNN_ERR_ARG,
                "qk_norm: rot must be even and lie in [0, dim]");
    SNN_REQUIRE(d->q_heads >= 0 && d->k_heads >= 0 && d->q_heads <= 65536 && d->k_heads <= 65536, SNN_ERR_ARG,
                "qk_norm: heads must lie in [0, 65536]");
    SNN_REQUIRE(d->eps >= 0.0f, SNN_ERR_ARG, "qk_norm: eps must not be negative");
    SNN_REQUIRE(d->rot == 0 || d->pos_type == SNN_I32 || d->pos_type == SNN_I64, SNN_ERR_ARG,
                "qk_norm: positions must be SNN_I32 or SNN_I64");
}
int64_t rows_of(const snn_qk* d) { return d->n_seq * d->n_steps; }

Heads heads_of(const snn_qk* d, const snn_heads* h, int64_t heads, const char* name, bool written) {
    const int size = snnb::elem_size(d->type);
    SNN_REQUIRE(h && h->data, SNN_ERR_ARG, std::string("qk_norm: null ") + name);
    SNN_REQUIRE((uintptr_t)h->data % size == 0, SNN_ERR_ARG, std::string("qk_norm: misaligned ") + name);
    const int64_t ss = d->n_seq > 1 ? h->seq_stride : 0, st = d->n_steps > 1 ? h->step_stride : 0;
    const int64_t hs = heads > 1 ? h->head_stride : 0, most = 1ll << 46;
    SNN_REQUIRE(ss >= 0 && st >= 0 && hs >= 0 && ss <= most / std::max<int64_t>(d->n_seq, 1) &&
                    st <= most / std::max<int64_t>(d->n_steps, 1) && hs <= most / std::max<int64_t>(heads, 1),
                SNN_ERR_ARG, std::string("qk_norm: bad strides of ") + name);
    if (written)
        SNN_REQUIRE(snnb::apart({{d->n_seq, ss}, {d->n_steps, st}, {heads, hs}}, d->dim), SNN_ERR_ARG,
                    std::string("qk_norm: rows overlap in ") + name);
    return {h->data, ss, st, hs};
}

struct Plan {
    int per_tile, ctas;
};
// Rows of a tile: up to 8, as far as that leaves eight CTAs an SM.  With gradients of
// weights each CTA leaves a row of sums, so they are at most four an SM.
Plan plan_of(const snn_qk* d, bool grad) {
    Plan p;
    const int64_t n = rows_of(d);
    p.per_tile = (int)std::min<int64_t>(MAX_ROWS, std::max<int64_t>(1, n / (8 * SMS)));
    const int64_t tiles = (n + p.per_tile - 1) / p.per_tile;
    p.ctas = (int)std::min<int64_t>(tiles, grad ? 4 * SMS : 64 * SMS);
    return p;
}

template <typename T, int V, int SL, bool IN, bool GRAD>
void launch(const NormArgs& A, int ctas, int G, cudaStream_t st) {
    k_qk_norm<T, V, SL, IN, GRAD><<<ctas, THREADS, (size_t)A.per_tile * (A.rot / 2) * 8, st>>>(A, G);
    SNN_CUDA(cudaGetLastError());
}
template <typename T, int V, bool GRAD>
void by_slots(const NormArgs& A, int ctas, cudaStream_t st) {
    const int words = A.dim / V, slots = (words + 1) / 2;
    int G = 1;
    while (G < 32 && G < slots) G *= 2;
    const int per = (slots + G - 1) / G;
    const bool in = V > 1 && A.adjacent;
    constexpr int MOST = MAX_DIM / V / 64;  // slots a lane may have
    if constexpr (MOST >= 2)
        if (per > 1) {
            if (in) launch<T, V, MOST, V != 1, GRAD>(A, ctas, G, st);
            else launch<T, V, MOST, false, GRAD>(A, ctas, G, st);
            return;
        }
    if (in) launch<T, V, 1, V != 1, GRAD>(A, ctas, G, st);
    else launch<T, V, 1, false, GRAD>(A, ctas, G, st);
}

template <bool GRAD>
void run(const snn_qk* d, NormArgs& A, cudaStream_t st) {
    const Plan p = plan_of(d, GRAD);
    A.per_tile = p.per_tile;
    const int size = snnb::elem_size(d->type);
    // The widest word that rows, heads and (pairs of halves) the halves consist of
    auto fits = [&](int v) {
        if (d->dim % v || (!A.adjacent && A.rot % (2 * v))) return false;
        for (const Side& S : A.side)
            for (const Heads& h : {S.x, S.y, S.dx})
                if (h.p && ((uintptr_t)h.p % (v * size) || h.ss % v || h.st % v || h.hs % v)) return false;
        return true;
    };
    snnb::with_elem(d->type, [&](auto t) {
        using T = decltype(t);
        constexpr int W = 16 / (int)sizeof(T);
        if (fits(W)) by_slots<T, W, GRAD>(A, p.ctas, st);
        else if (sizeof(T) == 2 && fits(4)) by_slots<T, 4, GRAD>(A, p.ctas, st);
        else if (fits(2)) by_slots<T, 2, GRAD>(A, p.ctas, st);
        else by_slots<T, 1, GRAD>(A, p.ctas, st);
    });
}

NormArgs base_args(const snn_qk* d, const void* positions, const float* freqs) {
    NormArgs A;
    memset(&A, 0, sizeof(A));
    A.rows = rows_of(d);
    A.steps = std::max<int64_t>(1, d->n_steps);
    A.dim = (int)d->dim;
    A.rot = (int)d->rot;
    A.adjacent = (d->flags & SNN_QK_ADJACENT) != 0;
    A.eps = d->eps;
    A.inv_count = d->flags & SNN_QK_UNIT ? 1.0f : 1.0f / (float)d->dim;
    if (d->rot && A.rows) {
        A.pos64 = d->pos_type == SNN_I64;
        SNN_REQUIRE(positions && (uintptr_t)positions % (A.pos64 ? 8 : 4) == 0, SNN_ERR_ARG,
                    "qk_norm: null or misaligned positions");
        SNN_REQUIRE(freqs && (uintptr_t)freqs % 4 == 0, SNN_ERR_ARG, "qk_norm: null or misaligned freqs");
        A.pos = positions;
        A.freqs = freqs;
    }
    return A;
}
void check_weight(const void* w) {
    SNN_REQUIRE((uintptr_t)w % 4 == 0, SNN_ERR_ARG, "qk_norm: misaligned weights");
}

}  // namespace

namespace snnb {

void qk_norm(const snn_qk* d, const snn_heads* q, const snn_heads* k, const float* wq, const float* wk,
             const void* positions, const float* freqs, const snn_heads* yq, const snn_heads* yk, cudaStream_t st) {
    check_desc(d);
    NormArgs A = base_args(d, positions, freqs);
    if (A.rows == 0) return;
    const snn_heads *x[2] = {q, k}, *y[2] = {yq, yk};
    const int64_t heads[2] = {d->q_heads, d->k_heads};
    const float* w[2] = {wq, wk};
    for (int i = 0; i < 2; ++i) {
        if (heads[i] == 0) continue;
        check_weight(w[i]);
        Side& S = A.side[i];
        S.x = heads_of(d, x[i], heads[i], i ? "k" : "q", false);
        S.y = heads_of(d, y[i], heads[i], i ? "yk" : "yq", true);
        S.w = w[i];
        S.heads = (int)heads[i];
    }
    if (d->q_heads + d->k_heads) run<false>(d, A, st);
}

int64_t qk_norm_grad_workspace(const snn_qk* d) {
    check_desc(d);
    return (int64_t)plan_of(d, true).ctas * 2 * d->dim * 4;
}

void qk_norm_grad(const snn_qk* d, const snn_heads* q, const snn_heads* k, const float* wq, const float* wk,
                  const void* positions, const float* freqs, const snn_heads* dyq, const snn_heads* dyk,
                  const snn_heads* dq, const snn_heads* dk, float* dwq, float* dwk, void* work, int64_t work_bytes,
                  cudaStream_t st) {
    check_desc(d);
    NormArgs A = base_args(d, positions, freqs);
    const snn_heads *x[2] = {q, k}, *y[2] = {dyq, dyk}, *dx[2] = {dq, dk};
    const int64_t heads[2] = {d->q_heads, d->k_heads};
    const float* w[2] = {wq, wk};
    float* dw[2] = {dwq, dwk};
    bool sums = false;
    for (int i = 0; i < 2; ++i) {
        check_weight(w[i]);
        check_weight(dw[i]);
        if (dw[i] && (A.rows == 0 || heads[i] == 0)) SNN_CUDA(cudaMemsetAsync(dw[i], 0, (size_t)d->dim * 4, st));
        if (A.rows == 0 || heads[i] == 0) continue;
        Side& S = A.side[i];
        S.x = heads_of(d, x[i], heads[i], i ? "k" : "q", false);
        S.y = heads_of(d, y[i], heads[i], i ? "dyk" : "dyq", false);
        S.dx = heads_of(d, dx[i], heads[i], i ? "dk" : "dq", true);
        S.w = w[i];
        S.heads = (int)heads[i];
        S.dw = dw[i];
        if (dw[i]) {
            const int64_t need = qk_norm_grad_workspace(d);
            SNN_REQUIRE(work && (uintptr_t)work % 256 == 0 && work_bytes >= need, SNN_ERR_ARG,
                        "qk_norm: workspace null, misaligned or too small");
            S.part = (float*)work + (i ? (int64_t)plan_of(d, true).ctas * d->dim : 0);
            sums = true;
        }
    }
    if (!A.side[0].x.p && !A.side[1].x.p) return;
    run<true>(d, A, st);
    if (sums) {
        k_qk_norm_sum<<<dim3((unsigned)((d->dim + 31) / 32), 2), 1024, 0, st>>>(A, plan_of(d, true).ctas);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
