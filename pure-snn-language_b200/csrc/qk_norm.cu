// qk_norm.cu - norms of queries and keys for each head with the position
// rotation in the same pass (snn_qk_norm), and their gradients.
//
//   n = x r,  r = 1 / sqrt(sum x^2 / count + eps),  y = turn(n w)
//   z = turn^-1(dy),  dw = sum z n,  dx = r (z w - n sum(z w n) / count)
// Bound by memory: every element is read once and written once.  A group of G
// lanes takes a head, a lane whole words of up to 16 bytes of it such that both
// elements of a rotated pair are its own, so that nothing but the sum of squares
// crosses lanes.  Cosines and sines of a row are made once for all of its heads of both
// sides, in shared memory, where the weights lie too (in registers, both cost two of five
// CTAs an SM, and more time than the reads).  Angles are products in 64 bits (a position
// of 1e5 has an angle whose f32 would be off by 4e-3), reduced to a turn before the f32 sine.
// 65,536 rows x 32 heads of 128 bf16: kernel 221 us, 165 at the copy rate; gradients of 32,768 x 20 x
// 100 f32 215 of 121.
#include <algorithm>
#include "elem.h"

namespace {
using snnb::from_f32;
using snnb::to_f32;
constexpr int SMS = 148, THREADS = 256, MAX_DIM = 512, MAX_ROWS = 16;

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
    int dim, rot, per_tile, places, pos64, adjacent;  // places: of a row's cosines and sines
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
// Cosine and sine of pair j, and weight j, lie at place_of<V>(j): lanes read theirs side by side
template <int V>
__device__ __forceinline__ int place_of(int j, int n) { return j % V * ((n + V - 1) / V) + j / V; }
// The pairs of the two words of slot s turned (BACK: the other way), its pairs being s V .. s V +
// V - 1.  IN: they lie inside a word.
template <int V, bool IN, bool BACK>
__device__ __forceinline__ void turn(int half, const float2* cs, int s, float (&a)[V], float (&b)[V]) {
    if (s * V >= half) return;
    const int step = (half + V - 1) / V;
    auto pair = [&](float& u, float& v, int i) {
        const float2 c = cs[i * step + s];
        const float si = BACK ? -c.y : c.y, x = u, y = v;
        u = fmaf(x, c.x, -(y * si));
        v = fmaf(x, si, y * c.x);
    };
    if constexpr (IN && V > 1) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if (s * V + i < half) pair(a[2 * i], a[2 * i + 1], i);
            if (s * V + i + V / 2 < half) pair(b[2 * i], b[2 * i + 1], i + V / 2);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) pair(a[i], b[i], i);
    }
}
template <typename T, int V>
__device__ __forceinline__ Word<T, V> word_of(const float (&o)[V]) {
    Word<T, V> x;
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(o[i], o[i + 1]);
                x.v[i] = __low2half(h);
                x.v[i + 1] = __high2half(h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(o[i], o[i + 1]);
                x.v[i] = __low2bfloat16(h);
                x.v[i + 1] = __high2bfloat16(h);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(o[i]);
    }
    return x;
}

// V elements a word, SL slots of two words a lane, G lanes a head
// CTAs that an SM has registers for
__host__ __device__ constexpr int resident(int v, int sl, bool grad) { return v * sl > 8 ? 2 : grad ? (v == 8 ? 2 : 3) : 4; }
template <typename T, int V, int SL, bool IN, bool GRAD>
__global__ void __launch_bounds__(THREADS, resident(V, SL, GRAD)) k_qk_norm(const __grid_constant__ NormArgs A, int G) {
    extern __shared__ float2 tables[];  // [2][rows of a tile][places]
    __shared__ float weight[2][MAX_DIM], sum[GRAD ? MAX_DIM : 1];
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
    for (int i = threadIdx.x; i < A.dim; i += THREADS) {
        weight[0][place_of<V>(i, A.dim)] = A.side[0].w ? A.side[0].w[i] : 1.0f;
        weight[1][place_of<V>(i, A.dim)] = A.side[1].w ? A.side[1].w[i] : 1.0f;
    }
    auto load = [&](const T* p, int w, float (&o)[V]) {
        W x = {};
        if (w < words) x = *reinterpret_cast<const W*>(p + w * V);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = to_f32(x.v[i]);
    };
    auto store = [&](T* p, int w, const float (&o)[V]) {
        if (w < words) *reinterpret_cast<W*>(p + w * V) = word_of<T, V>(o);
    };
    // o times the weights of word w
    auto weigh = [&](const float* wt, int w, float (&o)[V]) {
        if (w >= words) return;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] *= wt[i * words + w];
    };
    float da[2][GRAD ? SL : 1][V] = {}, db[2][GRAD ? SL : 1][V] = {};
    const int per_row = groups / A.per_tile, r = group / per_row;  // groups that take a row's heads in turn
    auto heads = [&](auto which_, const float2* c, long long row) {
        constexpr int which = decltype(which_)::value;
        const Side& S = A.side[which];
        int head = group - r * per_row;
        if (head >= S.heads) return;
        const T* x = reinterpret_cast<const T*>(S.x.p) + row_at(S.x, A, row) + head * S.x.hs;
        T* y = reinterpret_cast<T*>(S.y.p) + row_at(S.y, A, row) + head * S.y.hs;
        T* dx = GRAD ? reinterpret_cast<T*>(S.dx.p) + row_at(S.dx, A, row) + head * S.dx.hs : nullptr;
        // (the loop's end is the same for all lanes of a group: they shuffle among themselves)
#pragma unroll 1
        for (; head < S.heads; head += per_row, x += per_row * S.x.hs, y += per_row * S.y.hs, dx += GRAD ? per_row * S.dx.hs : 0) {
            float a[SL][V], b[SL][V];
            [[maybe_unused]] float za[GRAD ? SL : 1][V], zb[GRAD ? SL : 1][V];
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
            const float inv = rsqrtf(fmaf(all(sq), A.inv_count, A.eps));
#pragma unroll
            for (int i = 0; i < SL; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    a[i][j] *= inv;
                    b[i][j] *= inv;
                }
            if constexpr (!GRAD) {
#pragma unroll
                for (int i = 0; i < SL; ++i) {
                    if (S.w) {
                        weigh(weight[which], wa[i], a[i]);
                        weigh(weight[which], wb[i], b[i]);
                    }
                    turn<V, IN, false>(half, c, lane + i * G, a[i], b[i]);
                    store(y, wa[i], a[i]);
                    store(y, wb[i], b[i]);
                }
            } else {
                float dot = 0.0f;
#pragma unroll
                for (int i = 0; i < SL; ++i) {
                    turn<V, IN, true>(half, c, lane + i * G, za[i], zb[i]);
                    if (S.part) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            da[which][i][j] = fmaf(za[i][j], a[i][j], da[which][i][j]);
                            db[which][i][j] = fmaf(zb[i][j], b[i][j], db[which][i][j]);
                        }
                    }
                    if (S.w) {
                        weigh(weight[which], wa[i], za[i]);
                        weigh(weight[which], wb[i], zb[i]);
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) dot = fmaf(za[i][j], a[i][j], fmaf(zb[i][j], b[i][j], dot));
                }
                dot = all(dot) * A.inv_count;
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
    };
    auto table = [&](long long tile, float2* cs) {
        const int n = (int)min((long long)A.per_tile, A.rows - tile);
        for (int i = threadIdx.x; i < n * half; i += THREADS) {
            const int k = i / half;
            const long long at = tile + k;
            const double pos = A.pos64 ? (double)reinterpret_cast<const long long*>(A.pos)[at]
                                       : (double)reinterpret_cast<const int*>(A.pos)[at];
            const double turns = pos * (double)A.freqs[i - k * half] * 0.15915494309189533577;  // 1 / (2 pi)
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            cs[k * A.places + place_of<V>(i - k * half, half)] = make_float2(c, s);
        }
    };
    const long long step = (long long)gridDim.x * A.per_tile;
    long long tile = (long long)blockIdx.x * A.per_tile;
    float2 *now = tables, *next = tables + A.per_tile * A.places;
    if (tile < A.rows) table(tile, now);
#pragma unroll 1
    for (; tile < A.rows; tile += step) {
        __syncthreads();  // this tile's table is there, the other one's is no longer read
        if (tile + step < A.rows) table(tile + step, next);
        if (tile + r < A.rows) {
            heads(std::integral_constant<int, 0>(), now + r * A.places, tile + r);
            heads(std::integral_constant<int, 1>(), now + r * A.places, tile + r);
        }
        float2* t = now;
        now = next;
        next = t;
    }
    if constexpr (GRAD) {  // the groups' sums, one group after the other
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float* part = A.side[which].part;
            if (!part) continue;
#pragma unroll 1
            for (int k = 0; k < groups; ++k) {
                __syncthreads();
                if (group == k)
#pragma unroll
                    for (int i = 0; i < SL; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const int ea = wa[i] * V + j, eb = wb[i] * V + j;
                            if (wa[i] < words) sum[ea] = k ? sum[ea] + da[which][i][j] : da[which][i][j];
                            if (wb[i] < words) sum[eb] = k ? sum[eb] + db[which][i][j] : db[which][i][j];
                        }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < A.dim; i += THREADS) part[(long long)blockIdx.x * A.dim + i] = sum[i];
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
#pragma unroll 8
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

// The widest word that rows, heads and (pairs of halves) the halves consist of
int width_of(const snn_qk* d, const NormArgs& A) {
    const int size = snnb::elem_size(d->type);
    int v = 16 / size;
    auto fits = [&] {
        if (d->dim % v || (!A.adjacent && A.rot % (2 * v))) return false;
        for (const Side& S : A.side)
            for (const Heads& h : {S.x, S.y, S.dx})
                if (h.p && ((uintptr_t)h.p % (v * size) || h.ss % v || h.st % v || h.hs % v)) return false;
        return true;
    };
    while (v > 1 && !fits()) v /= 2;
    return v;
}
int lanes_of(const snn_qk* d, int v) {  // of a head
    const int slots = ((int)d->dim / v + 1) / 2;
    int G = 1;
    while (G < 32 && G < slots) G *= 2;
    return G;
}
// Rows of a tile: a power of two up to 16 and the groups of a CTA, as far as that leaves eight CTAs an SM.
int rows_of_tile(const snn_qk* d, int v) {
    int r = 1;
    while (r < MAX_ROWS && r < THREADS / lanes_of(d, v) && rows_of(d) >= 2ll * r * 8 * SMS) r *= 2;
    return r;
}
// CTAs of a gradient at most: each leaves a row of sums
int most_ctas(const snn_qk* d) { return (int)std::min<int64_t>(std::max<int64_t>(1, rows_of(d)), 3 * SMS); }

template <typename T, int V, int SL, bool IN, bool GRAD>
int launch(const NormArgs& A, int tiles, int G, cudaStream_t st) {
    // with sums of weights' gradients, and where it fills the SMs, one round of CTAs
    const int ctas = std::min(tiles, (GRAD ? 1 : 4) * resident(V, SL, GRAD) * SMS);
    auto* kernel = k_qk_norm<T, V, SL, IN, GRAD>;
    const size_t smem = (size_t)2 * A.per_tile * A.places * 8;
    if (smem > 40 * 1024) SNN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<ctas, THREADS, smem, st>>>(A, G);
    SNN_CUDA(cudaGetLastError());
    return ctas;
}
// the number of CTAs
template <bool GRAD>
int run(const snn_qk* d, NormArgs& A, cudaStream_t st) {
    const int v = width_of(d, A), G = lanes_of(d, v), slots = ((int)d->dim / v + 1) / 2;
    A.per_tile = rows_of_tile(d, v);
    A.places = (A.rot / 2 + v - 1) / v * v;
    const int tiles = (int)std::min<int64_t>(1 << 30, (rows_of(d) + A.per_tile - 1) / A.per_tile);
    int ctas = 0;
    auto by_slots = [&](auto t, auto vv) {
        using T = decltype(t);
        constexpr int V = decltype(vv)::value, MOST = MAX_DIM / V / 64;  // slots that a lane may have
        const bool in = V > 1 && A.adjacent;
        if constexpr (MOST >= 2)
            if (slots > G) {
                if (in) ctas = launch<T, V, MOST, V != 1, GRAD>(A, tiles, G, st);
                else ctas = launch<T, V, MOST, false, GRAD>(A, tiles, G, st);
                return;
            }
        if (in) ctas = launch<T, V, 1, V != 1, GRAD>(A, tiles, G, st);
        else ctas = launch<T, V, 1, false, GRAD>(A, tiles, G, st);
    };
    snnb::with_elem(d->type, [&](auto t) {
        constexpr int W = 16 / (int)sizeof(t);
        if (v == W) by_slots(t, std::integral_constant<int, W>());
        else if (v == 4) by_slots(t, std::integral_constant<int, 4>());
        else if (v == 2) by_slots(t, std::integral_constant<int, 2>());
        else by_slots(t, std::integral_constant<int, 1>());
    });
    return ctas;
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
    return (int64_t)most_ctas(d) * 2 * d->dim * 4;
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
            S.part = (float*)work + (i ? (int64_t)most_ctas(d) * d->dim : 0);
            sums = true;
        }
    }
    for (int i = 0; i < 2; ++i)  // (all has been looked at)
        if (dw[i] && !A.side[i].x.p) SNN_CUDA(cudaMemsetAsync(dw[i], 0, (size_t)d->dim * 4, st));
    if (!A.side[0].x.p && !A.side[1].x.p) return;
    const int ctas = run<true>(d, A, st);
    if (sums) {
        k_qk_norm_sum<<<dim3((unsigned)((d->dim + 31) / 32), 2), 1024, 0, st>>>(A, ctas);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
