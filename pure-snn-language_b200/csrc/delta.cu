// delta.cu - the delta-rule scan (snn_delta_scan): arguments, the choice of kernels,
// and the kernel for single steps.
#include "delta_tile.h"

namespace snnb_delta {
template <> DeltaSizes delta_sizes<float>();
template <> DeltaSizes delta_sizes<__nv_bfloat16>();
template <> DeltaSizes delta_sizes<__half>();
template <> void launch_prep<float>(const DeltaArgs&, cudaStream_t);
template <> void launch_prep<__nv_bfloat16>(const DeltaArgs&, cudaStream_t);
template <> void launch_prep<__half>(const DeltaArgs&, cudaStream_t);
template <> void launch_scan<float>(const DeltaArgs&, int, cudaStream_t);
template <> void launch_scan<__nv_bfloat16>(const DeltaArgs&, int, cudaStream_t);
template <> void launch_scan<__half>(const DeltaArgs&, int, cudaStream_t);
template <> void launch_grads<float>(const DeltaArgs&, int, cudaStream_t);
template <> void launch_grads<__nv_bfloat16>(const DeltaArgs&, int, cudaStream_t);
template <> void launch_grads<__half>(const DeltaArgs&, int, cudaStream_t);
}  // namespace snnb_delta

namespace {
using namespace snnb_delta;
constexpr int MAX_K = 128;

// ---- few steps: the recurrence itself ------------------------------------------------
// A CTA takes 32 V columns of a head's state, a warp every sixteenth row of it, in registers
// from the first step to the last.  Bound by the state's way from memory and back: 16
// warps of 64 registers, two CTAs an SM, have 128 kB of it in flight (64 streams x 8 heads
// x 128 x 128 bf16: kernel with 8 warps of 215 registers 22.8 us, this one 18, of 10.4 at the copy rate).
constexpr int STEP_WARPS = 16;
template <typename T, int V>
__global__ void __launch_bounds__(32 * STEP_WARPS, 2) k_delta_steps(const __grid_constant__ DeltaArgs A) {
    constexpr int R = MAX_K / STEP_WARPS;  // rows of a warp
    __shared__ float factor[3];  // what a decay takes off, what it leaves, the rate
    __shared__ __align__(16) float key[MAX_K], query[MAX_K], part[STEP_WARPS][2][32 * V];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int head = blockIdx.y, col = ((int)blockIdx.z * 32 + lane) * V, kh = head / A.group;
    const bool on = col < A.vdim;
    struct alignas(4 * V) F {
        float v[V];
    };
    for (long long s = blockIdx.x; s < A.n_seq; s += gridDim.x) {
        const Span sp = span_of(A, s);
        const long long at = (s * A.heads + head) * (long long)A.kdim * A.vdim + col;
        F S[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int d = i * STEP_WARPS + warp;
            if (A.h0 && on && d < A.kdim) S[i] = *reinterpret_cast<const F*>(A.h0 + at + (long long)d * A.vdim);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) S[i].v[j] = 0.0f;
        }
        for (int t = 0; t < sp.len; ++t) {
            if (tid < MAX_K) {
                key[tid] = tid < A.kdim ? to_f32(((const T*)A.k.p)[row_at(A, A.k, s, sp, t) + kh * A.k.hs + tid]) : 0.0f;
            } else if (tid < 2 * MAX_K) {
                const int d = tid - MAX_K;
                query[d] = d < A.kdim ? to_f32(((const T*)A.q.p)[row_at(A, A.q, s, sp, t) + kh * A.q.hs + d]) : 0.0f;
            }
            if (tid == 2 * MAX_K) {
                const float l = log_decay(A, ((const T*)A.gate.p)[row_at(A, A.gate, s, sp, t) + head * A.gate.hs]);
                factor[0] = -expm1f(l);  // 1 - a keeps its bits where a is near 1
                factor[1] = expf(l);
                factor[2] = rate_of(A, ((const T*)A.beta.p)[row_at(A, A.beta, s, sp, t) + head * A.beta.hs]);
            }
            struct alignas(sizeof(T) * V) E {
                T v[V];
            } vt;
            const T* vp = (const T*)A.v.p + row_at(A, A.v, s, sp, t) + head * A.v.hs + col;
            if (on && A.v.word >= (int)sizeof(E)) {
                vt = *reinterpret_cast<const E*>(vp);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) vt.v[j] = on ? vp[j] : from_f32<T>(0.0f);
            }
            __syncthreads();
            const float lost = factor[0], kept = factor[1], rate = factor[2];
            const bool little = lost < 0.5f;
            float k[R], dk[V] = {}, dq[V] = {}, kq = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                k[i] = key[i * STEP_WARPS + warp];
                const float q = query[i * STEP_WARPS + warp];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    S[i].v[j] = little ? fmaf(-lost, S[i].v[j], S[i].v[j]) : kept * S[i].v[j];
                    dk[j] = fmaf(k[i], S[i].v[j], dk[j]);
                    dq[j] = fmaf(q, S[i].v[j], dq[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < MAX_K / 32; ++i) kq = fmaf(key[i * 32 + lane], query[i * 32 + lane], kq);
#pragma unroll
            for (int o = 16; o; o >>= 1) kq += __shfl_xor_sync(~0u, kq, o);
            F pk, pq;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                pk.v[j] = dk[j];
                pq.v[j] = dq[j];
            }
            *reinterpret_cast<F*>(&part[warp][0][lane * V]) = pk;
            *reinterpret_cast<F*>(&part[warp][1][lane * V]) = pq;
            __syncthreads();
            float sk[V] = {}, sq[V] = {};
#pragma unroll
            for (int w = 0; w < STEP_WARPS; ++w) {
                const F f = *reinterpret_cast<const F*>(&part[w][0][lane * V]);
#pragma unroll
                for (int j = 0; j < V; ++j) sk[j] += f.v[j];
            }
            if (warp == 0)  // this one answers
#pragma unroll
                for (int w = 0; w < STEP_WARPS; ++w) {
                    const F f = *reinterpret_cast<const F*>(&part[w][1][lane * V]);
#pragma unroll
                    for (int j = 0; j < V; ++j) sq[j] += f.v[j];
                }
            E yt;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = rate * (to_f32(vt.v[j]) - sk[j]);
#pragma unroll
                for (int i = 0; i < R; ++i) S[i].v[j] = fmaf(k[i], u, S[i].v[j]);
                yt.v[j] = from_f32<T>(A.scale * fmaf(kq, u, sq[j]));
            }
            if (warp == 0 && on) {
                T* yp = (T*)A.y.p + row_at(A, A.y, s, sp, t) + head * A.y.hs + col;
                if (A.y.word >= (int)sizeof(E)) {
                    *reinterpret_cast<E*>(yp) = yt;
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) yp[j] = yt.v[j];
                }
            }
        }
        if (A.h && on)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i * STEP_WARPS + warp < A.kdim) *reinterpret_cast<F*>(A.h + at + (long long)(i * STEP_WARPS + warp) * A.vdim) = S[i];
    }
    if (A.zero) zero_rest<T>(A, A.y, A.heads, A.vdim, ((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x,
                             (long long)gridDim.x * gridDim.y * gridDim.z);
}

// Where the segments start from: starts[g + 1], which holds what segment g makes of nothing, gains its
// steps' product times starts[g], one segment after the other.  A CTA takes 16 columns of a
// head, in shared memory from one segment to the next; the next product is on its way
// meanwhile.  A thread has 8 columns of a row.  (6 products of 16 heads of 128 x 128: kernel 40 us.)
constexpr int JOIN_COLS = 16, JOIN_ROW = MAX_K + 4, JOIN_SMEM = (2 * MAX_K * JOIN_ROW + MAX_K * JOIN_COLS) * 4;
__global__ void __launch_bounds__(256) k_delta_join(const __grid_constant__ DeltaArgs A) {
    extern __shared__ __align__(16) float join[];  // two products [MAX_K][JOIN_ROW], a state [MAX_K][JOIN_COLS]
    float* S = join + 2 * MAX_K * JOIN_ROW;
    const int tid = threadIdx.x, head = blockIdx.y, c0 = (int)blockIdx.z * JOIN_COLS;
    const int d = tid >> 1, c = (tid & 1) * 8, kdim = A.kdim, kpad = (kdim + 3) / 4 * 4;
    const long long s = blockIdx.x, size = (long long)kdim * A.vdim;
    const Span sp = span_of(A, s);
    const long long first = item_at(A, s, sp);
    const int all = (sp.len + C - 1) / C, last = (all + A.seg - 1) / A.seg - 1;
    auto unit = [&](int g) { return (first + g) * A.heads + head; };
    auto load = [&](int g) {
        const float* M = A.maps + unit(g) * kdim * kdim;
        float* to = join + (g & 1) * MAX_K * JOIN_ROW;
        if (kdim == kpad) {
            for (int i = tid; i < kdim * (kdim / 4); i += 256) {
                const int r = i / (kdim / 4), k = i % (kdim / 4) * 4;
                copy16(to + r * JOIN_ROW + k, M + r * kdim + k, true);
            }
        } else {
            for (int i = tid; i < kdim * kpad; i += 256) {
                const int r = i / kpad, k = i % kpad;
                to[r * JOIN_ROW + k] = k < kdim ? M[r * kdim + k] : 0.0f;
            }
        }
        copies_end();
    };
    if (last < 2) return;
    load(1);
    for (int i = tid; i < MAX_K * JOIN_COLS; i += 256) {
        const int r = i / JOIN_COLS, cc = c0 + i % JOIN_COLS;
        S[i] = r < kdim && cc < A.vdim ? A.starts[unit(1) * size + (long long)r * A.vdim + cc] : 0.0f;
    }
    for (int g = 1; g < last; ++g) {
        if (g + 1 < last) load(g + 1);
        else copies_end();
        float* to = A.starts + unit(g + 1) * size + (long long)d * A.vdim + c0 + c;
        float sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = d < kdim && c0 + c + j < A.vdim ? to[j] : 0.0f;
        copies_wait<1>();
        __syncthreads();
        const float* M = join + (g & 1) * MAX_K * JOIN_ROW + d * JOIN_ROW;
        if (d < kdim)
#pragma unroll 2
            for (int k = 0; k < kpad; k += 4) {
                const float4 m = *reinterpret_cast<const float4*>(M + k);
                const float mk[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(S + (k + e) * JOIN_COLS + c + j);
                        sum[j] = fmaf(mk[e], v.x, sum[j]);
                        sum[j + 1] = fmaf(mk[e], v.y, sum[j + 1]);
                        sum[j + 2] = fmaf(mk[e], v.z, sum[j + 2]);
                        sum[j + 3] = fmaf(mk[e], v.w, sum[j + 3]);
                    }
            }
        __syncthreads();  // S and the product are no longer read
        if (d < kdim)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                S[d * JOIN_COLS + c + j] = sum[j];
                if (c0 + c + j < A.vdim) to[j] = sum[j];
            }
    }
    copies_wait<0>();
}

// the rows of no sequence where there is no sequence at all
template <typename T>
__global__ void __launch_bounds__(256) k_delta_zero(const __grid_constant__ DeltaArgs A, Heads r, int heads, int width) {
    zero_rest<T>(A, r, heads, width, blockIdx.x, gridDim.x);
}

void check_desc(const snn_delta* d) {
    SNN_REQUIRE(d, SNN_ERR_ARG, "delta: null description");
    SNN_REQUIRE(snnb::elem_type_ok(d->type), SNN_ERR_ARG, "delta: type must be SNN_F32, SNN_BF16 or SNN_F16");
    SNN_REQUIRE((d->flags & ~(SNN_SCAN_LOGIT | SNN_SCAN_ZERO)) == 0, SNN_ERR_ARG, "delta: unknown flags");
    SNN_REQUIRE(d->n_seq >= 0 && d->n_seq <= (1ll << 30), SNN_ERR_ARG, "delta: n_seq must lie in [0, 2^30]");
    SNN_REQUIRE(d->n_steps >= 0 && d->n_steps <= (1ll << 30), SNN_ERR_ARG, "delta: n_steps must lie in [0, 2^30]");
    SNN_REQUIRE(d->k_heads >= 1 && d->heads >= d->k_heads && d->heads <= 65535 && d->heads % d->k_heads == 0, SNN_ERR_ARG,
                "delta: heads must be a multiple of k_heads, at most 65535");
    SNN_REQUIRE(d->k_dim >= 1 && d->k_dim <= MAX_K, SNN_ERR_ARG, "delta: k_dim must lie in [1, 128]");
    SNN_REQUIRE(d->v_dim >= 1 && d->v_dim <= 1024, SNN_ERR_ARG, "delta: v_dim must lie in [1, 1024]");
    const int64_t slots = d->offsets ? d->n_steps / C + d->n_seq : d->n_seq * ((d->n_steps + C - 1) / C);
    SNN_REQUIRE(slots < (1ll << 31) && (slots + d->n_seq) <= (1ll << 46) / (d->heads * d->v_dim * 128 * 4), SNN_ERR_ARG,
                "delta: more than 2^46 bytes of states");
}
int64_t slots_of(const snn_delta* d) {
    return d->offsets ? d->n_steps / C + d->n_seq : d->n_seq * ((d->n_steps + C - 1) / C);
}
int64_t mean_steps(const snn_delta* d) { return d->offsets ? d->n_steps / std::max<int64_t>(d->n_seq, 1) : d->n_steps; }

Heads heads_of(const snn_delta* d, const snn_heads* h, int64_t heads, int64_t width, const char* name, bool written = false) {
    const int size = snnb::elem_size(d->type);
    const bool rows = d->n_steps > 0 && (d->offsets || d->n_seq > 0);
    SNN_REQUIRE(h && (h->data || !rows), SNN_ERR_ARG, std::string("delta: null ") + name);
    SNN_REQUIRE((uintptr_t)h->data % size == 0, SNN_ERR_ARG, std::string("delta: misaligned ") + name);
    const int64_t seqs = d->offsets ? 1 : d->n_seq, most = 1ll << 46;
    const int64_t ss = seqs > 1 ? h->seq_stride : 0, st = d->n_steps > 1 ? h->step_stride : 0, hs = heads > 1 ? h->head_stride : 0;
    SNN_REQUIRE(ss >= 0 && st >= 0 && hs >= 0 && ss <= most / std::max<int64_t>(seqs, 1) &&
                    st <= most / std::max<int64_t>(d->n_steps, 1) && hs <= most / heads,
                SNN_ERR_ARG, std::string("delta: bad strides of ") + name);
    if (written)
        SNN_REQUIRE(snnb::apart({{seqs, ss}, {d->n_steps, st}, {heads, hs}}, width), SNN_ERR_ARG,
                    std::string("delta: rows overlap in ") + name);
    int word = 16;  // bytes
    while (word > size && ((uintptr_t)h->data % word || ss * size % word || st * size % word || hs * size % word || width * size % word))
        word /= 2;
    return {h->data, ss, st, hs, word};
}
// a gate's or rate's rows: a head beside the other
Heads gates_of(const snn_delta* d, const snn_rows* r, const char* name, bool written = false) {
    SNN_REQUIRE(r, SNN_ERR_ARG, std::string("delta: null ") + name);
    const snn_heads h = {r->data, r->seq_stride, r->step_stride, 1};
    Heads o = heads_of(d, &h, d->heads, 1, name, written);
    o.hs = 1;
    return o;
}
void check_states(std::initializer_list<const void*> p) {
    for (const void* q : p) SNN_REQUIRE((uintptr_t)q % 4 == 0, SNN_ERR_ARG, "delta: misaligned states");
}

DeltaSizes sizes_of(const snn_delta* d) {
    DeltaSizes z{};
    snnb::with_elem(d->type, [&](auto t) { z = delta_sizes<decltype(t)>(); });
    return z;
}
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t vpad_of(const snn_delta* d) { return (d->v_dim + 7) / 8 * 8; }
// T and P, keys, factors, then (kept for the gradient) states and U
struct Layout {
    int64_t keys, factors, states, u, all, kept_all;
    int64_t starts, maps, cut;  // of a workspace for segments: their offsets in it, its size
};
// Chunks of a segment (0: sequences stay whole) and how many segments there are (packed: at most).  Few heads leave
// most SMs empty for long: then sequences are cut, a first run makes what each segment makes of no
// state and the product of its steps (twice the columns, no results), those are joined, and all segments
// run at once.  That is 2.7 times the work (about), so it takes four segments and more, as many as
// give every SM eight warps; a segment has at least 8 chunks.  1 x 16,384 steps x 16 heads of 128 x 128 f16: whole
// 1,300 us, by 8 segments 630 for both runs, 40 to join.  Packed sequences may be of any lengths: segments are of the mean's
// size, and numbered as their chunks are, by their rows' place.
struct Cut {
    int seg;
    int64_t items;
};
Cut segments_of(const snn_delta* d) {
    const int64_t chunks = (mean_steps(d) + C - 1) / C, warps = d->n_seq * d->heads * ((d->v_dim + 15) / 16);
    int64_t g = 1;
    while (g < 16 && warps * g * 2 <= 8 * SMS && chunks >= 16 * g) g *= 2;
    if (g < 4 || d->n_seq > 64) return {0, d->n_seq};
    const int64_t seg = (chunks + g - 1) / g;
    return {(int)seg, d->offsets ? d->n_steps / (seg * C) + d->n_seq : d->n_seq * ((chunks + seg - 1) / seg)};
}
Layout layout_of(const snn_delta* d) {
    const DeltaSizes z = sizes_of(d);
    const int64_t units = slots_of(d) * d->heads, kd = d->k_dim <= 64 ? 64 : 128;
    Layout l;
    l.keys = round256(units * z.squares);
    l.factors = l.keys + round256(slots_of(d) * d->k_heads * 2 * C * (kd + PAD) * z.key);
    l.all = l.states = l.factors + round256(units * SC * 4);
    l.u = l.states + round256(units * d->v_dim * (kd + PAD) * z.kept);
    l.kept_all = l.u + round256(units * z.planes * C * vpad_of(d) * z.kept);
    const Cut cut = segments_of(d);
    l.starts = 0;
    l.maps = cut.seg ? round256(cut.items * d->heads * d->k_dim * d->v_dim * 4) : 0;
    l.cut = cut.seg ? l.maps + round256(cut.items * d->heads * d->k_dim * d->k_dim * 4) : 0;
    return l;
}
// Up to 8 steps one by one (64 x 8 heads of 128 x 128 bf16, us by 4 and 8 steps: 32, 55; as a chunk 74).  The
// mean decides for all: packed lengths lie on the device.  A long sequence among single steps is then slow: 63
// of one step and one of 400, 8 heads, 811 us (141 as chunks, 77 as two calls).
bool by_steps(const snn_delta* d) { return mean_steps(d) <= 8; }

DeltaArgs base_args(const snn_delta* d, const snn_heads* q, const snn_heads* k, const snn_heads* v, const snn_rows* gate,
                    const snn_rows* beta) {
    SNN_REQUIRE((uintptr_t)d->offsets % 8 == 0, SNN_ERR_ARG, "delta: misaligned offsets");
    DeltaArgs A;
    memset(&A, 0, sizeof(A));
    A.q = heads_of(d, q, d->k_heads, d->k_dim, "q");
    A.k = heads_of(d, k, d->k_heads, d->k_dim, "k");
    A.v = heads_of(d, v, d->heads, d->v_dim, "v");
    A.gate = gates_of(d, gate, "gate");
    A.beta = gates_of(d, beta, "beta");
    A.off = d->offsets;
    A.n_seq = d->n_seq;
    A.slots = slots_of(d);
    A.n_steps = (int)d->n_steps;
    A.hk = (int)d->k_heads;
    A.heads = (int)d->heads;
    A.group = (int)(d->heads / d->k_heads);
    A.kdim = (int)d->k_dim;
    A.vdim = (int)d->v_dim;
    A.vpad = (int)vpad_of(d);
    A.logit = (d->flags & SNN_SCAN_LOGIT) != 0;
    A.zero = d->offsets && (d->flags & SNN_SCAN_ZERO) != 0;
    A.scale = d->scale;
    A.items = d->n_seq;
    return A;
}
void zero_rows(const snn_delta* d, const DeltaArgs& A, const Heads& r, int heads, int width, cudaStream_t st) {
    if (!A.zero || !r.p || d->n_steps == 0) return;
    snnb::with_elem(d->type, [&](auto t) { k_delta_zero<decltype(t)><<<4 * SMS, 256, 0, st>>>(A, r, heads, width); });
    SNN_CUDA(cudaGetLastError());
}

// Warps of a CTA.  A chunk's K, Q, T and P fill a CTA's shared memory (one CTA an SM), and
// serve its warps, each with 16 columns of the state.  Up to four warps have a tensor core
// each (5.1 us a chunk of 128 x 16, f16); eight share them (7.3), but CTAs that do not fit on
// the SMs at once are a second round.
int warps_of(const snn_delta* d, int64_t items) {
    int best = 1;
    double least = 1e300;
    for (int nw = 1; nw <= 8; nw *= 2) {
        const int64_t ctas = items * d->heads * ((d->v_dim + 16 * nw - 1) / (16 * nw));
        const double cost = (double)((ctas + SMS - 1) / SMS) * (nw == 8 ? 1.45 : 1.0);
        if (nw > 1 && 16 * nw >= 2 * d->v_dim) break;  // no warp without columns where fewer do
        if (cost <= least) {
            least = cost;
            best = nw;
        }
    }
    return best;
}

void check_work(const void* work, int64_t bytes, int64_t needed, const char* name) {
    SNN_REQUIRE(needed == 0 || (work && (uintptr_t)work % 256 == 0 && bytes >= needed), SNN_ERR_ARG,
                std::string("delta: ") + name + " null, misaligned or too small");
}

}  // namespace

namespace snnb {

int64_t delta_scan_saved(const snn_delta* d) {
    check_desc(d);
    return layout_of(d).kept_all;
}
int64_t delta_scan_workspace(const snn_delta* d, bool with_saved) {
    check_desc(d);
    const Layout l = layout_of(d);
    return with_saved ? l.cut : by_steps(d) ? 0 : l.cut + l.all;
}

void delta_scan(const snn_delta* d, const snn_heads* q, const snn_heads* k, const snn_heads* v, const snn_rows* gate,
                const snn_rows* beta, const float* h0, const snn_heads* y, float* h, void* saved, int64_t saved_bytes,
                void* work, int64_t work_bytes, cudaStream_t st) {
    check_desc(d);
    DeltaArgs A = base_args(d, q, k, v, gate, beta);
    A.y = heads_of(d, y, d->heads, d->v_dim, "y", true);
    check_states({h0, h});
    A.h0 = h0;
    A.h = h;
    if (d->n_seq == 0) return zero_rows(d, A, A.y, A.heads, A.vdim, st);
    const Layout l = layout_of(d);
    if (!saved && by_steps(d)) {
        const bool wide = d->v_dim % 4 == 0 && (uintptr_t)h0 % 16 == 0 && (uintptr_t)h % 16 == 0 && d->v_dim > 32;
        with_elem(d->type, [&](auto t) {
            using T = decltype(t);
            const int cols = wide ? 128 : 32;
            const dim3 grid((unsigned)d->n_seq, (unsigned)d->heads, (unsigned)((d->v_dim + cols - 1) / cols));
            if (wide) k_delta_steps<T, 4><<<grid, 32 * STEP_WARPS, 0, st>>>(A);
            else k_delta_steps<T, 1><<<grid, 32 * STEP_WARPS, 0, st>>>(A);
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    // the workspace: what cut sequences want, then, without saved, what it would hold of the chunks
    char* base = (char*)saved;
    if (saved) check_work(saved, saved_bytes, l.kept_all, "saved");
    check_work(work, work_bytes, saved ? l.cut : l.cut + l.all, "workspace");
    if (!saved) base = (char*)work + l.cut;
    A.squares = base;
    A.keys = base + l.keys;
    A.factors = (float*)(base + l.factors);
    if (saved) {
        A.states = base + l.states;
        A.u = base + l.u;
    }
    const Cut cut = segments_of(d);
    A.seg = cut.seg;
    A.items = cut.items;
    A.starts = (float*)work;
    A.maps = (float*)((char*)work + l.maps);
    with_elem(d->type, [&](auto t) {
        using T = decltype(t);
        if (A.slots) launch_prep<T>(A, st);
        if (A.seg) {
            A.only = 1;
            launch_scan<T>(A, 8, st);
            A.only = 0;
            set_smem<k_delta_join>(JOIN_SMEM);
            const dim3 grid((unsigned)d->n_seq, (unsigned)d->heads, (unsigned)((d->v_dim + JOIN_COLS - 1) / JOIN_COLS));
            k_delta_join<<<grid, 256, JOIN_SMEM, st>>>(A);
            SNN_CUDA(cudaGetLastError());
        }
        launch_scan<T>(A, warps_of(d, A.items), st);
    });
}

}  // namespace snnb

namespace snnb {

int64_t delta_scan_grad_workspace(const snn_delta* d) {
    check_desc(d);
    const Layout l = layout_of(d);
    return l.kept_all - l.states;
}

void delta_scan_grad(const snn_delta* d, const snn_heads* q, const snn_heads* k, const snn_heads* v, const snn_rows* gate,
                     const snn_rows* beta, const void* saved, int64_t saved_bytes, const snn_heads* dy, const float* dh,
                     const snn_heads* dq, const snn_heads* dk, const snn_heads* dv, const snn_rows* dgate,
                     const snn_rows* dbeta, float* dh0, void* work, int64_t work_bytes, cudaStream_t st) {
    check_desc(d);
    SNN_REQUIRE(dy || dh || d->n_seq == 0, SNN_ERR_ARG, "delta: neither dy nor dh");
    DeltaArgs A = base_args(d, q, k, v, gate, beta);
    if (dy) A.dy = heads_of(d, dy, d->heads, d->v_dim, "dy");
    else A.dy.word = 16;
    A.dq = heads_of(d, dq, d->k_heads, d->k_dim, "dq", true);
    A.dk = heads_of(d, dk, d->k_heads, d->k_dim, "dk", true);
    A.dv = heads_of(d, dv, d->heads, d->v_dim, "dv", true);
    A.dgate = gates_of(d, dgate, "dgate", true);
    A.dbeta = gates_of(d, dbeta, "dbeta", true);
    check_states({dh, dh0});
    A.dh = dh;
    A.dh0 = dh0;
    const Layout l = layout_of(d);
    if (d->n_seq) {
        check_work(saved, saved_bytes, l.kept_all, "saved");
        check_work(work, work_bytes, l.kept_all - l.states, "workspace");
    }
    zero_rows(d, A, A.dq, A.hk, A.kdim, st);
    zero_rows(d, A, A.dk, A.hk, A.kdim, st);
    zero_rows(d, A, A.dv, A.heads, A.vdim, st);
    zero_rows(d, A, A.dgate, A.heads, 1, st);
    zero_rows(d, A, A.dbeta, A.heads, 1, st);
    if (d->n_seq == 0) return;
    char* base = (char*)saved;
    A.squares = base;
    A.keys = base + l.keys;
    A.factors = (float*)(base + l.factors);
    A.states = base + l.states;
    A.u = base + l.u;
    A.dstates = (char*)work;
    A.dr = (char*)work + (l.u - l.states);
    with_elem(d->type, [&](auto t) { launch_grads<decltype(t)>(A, warps_of(d, d->n_seq), st); });
}

}  // namespace snnb
