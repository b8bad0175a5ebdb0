// embed.cu - token drive: rows of a table picked by a token stream
// (snn_embed), and the table's gradient by sorted tokens (snn_embed_grad).
#include <algorithm>
#include "elem.h"

namespace {
using snnb::from_f32;
using snnb::to_f32;

// V elements that are loaded and stored as one word of at most 16 bytes
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};

template <typename TOK>
__device__ __forceinline__ unsigned token_at(const TOK* tok, long long i, unsigned vocab) {
    // outside [0, vocab): `vocab`
    const long long t = (long long)tok[i];
    return (unsigned long long)t < vocab ? (unsigned)t : vocab;
}

// ---- out[i] = scale * table[tok[i]] -----------------------------------------
// A warp per segment of SEG vectors of a row.
constexpr int E_THREADS = 256;
constexpr int E_UNROLL = 4;
template <typename TOK, typename TT, typename OT, int V>
__global__ void __launch_bounds__(E_THREADS) k_embed(const TOK* tok, long long n, const TT* table, unsigned vocab,
                                                     int dv, long long tstride, float scale, OT* out,
                                                     long long ostride, int segs) {
    const int lane = threadIdx.x & 31;
    const long long nw = (long long)gridDim.x * (E_THREADS / 32);
    for (long long w = (long long)blockIdx.x * (E_THREADS / 32) + (threadIdx.x >> 5); w < n * segs; w += nw) {
        const long long i = w / segs;
        const int c0 = (int)(w - i * segs) * (32 * E_UNROLL) + lane;
        const unsigned t = token_at(tok, i, vocab);
        const Pack<TT, V>* src = reinterpret_cast<const Pack<TT, V>*>(table + (long long)t * tstride);
        Pack<OT, V>* dst = reinterpret_cast<Pack<OT, V>*>(out + i * ostride);
        Pack<TT, V> in[E_UNROLL];
#pragma unroll
        for (int u = 0; u < E_UNROLL; ++u)
            if (t < vocab && c0 + u * 32 < dv) in[u] = src[c0 + u * 32];
#pragma unroll
        for (int u = 0; u < E_UNROLL; ++u) {
            if (c0 + u * 32 >= dv) continue;
            Pack<OT, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = from_f32<OT>(t < vocab ? scale * to_f32(in[u].v[k]) : 0.0f);
            dst[c0 + u * 32] = o;
        }
    }
}

// ---- the positions sorted by token -------------------------------------------
// Least significant digit first, 8 bits a pass; each pass counts the digits of
// every tile, sums them in (digit, tile) order and scatters in input order, so
// positions of one token stay in ascending order.
constexpr int S_THREADS = 256;
constexpr int S_PER = 8;
constexpr int S_TILE = S_THREADS * S_PER;
constexpr int S_BINS = 256;

struct Pair {
    unsigned key, pos;
};

template <typename TOK>
struct FromTokens {
    const TOK* tok;
    unsigned vocab;
    __device__ Pair operator()(long long i) const { return {token_at(tok, i, vocab), (unsigned)i}; }
};
struct FromPairs {
    const Pair* p;
    __device__ Pair operator()(long long i) const { return p[i]; }
};

template <typename SRC>
__global__ void __launch_bounds__(S_THREADS) k_sort_count(SRC src, long long n, int shift, unsigned* counts,
                                                          uint8_t* present) {
    __shared__ unsigned h[S_BINS];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long b = (long long)blockIdx.x * S_TILE;
#pragma unroll
    for (int u = 0; u < S_PER; ++u) {
        const long long i = b + u * S_THREADS + threadIdx.x;
        if (i < n) {
            const Pair p = src(i);
            atomicAdd(&h[(p.key >> shift) & (S_BINS - 1)], 1u);
            if (present) present[p.key] = 1;
        }
    }
    __syncthreads();
    counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x] = h[threadIdx.x];
}

// exclusive sum of m counts, one CTA
__global__ void __launch_bounds__(1024) k_sort_scan(unsigned* c, int m) {
    __shared__ unsigned ws[32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned base = 0;
    for (int b = 0; b < m; b += 1024) {
        const int i = b + threadIdx.x;
        const unsigned v = i < m ? c[i] : 0u;
        unsigned x = v;
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) ws[w] = x;
        __syncthreads();
        if (w == 0) {
            unsigned s = ws[lane];
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += y;
            }
            ws[lane] = s;
        }
        __syncthreads();
        if (i < m) c[i] = base + (w ? ws[w - 1] : 0u) + x - v;
        base += ws[31];
        __syncthreads();
    }
}

template <typename SRC>
__global__ void __launch_bounds__(S_THREADS) k_sort_scatter(SRC src, long long n, int shift, const unsigned* counts,
                                                            Pair* out) {
    constexpr int W = S_THREADS / 32;
    __shared__ unsigned wc[W][S_BINS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < W * S_BINS; i += S_THREADS) (&wc[0][0])[i] = 0;
    __syncthreads();
    // a warp's S_PER * 32 items are consecutive
    const long long b = (long long)blockIdx.x * S_TILE + w * (S_PER * 32) + lane;
    Pair p[S_PER];
    unsigned rank[S_PER];
#pragma unroll
    for (int u = 0; u < S_PER; ++u) {
        const long long i = b + u * 32;
        const bool in = i < n;
        if (in) p[u] = src(i);
        const unsigned live = __ballot_sync(~0u, in);
        if (in) {
            const unsigned d = (p[u].key >> shift) & (S_BINS - 1);
            const unsigned same = __match_any_sync(live, d);
            const unsigned before = __popc(same & ((1u << lane) - 1u));
            rank[u] = wc[w][d] + before;
            __syncwarp(live);
            if (before == 0) wc[w][d] += __popc(same);
            __syncwarp(live);
        }
    }
    __syncthreads();
    unsigned run = counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x];
    for (int k = 0; k < W; ++k) {
        const unsigned v = wc[k][threadIdx.x];
        wc[k][threadIdx.x] = run;
        run += v;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < S_PER; ++u)
        if (b + u * 32 < n) out[wc[w][(p[u].key >> shift) & (S_BINS - 1)] + rank[u]] = p[u];
}

// ---- sums over runs of one token ----------------------------------------------
// The sorted positions are cut into pieces of `per`; a CTA sums one piece for a
// tile of columns.  A run that lies inside a piece is finished there; the part
// of a run that came from the piece before goes to part[2 piece], the part that
// goes on into the next one to part[2 piece + 1] (a piece inside one run:
// part[2 piece] only).
constexpr int G_THREADS = 128;
constexpr int G_UNROLL = 8;
constexpr int G_MAX_PER = 1024;

template <typename DT, typename OT, int V>
__global__ void __launch_bounds__(G_THREADS) k_grad_pieces(const Pair* pair, int n, int per, const DT* dy, int dim,
                                                           long long dstride, float scale, OT* out,
                                                           long long ostride, unsigned vocab, int accumulate,
                                                           float* part) {
    __shared__ Pair sp[G_MAX_PER];
    const int piece = blockIdx.x;
    const int b = piece * per, m = min(per, n - b);
    for (int i = threadIdx.x; i < m; i += G_THREADS) sp[i] = pair[b + i];
    const unsigned prev = b > 0 ? pair[b - 1].key : ~0u;
    const unsigned next = b + m < n ? pair[b + m].key : ~0u;
    __syncthreads();
    const int c = ((int)blockIdx.y * G_THREADS + threadIdx.x) * V;
    if (c >= dim) return;
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    unsigned cur = sp[0].key;
    bool head = cur == prev;
    auto flush = [&](bool tail) {
        if (cur < vocab) {
            if (head || tail) {
                float* q = part + ((long long)2 * piece + (head ? 0 : 1)) * dim + c;
#pragma unroll
                for (int k = 0; k < V; ++k) q[k] = acc[k];
            } else {
                Pack<OT, V>* q = reinterpret_cast<Pack<OT, V>*>(out + (long long)cur * ostride + c);
                Pack<OT, V> o;
                if (accumulate) o = *q;
#pragma unroll
                for (int k = 0; k < V; ++k)
                    o.v[k] = from_f32<OT>(accumulate ? to_f32(o.v[k]) + scale * acc[k] : scale * acc[k]);
                *q = o;
            }
        }
        head = false;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    };
    for (int i0 = 0; i0 < m; i0 += G_UNROLL) {
        Pack<DT, V> in[G_UNROLL];
#pragma unroll
        for (int u = 0; u < G_UNROLL; ++u)
            if (i0 + u < m && sp[i0 + u].key < vocab)
                in[u] = *reinterpret_cast<const Pack<DT, V>*>(dy + (long long)sp[i0 + u].pos * dstride + c);
#pragma unroll
        for (int u = 0; u < G_UNROLL; ++u) {
            if (i0 + u >= m) break;
            const unsigned key = sp[i0 + u].key;
            if (key != cur) {
                flush(false);
                cur = key;
            }
            if (key < vocab) {
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += to_f32(in[u].v[k]);
            }
        }
    }
    flush(cur == next);
}

// The runs that cross pieces: the CTA of the piece a run starts in sums the
// run's parts in ascending order of pieces, J interleaved partial sums.
constexpr int J_GROUPS = 8;
template <typename OT>
__global__ void __launch_bounds__(32 * J_GROUPS) k_grad_join(const Pair* pair, int n, int per, int pieces, int dim,
                                                             float scale, OT* out, long long ostride, unsigned vocab,
                                                             int accumulate, const float* part) {
    const int piece = blockIdx.x;
    const int b = piece * per, e = min(b + per, n);
    if (e >= n) return;
    const unsigned key = pair[e - 1].key;
    if (key >= vocab || pair[e].key != key) return;
    if (pair[b].key == key && b > 0 && pair[b - 1].key == key) return;  // started earlier
    int lo = piece + 1, hi = pieces;  // pieces (piece, end) begin with this key
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pair[(long long)mid * per].key == key) lo = mid + 1;
        else hi = mid;
    }
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.y * 32 + lane;
    __shared__ float s[J_GROUPS][32];
    float acc = 0.0f;
    if (c < dim) {
        if (grp == 0) acc = part[((long long)2 * piece + 1) * dim + c];
        for (int q = piece + 1 + grp; q < lo; q += J_GROUPS) acc += part[(long long)2 * q * dim + c];
    }
    s[grp][lane] = acc;
    __syncthreads();
    if (grp == 0 && c < dim) {
        for (int g = 1; g < J_GROUPS; ++g) acc += s[g][lane];
        OT* q = out + (long long)key * ostride + c;
        *q = from_f32<OT>(accumulate ? to_f32(*q) + scale * acc : scale * acc);
    }
}

// rows of tokens that do not occur
template <typename OT>
__global__ void __launch_bounds__(256) k_grad_zero(const uint8_t* present, unsigned vocab, int dim, OT* out,
                                                   long long ostride) {
    for (unsigned v = blockIdx.x; v < vocab; v += gridDim.x) {
        if (present[v]) continue;
        for (int c = threadIdx.x; c < dim; c += 256) out[(long long)v * ostride + c] = from_f32<OT>(0.0f);
    }
}

int pieces_per(int64_t n) { return (int)std::min<int64_t>(G_MAX_PER, std::max<int64_t>(32, (n + 591) / 592)); }

struct GradWork {
    int64_t pairs_a, pairs_b, counts, present, part, bytes;
    int per, pieces, tiles;
};
GradWork grad_work(int64_t n, int64_t vocab, int64_t dim) {
    GradWork w;
    w.per = pieces_per(n);
    w.pieces = (int)((n + w.per - 1) / w.per);
    w.tiles = (int)((n + S_TILE - 1) / S_TILE);
    int64_t at = 0;
    auto take = [&](int64_t b) {
        const int64_t p = at;
        at += (b + 255) / 256 * 256;
        return p;
    };
    w.pairs_a = take(n * 8);
    w.pairs_b = take(n * 8);
    w.counts = take((int64_t)S_BINS * w.tiles * 4);
    w.present = take(vocab + 1);
    w.part = take((int64_t)2 * w.pieces * dim * 4);
    w.bytes = at;
    return w;
}

template <typename F>
void with_token(int32_t type, const void* tok, F&& f) {
    if (type == SNN_U8) f((const uint8_t*)tok);
    else if (type == SNN_I32) f((const int32_t*)tok);
    else f((const long long*)tok);
}

void check_tokens(const void* tok, int32_t type) {
    SNN_REQUIRE(type == SNN_U8 || type == SNN_I32 || type == SNN_I64, SNN_ERR_ARG,
                "embed: token type must be SNN_U8, SNN_I32 or SNN_I64");
    const int size = type == SNN_U8 ? 1 : type == SNN_I32 ? 4 : 8;
    SNN_REQUIRE(tok && (uintptr_t)tok % size == 0, SNN_ERR_ARG, "embed: null or misaligned tokens");
}

void check_rows(const void* p, int32_t type, int64_t dim, int64_t stride, const char* name, bool written) {
    SNN_REQUIRE(snnb::elem_type_ok(type), SNN_ERR_ARG,
                std::string("embed: type of ") + name + " must be SNN_F32, SNN_BF16 or SNN_F16");
    SNN_REQUIRE(p && (uintptr_t)p % snnb::elem_size(type) == 0, SNN_ERR_ARG,
                std::string("embed: null or misaligned ") + name);
    SNN_REQUIRE(stride >= (written ? dim : 0) && stride < (1ll << 32), SNN_ERR_ARG,
                std::string("embed: bad row stride of ") + name);
}

void check_sizes(int64_t n, int64_t vocab, int64_t dim) {
    SNN_REQUIRE(n >= 0 && n <= (1ll << 30), SNN_ERR_ARG, "embed: n must lie in [0, 2^30]");
    SNN_REQUIRE(vocab >= 1 && vocab < (1ll << 31), SNN_ERR_ARG, "embed: vocab must lie in [1, 2^31)");
    SNN_REQUIRE(dim >= 1 && dim < (1ll << 24), SNN_ERR_ARG, "embed: dim must lie in [1, 2^24)");
}

// whether rows at p, `stride` elements apart, can be accessed in words of v elements
bool fits(const void* p, int32_t type, int64_t dim, int64_t stride, int v) {
    const int word = std::min(16, snnb::elem_size(type) * v);
    return dim % v == 0 && (stride * snnb::elem_size(type)) % word == 0 && (uintptr_t)p % word == 0;
}

}  // namespace

namespace snnb {

void embed(const void* tokens, int32_t tok_type, int64_t n, const void* table, int32_t table_type, int64_t vocab,
           int64_t dim, int64_t table_stride, float scale, void* out, int32_t out_type, int64_t out_stride,
           cudaStream_t st) {
    check_sizes(n, vocab, dim);
    if (n == 0) return;
    check_tokens(tokens, tok_type);
    check_rows(table, table_type, dim, table_stride, "table", false);
    check_rows(out, out_type, dim, out_stride, "out", true);
    const int sms = device_sms();
    with_token(tok_type, tokens, [&](auto tok) {
        with_elem(table_type, [&](auto tt) {
            with_elem(out_type, [&](auto ot) {
                using TOK = std::remove_const_t<std::remove_pointer_t<decltype(tok)>>;
                using TT = decltype(tt);
                using OT = decltype(ot);
                auto go = [&](auto vc) {
                    constexpr int V = decltype(vc)::value;
                    const int dv = (int)(dim / V);
                    const int segs = (dv + 32 * E_UNROLL - 1) / (32 * E_UNROLL);
                    const int64_t ctas = std::min<int64_t>((n * segs + E_THREADS / 32 - 1) / (E_THREADS / 32),
                                                           (int64_t)sms * 32);
                    k_embed<TOK, TT, OT, V><<<(unsigned)ctas, E_THREADS, 0, st>>>(
                        tok, n, (const TT*)table, (unsigned)vocab, dv, table_stride, scale, (OT*)out, out_stride, segs);
                };
                auto ok = [&](int v) {
                    return fits(table, table_type, dim, table_stride, v) && fits(out, out_type, dim, out_stride, v);
                };
                if (ok(8)) go(std::integral_constant<int, 8>());
                else if (ok(4)) go(std::integral_constant<int, 4>());
                else go(std::integral_constant<int, 1>());
            });
        });
    });
    SNN_CUDA(cudaGetLastError());
}

int64_t embed_grad_workspace(int64_t n, int64_t vocab, int64_t dim) {
    check_sizes(n, vocab, dim);
    return grad_work(n, vocab, dim).bytes;
}

void embed_grad(const void* tokens, int32_t tok_type, int64_t n, const void* dy, int32_t dy_type, int64_t dim,
                int64_t dy_stride, float scale, void* dtable, int32_t dtable_type, int64_t vocab,
                int64_t dtable_stride, int32_t accumulate, void* work, int64_t work_bytes, cudaStream_t st) {
    check_sizes(n, vocab, dim);
    check_rows(dtable, dtable_type, dim, dtable_stride, "dtable", true);
    if (n > 0) {
        check_tokens(tokens, tok_type);
        check_rows(dy, dy_type, dim, dy_stride, "dy", false);
    }
    const GradWork L = grad_work(n, vocab, dim);
    SNN_REQUIRE(work && (uintptr_t)work % 256 == 0 && work_bytes >= L.bytes, SNN_ERR_ARG,
                "embed: workspace null, misaligned or too small");
    const int sms = device_sms();
    char* w = (char*)work;
    Pair* a = (Pair*)(w + L.pairs_a);
    Pair* b = (Pair*)(w + L.pairs_b);
    unsigned* counts = (unsigned*)(w + L.counts);
    uint8_t* present = accumulate ? nullptr : (uint8_t*)(w + L.present);
    float* part = (float*)(w + L.part);
    if (present) SNN_CUDA(cudaMemsetAsync(present, 0, (size_t)vocab + 1, st));
    if (n > 0) {
        int bits = 1;
        while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
        auto pass = [&](auto src, int shift, Pair* dst, uint8_t* mark) {
            k_sort_count<<<L.tiles, S_THREADS, 0, st>>>(src, (long long)n, shift, counts, mark);
            k_sort_scan<<<1, 1024, 0, st>>>(counts, S_BINS * L.tiles);
            k_sort_scatter<<<L.tiles, S_THREADS, 0, st>>>(src, (long long)n, shift, counts, dst);
        };
        with_token(tok_type, tokens, [&](auto tok) {
            using TOK = std::remove_const_t<std::remove_pointer_t<decltype(tok)>>;
            pass(FromTokens<TOK>{tok, (unsigned)vocab}, 0, a, present);
        });
        for (int shift = 8; shift < bits; shift += 8) {
            pass(FromPairs{a}, shift, b, (uint8_t*)nullptr);
            std::swap(a, b);
        }
        with_elem(dy_type, [&](auto dt) {
            with_elem(dtable_type, [&](auto ot) {
                using DT = decltype(dt);
                using OT = decltype(ot);
                auto go = [&](auto vc) {
                    constexpr int V = decltype(vc)::value;
                    const int64_t tile = (int64_t)G_THREADS * V;
                    const dim3 grid((unsigned)L.pieces, (unsigned)((dim + tile - 1) / tile));
                    k_grad_pieces<DT, OT, V><<<grid, G_THREADS, 0, st>>>(a, (int)n, L.per, (const DT*)dy, (int)dim,
                                                                        dy_stride, scale, (OT*)dtable, dtable_stride,
                                                                        (unsigned)vocab, accumulate, part);
                };
                auto ok = [&](int v) {
                    return fits(dy, dy_type, dim, dy_stride, v) && fits(dtable, dtable_type, dim, dtable_stride, v);
                };
                if (dy_type != SNN_F32 && ok(8)) go(std::integral_constant<int, 8>());
                else if (ok(4)) go(std::integral_constant<int, 4>());
                else go(std::integral_constant<int, 1>());
                k_grad_join<OT><<<dim3((unsigned)L.pieces, (unsigned)((dim + 31) / 32)), 32 * J_GROUPS, 0, st>>>(
                    a, (int)n, L.per, L.pieces, (int)dim, scale, (OT*)dtable, dtable_stride, (unsigned)vocab,
                    accumulate, part);
            });
        });
    }
    if (present)
        with_elem(dtable_type, [&](auto ot) {
            using OT = decltype(ot);
            k_grad_zero<OT><<<(unsigned)std::min<int64_t>(vocab, (int64_t)sms * 8), 256, 0, st>>>(
                present, (unsigned)vocab, (int)dim, (OT*)dtable, dtable_stride);
        });
    SNN_CUDA(cudaGetLastError());
}

}  // namespace snnb
