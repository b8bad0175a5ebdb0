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
// Least significant digit first, up to 9 bits a pass (vocabularies of up to 511
// tokens take one pass, up to 2^18 - 1 two).  A pass counts the digits of every
// tile and scatters in input order, so positions of one token stay in
// ascending order; a tile's offsets are sums over the counts (digit, tile),
// taken by every scattering CTA itself where there are few tiles, else by a
// scan between the two.
constexpr int S_THREADS = 512;
constexpr int S_PER = 8;
constexpr int S_TILE = S_THREADS * S_PER;
constexpr int S_BINS = 512;
constexpr int S_FEW = 96;  // tiles up to which a CTA sums the counts itself (192 KB of them)
static_assert(S_BINS == S_THREADS, "a thread per digit");

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

// exclusive sum of one value a thread over the CTA (1,024 threads at most)
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* ws, unsigned& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    unsigned x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) ws[w] = x;
    __syncthreads();
    if (w == 0) {
        unsigned s = lane < nw ? ws[lane] : 0u;
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, s, o);
            if (lane >= o) s += y;
        }
        ws[lane] = s;
    }
    __syncthreads();
    total = ws[nw - 1];
    const unsigned r = (w ? ws[w - 1] : 0u) + x - v;
    __syncthreads();
    return r;
}

template <typename SRC>
__global__ void __launch_bounds__(S_THREADS) k_sort_count(SRC src, long long n, int shift, int bins, unsigned* counts,
                                                          uint8_t* present) {
    __shared__ unsigned h[S_BINS];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long b = (long long)blockIdx.x * S_TILE;
    Pair p[S_PER];
#pragma unroll
    for (int u = 0; u < S_PER; ++u) {
        const long long i = b + u * S_THREADS + threadIdx.x;
        if (i < n) p[u] = src(i);
    }
#pragma unroll
    for (int u = 0; u < S_PER; ++u) {
        if (b + u * S_THREADS + threadIdx.x < n) {
            atomicAdd(&h[(p[u].key >> shift) & (bins - 1)], 1u);
            if (present) present[p[u].key] = 1;
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < bins) counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x] = h[threadIdx.x];
}

// exclusive sum of m counts, one CTA
__global__ void __launch_bounds__(1024) k_sort_scan(unsigned* c, int m) {
    __shared__ unsigned ws[32];
    unsigned base = 0;
    for (int b = 0; b < m; b += 4096) {
        unsigned v[4], sum = 0, total;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = b + threadIdx.x * 4 + k;
            v[k] = i < m ? c[i] : 0u;
            sum += v[k];
        }
        unsigned at = base + block_scan(sum, ws, total);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = b + threadIdx.x * 4 + k;
            if (i < m) c[i] = at;
            at += v[k];
        }
        base += total;
    }
}

// FEW: counts are as counted; otherwise summed already
template <typename SRC, bool FEW>
__global__ void __launch_bounds__(S_THREADS) k_sort_scatter(SRC src, long long n, int shift, int bins,
                                                            const unsigned* counts, Pair* out) {
    constexpr int W = S_THREADS / 32;
    __shared__ unsigned wc[W][S_BINS];
    __shared__ unsigned ws[32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    // a warp's S_PER * 32 items are consecutive
    const long long b = (long long)blockIdx.x * S_TILE + w * (S_PER * 32) + lane;
    Pair p[S_PER];
#pragma unroll
    for (int u = 0; u < S_PER; ++u)
        if (b + u * 32 < n) p[u] = src(b + u * 32);
    unsigned run = 0;  // of this thread's digit: items of smaller digits and of earlier tiles
    if (FEW) {
        unsigned before = 0, all = 0;
        if ((int)threadIdx.x < bins)
            for (int t = 0; t < (int)gridDim.x; ++t) {
                const unsigned v = counts[(size_t)threadIdx.x * gridDim.x + t];
                if (t < (int)blockIdx.x) before += v;
                all += v;
            }
        unsigned total;
        run = block_scan(all, ws, total) + before;
    } else if ((int)threadIdx.x < bins) {
        run = counts[(size_t)threadIdx.x * gridDim.x + blockIdx.x];
    }
    for (int i = threadIdx.x; i < W * S_BINS; i += S_THREADS) (&wc[0][0])[i] = 0;
    __syncthreads();
    unsigned rank[S_PER];
#pragma unroll
    for (int u = 0; u < S_PER; ++u) {
        const bool in = b + u * 32 < n;
        const unsigned live = __ballot_sync(~0u, in);
        if (in) {
            const unsigned d = (p[u].key >> shift) & (bins - 1);
            const unsigned same = __match_any_sync(live, d);
            const unsigned before = __popc(same & ((1u << lane) - 1u));
            rank[u] = wc[w][d] + before;
            __syncwarp(live);
            if (before == 0) wc[w][d] += __popc(same);
            __syncwarp(live);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const unsigned v = wc[k][threadIdx.x];
        wc[k][threadIdx.x] = run;
        run += v;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < S_PER; ++u)
        if (b + u * 32 < n) out[wc[w][(p[u].key >> shift) & (bins - 1)] + rank[u]] = p[u];
}

// ---- sums over runs of one token ----------------------------------------------
// N bytes in registers, as one load brings them (unpacked where they are used)
template <int N>
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
struct Raw<16> {
    using type = uint4;
};
__device__ __forceinline__ void add_raw(float (&acc)[4], const uint4& w, float) {
    acc[0] += __uint_as_float(w.x);
    acc[1] += __uint_as_float(w.y);
    acc[2] += __uint_as_float(w.z);
    acc[3] += __uint_as_float(w.w);
}
__device__ __forceinline__ void add_raw(float (&acc)[1], unsigned w, float) { acc[0] += __uint_as_float(w); }
__device__ __forceinline__ void add_raw(float (&acc)[8], const uint4& w, __nv_bfloat16) {
    const unsigned v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        acc[2 * k] += __uint_as_float(v[k] << 16);
        acc[2 * k + 1] += __uint_as_float(v[k] & 0xffff0000u);
    }
}
__device__ __forceinline__ void add_raw(float (&acc)[8], const uint4& w, __half) {
    const unsigned v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __half2 p;
        memcpy(&p, &v[k], 4);
        const float2 f = __half22float2(p);
        acc[2 * k] += f.x;
        acc[2 * k + 1] += f.y;
    }
}
__device__ __forceinline__ void add_raw(float (&acc)[1], unsigned short w, __nv_bfloat16) {
    acc[0] += __uint_as_float((unsigned)w << 16);
}
__device__ __forceinline__ void add_raw(float (&acc)[1], unsigned short w, __half) {
    acc[0] += __half2float(__ushort_as_half(w));
}

// V columns of a row of the gradient: stored, or added to what is there
template <typename OT, int V>
__device__ __forceinline__ void put_row(OT* q, const float (&acc)[V], float scale, int accumulate, int words) {
    if (words) {
        using P = Pack<OT, V>;
        P o;
        if (accumulate) o = *reinterpret_cast<const P*>(q);
#pragma unroll
        for (int k = 0; k < V; ++k)
            o.v[k] = from_f32<OT>(accumulate ? to_f32(o.v[k]) + scale * acc[k] : scale * acc[k]);
        *reinterpret_cast<P*>(q) = o;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) q[k] = from_f32<OT>(accumulate ? to_f32(q[k]) + scale * acc[k] : scale * acc[k]);
    }
}

struct GradArgs {
    const Pair* pair;
    int n, per, pieces, dim, accumulate, words;  // words: rows of the gradient are V elements wide words
    unsigned vocab;
    const void* dy;
    long long dstride;
    float scale;
    void* out;
    long long ostride;
    float* part;
    const uint8_t* present;
};

// The sorted positions are cut into pieces of `per`; blockDim.x threads sum one
// piece for V columns each.  A run that lies inside a piece is finished there;
// the part of a run that came from the piece before goes to part[2 piece], the
// part that goes on into the next one to part[2 piece + 1] (a piece inside one
// run: part[2 piece] only).  The CTAs behind the pieces clear the rows of
// tokens that do not occur.
constexpr int G_THREADS = 128;
constexpr int G_UNROLL = 8;
constexpr int G_SHARED = 2048;  // positions a CTA holds, all its pieces together

template <typename DT, typename OT, int V>
__global__ void __launch_bounds__(G_THREADS) k_grad_pieces(const GradArgs A, int ctas) {
    using R = typename Raw<sizeof(DT) * V>::type;
    const int c = ((int)blockIdx.y * blockDim.x + threadIdx.x) * V;
    OT* const out = reinterpret_cast<OT*>(A.out);
    if ((int)blockIdx.x >= ctas) {
        if (c >= A.dim) return;
        const float zero[V] = {};
        for (unsigned v = (blockIdx.x - ctas) * blockDim.y + threadIdx.y; v < A.vocab;
             v += (gridDim.x - ctas) * blockDim.y)
            if (!A.present[v]) put_row<OT, V>(out + (long long)v * A.ostride + c, zero, 1.0f, 0, A.words);
        return;
    }
    __shared__ Pair held[G_SHARED];
    const int first = blockIdx.x * blockDim.y * A.per;  // of the CTA's positions
    const int all = min(A.per * (int)blockDim.y, A.n - first);
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < all; i += blockDim.x * blockDim.y)
        held[i] = A.pair[first + i];
    const int piece = blockIdx.x * blockDim.y + threadIdx.y;
    const int b = piece * A.per, m = min(A.per, A.n - b);
    const unsigned prev = m > 0 && b > 0 ? A.pair[b - 1].key : ~0u;
    const unsigned next = m > 0 && b + m < A.n ? A.pair[b + m].key : ~0u;
    __syncthreads();
    if (c >= A.dim || m <= 0) return;
    const Pair* sp = held + (b - first);
    const char* dy = reinterpret_cast<const char*>(reinterpret_cast<const DT*>(A.dy) + c);
    const long long ds = A.dstride * (int)sizeof(DT);
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    unsigned cur = sp[0].key;
    bool head = cur == prev;
    auto flush = [&](bool tail) {
        if (cur < A.vocab) {
            if (head || tail) {
                float* q = A.part + ((long long)2 * piece + (head ? 0 : 1)) * A.dim + c;
#pragma unroll
                for (int k = 0; k < V; ++k) q[k] = acc[k];
            } else {
                put_row<OT, V>(out + (long long)cur * A.ostride + c, acc, A.scale, A.accumulate, A.words);
            }
        }
        head = false;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    };
    for (int i0 = 0; i0 < m; i0 += G_UNROLL) {
        R in[G_UNROLL];
        // rows of tokens outside the vocabulary are read too, not added
#pragma unroll
        for (int u = 0; u < G_UNROLL; ++u)
            in[u] = *reinterpret_cast<const R*>(dy + (long long)sp[min(i0 + u, m - 1)].pos * ds);
        if (i0 + G_UNROLL <= m && sp[i0 + G_UNROLL - 1].key == cur) {
            if (cur < A.vocab)
#pragma unroll
                for (int u = 0; u < G_UNROLL; ++u) add_raw(acc, in[u], DT());
            continue;
        }
#pragma unroll
        for (int u = 0; u < G_UNROLL; ++u) {
            if (i0 + u >= m) continue;
            const unsigned key = sp[i0 + u].key;
            if (key != cur) {
                flush(false);
                cur = key;
            }
            if (key < A.vocab) add_raw(acc, in[u], DT());
        }
    }
    flush(cur == next);
}

// The runs that cross pieces: the CTA of the piece a run starts in sums the
// run's parts, every J_GROUPS-th piece by one warp, the warps' sums in order.
constexpr int J_GROUPS = 8;
constexpr int J_COLS = 4;
template <typename OT>
__global__ void __launch_bounds__(32 * J_GROUPS) k_grad_join(const GradArgs A) {
    const int piece = blockIdx.x;
    const int b = piece * A.per, e = min(b + A.per, A.n);
    if (e >= A.n) return;
    const unsigned key = A.pair[e - 1].key, after = A.pair[e].key, at = A.pair[b].key;
    const unsigned before = b > 0 ? A.pair[b - 1].key : ~0u;
    if (key >= A.vocab || after != key) return;
    if (at == key && before == key) return;  // started earlier
    int lo = piece + 1, hi = A.pieces;  // pieces (piece, end) begin with this key
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (A.pair[(long long)mid * A.per].key == key) lo = mid + 1;
        else hi = mid;
    }
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    __shared__ float s[J_GROUPS][J_COLS][32];
    const int c0 = blockIdx.y * (32 * J_COLS) + lane;
    float acc[J_COLS] = {};
#pragma unroll
    for (int k = 0; k < J_COLS; ++k)
        if (grp == 0 && c0 + 32 * k < A.dim) acc[k] = A.part[((long long)2 * piece + 1) * A.dim + c0 + 32 * k];
#pragma unroll 4
    for (int q = piece + 1 + grp; q < lo; q += J_GROUPS)
#pragma unroll
        for (int k = 0; k < J_COLS; ++k)
            if (c0 + 32 * k < A.dim) acc[k] += A.part[(long long)2 * q * A.dim + c0 + 32 * k];
#pragma unroll
    for (int k = 0; k < J_COLS; ++k) s[grp][k][lane] = acc[k];
    __syncthreads();
    if (grp >= J_COLS) return;
    const int c = c0 + 32 * grp;
    if (c >= A.dim) return;
    float sum[1] = {0.0f};
    for (int g = 0; g < J_GROUPS; ++g) sum[0] += s[g][grp][lane];
    put_row<OT, 1>(reinterpret_cast<OT*>(A.out) + (long long)key * A.ostride + c, sum, A.scale, A.accumulate, 0);
}

// rows of a gradient without positions
template <typename OT>
__global__ void __launch_bounds__(256) k_grad_clear(unsigned vocab, int dim, OT* out, long long ostride) {
    for (unsigned v = blockIdx.x; v < vocab; v += gridDim.x)
        for (int c = threadIdx.x; c < dim; c += 256) out[(long long)v * ostride + c] = from_f32<OT>(0.0f);
}

// How the columns and positions are cut.  The order of the sums follows `per`,
// so it goes by n and dim alone: pieces such that SMS * 8 CTAs' worth of threads
// have one each, of 32 to 1,024 positions.
constexpr int SMS = 148;
int pieces_per(int64_t n, int64_t dim) {
    const int64_t cols = (dim + 1023) / 1024, wanted = std::max<int64_t>(1, SMS * 8 / cols);
    return (int)std::min<int64_t>(1024, std::max<int64_t>(32, (n + wanted - 1) / wanted));
}

struct GradWork {
    int64_t pairs_a, pairs_b, counts, present, part, bytes;
    int per, pieces, tiles;
};
GradWork grad_work(int64_t n, int64_t vocab, int64_t dim) {
    GradWork w;
    w.per = pieces_per(n, dim);
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
    w.bytes = std::max<int64_t>(at, 256);
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
    char* w = (char*)work;
    Pair* a = (Pair*)(w + L.pairs_a);
    Pair* b = (Pair*)(w + L.pairs_b);
    unsigned* counts = (unsigned*)(w + L.counts);
    uint8_t* present = accumulate ? nullptr : (uint8_t*)(w + L.present);
    float* part = (float*)(w + L.part);
    if (n == 0) {
        if (present)
            with_elem(dtable_type, [&](auto ot) {
                using OT = decltype(ot);
                k_grad_clear<OT><<<(unsigned)std::min<int64_t>(vocab, SMS * 8), 256, 0, st>>>(
                    (unsigned)vocab, (int)dim, (OT*)dtable, dtable_stride);
            });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    if (present) SNN_CUDA(cudaMemsetAsync(present, 0, (size_t)vocab + 1, st));
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
    const int passes = (bits + 8) / 9, digit = (bits + passes - 1) / passes, bins = 1 << digit;
    auto pass = [&](auto src, int shift, Pair* dst, uint8_t* mark) {
        using SRC = decltype(src);
        k_sort_count<<<L.tiles, S_THREADS, 0, st>>>(src, (long long)n, shift, bins, counts, mark);
        if (L.tiles <= S_FEW) {
            k_sort_scatter<SRC, true><<<L.tiles, S_THREADS, 0, st>>>(src, (long long)n, shift, bins, counts, dst);
        } else {
            k_sort_scan<<<1, 1024, 0, st>>>(counts, bins * L.tiles);
            k_sort_scatter<SRC, false><<<L.tiles, S_THREADS, 0, st>>>(src, (long long)n, shift, bins, counts, dst);
        }
    };
    with_token(tok_type, tokens, [&](auto tok) {
        using TOK = std::remove_const_t<std::remove_pointer_t<decltype(tok)>>;
        pass(FromTokens<TOK>{tok, (unsigned)vocab}, 0, a, present);
    });
    for (int k = 1; k < passes; ++k) {
        pass(FromPairs{a}, k * digit, b, (uint8_t*)nullptr);
        std::swap(a, b);
    }
    GradArgs A;
    A.pair = a;
    A.n = (int)n;
    A.per = L.per;
    A.pieces = L.pieces;
    A.dim = (int)dim;
    A.accumulate = accumulate != 0;
    A.vocab = (unsigned)vocab;
    A.dy = dy;
    A.dstride = dy_stride;
    A.scale = scale;
    A.out = dtable;
    A.ostride = dtable_stride;
    A.part = part;
    A.present = present;
    with_elem(dy_type, [&](auto dt) {
        with_elem(dtable_type, [&](auto ot) {
            using DT = decltype(dt);
            using OT = decltype(ot);
            auto go = [&](auto vc) {
                constexpr int V = decltype(vc)::value;
                A.words = fits(dtable, dtable_type, dim, dtable_stride, V);
                int tx = 1;  // threads a row of a piece, a power of two
                while (tx < G_THREADS && (int64_t)tx * V < dim) tx *= 2;
                const int ty = std::min(G_THREADS / tx, G_SHARED / L.per);
                const unsigned ctas = (unsigned)((L.pieces + ty - 1) / ty);
                const unsigned clear = present ? (unsigned)std::min<int64_t>((vocab + ty - 1) / ty, SMS * 4) : 0u;
                const unsigned cols = (unsigned)((dim + (int64_t)tx * V - 1) / ((int64_t)tx * V));
                k_grad_pieces<DT, OT, V><<<dim3(ctas + clear, cols), dim3(tx, ty), 0, st>>>(A, (int)ctas);
            };
            constexpr int V16 = 16 / (int)sizeof(DT);
            if (fits(dy, dy_type, dim, dy_stride, V16)) go(std::integral_constant<int, V16>());
            else go(std::integral_constant<int, 1>());
            k_grad_join<OT><<<dim3((unsigned)L.pieces, (unsigned)((dim + 32 * J_COLS - 1) / (32 * J_COLS))),
                              32 * J_GROUPS, 0, st>>>(A);
        });
    });
    SNN_CUDA(cudaGetLastError());
}

}  // namespace snnb
