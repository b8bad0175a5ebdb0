// embed.cu - token drive: rows of a table picked by a token stream
// (snn_embed), and the table's gradient by sorted tokens (snn_embed_grad).
#include <algorithm>
#include "elem.h"

namespace {
constexpr int SMS = 148;  // multiprocessors of a B200
using snnb::from_f32;
using snnb::to_f32;

// V elements that are stored as one word of at most 16 bytes
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};
// N bytes in registers, as one load (32: two) brings them; unpacked where they
// are used, so that loads stay in flight
struct Raw32 {
    uint4 lo, hi;
};
template <int N> struct Raw;
template <> struct Raw<2> { using type = unsigned short; };
template <> struct Raw<4> { using type = unsigned; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<32> { using type = Raw32; };

__device__ __forceinline__ void unpack(float* o, unsigned w, float) { o[0] = __uint_as_float(w); }
__device__ __forceinline__ void unpack(float* o, unsigned w, __nv_bfloat16) {
    o[0] = __uint_as_float(w << 16);
    o[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack(float* o, unsigned w, __half) {
    __half2 p;
    memcpy(&p, &w, 4);
    const float2 f = __half22float2(p);
    o[0] = f.x;
    o[1] = f.y;
}
__device__ __forceinline__ void unpack(float* o, unsigned short w, __nv_bfloat16) {
    o[0] = __uint_as_float((unsigned)w << 16);
}
__device__ __forceinline__ void unpack(float* o, unsigned short w, __half) { o[0] = __half2float(__ushort_as_half(w)); }
template <typename T>
__device__ __forceinline__ void unpack(float* o, const uint2& w, T t) {
    constexpr int E = 4 / (int)sizeof(T);
    unpack(o, w.x, t);
    unpack(o + E, w.y, t);
}
template <typename T>
__device__ __forceinline__ void unpack(float* o, const uint4& w, T t) {
    constexpr int E = 4 / (int)sizeof(T);
    unpack(o, w.x, t);
    unpack(o + E, w.y, t);
    unpack(o + 2 * E, w.z, t);
    unpack(o + 3 * E, w.w, t);
}
template <typename T>
__device__ __forceinline__ void unpack(float* o, const Raw32& w, T t) {
    constexpr int E = 16 / (int)sizeof(T);
    unpack(o, w.lo, t);
    unpack(o + E, w.hi, t);
}

template <typename TOK>
__device__ __forceinline__ unsigned token_at(const TOK* tok, long long i, unsigned vocab) {
    // outside [0, vocab): `vocab`
    const long long t = (long long)tok[i];
    return (unsigned long long)t < vocab ? (unsigned)t : vocab;
}

// ---- out[i] = scale * table[tok[i]] -----------------------------------------
// A warp takes up to 32 * e_unroll words of a row, all in flight at once.  Bound by the writes of the
// rows (and their reads, where the table is large).
constexpr int E_THREADS = 256;
template <int V>
constexpr int e_unroll = V >= 4 ? 4 : V == 2 ? 8 : 16;
template <typename TOK, typename TT, typename OT, int V>
__global__ void __launch_bounds__(E_THREADS) k_embed(const TOK* tok, long long n, const TT* table, unsigned vocab,
                                                     int dv, long long tstride, float scale, OT* out,
                                                     long long ostride, int segs) {
    using R = typename Raw<sizeof(TT) * V>::type;
    constexpr int E_UNROLL = e_unroll<V>;
    const int lane = threadIdx.x & 31;
    const long long nw = (long long)gridDim.x * (E_THREADS / 32);
    for (long long w = (long long)blockIdx.x * (E_THREADS / 32) + (threadIdx.x >> 5); w < n * segs; w += nw) {
        const long long i = segs == 1 ? w : w / segs;
        const int c0 = (int)(w - i * segs) * (32 * E_UNROLL) + lane;
        const unsigned t = token_at(tok, i, vocab);
        // a token outside the vocabulary reads row 0 and writes zeros
        const R* src = reinterpret_cast<const R*>(table + (long long)(t < vocab ? t : 0u) * tstride);
        Pack<OT, V>* dst = reinterpret_cast<Pack<OT, V>*>(out + i * ostride);
        R in[E_UNROLL];
#pragma unroll
        for (int u = 0; u < E_UNROLL; ++u) in[u] = src[min(c0 + u * 32, dv - 1)];
#pragma unroll
        for (int u = 0; u < E_UNROLL; ++u) {
            if (c0 + u * 32 >= dv) break;
            float f[V];
            unpack(f, in[u], TT());
            Pack<OT, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = from_f32<OT>(t < vocab ? scale * f[k] : 0.0f);
            dst[c0 + u * 32] = o;
        }
    }
}

// A kernel launched as the dependent of the one before (launch_next) starts
// while that one still runs: it must call after_previous() before it touches
// what earlier kernels write.  let_next() allows the next kernel to start; it
// comes after after_previous(), so that what ran before the previous kernel is
// complete for the next one's start.  In every kernel at least one CTA waits, so
// that what follows the call on the stream finds all of its kernels done.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... Q>
void launch_next(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t st, Q&&... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    SNN_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

// ---- the positions sorted by token -------------------------------------------
// Least significant digit first, up to 9 bits a pass (vocabularies of up to 511
// tokens take one pass, up to 2^18 - 1 two).  A pass counts the digits of every
// tile and scatters in input order, so positions of one token stay in
// ascending order.  Launches are what a short sort costs: up to S_OWN items
// every scattering CTA counts them all itself (one launch a pass), beyond there
// are three: counts by tile, their sums by digit, the scatter.
constexpr int S_THREADS = 512;
constexpr int S_PER = 4, S_OWN_PER = 2;  // items a thread
constexpr int S_OWN = 32768;
constexpr int S_TILE = S_THREADS * S_PER;
constexpr int S_BINS = 512;
static_assert(S_BINS == S_THREADS, "a thread per digit");

struct Pair {
    unsigned key, pos;
};

// The gradient's rows set to zero by CTAs of the first sorting kernel, most of
// whose SMs are idle: rows that do not occur stay zero, the others are written
// again by the sums.
struct Clear {
    char* p;
    long long rows, row_bytes, stride;  // contiguous rows count as one
    int word;                           // 16, 4 or 2 bytes a store
    int ctas;                           // 0: nothing to clear
};
__device__ __forceinline__ void clear_rows(const Clear& C, int cta) {
    const long long step = (long long)C.ctas * blockDim.x, t = (long long)cta * blockDim.x + threadIdx.x;
    if (C.word == 16) {
        const long long per = C.row_bytes / 16;
        if (C.rows == 1) {
            for (long long i = t; i < per; i += step) reinterpret_cast<uint4*>(C.p)[i] = make_uint4(0, 0, 0, 0);
            for (long long i = per * 16 + t * 2; i < C.row_bytes; i += step * 2) *reinterpret_cast<unsigned short*>(C.p + i) = 0;
        } else {
            for (long long r = cta; r < C.rows; r += C.ctas)
                for (long long i = threadIdx.x; i < per; i += blockDim.x)
                    reinterpret_cast<uint4*>(C.p + r * C.stride)[i] = make_uint4(0, 0, 0, 0);
        }
    } else {
        const long long per = C.row_bytes / C.word;
        for (long long r = cta; r < C.rows; r += C.ctas)
            for (long long i = threadIdx.x; i < per; i += blockDim.x) {
                if (C.word == 4) reinterpret_cast<unsigned*>(C.p + r * C.stride)[i] = 0;
                else reinterpret_cast<unsigned short*>(C.p + r * C.stride)[i] = 0;
            }
    }
}

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

__global__ void __launch_bounds__(S_THREADS) k_clear(Clear clear) { clear_rows(clear, blockIdx.x); }

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

template <typename SRC, int PER>
__global__ void __launch_bounds__(S_THREADS) k_sort_count(SRC src, long long n, int shift, int bins, unsigned* counts,
                                                          int tiles, Clear clear) {
    __shared__ unsigned h[S_BINS];
    after_previous();
    let_next();
    if ((int)blockIdx.x >= tiles) return clear_rows(clear, blockIdx.x - tiles);
    h[threadIdx.x] = 0;
    __syncthreads();
    const long long b = (long long)blockIdx.x * (S_THREADS * PER);
    Pair p[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const long long i = b + u * S_THREADS + threadIdx.x;
        if (i < n) p[u] = src(i);
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        if (b + u * S_THREADS + threadIdx.x < n) atomicAdd(&h[(p[u].key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    if ((int)threadIdx.x < bins)
        counts[(size_t)threadIdx.x * tiles + blockIdx.x] = h[threadIdx.x];
}

// per digit: exclusive sums of the tiles' counts, and the digit's total
__global__ void __launch_bounds__(256) k_sort_scan(unsigned* counts, int tiles, unsigned* totals) {
    __shared__ unsigned ws[32];
    after_previous();
    let_next();
    unsigned* c = counts + (size_t)blockIdx.x * tiles;
    unsigned base = 0;
    for (int b = 0; b < tiles; b += 256) {
        const int i = b + threadIdx.x;
        const unsigned v = i < tiles ? c[i] : 0u;
        unsigned total;
        const unsigned at = block_scan(v, ws, total);
        if (i < tiles) c[i] = base + at;
        base += total;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = base;
}

// OWN: the CTA counts all n items itself; else counts and totals are from the scan
template <typename SRC, bool OWN, int PER>
__global__ void __launch_bounds__(S_THREADS) k_sort_scatter(SRC src, long long n, int shift, int bins,
                                                            const unsigned* counts, const unsigned* totals, Pair* out,
                                                            int tiles, Clear clear) {
    constexpr int W = S_THREADS / 32;
    __shared__ unsigned wc[W][S_BINS];
    __shared__ unsigned ws[32];
    after_previous();
    let_next();
    if ((int)blockIdx.x >= tiles) return clear_rows(clear, blockIdx.x - tiles);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    // a warp's PER * 32 items are consecutive
    const long long tile = (long long)blockIdx.x * (S_THREADS * PER), b = tile + w * (PER * 32) + lane;
    Pair p[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u)
        if (b + u * 32 < n) p[u] = src(b + u * 32);
    unsigned run = 0, total;  // of this thread's digit: items of smaller digits and of earlier tiles
    if (OWN) {
        wc[0][threadIdx.x] = wc[1][threadIdx.x] = 0;
        __syncthreads();
#pragma unroll 8
        for (int i = threadIdx.x; i < (int)n; i += S_THREADS) {
            const unsigned d = (src(i).key >> shift) & (bins - 1);
            atomicAdd(&wc[i < (int)tile ? 0 : 1][d], 1u);
        }
        __syncthreads();
        const unsigned before = wc[0][threadIdx.x];
        run = block_scan(before + wc[1][threadIdx.x], ws, total) + before;
    } else {
        const bool in = (int)threadIdx.x < bins;
        const unsigned before = in ? counts[(size_t)threadIdx.x * tiles + blockIdx.x] : 0u;
        run = block_scan(in ? totals[threadIdx.x] : 0u, ws, total) + before;
    }
    for (int i = threadIdx.x; i < W * S_BINS; i += S_THREADS) (&wc[0][0])[i] = 0;
    __syncthreads();
    unsigned rank[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
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
    for (int u = 0; u < PER; ++u)
        if (b + u * 32 < n) out[wc[w][(p[u].key >> shift) & (bins - 1)] + rank[u]] = p[u];
}

// ---- sums over runs of one token ----------------------------------------------
template <int V, typename R, typename T>
__device__ __forceinline__ void add_raw(float (&acc)[V], const R& w, T t) {
    float f[V];
    unpack(f, w, t);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += f[k];
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
};

// The sorted positions are cut into pieces of `per`; blockDim.x threads sum one
// piece for V columns each.  A run that lies inside a piece is finished there;
// the part of a run that came from the piece before goes to part[2 piece], the
// part that goes on into the next one to part[2 piece + 1] (a piece inside one
// run: part[2 piece] only).  8 CTAs an SM leave 64 registers, of which 16-bit
// gradients summed to f32 by 8 columns a thread spill 22 bytes, the other forms
// none.
constexpr int G_THREADS = 128;
template <typename R>
constexpr int g_unroll = sizeof(R) >= 8 ? 8 : 16;  // rows in flight a thread
constexpr int G_SHARED = 2048;  // positions a CTA holds, all its pieces together

template <typename DT, typename OT, int V>
__global__ void __launch_bounds__(G_THREADS, 8) k_grad_pieces(const GradArgs A) {
    using R = typename Raw<sizeof(DT) * V>::type;
    constexpr int G_UNROLL = g_unroll<R>;
    const int c = ((int)blockIdx.y * blockDim.x + threadIdx.x) * V;
    OT* const out = reinterpret_cast<OT*>(A.out);
    __shared__ Pair held[G_SHARED];
    after_previous();
    let_next();
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

// The runs that cross pieces: the CTA of the piece a run starts in (found from
// the sorted tokens while the pieces are still summed) sums the run's parts, every J_GROUPS-th piece by one warp, the warps' sums in order.
constexpr int J_GROUPS = 8;
constexpr int J_COLS = 4;
template <typename OT>
__global__ void __launch_bounds__(32 * J_GROUPS) k_grad_join(const GradArgs A) {
    const int piece = blockIdx.x;
    const int b = piece * A.per, e = min(b + A.per, A.n);
    const unsigned key = A.pair[e - 1].key, after = e < A.n ? A.pair[e].key : ~0u, at = A.pair[b].key;
    const unsigned before = b > 0 ? A.pair[b - 1].key : ~0u;
    if (key >= A.vocab || after != key || (at == key && before == key)) {  // no run begins here and goes on
        // one CTA waits in any case: this kernel does not end before the one it depends on
        if (blockIdx.x == 0 && blockIdx.y == 0) after_previous();
        return;
    }
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
    int lo = piece + 1;  // becomes the end of the pieces that begin with this key
    for (bool more = true; more; lo += 128) {
        unsigned in[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long q = lo + k * 32 + lane;
            in[k] = __ballot_sync(~0u, q < A.pieces && A.pair[q * A.per].key == key);
        }
        int run = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (run == k * 32) run += in[k] == ~0u ? 32 : __ffs(~in[k]) - 1;
        more = run == 128;
        if (!more) lo += run - 128;
    }
    after_previous();  // the pieces' sums
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

// Short calls in one launch: a CTA sorts all n tokens in shared memory (a
// bitonic network over token * 2048 + position, so equal tokens keep their
// order) and sums for 8 * V columns; groups of 8 threads take consecutive parts
// of the sorted positions, and the group a run starts in joins its parts.
// 512 bytes by 500 columns in f32: 29 us by the kernels above, 11 by this one.
constexpr int T_THREADS = 512, T_COLS = 8, T_GROUPS = T_THREADS / T_COLS;
constexpr int T_N = 2048, T_VOCAB = 4096;

template <typename TOK, typename DT, typename OT, int V>
__global__ void __launch_bounds__(T_THREADS) k_grad_small(const TOK* tok, const GradArgs A) {
    using R = typename Raw<sizeof(DT) * V>::type;
    constexpr int G_UNROLL = 8;
    __shared__ unsigned key[T_N];
    __shared__ unsigned seen[T_VOCAB / 32 + 1];
    __shared__ float part[T_GROUPS][2][T_COLS * V];
    // element e * T_THREADS + thread: partners within a thread, a warp, or the CTA
    constexpr int E = T_N / T_THREADS;
    unsigned v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = e * T_THREADS + threadIdx.x;
        v[e] = i < A.n ? token_at(tok, i, A.vocab) << 11 | i : ~0u;
    }
    for (int i = threadIdx.x; i < T_VOCAB / 32 + 1; i += T_THREADS) seen[i] = 0;
    const int held = A.n <= T_THREADS ? 1 : E;
    const int size = held * T_THREADS;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            if (j >= T_THREADS) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int o = e ^ (j / T_THREADS);
                    if (o > e && o < E) {
                        const unsigned lo = min(v[e], v[o]), hi = max(v[e], v[o]);
                        const bool up = ((e * T_THREADS) & k) == 0;
                        v[e] = up ? lo : hi;
                        v[o] = up ? hi : lo;
                    }
                }
                continue;
            }
            if (j >= 32) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (e < held) key[e * T_THREADS + threadIdx.x] = v[e];
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (e >= held) continue;
                const int i = e * T_THREADS + threadIdx.x;
                const unsigned o = j >= 32 ? key[i ^ j] : __shfl_xor_sync(~0u, v[e], j);
                v[e] = ((i & j) == 0) == ((i & k) == 0) ? min(v[e], o) : max(v[e], o);
            }
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < held) key[e * T_THREADS + threadIdx.x] = v[e];
    __syncthreads();
    for (int i = threadIdx.x; i < A.n; i += T_THREADS) atomicOr(&seen[key[i] >> 16], 1u << (key[i] >> 11 & 31));
    __syncthreads();
    const int x = threadIdx.x % T_COLS, g = threadIdx.x / T_COLS;
    const int c = (blockIdx.x * T_COLS + x) * V;
    const bool live = c < A.dim;
    const int per = (A.n + T_GROUPS - 1) / T_GROUPS, b = g * per, m = min(per, A.n - b);
    OT* const out = reinterpret_cast<OT*>(A.out) + c;
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    if (live && m > 0) {
        const char* dy = reinterpret_cast<const char*>(reinterpret_cast<const DT*>(A.dy) + c);
        const long long ds = A.dstride * (int)sizeof(DT);
        unsigned cur = key[b] >> 11;
        bool head = b > 0 && key[b - 1] >> 11 == cur;
        for (int i0 = 0; i0 <= m; i0 += G_UNROLL) {
            R in[G_UNROLL];
#pragma unroll
            for (int u = 0; u < G_UNROLL; ++u)
                if (i0 < m) in[u] = *reinterpret_cast<const R*>(dy + (long long)(key[b + min(i0 + u, m - 1)] & (T_N - 1)) * ds);
#pragma unroll
            for (int u = 0; u < G_UNROLL; ++u) {
                const int i = i0 + u;
                if (i > m) break;
                // i == m: the position behind the part, which ends its last run
                const unsigned t = b + i < A.n ? key[b + i] >> 11 : ~0u;
                if (t != cur || i == m) {
                    const bool tail = i == m && t == cur;
                    if (cur < A.vocab) {
                        if (head || tail) {
#pragma unroll
                            for (int k = 0; k < V; ++k) part[g][head ? 0 : 1][x * V + k] = acc[k];
                        } else {
                            put_row<OT, V>(out + (long long)cur * A.ostride, acc, A.scale, A.accumulate, A.words);
                        }
                    }
                    head = false;
                    cur = t;
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
                }
                if (i < m && t < A.vocab) add_raw(acc, in[u], DT());
            }
        }
    }
    __syncthreads();
    if (!live) return;
    if (m > 0 && b + m < A.n) {
        const unsigned last = key[b + m - 1] >> 11;
        const bool started = key[b] >> 11 != last || b == 0 || key[b - 1] >> 11 != last;
        if (last < A.vocab && key[b + m] >> 11 == last && started) {
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = part[g][1][x * V + k];
            for (int q = g + 1; q < T_GROUPS && q * per < A.n && key[q * per] >> 11 == last; ++q)
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += part[q][0][x * V + k];
            put_row<OT, V>(out + (long long)last * A.ostride, acc, A.scale, A.accumulate, A.words);
        }
    }
    if (A.accumulate) return;
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.0f;
    for (unsigned v = g; v < A.vocab; v += T_GROUPS)
        if (!(seen[v >> 5] >> (v & 31) & 1u)) put_row<OT, V>(out + (long long)v * A.ostride, acc, 1.0f, 0, A.words);
}

// How the columns and positions are cut.  The order of the sums follows `per`,
// so it goes by n and dim alone: pieces such that SMS * 8 CTAs' worth of threads
// have one each, of 32 to 1,024 positions.
int pieces_per(int64_t n, int64_t dim) {
    const int64_t cols = (dim + 1023) / 1024, wanted = std::max<int64_t>(1, SMS * 8 / cols);
    return (int)std::min<int64_t>(1024, std::max<int64_t>(32, (n + wanted - 1) / wanted));
}

struct GradWork {
    int64_t pairs_a, pairs_b, counts, totals, part, bytes;
    int per, pieces, tiles;
    bool small;
};
GradWork grad_work(int64_t n, int64_t vocab, int64_t dim) {
    GradWork w;
    w.per = pieces_per(n, dim);
    w.pieces = (int)((n + w.per - 1) / w.per);
    w.tiles = (int)((n + S_TILE - 1) / S_TILE);
    w.small = n <= T_N && vocab <= T_VOCAB;
    if (w.small) n = w.pieces = w.tiles = 0;
    int64_t at = 0;
    auto take = [&](int64_t b) {
        const int64_t p = at;
        at += (b + 255) / 256 * 256;
        return p;
    };
    w.pairs_a = take(n * 8);
    w.pairs_b = take(n * 8);
    w.counts = take((int64_t)S_BINS * w.tiles * 4);
    w.totals = take(S_BINS * 4);
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
    SNN_REQUIRE(dim >= 1 && dim <= (1ll << 22), SNN_ERR_ARG, "embed: dim must lie in [1, 2^22]");
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
                    const int segs = (dv + 32 * e_unroll<V> - 1) / (32 * e_unroll<V>);
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
                else if (ok(2)) go(std::integral_constant<int, 2>());
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
    unsigned *counts = (unsigned*)(w + L.counts), *totals = (unsigned*)(w + L.totals);
    GradArgs A;
    A.pair = nullptr;
    A.n = (int)n;
    A.per = L.per;
    A.pieces = L.pieces;
    A.dim = (int)dim;
    A.accumulate = accumulate != 0;
    A.words = 0;
    A.vocab = (unsigned)vocab;
    A.dy = dy;
    A.dstride = dy_stride;
    A.scale = scale;
    A.out = dtable;
    A.ostride = dtable_stride;
    A.part = (float*)(w + L.part);
    // f(DT(), OT(), V): the types and the columns a thread takes
    auto typed = [&](auto&& f) {
        with_elem(dy_type, [&](auto dt) {
            with_elem(dtable_type, [&](auto ot) {
                constexpr int V4 = 4 / (int)sizeof(dt);
                auto ok = [&](int v) { return n > 0 && fits(dy, dy_type, dim, dy_stride, v); };
                auto go = [&](auto vc) {
                    A.words = fits(dtable, dtable_type, dim, dtable_stride, decltype(vc)::value);
                    f(dt, ot, vc);
                };
                if (ok(4 * V4)) go(std::integral_constant<int, 4 * V4>());
                else if (ok(2 * V4)) go(std::integral_constant<int, 2 * V4>());
                else if (V4 > 1 && ok(V4)) go(std::integral_constant<int, V4>());
                else go(std::integral_constant<int, 1>());
            });
        });
    };
    if (L.small) {
        with_token(tok_type, tokens, [&](auto tok) {
            using TOK = std::remove_const_t<std::remove_pointer_t<decltype(tok)>>;
            typed([&](auto dt, auto ot, auto vc) {
                constexpr int V = decltype(vc)::value;
                const unsigned ctas = (unsigned)((dim + T_COLS * V - 1) / (T_COLS * V));
                k_grad_small<TOK, decltype(dt), decltype(ot), V><<<ctas, T_THREADS, 0, st>>>(tok, A);
            });
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const int size = elem_size(dtable_type);
    Clear clear = {(char*)dtable, vocab, dim * size, dtable_stride * size, 0, 0};
    if (!accumulate) {
        const bool aligned = (uintptr_t)dtable % 16 == 0;
        const int64_t all = clear.rows * clear.row_bytes;
        clear.word = aligned && clear.row_bytes % 16 == 0 && clear.stride % 16 == 0 ? 16 : size;
        if (aligned && clear.stride == clear.row_bytes) {  // one stretch of memory
            clear.rows = 1;
            clear.row_bytes = all;
            clear.word = 16;
        }
        clear.ctas = (int)std::min<int64_t>(SMS * 3, (all + (1 << 14) - 1) >> 14);
    }
    if (n == 0) {
        if (clear.ctas) k_clear<<<(unsigned)clear.ctas, S_THREADS, 0, st>>>(clear);
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const Clear nothing = {nullptr, 0, 0, 0, 0, 0};
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
    const int passes = (bits + 8) / 9, digit = (bits + passes - 1) / passes, bins = 1 << digit;
    bool later = false;  // the first kernel waits for all work before the call
    auto pass = [&](auto src, int shift, Pair* dst, const Clear& C) {
        using SRC = decltype(src);
        auto start = [&](auto kernel, int ctas, auto... args) {
            if (later) launch_next(kernel, dim3(ctas), dim3(S_THREADS), st, args...);
            else kernel<<<ctas, S_THREADS, 0, st>>>(args...);
            later = true;
        };
        if (n <= S_OWN) {
            const int tiles = (int)((n + S_THREADS * S_OWN_PER - 1) / (S_THREADS * S_OWN_PER));
            start(k_sort_scatter<SRC, true, S_OWN_PER>, tiles + C.ctas, src, (long long)n, shift, bins, counts, totals,
                  dst, tiles, C);
            return;
        }
        start(k_sort_count<SRC, S_PER>, L.tiles + C.ctas, src, (long long)n, shift, bins, counts, L.tiles, C);
        launch_next(k_sort_scan, dim3(bins), dim3(256), st, counts, L.tiles, totals);
        launch_next(k_sort_scatter<SRC, false, S_PER>, dim3(L.tiles), dim3(S_THREADS), st, src, (long long)n, shift, bins,
                    counts, totals, dst, L.tiles, nothing);
    };
    with_token(tok_type, tokens, [&](auto tok) {
        using TOK = std::remove_const_t<std::remove_pointer_t<decltype(tok)>>;
        pass(FromTokens<TOK>{tok, (unsigned)vocab}, 0, a, clear);
    });
    for (int k = 1; k < passes; ++k) {
        pass(FromPairs{a}, k * digit, b, nothing);
        std::swap(a, b);
    }
    A.pair = a;
    typed([&](auto dt, auto ot, auto vc) {
        using OT = decltype(ot);
        constexpr int V = decltype(vc)::value;
        int tx = 1;  // threads a row of a piece, a power of two
        while (tx < G_THREADS && (int64_t)tx * V < dim) tx *= 2;
        const int ty = std::min(G_THREADS / tx, G_SHARED / L.per);
        const unsigned ctas = (unsigned)((L.pieces + ty - 1) / ty);
        const unsigned cols = (unsigned)((dim + (int64_t)tx * V - 1) / ((int64_t)tx * V));
        launch_next(k_grad_pieces<decltype(dt), OT, V>, dim3(ctas, cols), dim3(tx, ty), st, A);
        launch_next(k_grad_join<OT>, dim3((unsigned)L.pieces, (unsigned)((dim + 32 * J_COLS - 1) / (32 * J_COLS))),
                    dim3(32 * J_GROUPS), st, A);
    });
    SNN_CUDA(cudaGetLastError());
}

}  // namespace snnb
