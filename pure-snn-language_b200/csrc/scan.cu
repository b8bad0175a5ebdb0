// scan.cu - leaky scans (snn_leaky_scan, snn_leaky_scan_grad): the linear
// recurrence h_t = a_t h_{t-1} + u_t along sequences, and its gradients:
// arguments, the choice of kernels, and the kernel for short sequences.
#include "scan_tile.h"

namespace {
using namespace snnb_scan;

// ---- short sequences: a thread per sequence and V channels, a step at a time ----
template <typename T, int GM, bool RASTER, int V>
__global__ void __launch_bounds__(128) k_scan_steps(const ScanArgs A) {
    using X = InWord<T, V, RASTER>;
    const int c = (int)(blockIdx.x * 128 + threadIdx.x) * V;
    for (long long s = blockIdx.y; s < A.n_seq && c < A.D; s += gridDim.y) {
        const Span sp = span_of(A, s);
        constexpr bool LO = is_logit<GM>;
        Decay<V, LO> d;
        Vec<V> rest;
        if (per_channel<GM>) channel_decays<GM>(A, c, V, d, rest);
        Vec<V> h = load_f32<V>(A.h0 + s * A.D + c, A.h0 != nullptr);
        constexpr int U = 4;  // steps whose rows are loaded before the first is used
        for (int t0 = 0; t0 < sp.len; t0 += U) {
            Word<T, V> g[U];
            X xw[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int t = min(t0 + i, sp.len - 1);
                if (!per_channel<GM>)
                    g[i] = *reinterpret_cast<const Word<T, V>*>(reinterpret_cast<const T*>(A.gate.p) +
                                                                row_at(A, A.gate, s, sp, t) + c);
                const long long xr = row_at(A, A.x, s, sp, t);
                xw[i] = RASTER ? *reinterpret_cast<const X*>(reinterpret_cast<const unsigned*>(A.x.p) + xr + (c >> 5))
                               : *reinterpret_cast<const X*>(reinterpret_cast<const T*>(A.x.p) + xr + c);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int t = t0 + i;
                if (t >= sp.len) break;
                if (A.saved && t % BLOCK == 0) store_f32<V>(A.saved + (sp.block0 + t / BLOCK) * A.D + c, h);
                if (!per_channel<GM>) decays<T, GM>(Unpack<T>::get(g[i]), d, rest);
                Vec<V> u = in_values<T, V, RASTER>(xw[i], c);
                if (A.leaky) u = vmul(rest, u);
                const Vec<V> before = h;
                h = d.step(h, u);
                if constexpr (short_logit<T, GM>) {  // an infinite state stays so
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if (fabsf(before.v[k]) > FLT_MAX) h.v[k] = fmaf(d.a.v[k], before.v[k], u.v[k]);
                }
                *reinterpret_cast<Word<T, V>*>(reinterpret_cast<T*>(A.y.p) + row_at(A, A.y, s, sp, t) + c) =
                    Unpack<T>::put(h);
            }
        }
        if (A.h) store_f32<V>(A.h + s * A.D + c, h);
    }
    if (A.zero) zero_rest<T>(A, A.y, (long long)blockIdx.y * gridDim.x + blockIdx.x, (long long)gridDim.x * gridDim.y);
}

// the same rows where there is no sequence at all
template <typename T>
__global__ void __launch_bounds__(128) k_scan_zero(const ScanArgs A, Rows r) {
    zero_rest<T>(A, r, blockIdx.x, gridDim.x);
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

// The states (GRAD: r) that the chunks of a sequence start from, from their
// maps; in place of map_h.  A warp per consecutive part of the chunks joins its
// maps, the parts' maps give each its first state.
template <bool GRAD, bool KEEP, bool OVER>
__global__ void k_scan_join(const ScanArgs A) {
    __shared__ Vec<1> sa[32][32], sl[32][32], sh[32][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, groups = blockDim.x >> 5;
    const int c = (int)blockIdx.x * 32 + lane;
    for (long long s = blockIdx.y; s < A.n_seq; s += gridDim.y) {
        const Span sp = span_of(A, s);
        const int n = max(1, (sp.len + A.chunk - 1) / A.chunk);
        const long long j0 = chunk0_of(A, s);
        // position p of the chain: chunk j0 + p, or from the last one back
        auto at = [&](int p) { return (j0 + (GRAD ? n - 1 - p : p)) * A.D + c; };
        const int per = (n + groups - 1) / groups, lo = min(n, g * per), hi = min(n, lo + per);
        Vec<1> a = {1.0f}, l = {0.0f}, h = {0.0f};
        if (c < A.D)
#pragma unroll 8
            for (int p = lo; p < min(hi, n - 1); ++p) {
                const Vec<1> ma = {A.map_a[at(p)]}, ml = {KEEP ? A.map_l[at(p)] : 0.0f}, mh = {A.map_h[at(p)]};
                h = OVER ? mapped<KEEP>(ma, ml, h, mh) : plain<KEEP>(ma, ml, h, mh);
                if (KEEP) span_times(ma, ml, a, l);
                else a = vmul(ma, a);
            }
        sa[g][lane] = a;
        sl[g][lane] = l;
        sh[g][lane] = h;
        __syncthreads();
        if (c < A.D) {
            h.v[0] = !GRAD && A.h0 ? A.h0[s * A.D + c] : 0.0f;
            for (int k = 0; k < g; ++k) h = OVER ? mapped<KEEP>(sa[k][lane], sl[k][lane], h, sh[k][lane]) : plain<KEEP>(sa[k][lane], sl[k][lane], h, sh[k][lane]);
#pragma unroll 8
            for (int p = lo; p < hi; ++p) {
                const bool map = p < n - 1;
                const Vec<1> ma = {map ? A.map_a[at(p)] : 0.0f}, ml = {map && KEEP ? A.map_l[at(p)] : 0.0f};
                const Vec<1> mh = {map ? A.map_h[at(p)] : 0.0f};
                A.map_h[at(p)] = h.v[0];
                h = OVER ? mapped<KEEP>(ma, ml, h, mh) : plain<KEEP>(ma, ml, h, mh);
            }
        }
        __syncthreads();
    }
}

void check_desc(const snn_scan* d) {
    SNN_REQUIRE(d, SNN_ERR_ARG, "null scan description");
    SNN_REQUIRE(snnb::elem_type_ok(d->type), SNN_ERR_ARG, "scan: type must be SNN_F32, SNN_BF16 or SNN_F16");
    SNN_REQUIRE((d->flags & ~(SNN_SCAN_LOGIT | SNN_SCAN_LEAKY | SNN_SCAN_CHANNEL | SNN_SCAN_RASTER | SNN_SCAN_ZERO)) == 0,
                SNN_ERR_ARG, "scan: unknown flags");
    SNN_REQUIRE(d->n_seq >= 0 && d->n_seq < (1ll << 31), SNN_ERR_ARG, "scan: n_seq must lie in [0, 2^31)");
    SNN_REQUIRE(d->n_channels >= 1 && d->n_channels < (1ll << 30), SNN_ERR_ARG,
                "scan: n_channels must lie in [1, 2^30)");
    SNN_REQUIRE(d->n_steps >= 0 && d->n_steps <= (1ll << 30), SNN_ERR_ARG, "scan: n_steps must lie in [0, 2^30]");
    const int64_t rows = std::max<int64_t>(1, d->offsets ? d->n_steps + d->n_seq : d->n_steps * d->n_seq);
    SNN_REQUIRE(rows <= (1ll << 46) / d->n_channels, SNN_ERR_ARG, "scan: more than 2^46 elements");
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

void check_states(std::initializer_list<const void*> p) {
    for (const void* q : p) SNN_REQUIRE((uintptr_t)q % 4 == 0, SNN_ERR_ARG, "scan: misaligned states");
}

ScanArgs base_args(const snn_scan* d, const snn_rows* gate, const snn_rows* x) {
    SNN_REQUIRE((uintptr_t)d->offsets % 8 == 0, SNN_ERR_ARG, "scan: misaligned offsets");
    ScanArgs A;
    memset(&A, 0, sizeof(A));
    A.off = d->offsets;
    A.n_seq = d->n_seq;
    A.n_steps = (int)d->n_steps;
    A.D = (int)d->n_channels;
    A.logit = (d->flags & SNN_SCAN_LOGIT) != 0;
    A.leaky = (d->flags & SNN_SCAN_LEAKY) != 0;
    A.zero = d->offsets && (d->flags & SNN_SCAN_ZERO) != 0;
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

int gate_mode(const snn_scan* d) {
    return (d->flags & SNN_SCAN_CHANNEL ? GATE_CHANNEL : GATE_VALUE) + (d->flags & SNN_SCAN_LOGIT ? 1 : 0);
}

constexpr int SMS = 148;
int64_t mean_steps(const snn_scan* d) { return d->offsets ? d->n_steps / std::max<int64_t>(d->n_seq, 1) : d->n_steps; }

// Grid of the kernels.  The sizes alone decide (the sums of a channel gate's
// gradient follow the grid).  A cluster per (tile of channels, worker), a worker
// for each sequence up to 32 CTAs an SM, the rest taken in turn; where that
// leaves SMs empty, a cluster of up to MAX_CLUSTER CTAs along the steps.  Packed
// sequences may differ in length and end at different times: four times the
// CTAs, so that the longest is split too (24 sequences of 40,003 rows by 1,001
// channels, us by 2 / 4 / 8 CTAs an SM: forward 117 / 101 / 88, gradient 249 /
// 177 / 160, by 8 with the present joins 87 / 156).  The mean
// length stands for the longest: one sequence of 30,000 rows beside 255 of one
// row, by 2,048 channels in bf16, goes to single warps and takes 1.2 ms forward,
// where 16 of equal lengths take 0.14.
// Where even clusters leave most SMs empty for long, the sequences are cut into
// chunks: a first kernel reads them for their maps, a second joins the maps,
// and the chunks run as sequences of their own.  That reads the inputs twice and
// costs 20 us (gradient 25) however little there is, so it takes long
// sequences of few (tile, sequence) items, by clusters / by chunks in us:
//   1 x 50,000 x 64 f32 (2 items)           forward 102 / 31   gradient 221 / 39
//   39 packed, 1,997,736 rows x 33, per channel (39)  670 / 284          1267 / 592
//   1 x 50,021 x 1,000 f32 (32)                       162 / 198           292 / 234
//   2 packed, 20,106 x 59 f32 (4)                      33 / 29             61 / 39
//   100 packed, 2,000,000 x 30, per channel (100)     285 / 162           605 / 373
//   120 packed, 2,400,000 x 20 f32, per channel (120) 246 / 151           518 / 242
//   3 packed, 30,000 x 2,000 bf16 (96)                131 / 141           238 / 280
//   1 x 2,000 x 512 bf16 (8)                           12 / 23             16 / 29
Plan plan_of(const snn_scan* d, bool grad) {
    const int width = 128 / snnb::elem_size(d->type), tile = grad ? Bwd::TT : Fwd::TT;
    Plan p;
    p.ctiles = (int)((d->n_channels + width - 1) / width);
    p.workers = (int)std::min<int64_t>(d->n_seq, std::max(32, 32 * SMS / p.ctiles));
    p.cluster = 1;
    p.chunk = 0;
    p.n_chunks = 0;
    const int64_t rows = d->offsets ? d->n_steps : d->n_seq * d->n_steps, items = (int64_t)p.ctiles * d->n_seq;
    if (mean_steps(d) >= (grad ? 6144 : 12288) && items <= (d->offsets ? (p.ctiles <= 8 ? 160 : 48) : grad ? 36 : 16)) {
        const int64_t warps = SMS * (grad ? 8 : 12) * (d->flags & SNN_SCAN_CHANNEL ? 2 : 1);
        const int64_t c = (rows * p.ctiles + warps - 1) / warps;
        // (at least 96 steps: 1 x 20,000 x 300 bf16 gradient 65 us by 128, 59 by 96,
        // 59 by 64; 1 x 50,000 x 64 f32 forward 34, 33, 38)
        p.chunk = (int)std::max<int64_t>(96, (c + 15) / 16 * 16);
        p.n_chunks = rows / p.chunk + d->n_seq;
        p.workers = (int)std::min<int64_t>(p.n_chunks, std::max(32, 32 * SMS / p.ctiles));
        p.shape = 2;
        return p;
    }
    const int64_t wanted = (d->offsets ? 8 : 2) * SMS, ctas = (int64_t)p.ctiles * p.workers;
    while (p.cluster < MAX_CLUSTER && ctas * p.cluster < wanted && (int64_t)tile * p.cluster < mean_steps(d))
        p.cluster *= 2;
    // Without clusters: 16 x 4,096 x 2,048 in bf16 (512 items) gradient 335 us by
    // tiles, 273 by the smaller ones, 376 by single warps (forward 163 / - / 172);
    // a raster of 1,000 x 55,000 (1,719 items) forward 55 / - / 47, gradient 132 /
    // - / 81.
    p.shape = p.cluster > 1 || ctas < 3 * SMS ? 0 : ctas < 8 * SMS ? 1 : 2;
    return p;
}
// workspace: the maps of the chunks, then a channel gate's sums
int64_t map_floats(const snn_scan* d, const Plan& p) { return (p.n_chunks * d->n_channels + 63) / 64 * 64; }
int64_t work_bytes_of(const snn_scan* d, const Plan& p, bool grad) {
    const int64_t sums = grad && (d->flags & SNN_SCAN_CHANNEL) ? (int64_t)p.workers * p.cluster * d->n_channels : 0;
    return (3 * map_floats(d, p) + sums) * 4;
}
void check_work(const void* work, int64_t bytes, int64_t needed) {
    SNN_REQUIRE(needed == 0 || (work && (uintptr_t)work % 256 == 0 && bytes >= needed), SNN_ERR_ARG,
                "scan: workspace null, misaligned or too small");
}

// the kernels of a plan
template <bool GRAD>
void run_plan(const snn_scan* d, int words, const Plan& p, void* work, ScanArgs& A, cudaStream_t st) {
    A.chunk = p.chunk;
    A.n_chunks = p.n_chunks;
    A.map_a = (float*)work;
    A.map_l = (float*)work + map_floats(d, p);
    A.map_h = (float*)work + 2 * map_floats(d, p);
    const int gm = gate_mode(d);
    const bool raster = (d->flags & SNN_SCAN_RASTER) != 0;
    snnb::with_elem(d->type, [&](auto t) {
        using T = decltype(t);
        if (p.chunk) {
            launch_tiles<GRAD, T>(gm, raster, words, true, p, A, st);
            const int64_t mean = p.n_chunks / d->n_seq;
            int groups = 1;
            while (groups < 32 && groups * 4 < mean) groups *= 2;
            const dim3 grid((unsigned)((d->n_channels + 31) / 32), (unsigned)std::min<int64_t>(d->n_seq, 65535));
            if (A.logit) k_scan_join<GRAD, true, false><<<grid, 32 * groups, 0, st>>>(A);
            else if (gm == GATE_VALUE && sizeof(T) == 2) k_scan_join<GRAD, false, true><<<grid, 32 * groups, 0, st>>>(A);
            else k_scan_join<GRAD, true, true><<<grid, 32 * groups, 0, st>>>(A);
            SNN_CUDA(cudaGetLastError());  // the launch after it does not report this one
        }
        launch_tiles<GRAD, T>(gm, raster, words, false, p, A, st);
    });
}

// no sequence: all rows of r are rows of no sequence
void zero_rows(const snn_scan* d, const ScanArgs& A, const Rows& r, cudaStream_t st) {
    if (!A.zero || !r.p || d->n_steps == 0) return;
    snnb::with_elem(d->type, [&](auto t) {
        k_scan_zero<decltype(t)><<<(unsigned)std::min<int64_t>(d->n_steps, 8 * SMS), 128, 0, st>>>(A, r);
    });
    SNN_CUDA(cudaGetLastError());
}

// whether r's rows are words of `bytes` from the first element on
bool fits(const Rows& r, int size, int bytes) {
    return (uintptr_t)r.p % bytes == 0 && r.ss * size % bytes == 0 && r.st * size % bytes == 0;
}
// The words that rows are staged in (see Rower); written rows go in 4-byte
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

}  // namespace

namespace snnb {

int64_t leaky_scan_saved(const snn_scan* d) {
    check_desc(d);
    return saved_floats(d);
}

int64_t leaky_scan_workspace(const snn_scan* d, bool grad) {
    check_desc(d);
    return d->n_seq ? work_bytes_of(d, plan_of(d, grad), grad) : 0;
}

void leaky_scan(const snn_scan* d, const snn_rows* gate, const snn_rows* x, const float* h0,
                const snn_rows* y, float* h, float* saved, void* work, int64_t work_bytes, cudaStream_t st) {
    check_desc(d);
    if (d->n_seq == 0 && !(d->offsets && (d->flags & SNN_SCAN_ZERO))) return;
    ScanArgs A = base_args(d, gate, x);
    A.y = rows_of(d, y, "y", d->n_channels, elem_size(d->type), true);
    if (d->n_seq == 0) return zero_rows(d, A, A.y, st);
    check_states({h0, h, saved});
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
        with_elem(d->type, [&](auto t) {
            auto go = [&](auto gm) {
                using T = decltype(t);
                constexpr int GM = decltype(gm)::value;
                if (raster_x)
                    vec == 2 ? k_scan_steps<T, GM, true, 2><<<grid, 128, 0, st>>>(A)
                             : k_scan_steps<T, GM, true, 1><<<grid, 128, 0, st>>>(A);
                else
                    vec == 2 ? k_scan_steps<T, GM, false, 2><<<grid, 128, 0, st>>>(A)
                             : k_scan_steps<T, GM, false, 1><<<grid, 128, 0, st>>>(A);
            };
            const int gm = gate_mode(d);
            if (gm == GATE_VALUE) go(std::integral_constant<int, GATE_VALUE>());
            else if (gm == GATE_LOGIT) go(std::integral_constant<int, GATE_LOGIT>());
            else if (gm == GATE_CHANNEL) go(std::integral_constant<int, GATE_CHANNEL>());
            else go(std::integral_constant<int, GATE_CHANNEL_LOGIT>());
        });
        SNN_CUDA(cudaGetLastError());
        return;
    }
    const Plan p = plan_of(d, false);
    check_work(work, work_bytes, work_bytes_of(d, p, false));
    run_plan<false>(d, words, p, work, A, st);
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
        if (!(d->offsets && (d->flags & SNN_SCAN_ZERO))) return;
    }
    const int size = elem_size(d->type);
    SNN_REQUIRE(saved || d->n_seq == 0, SNN_ERR_ARG, "scan: null saved");
    ScanArgs A = base_args(d, gate, x);
    check_states({saved, dh, dh0});
    A.saved = const_cast<float*>(saved);
    A.dh = dh;
    A.dh0 = dh0;
    if (dy) A.y = rows_of(d, dy, "dy", d->n_channels, size);
    if (dx) A.dx = rows_of(d, dx, "dx", d->n_channels, size, true);
    if (dgate && channel) {
        SNN_REQUIRE(dgate->data && (uintptr_t)dgate->data % 4 == 0, SNN_ERR_ARG, "scan: null or misaligned dgate");
        A.dgate = {dgate->data, 0, 0};
    } else if (dgate) {
        A.dgate = rows_of(d, dgate, "dgate", d->n_channels, size, true);
    }
    if (d->n_seq == 0) {
        zero_rows(d, A, A.dx, st);
        if (!channel) zero_rows(d, A, A.dgate, st);
        return;
    }
    const Rows none = {nullptr, 0, 0};
    const int words = copy_words(d, {channel ? none : A.gate, d->flags & SNN_SCAN_RASTER ? none : A.x, A.y},
                                 {channel ? none : A.dgate, A.dx});
    const Plan p = plan_of(d, true);
    check_work(work, work_bytes, work_bytes_of(d, p, true));
    if (channel && dgate) A.part = (float*)work + 3 * map_floats(d, p);
    run_plan<true>(d, words, p, work, A, st);
    if (A.part) {
        k_scan_gate_sum<<<(unsigned)((d->n_channels + 31) / 32), 256, 0, st>>>(A, p.workers * p.cluster);
        SNN_CUDA(cudaGetLastError());
    }
}

}  // namespace snnb
