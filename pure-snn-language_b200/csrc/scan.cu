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
    float* part;   // per-worker sums of a channel gate's gradient
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

template <typename T, int GM, bool RASTER>
__global__ void __launch_bounds__(128) k_scan_grad_seq(const ScanArgs A) {
    const int c = (int)(blockIdx.x * 128 + threadIdx.x);
    if (c >= A.D) return;
    float sum = 0.0f;
    const Decay fixed = GM == GATE_CHANNEL ? decay_channel(A, c) : Decay();
    for (long long s = blockIdx.y; s < A.n_seq; s += gridDim.y) {
        const Span sp = span_of(A, s);
        float r = A.dh ? A.dh[s * A.D + c] : 0.0f;  // gradient that reaches h_t from later steps
        for (long long b = (sp.len + BLOCK - 1) / BLOCK - 1; b >= 0; --b) {
            float past[BLOCK];
            float h = A.saved[(sp.block0 + b) * A.D + c];
            const int n = (int)min((long long)BLOCK, sp.len - b * BLOCK);
            for (int i = 0; i < n; ++i) {
                const long long t = b * BLOCK + i;
                past[i] = h;
                const Decay d = decay_at<T, GM>(A, row_at(A, A.gate, s, sp, t), c, fixed);
                float u = input_at<T, RASTER>(A, row_at(A, A.x, s, sp, t), c);
                if (A.leaky) u = d.rest() * u;
                h = d.step(h, u);
            }
            for (int i = n - 1; i >= 0; --i) {
                const long long t = b * BLOCK + i;
                const Decay d = decay_at<T, GM>(A, row_at(A, A.gate, s, sp, t), c, fixed);
                float g = r;
                if (A.y.p) g += to_f32(reinterpret_cast<const T*>(A.y.p)[row_at(A, A.y, s, sp, t) + c]);
                float e = past[i];
                if (A.leaky) e -= input_at<T, RASTER>(A, row_at(A, A.x, s, sp, t), c);
                const float da = g * e;
                if (GM == GATE_CHANNEL) sum += da;
                else if (A.dgate.p)
                    reinterpret_cast<T*>(A.dgate.p)[row_at(A, A.dgate, s, sp, t) + c] =
                        from_f32<T>(GM == GATE_LOGIT ? da * d.slope() : da);
                if (A.dx.p)
                    reinterpret_cast<T*>(A.dx.p)[row_at(A, A.dx, s, sp, t) + c] = from_f32<T>(A.leaky ? d.rest() * g : g);
                r = d.times(g);
            }
        }
        if (A.dh0) A.dh0[s * A.D + c] = r;
    }
    if (GM == GATE_CHANNEL && A.part) A.part[(long long)blockIdx.y * A.D + c] = sum;
}

// dgate of a channel gate: the workers' sums in ascending order
__global__ void __launch_bounds__(128) k_scan_gate_sum(const ScanArgs A, int workers) {
    const int c = (int)(blockIdx.x * 128 + threadIdx.x);
    if (c >= A.D) return;
    float sum = 0.0f;
    for (int w = 0; w < workers; ++w) sum += A.part[(long long)w * A.D + c];
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

int seq_workers(const snn_scan* d) { return (int)std::min<int64_t>(d->n_seq, 1024); }

}  // namespace

namespace snnb {

int64_t leaky_scan_saved(const snn_scan* d) {
    check_desc(d);
    return saved_floats(d);
}

int64_t leaky_scan_grad_workspace(const snn_scan* d) {
    check_desc(d);
    return d->flags & SNN_SCAN_CHANNEL ? (int64_t)seq_workers(d) * d->n_channels * 4 : 0;
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
    const dim3 grid((unsigned)((d->n_channels + 127) / 128), (unsigned)seq_workers(d));
    dispatch(d, [&](auto t, auto gm, auto raster) {
        k_scan_seq<decltype(t), decltype(gm)::value, decltype(raster)::value != 0><<<grid, 128, 0, st>>>(A);
    });
    SNN_CUDA(cudaGetLastError());
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
    const dim3 grid((unsigned)((d->n_channels + 127) / 128), (unsigned)seq_workers(d));
    dispatch(d, [&](auto t, auto gm, auto raster) {
        k_scan_grad_seq<decltype(t), decltype(gm)::value, decltype(raster)::value != 0><<<grid, 128, 0, st>>>(A);
    });
    if (A.part) k_scan_gate_sum<<<grid.x, 128, 0, st>>>(A, seq_workers(d));
    SNN_CUDA(cudaGetLastError());
}

}  // namespace snnb
