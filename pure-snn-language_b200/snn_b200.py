"""Python binding of the B200 SNN core (libsnn_b200.so, C ABI in
include/snn_b200.h).

Mirrors the reference host API (TSOFTP-afk/pure-snn-language):
``Network`` plays the role of ``stage2e::BioMechanismScheduler`` +
``MemoryAllocator`` (src/stage2e/scheduler.cuh:66-224) and of
``SNNNetwork`` (src/include/network.h:11-95): build by columns and layers,
step / run with byte injection, read state and counters, save / load.

The library must be built (``make -C pure-snn-language_b200``); importing this
module on a machine without the built library, or creating a network without
a CUDA device, raises instead of falling back to anything else.
"""
import ctypes as C
import functools
import os
import struct

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsnn_b200.so")
# the same core built with the reference's arithmetic (CUDA expf, compiler
# contraction of plain expressions) instead of the canonical one
REFMATH_LIB_PATH = os.path.join(HERE, "libsnn_b200_refmath.so")

SNN_OK = 0
ERRORS = {1: "SNN_ERR_ARG", 2: "SNN_ERR_CUDA", 3: "SNN_ERR_OOM", 4: "SNN_ERR_STATE",
          5: "SNN_ERR_IO", 6: "SNN_ERR_UNSUPPORTED", 7: "SNN_ERR_NO_DEVICE"}
MODEL_STAGE2E, MODEL_STAGE0, MODEL_PROP = 0, 1, 2
PROP_PLAIN, PROP_STDP, PROP_STP = 0, 1, 2
PRESET_REF, PRESET_BASELINE = 0, 1
CORPUS_TEXT_FILTER = 1
QK_UNIT, QK_ADJACENT = 1, 2
SCAN_LOGIT, SCAN_LEAKY, SCAN_CHANNEL, SCAN_RASTER, SCAN_ZERO = 1, 2, 4, 8, 32
FMT_NATIVE, FMT_SNN2_V1, FMT_SCKP_V2, FMT_RAW_F32 = 0, 1, 2, 3

STATE = {
    "V": (0, np.float32, "N"), "w": (1, np.float32, "N"), "s": (2, np.float32, "N"),
    "fr": (3, np.float32, "N"), "ca_neuron": (4, np.float32, "N"),
    "input": (5, np.float32, "N"), "nmda_cur": (6, np.float32, "N"),
    "last": (7, np.int32, "N"), "ref": (8, np.int32, "N"), "x_post": (9, np.float32, "N"),
    "thresh_off": (10, np.int32, "N"),
    "alpha": (20, np.float32, "S"), "beta": (21, np.float32, "S"),
    "weight": (22, np.float32, "S"), "x_pre": (23, np.float32, "S"),
    "nmda": (24, np.float32, "S"), "ca": (25, np.float32, "S"),
    "R": (26, np.float32, "S"), "u": (27, np.float32, "S"), "elig": (28, np.float32, "S"),
    "camkii_act": (29, np.float32, "S"), "autophos": (30, np.float32, "S"),
    "e1": (31, np.float32, "S"), "e2": (32, np.float32, "S"),
    "ampa": (33, np.float32, "S"), "last_pre": (34, np.float32, "S"),
    "post": (40, np.int32, "S"), "delay": (41, np.uint8, "S"), "row_ptr": (42, np.int32, "N1"),
    "flags": (43, np.uint8, "S"), "gates": (50, np.float32, "G4"),
    "modulators": (51, np.float32, "4"), "byte_hist": (52, np.int32, "256"),
    "neuron_byte_counts": (53, np.int32, "N256"),
}


class SnnError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code


class Config(C.Structure):
    _fields_ = [("model", C.c_int32), ("preset", C.c_int32), ("device", C.c_int32),
                ("e0", C.c_int32), ("phase_offset", C.c_int32), ("raster_steps", C.c_int32),
                ("prop_mode", C.c_int32), ("prop_rate", C.c_float), ("prop_w_max", C.c_float),
                ("prop_push", C.c_int32), ("reserved", C.c_int32 * 6)]


class TopologySpec(C.Structure):
    _fields_ = [("n_columns", C.c_int32), ("l4", C.c_int32), ("l23", C.c_int32),
                ("l5", C.c_int32), ("l6", C.c_int32), ("pf_groups", C.c_int32),
                ("pf_group_size", C.c_int32), ("deg_intra", C.c_int32), ("deg_inter", C.c_int32),
                ("deg_l5_pf", C.c_int32), ("deg_pf_self", C.c_int32),
                ("deg_pf_assoc", C.c_int32), ("total_synapses", C.c_int64),
                ("seed", C.c_uint32), ("rule", C.c_int32), ("reserved", C.c_int32 * 8)]


class Counters(C.Structure):
    _fields_ = [("step", C.c_int64), ("total_spikes", C.c_int64), ("arrivals", C.c_int64),
                ("dispatched", C.c_int64), ("dropped_ref", C.c_int64),
                ("ltp_visits", C.c_int64), ("burst_spikes", C.c_int64),
                ("n_neurons", C.c_int64), ("n_synapses", C.c_int64), ("n_groups", C.c_int64),
                ("last_spikes", C.c_int32), ("last_byte", C.c_int32),
                ("modeled_bytes", C.c_double), ("local_lo", C.c_int64), ("local_hi", C.c_int64),
                ("reserved", C.c_int64 * 4)]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_ if k != "reserved"}


class Semantic(C.Structure):
    _fields_ = [("silhouette", C.c_double), ("js_mean", C.c_double), ("js_max", C.c_double),
                ("column_ratio", C.c_double), ("grand_total", C.c_double),
                ("n_columns", C.c_int32), ("nonzero_columns", C.c_int32),
                ("layer_delay", C.c_double * 5), ("layer_delay_n", C.c_int32 * 5),
                ("layer_sig", C.c_int32 * 5), ("layer_act", C.c_int32 * 5),
                ("layer_chi2_mean", C.c_double * 5), ("reserved", C.c_int32 * 8)]

    def as_dict(self):
        out = {}
        for k, _ in self._fields_:
            if k == "reserved":
                continue
            v = getattr(self, k)
            out[k] = list(v) if hasattr(v, "__len__") else v
        return out


class Profile(C.Structure):
    _fields_ = [("steps", C.c_int64), ("n_kernels", C.c_int32), ("reserved0", C.c_int32),
                ("kernel_ms", C.c_double * 8), ("launches", C.c_int64 * 8),
                ("step_ms", C.c_double), ("names", (C.c_char * 32) * 8)]

    def as_dict(self):
        k = self.n_kernels
        return {"steps": self.steps, "step_ms": self.step_ms,
                "kernels": {self.names[i].value.decode(): {"ms": self.kernel_ms[i],
                                                           "launches": self.launches[i]}
                            for i in range(k)}}


EXPORTS = ["snn_config_init", "snn_topology_init", "snn_create", "snn_destroy",
           "snn_last_error", "snn_version", "snn_build_columns", "snn_set_corpus", "snn_step",
           "snn_run", "snn_synchronize", "snn_get_spikes", "snn_get_state", "snn_get_counters",
           "snn_set_dopamine", "snn_set_e0", "snn_save", "snn_load", "snn_stream_generate",
           "snn_set_profiling", "snn_get_profile", "snn_propagate", "snn_propagate_static",
           "snn_nccl_unique_id", "snn_set_shard", "snn_shard_plan", "snn_semantic_eval",
           "snn_set_corpus_ex", "snn_load_text_corpus", "snn_byte_classes", "snn_embed",
           "snn_embed_grad", "snn_embed_grad_workspace", "snn_leaky_scan", "snn_leaky_scan_saved", "snn_leaky_scan_workspace",
           "snn_leaky_scan_grad", "snn_leaky_scan_grad_workspace", "snn_qk_norm", "snn_qk_norm_grad",
           "snn_qk_norm_grad_workspace", "snn_adamw", "snn_delta_scan", "snn_delta_scan_saved",
           "snn_delta_scan_workspace", "snn_delta_scan_grad", "snn_delta_scan_grad_workspace"]

_lib = None
_lib_refmath = None


def lib(refmath=False):
    """Load libsnn_b200.so, or with refmath=True libsnn_b200_refmath.so
    (raises if it was not built)."""
    global _lib, _lib_refmath
    if refmath:
        if _lib_refmath is None:
            _lib_refmath = _load(REFMATH_LIB_PATH)
        return _lib_refmath
    if _lib is None:
        _lib = _load(LIB_PATH)
    return _lib


def _load(path):
    if not os.path.exists(path):
        raise OSError(f"{path} is missing: build it with `make -C {HERE}`")
    L = C.CDLL(path)
    vp = C.c_void_p
    L.snn_config_init.argtypes = [C.POINTER(Config), C.c_int32, C.c_int32]
    L.snn_topology_init.argtypes = [C.POINTER(TopologySpec), C.c_int32, C.c_int32]
    L.snn_create.argtypes = [C.POINTER(Config), C.POINTER(vp)]
    L.snn_destroy.argtypes = [vp]
    L.snn_destroy.restype = None
    L.snn_last_error.argtypes = [vp]
    L.snn_last_error.restype = C.c_char_p
    L.snn_version.restype = C.c_char_p
    L.snn_build_columns.argtypes = [vp, C.POINTER(TopologySpec)]
    L.snn_set_corpus.argtypes = [vp, vp, C.c_int64]
    L.snn_set_corpus_ex.argtypes = [vp, vp, C.c_int64, C.c_int32, vp]
    L.snn_load_text_corpus.argtypes = [vp, C.c_char_p, vp]
    L.snn_byte_classes.argtypes = [vp, C.c_int64, vp, C.c_int32]
    L.snn_step.argtypes = [vp, C.c_int32, C.c_int32, C.c_int32]
    L.snn_run.argtypes = [vp, C.c_int32, vp, C.c_int64, C.c_int32, vp, vp]
    L.snn_synchronize.argtypes = [vp]
    L.snn_get_spikes.argtypes = [vp, vp, C.c_int64]
    L.snn_get_state.argtypes = [vp, C.c_int32, vp, C.c_int64]
    L.snn_get_counters.argtypes = [vp, C.POINTER(Counters)]
    L.snn_semantic_eval.argtypes = [vp, C.c_int64, C.POINTER(Semantic), vp, C.c_int64]
    L.snn_set_dopamine.argtypes = [vp, C.c_float]
    L.snn_set_e0.argtypes = [vp, C.c_int32]
    L.snn_save.argtypes = [vp, C.c_char_p, C.c_int32]
    L.snn_load.argtypes = [vp, C.c_char_p, C.c_int32]
    L.snn_stream_generate.argtypes = [vp, C.c_int64, C.c_uint64, C.c_double, C.c_double]
    L.snn_set_profiling.argtypes = [vp, C.c_int32]
    L.snn_get_profile.argtypes = [vp, C.POINTER(Profile)]
    L.snn_propagate.argtypes = [vp, vp, C.c_int64, C.c_int32, vp, vp, C.c_int64, C.c_int32, vp]
    L.snn_propagate_static.argtypes = L.snn_propagate.argtypes
    L.snn_nccl_unique_id.argtypes = [vp, C.c_int64]
    L.snn_set_shard.argtypes = [vp, C.c_int32, C.c_int32, vp, C.c_int64]
    i32, i64 = C.c_int32, C.c_int64
    L.snn_embed.argtypes = [vp, i32, i64, vp, i32, i64, i64, i64, C.c_float, vp, i32, i64, vp]
    L.snn_embed_grad_workspace.argtypes = [i64, i64, i64, vp]
    L.snn_embed_grad.argtypes = [vp, i32, i64, vp, i32, i64, i64, C.c_float, vp, i32, i64, i64,
                                 i32, vp, i64, vp]
    ps = pr = C.c_char_p  # snn_scan, snn_rows: packed bytes
    L.snn_leaky_scan_saved.argtypes = [ps, vp]
    L.snn_leaky_scan.argtypes = [ps, pr, pr, vp, pr, vp, vp, vp, i64, vp]
    L.snn_leaky_scan_workspace.argtypes = [ps, vp]
    L.snn_leaky_scan_grad_workspace.argtypes = [ps, vp]
    L.snn_leaky_scan_grad.argtypes = [ps, pr, pr, vp, pr, vp, pr, pr, vp, vp, i64, vp]
    L.snn_qk_norm.argtypes = [ps, pr, pr, vp, vp, vp, vp, pr, pr, vp]
    L.snn_qk_norm_grad_workspace.argtypes = [ps, vp]
    L.snn_qk_norm_grad.argtypes = [ps, pr, pr, vp, vp, vp, vp, pr, pr, pr, pr, vp, vp, vp, i64, vp]
    L.snn_delta_scan_saved.argtypes = [ps, vp]
    L.snn_delta_scan_workspace.argtypes = [ps, i32, vp]
    L.snn_delta_scan_grad_workspace.argtypes = [ps, vp]
    L.snn_delta_scan.argtypes = [ps, pr, pr, pr, pr, pr, vp, pr, vp, vp, i64, vp, i64, vp]
    L.snn_delta_scan_grad.argtypes = [ps, pr, pr, pr, pr, pr, vp, i64, pr, vp, pr, pr, pr, pr, pr, vp, vp, i64, vp]
    L.snn_adamw.argtypes = [vp, i64, i32, ps, vp]
    L.snn_shard_plan.argtypes = [C.POINTER(TopologySpec), C.c_int32, C.c_int32, vp, C.c_int32]
    return L


def propagate(post, w, fanout, spikes, acc, frac_bits=24, stream=None, static=False):
    """snn_propagate on torch CUDA tensors (int32 post[n_pre*fanout],
    float32 w[...], uint8 spikes[n_pre], int32 acc[n_post], accumulated in
    place) on `stream` (a torch.cuda.Stream, default: the current stream).
    static=True calls snn_propagate_static (no allocation, n_pre <= 2^20)."""
    import torch
    for t_, dt in ((post, torch.int32), (w, torch.float32), (spikes, torch.uint8), (acc, torch.int32)):
        if not (t_.is_cuda and t_.dtype == dt and t_.is_contiguous()):
            raise SnnError(1, "propagate wants contiguous CUDA tensors int32/float32/uint8/int32")
    st = stream if stream is not None else torch.cuda.current_stream(acc.device)
    fn = lib().snn_propagate_static if static else lib().snn_propagate
    rc = fn(post.data_ptr(), w.data_ptr(), spikes.numel(), fanout, spikes.data_ptr(),
            acc.data_ptr(), acc.numel(), frac_bits, st.cuda_stream)
    if rc:
        raise SnnError(rc, lib().snn_last_error(None).decode())


_T = None  # torch, from the first call of an operator on


def _torch():
    global _T, _ELEM, _TOKEN
    import torch
    _ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    _TOKEN = {torch.uint8: 8, torch.int32: 9, torch.int64: 10}
    _T = torch
    return torch


def _elem(dtype):
    """SNN_F32 / SNN_BF16 / SNN_F16 of a torch dtype."""
    c = _ELEM.get(dtype)
    if c is None:
        raise SnnError(1, f"element type must be float32, bfloat16 or float16, not {dtype}")
    return c


def _require(ok, msg):
    if not ok:
        raise SnnError(1, msg)


def _check(rc):
    if rc:
        raise SnnError(rc, lib().snn_last_error(None).decode())


def _call(fn, dev, stream, *args):
    """fn(*args, stream) with `dev` current, on `stream` (default: the
    device's current stream)."""
    if stream is None:
        raw = _T._C._cuda_getCurrentRawStream(dev.index)
    else:
        _require(stream.device == dev, f"the stream is on {stream.device}, the tensors on {dev}")
        raw = stream.cuda_stream
    if _T._C._cuda_getDevice() == dev.index:
        rc = fn(*args, raw)
    else:
        with _T.cuda.device(dev):
            rc = fn(*args, raw)
    if rc:
        raise SnnError(rc, lib().snn_last_error(None).decode())


def _new(dev, stream, shape, dtype):
    """A contiguous new tensor whose memory belongs to `stream` (the one it is used on)."""
    if stream is not None:
        with _T.cuda.stream(stream):
            return _T.empty(shape, dtype=dtype, device=dev)
    n = len(shape)  # with strides given an allocation takes 1.5 us, without 2.3
    if n == 2:
        return _T.empty_strided(shape, (shape[1], 1), dtype=dtype, device=dev)
    if n == 3:
        return _T.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=dtype, device=dev)
    if n == 1:
        return _T.empty_strided(shape, (1,), dtype=dtype, device=dev)
    return _T.empty(shape, dtype=dtype, device=dev)


def _cuda(t, name, dev):
    if t.device != dev:
        raise SnnError(1, f"{name} must be a CUDA tensor on {dev}, not on {t.device}")


def _tokens(tokens):
    """(device, type code) of a token tensor."""
    if not (tokens.is_cuda and tokens.is_contiguous()):
        raise SnnError(1, "tokens must be a contiguous CUDA tensor")
    code = _TOKEN.get(tokens.dtype)
    if code is None:
        raise SnnError(1, f"tokens must be uint8, int32 or int64, not {tokens.dtype}")
    return tokens.device, code


def _row_stride(t, name):
    """The stride of t's rows (its last dimension, of unit stride)."""
    if t.is_contiguous():
        return t.shape[-1]
    _require(t.dim() == 2 and (t.shape[1] == 1 or t.stride(1) == 1), f"{name} wants unit column "
             "stride and, unless it is contiguous, two dimensions")
    return t.stride(0)


def embed(tokens, table, scale=1.0, dtype=None, out=None, stream=None):
    """The drive rows of a token stream (snn_embed): scale * table[tokens].

    tokens: contiguous uint8 / int32 / int64 CUDA tensor of any shape; table
    [vocab, dim] in float32 / bfloat16 / float16, unit column stride.  Returns
    tokens.shape + (dim,) in `dtype` (default: the table's), or `out`.  A
    token outside [0, vocab) gives zeros.  Runs on `stream` (default: the
    current stream of the tensors' device), on which new results are made.
    autograd does not see these operators: embed_grad is the gradient."""
    if _T is None:
        _torch()
    dev, tok = _tokens(tokens)
    if table.device != dev:
        _cuda(table, "table", dev)
    size = table.shape
    if len(size) != 2 or size[0] < 1 or size[1] < 1:
        raise SnnError(1, "table must be [vocab, dim] and not empty")
    vocab, dim = size
    shape = (*tokens.shape, dim)
    if out is None:
        dtype = dtype or table.dtype
        out = _new(dev, stream, shape, dtype)
        ostride = dim
    else:
        _cuda(out, "out", dev)
        _require(out.shape == shape and (dtype is None or dtype == out.dtype),
                 "out must be tokens.shape + (dim,) of the wanted dtype")
        dtype = out.dtype
        ostride = _row_stride(out, "out")
    _call(_lib.snn_embed if _lib else lib().snn_embed, dev, stream, tokens.data_ptr(), tok, tokens.numel(),
          table.data_ptr(), _elem(table.dtype), vocab, dim, _row_stride(table, "table"), scale,
          out.data_ptr(), _elem(dtype), ostride)
    return out


@functools.lru_cache(maxsize=1024)
def _embed_work(n, vocab, dim):
    """Workspace bytes of embed_grad's sizes."""
    size = C.c_int64()
    _check(lib().snn_embed_grad_workspace(n, vocab, dim, C.byref(size)))
    return size.value


def embed_grad(tokens, dy, vocab=None, scale=1.0, dtype=None, out=None, accumulate=False, stream=None):
    """Gradient of `embed` for its table (snn_embed_grad): [vocab, dim] with
    scale * the sum of dy over the positions of each token, in f32 over the
    positions sorted by token (equal calls give equal bits), rounded once.

    tokens as for `embed`; dy tokens.shape + (dim,).  Returns a new tensor of
    `dtype` (default float32), or `out`; with accumulate=True the sum is added
    to `out` and rows that do not occur are not touched."""
    if _T is None:
        _torch()
    dev, tok = _tokens(tokens)
    _cuda(dy, "dy", dev)
    n = tokens.numel()
    if dy.dim() < 1 or dy.shape[:-1] != tokens.shape or dy.shape[-1] < 1:
        raise SnnError(1, "dy must be tokens.shape + (dim,)")
    dim = dy.shape[-1]
    if out is None:
        _require(vocab is not None and vocab >= 1 and not accumulate,
                 "give a positive vocab, or out (accumulate wants out)")
        out = _new(dev, stream, (vocab, dim), dtype or _T.float32)
        ostride = dim
    else:
        _cuda(out, "out", dev)
        _require(out.dim() == 2 and out.shape[1] == dim and out.shape[0] >= 1
                 and vocab in (None, out.shape[0]) and (dtype is None or dtype == out.dtype),
                 "out must be [vocab, dim] of the wanted dtype")
        vocab = out.shape[0]
        ostride = _row_stride(out, "out")
    size = _embed_work(n, vocab, dim)
    work = _new(dev, stream, (size,), _T.uint8)
    _call(lib().snn_embed_grad, dev, stream, tokens.data_ptr(), tok, n, dy.data_ptr(), _elem(dy.dtype),
          dim, _row_stride(dy, "dy"), scale, out.data_ptr(), _elem(out.dtype), vocab, ostride,
          1 if accumulate else 0, work.data_ptr(), size)
    return out


_SCAN = struct.Struct("=iiqqqQ")  # snn_scan
_ROWS = struct.Struct("=Qqq")     # snn_rows


def _scan_rows(t, name, shape, dtype):
    """snn_rows of a tensor [steps, c] (packed) or [sequences, steps, c]."""
    if t.shape != shape or t.dtype != dtype:
        raise SnnError(1, f"{name} must be {tuple(shape)} in {dtype}, not {tuple(t.shape)} in {t.dtype}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] != 1:
        raise SnnError(1, f"{name} wants unit channel stride")
    return _ROWS.pack(t.data_ptr(), st[0], st[-2])


def _scan_args(gate, x, logit, leaky, offsets, dtype, zero):
    """(snn_scan, gate rows, x rows, dtype of y, its shape, the states' shape, _scan_sizes); zero: rows of no
    sequence become zero in what the call writes"""
    if _T is None:
        _torch()
    dev, xt, shape = x.device, x.dtype, x.shape
    if dev.type != "cuda":
        raise SnnError(1, "x must be a CUDA tensor")
    if gate.device != dev:
        _cuda(gate, "gate", dev)
    if len(shape) != (3 if offsets is None else 2):
        raise SnnError(1, "x must be [sequences, steps, channels], or [rows, channels] with offsets")
    flags = (SCAN_LOGIT if logit else 0) | (SCAN_LEAKY if leaky else 0)
    if xt in _ELEM:
        if dtype is not None and dtype != xt:
            raise SnnError(1, "y has x's dtype")
        dtype, d = xt, shape[-1]
        xr = _scan_rows(x, "x", shape, xt)
    else:
        _require(xt in (_T.int32, _T.uint32),
                 "x must be float32, bfloat16 or float16, or the int32 or uint32 words of a raster")
        dtype, d = dtype or _T.float32, gate.shape[-1]
        flags |= SCAN_RASTER
        xr = _scan_rows(x, "x", (*shape[:-1], (d + 31) // 32), xt)
        shape = (*shape[:-1], d)
    if d < 1:
        raise SnnError(1, "no channels")
    if offsets is None:
        n_seq, off = shape[0], 0
    else:
        _cuda(offsets, "offsets", dev)
        _require(offsets.dtype == _T.int64 and offsets.dim() == 1 and offsets.is_contiguous()
                 and offsets.numel() >= 1, "offsets must be contiguous int64 [sequences + 1]")
        n_seq, off = offsets.numel() - 1, offsets.data_ptr()
        if zero:
            flags |= SCAN_ZERO
    if gate.dim() == 1:
        _require(gate.shape[0] == d and gate.dtype == _T.float32 and gate.is_contiguous(),
                 "a gate per channel must be contiguous float32 [channels]")
        g = _ROWS.pack(gate.data_ptr(), 0, 0)
        flags |= SCAN_CHANNEL
    else:
        g = _scan_rows(gate, "gate", shape, dtype)
    kind = _elem(dtype)
    return (_SCAN.pack(kind, flags, n_seq, shape[-2], d, off), g, xr, dtype, shape, (n_seq, d),
            _scan_sizes(kind, flags, n_seq, shape[-2], d, offsets is not None))


def _state(t, name, shape, dev):
    """Address of a float32 state tensor, or None."""
    if t is None:
        return None
    _cuda(t, name, dev)
    if t.shape != shape or t.dtype != _T.float32 or not t.is_contiguous():
        raise SnnError(1, f"{name} must be contiguous float32 {tuple(shape)}")
    return t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _scan_sizes(kind, flags, n_seq, n_steps, channels, packed):
    """(floats of saved, workspace bytes forward, gradient) of a scan's sizes."""
    desc, size, L, out = _SCAN.pack(kind, flags, n_seq, n_steps, channels, 8 if packed else 0), C.c_int64(), lib(), []
    for fn in (L.snn_leaky_scan_saved, L.snn_leaky_scan_workspace, L.snn_leaky_scan_grad_workspace):
        _check(fn(desc, C.byref(size)))
        out.append(size.value)
    return tuple(out)


def leaky_scan(gate, x, h0=None, logit=False, leaky=False, offsets=None, dtype=None, out=None,
               h_out=None, save=False, stream=None):
    """Leaky integration along whole sequences (snn_leaky_scan):
    h_t = a_t h_{t-1} + u_t with a = gate, or 1 / (1 + exp(-gate)) (logit),
    and u = x, or (1 - a) x (leaky).

    x: [sequences, steps, channels] or, with offsets (int64 [sequences + 1]),
    packed [rows, channels] in float32 / bfloat16 / float16; or the spike
    raster of Network.run (int32 / uint32 words, y in `dtype`, default
    float32).  gate: x's form and dtype, or float32 [channels].  h0: float32
    [sequences, channels] (default zeros).  Returns (y, h), h the float32
    states after the last steps; with save=True also what leaky_scan_grad
    needs.  `out` takes y; `h_out` takes h and may be h0, so that a stream of
    single steps keeps its state in place.  Rows of no sequence (before
    offsets[0], from offsets[-1] on) are zero in a new y and not written in
    `out`.  autograd does not see this call: leaky_scan_grad is the gradient."""
    desc, g, xr, dtype, shape, state, sizes = _scan_args(gate, x, logit, leaky, offsets, dtype, out is None)
    dev = x.device
    if out is None:
        out = _new(dev, stream, shape, dtype)
        d = shape[-1]
        yr = _ROWS.pack(out.data_ptr(), shape[-2] * d, d)
    else:
        _cuda(out, "out", dev)
        yr = _scan_rows(out, "out", shape, dtype)
    if h_out is None:
        h_out = _new(dev, stream, state, _T.float32)
        hp = h_out.data_ptr()
    else:
        hp = _state(h_out, "h_out", state, dev)
    saved = sp = wp = None
    if save:
        saved = _new(dev, stream, (sizes[0],), _T.float32)
        sp = saved.data_ptr()
    if sizes[1]:
        work = _new(dev, stream, (sizes[1],), _T.uint8)
        wp = work.data_ptr()
    _call(lib().snn_leaky_scan, dev, stream, desc, g, xr,
          None if h0 is None else _state(h0, "h0", state, dev), yr, hp, sp, wp, sizes[1])
    return (out, h_out, saved) if save else (out, h_out)


def leaky_scan_grad(gate, x, dy, saved, dh=None, logit=False, leaky=False, offsets=None,
                    need_gate=True, need_x=True, need_h0=True, stream=None):
    """Gradients of leaky_scan (snn_leaky_scan_grad) from those of y (dy, None
    for none) and of the final states (dh): returns (dgate, dx, dh0), each
    None where it is not needed (dx of a raster never is).  gate, x, logit,
    leaky and offsets as in the forward call with save=True, `saved` its
    result.  dgate has gate's shape and dtype (a gate per channel: the sum over
    all steps), dx x's, dh0 is float32 [sequences, channels].  Rows of no
    sequence have the gradient 0."""
    raster = not x.dtype.is_floating_point
    kind = None  # a raster's gradients have dy's type, without dy that of a gate per step
    if raster:
        kind = dy.dtype if dy is not None else gate.dtype if gate.dim() > 1 else None
    desc, g, xr, dtype, shape, state, sizes = _scan_args(gate, x, logit, leaky, offsets, kind, True)
    dev = x.device
    if dy is None and dh is None:
        raise SnnError(1, "neither dy nor dh is given")
    _cuda(saved, "saved", dev)
    if saved.dtype != _T.float32 or saved.numel() != sizes[0] or not saved.is_contiguous():
        raise SnnError(1, "saved is not what the forward call of these sizes gives")
    dyr = dgate = dgr = dx = dxr = dh0 = hp = wp = None
    d = shape[-1]
    if dy is not None:
        _cuda(dy, "dy", dev)
        dyr = _scan_rows(dy, "dy", shape, dtype)
    if need_gate:
        dgate = _new(dev, stream, gate.shape, gate.dtype)
        dgr = _ROWS.pack(dgate.data_ptr(), shape[-2] * d, d)
    if need_x and not raster:
        dx = _new(dev, stream, shape, dtype)
        dxr = _ROWS.pack(dx.data_ptr(), shape[-2] * d, d)
    if need_h0:
        dh0 = _new(dev, stream, state, _T.float32)
        hp = dh0.data_ptr()
    if sizes[2]:
        work = _new(dev, stream, (sizes[2],), _T.uint8)
        wp = work.data_ptr()
    _call(lib().snn_leaky_scan_grad, dev, stream, desc, g, xr, saved.data_ptr(), dyr,
          None if dh is None else _state(dh, "dh", state, dev), dgr, dxr, hp, wp, sizes[2])
    return dgate, dx, dh0


_QK = struct.Struct("=iiqqqqqqif")  # snn_qk
_HEADS = struct.Struct("=Qqqq")     # snn_heads


def _heads(t, name, shape, dtype):
    """snn_heads of a tensor [rows, heads, dim] or [sequences, steps, heads, dim]."""
    if t.shape != shape or t.dtype != dtype:
        raise SnnError(1, f"{name} must be {tuple(shape)} in {dtype}, not {tuple(t.shape)} in {t.dtype}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] != 1:
        if t.numel() == 0:  # (torch gives these any strides)
            return _HEADS.pack(0, 0, 0, 0)
        raise SnnError(1, f"{name} wants unit stride in its last dimension")
    return _HEADS.pack(t.data_ptr(), st[0], st[-3], st[-2])


def _new_heads(dev, stream, shape, dtype):
    """(a new tensor of heads, its snn_heads)"""
    d = shape[-1]
    n = shape[-2] * d
    if stream is not None:
        t = _new(dev, stream, tuple(shape), dtype)
    elif len(shape) == 4:  # (as in _new)
        t = _T.empty_strided(shape, (shape[1] * n, n, d, 1), dtype=dtype, device=dev)
    else:
        t = _T.empty_strided(shape, (n, d, 1), dtype=dtype, device=dev)
    return t, _HEADS.pack(t.data_ptr(), shape[-3] * n, n, d)


def _qk_args(q, k, wq, wk, positions, freqs, eps, unit, adjacent):
    """(device, snn_qk, (rows of q, of k), (addresses of the weights), address of positions, of freqs)"""
    if _T is None:
        _torch()
    some = q if q is not None else k
    _require(some is not None, "neither q nor k is given")
    dev, shape, dtype = some.device, some.shape, some.dtype
    if dev.type != "cuda":
        raise SnnError(1, "q and k must be CUDA tensors")
    if len(shape) not in (3, 4) or shape[-1] < 1:
        raise SnnError(1, "q and k must be [rows, heads, dim] or [sequences, steps, heads, dim]")
    dim, lead = shape[-1], shape[:-2]
    hq = hk = 0
    rq = rk = pq = pk = pp = fp = None
    if q is not None:
        hq = shape[-2]
        rq, pq = _heads(q, "q", shape, dtype), _qk_weight(wq, "q_weight", dim, dev)
    if k is not None:
        if k.device != dev:
            _cuda(k, "k", dev)
        hk = k.shape[-2] if k.dim() == len(shape) else 0
        rk, pk = _heads(k, "k", (*lead, hk, dim), dtype), _qk_weight(wk, "k_weight", dim, dev)
    rot, pos_type = 0, 9
    if (positions is None) != (freqs is None):
        raise SnnError(1, "positions and freqs are given together")
    if freqs is not None:
        if freqs.device != dev or positions.device != dev:
            _cuda(freqs, "freqs", dev)
            _cuda(positions, "positions", dev)
        rot, pos_type = 2 * freqs.numel(), _TOKEN.get(positions.dtype)
        if freqs.dim() != 1 or freqs.dtype != _T.float32 or not freqs.is_contiguous() or rot > dim:
            raise SnnError(1, "freqs must be contiguous float32 of at most dim / 2 elements")
        if positions.shape != lead or pos_type not in (9, 10) or not positions.is_contiguous():
            raise SnnError(1, "positions must be contiguous int32 or int64, one for each row")
        pp, fp = positions.data_ptr(), freqs.data_ptr()
    n_seq, n_steps = lead if len(lead) == 2 else (1, lead[0])
    desc = _QK.pack(_elem(dtype), (QK_UNIT if unit else 0) | (QK_ADJACENT if adjacent else 0), n_seq, n_steps, hq, hk, dim, rot,
                    pos_type, eps)
    return dev, desc, (rq, rk), (pq, pk), pp, fp


def _qk_weight(w, name, dim, dev):
    """Address of a side's weights, or None."""
    if w is None:
        return None
    _cuda(w, name, dev)
    if w.shape != (dim,) or w.dtype != _T.float32 or not w.is_contiguous():
        raise SnnError(1, f"{name} must be contiguous float32 [dim]")
    return w.data_ptr()


def _qk_results(dev, stream, q, k, out):
    """(the results for q and k, new or those of out; their snn_heads)"""
    res, to = [None, None], [None, None]
    for i, x in enumerate((q, k)):
        if x is None:
            continue
        if out[i] is None:
            res[i], to[i] = _new_heads(dev, stream, x.shape, x.dtype)
        else:
            _cuda(out[i], "out", dev)
            res[i], to[i] = out[i], _heads(out[i], "out", x.shape, x.dtype)
    return res, to


def qk_norm(q, k, q_weight=None, k_weight=None, positions=None, freqs=None, eps=1e-6, unit=False,
            adjacent=False, out=(None, None), stream=None):
    """Norms of queries and keys for each head, then the position rotation
    (snn_qk_norm): y = turn(x / sqrt(mean x^2 + eps) * weight); unit=True takes
    the sum in place of the mean (rows of unit length).

    q, k: [rows, heads, dim] or [sequences, steps, heads, dim] in float32 / bfloat16
    / float16, any strides but a unit one of dim; the heads may differ in number,
    either may be None.  Weights: float32 [dim].  positions: int32 / int64, one for each row,
    and freqs: float32, the angle a position of each rotated pair (at most dim / 2 pairs; the
    elements behind them are not rotated); pairs lie half of the rotated elements
    apart, with adjacent=True beside one another.  Returns (yq, yk), new
    tensors or `out`, which may be (q, k).  autograd does not see this call:
    qk_norm_grad is the gradient."""
    dev, desc, rows, weights, pp, fp = _qk_args(q, k, q_weight, k_weight, positions, freqs, eps, unit, adjacent)
    res, to = _qk_results(dev, stream, q, k, out)
    _call(lib().snn_qk_norm, dev, stream, desc, *rows, *weights, pp, fp, *to)
    return tuple(res)


@functools.lru_cache(maxsize=1024)
def _qk_work(desc):
    size = C.c_int64()
    _check(lib().snn_qk_norm_grad_workspace(desc, C.byref(size)))
    return size.value


def qk_norm_grad(q, k, dyq, dyk, q_weight=None, k_weight=None, positions=None, freqs=None, eps=1e-6,
                 unit=False, adjacent=False, out=(None, None), stream=None):
    """Gradients of qk_norm (snn_qk_norm_grad) from those of its results: (dq, dk,
    dq_weight, dk_weight), the last two float32 [dim], None without that weight.
    Arguments as for qk_norm; `out` takes (dq, dk) and may be (dyq, dyk)."""
    dev, desc, rows, weights, pp, fp = _qk_args(q, k, q_weight, k_weight, positions, freqs, eps, unit, adjacent)
    dy, dw, dwp = [None, None], [None, None], [None, None]
    for i, (x, g, name) in enumerate(((q, dyq, "dyq"), (k, dyk, "dyk"))):
        if x is None:
            continue
        _require(g is not None, f"{name} is missing")
        _cuda(g, name, dev)
        dy[i] = _heads(g, name, x.shape, x.dtype)
        if weights[i] is not None:
            dw[i] = _new(dev, stream, (x.shape[-1],), _T.float32)
            dwp[i] = dw[i].data_ptr()
    res, to = _qk_results(dev, stream, q, k, out)
    size, wp = 0, None
    if dwp != [None, None]:
        size = _qk_work(desc)
        work = _new(dev, stream, (size,), _T.uint8)
        wp = work.data_ptr()
    _call(lib().snn_qk_norm_grad, dev, stream, desc, *rows, *weights, pp, fp, *dy, *to, *dwp, wp, size)
    return (*res, *dw)


_DELTA = struct.Struct("=iiqqqqqqQfi")  # snn_delta


def _gate_rows(t, name, shape, dtype):
    """_scan_rows, of tensors without elements too (torch gives these any strides)"""
    if t.shape == shape and t.dtype == dtype and t.numel() == 0:
        return _ROWS.pack(0, 0, 0)
    return _scan_rows(t, name, shape, dtype)


def _delta_args(q, k, v, gate, beta, scale, logit, offsets, zero):
    """(snn_delta, (snn_heads of q, k, v, snn_rows of gate, beta), the states' shape, _delta_sizes)"""
    if _T is None:
        _torch()
    dev, dtype, shape, qs = v.device, v.dtype, v.shape, q.shape
    if dev.type != "cuda":
        raise SnnError(1, "v must be a CUDA tensor")
    for t, name in ((q, "q"), (k, "k"), (gate, "gate"), (beta, "beta")):
        if t.device != dev:
            _cuda(t, name, dev)
    if len(shape) != (4 if offsets is None else 3) or len(qs) != len(shape):
        raise SnnError(1, "q, k and v must be [sequences, steps, heads, dim], or [rows, heads, dim] with offsets")
    lead, heads, dv, hk, dk = shape[:-2], shape[-2], shape[-1], qs[-2], qs[-1]
    if not (hk and dk and dv and heads and heads % hk == 0):
        raise SnnError(1, "the heads of v must be a multiple of those of q and k, no dimension of heads empty")
    rows = (_heads(q, "q", (*lead, hk, dk), dtype), _heads(k, "k", (*lead, hk, dk), dtype), _heads(v, "v", shape, dtype),
            _gate_rows(gate, "gate", (*lead, heads), dtype), _gate_rows(beta, "beta", (*lead, heads), dtype))
    flags = SCAN_LOGIT if logit else 0
    if offsets is None:
        n_seq, off = shape[0], 0
    else:
        _cuda(offsets, "offsets", dev)
        _require(offsets.dtype == _T.int64 and offsets.dim() == 1 and offsets.is_contiguous()
                 and offsets.numel() >= 1, "offsets must be contiguous int64 [sequences + 1]")
        n_seq, off = offsets.numel() - 1, offsets.data_ptr()
        if zero:
            flags |= SCAN_ZERO
    kind, n = _elem(dtype), shape[-3]
    return (_DELTA.pack(kind, flags, n_seq, n, hk, heads, dk, dv, off, scale, 0), rows, (n_seq, heads, dk, dv),
            _delta_sizes(kind, n_seq, n, hk, heads, dk, dv, offsets is not None))


@functools.lru_cache(maxsize=1024)
def _delta_sizes(kind, n_seq, n, hk, heads, dk, dv, packed):
    """(bytes of saved, workspace bytes forward, with saved, gradient) of a delta-rule scan's sizes."""
    desc, size, L, out = _DELTA.pack(kind, 0, n_seq, n, hk, heads, dk, dv, 8 if packed else 0, 1.0, 0), C.c_int64(), lib(), []
    for fn, how in ((L.snn_delta_scan_saved, ()), (L.snn_delta_scan_workspace, (0,)), (L.snn_delta_scan_workspace, (1,)),
                    (L.snn_delta_scan_grad_workspace, ())):
        _check(fn(desc, *how, C.byref(size)))
        out.append(size.value)
    return tuple(out)


def delta_scan(q, k, v, gate, beta, h0=None, scale=1.0, logit=False, offsets=None, out=None, h_out=None,
               save=False, stream=None):
    """Delta-rule scan along whole sequences (snn_delta_scan): a state matrix S of
    fast synapses for each head, S' = a_t S, u = b_t (v_t - S'^T k_t), S = S' + k_t u^T,
    y_t = scale S^T q_t with a = exp(gate), b = beta, or both logistic (logit).

    q, k: [sequences, steps, key heads, dk] or, with offsets (int64 [sequences
    + 1]), packed [rows, key heads, dk]; v likewise with `heads`, a multiple of the key
    heads, and dv; gate, beta: [.., heads]; all float32, bfloat16 or float16 alike, of any
    strides but a unit last one; dk <= 128, dv <= 1024.  Keys are wanted of unit length
    (qk_norm with unit=True).  h0: float32 [sequences, heads, dk, dv] (default
    zeros).  Returns (y, h), h the float32 states after the last steps; with
    save=True also what delta_scan_grad needs.  `out` takes y; `h_out` takes h and
    may be h0, so that a stream of single steps keeps its state in place.  Rows of no
    sequence are zero in a new y and not written in `out`.  autograd does not see this
    call: delta_scan_grad is the gradient."""
    desc, rows, state, sizes = _delta_args(q, k, v, gate, beta, scale, logit, offsets, out is None)
    dev = v.device
    if out is None:
        out, yr = _new_heads(dev, stream, v.shape, v.dtype)
    else:
        _cuda(out, "out", dev)
        yr = _heads(out, "out", v.shape, v.dtype)
    if h_out is None:
        h_out = _new_heads(dev, stream, state, _T.float32)[0]
        hp = h_out.data_ptr()
    else:
        hp = _state(h_out, "h_out", state, dev)
    saved = sp = wp = None
    if save:
        saved = _new(dev, stream, (sizes[0],), _T.uint8)
        sp = saved.data_ptr()
    size = sizes[2] if save else sizes[1]
    if size:
        work = _new(dev, stream, (size,), _T.uint8)
        wp = work.data_ptr()
    _call(lib().snn_delta_scan, dev, stream, desc, *rows, None if h0 is None else _state(h0, "h0", state, dev), yr, hp,
          sp, sizes[0], wp, size)
    return (out, h_out, saved) if save else (out, h_out)


def delta_scan_grad(q, k, v, gate, beta, dy, saved, dh=None, scale=1.0, logit=False, offsets=None, need_h0=True,
                    stream=None):
    """Gradients of delta_scan (snn_delta_scan_grad) from those of y (dy, None for
    none) and of the final states (dh): (dq, dk, dv, dgate, dbeta, dh0) of the forms of their
    inputs, dh0 None where it is not needed.  The other arguments as in the forward call
    with save=True, `saved` its result.  Rows of no sequence have the gradient 0."""
    desc, rows, state, sizes = _delta_args(q, k, v, gate, beta, scale, logit, offsets, True)
    dev, dtype = v.device, v.dtype
    if dy is None and dh is None:
        raise SnnError(1, "neither dy nor dh is given")
    _cuda(saved, "saved", dev)
    if saved.dtype != _T.uint8 or saved.numel() != sizes[0] or not saved.is_contiguous():
        raise SnnError(1, "saved is not what the forward call of these sizes gives")
    dyr = None
    if dy is not None:
        _cuda(dy, "dy", dev)
        dyr = _heads(dy, "dy", v.shape, dtype)
    dq, dqr = _new_heads(dev, stream, q.shape, dtype)
    dk, dkr = _new_heads(dev, stream, k.shape, dtype)
    dv, dvr = _new_heads(dev, stream, v.shape, dtype)
    dgate, dbeta = _new(dev, stream, gate.shape, dtype), _new(dev, stream, gate.shape, dtype)
    n = gate.shape[-1]
    gr, br = (_ROWS.pack(t.data_ptr(), gate.shape[-2] * n, n) for t in (dgate, dbeta))
    dh0 = hp = wp = None
    if need_h0:
        dh0 = _new(dev, stream, state, _T.float32)
        hp = dh0.data_ptr()
    if sizes[3]:
        work = _new(dev, stream, (sizes[3],), _T.uint8)
        wp = work.data_ptr()
    _call(lib().snn_delta_scan_grad, dev, stream, desc, *rows, saved.data_ptr(), sizes[0], dyr,
          None if dh is None else _state(dh, "dh", state, dev), dqr, dkr, dvr, gr, br, hp, wp, sizes[3])
    return dq, dk, dv, dgate, dbeta, dh0


_ADAMW_TENSOR = np.dtype([(i, np.uint64) for i in ("p", "g", "m", "v", "ms", "vs", "copy")] + [
    ("n", np.int64), ("g_type", np.int32), ("copy_type", np.int32)])  # snn_adamw_tensor
_ADAMW_RULE = struct.Struct("=ddddddqQ")                              # snn_adamw_rule


class AdamW:
    """AdamW over a list of parameters (snn_adamw), a launch for up to 400 tensors.

    params: contiguous float32 CUDA tensors of one device, no two of which overlap.
    bits: how the moments are held, 32, or 8 (e4m3 values with a float32 scale
    for every 256 elements; of second moments the root).  copies: None, or
    for each parameter a bfloat16 or float16 tensor that takes its rounded
    values (entries may be None).  The moments are the lists m and v (with
    8 bits float8_e4m3fn, their scales in m_scale and v_scale), zeros at
    first; moments=(m, v, m_scale, v_scale) takes those of an earlier run over.
    All these tensors stay where they are: a step refuses one that has been replaced
    or has moved (m[i].copy_(..) restores a moment)."""

    def __init__(self, params, bits=32, copies=None, moments=None):
        T = _torch()
        self.params, self.bits = list(params), bits
        _require(bits in (32, 8), "moments have 32 or 8 bits")
        _require(len(self.params) > 0, "no parameters")
        self.device = dev = self.params[0].device
        kind = T.float32 if bits == 32 else T.float8_e4m3fn
        n = len(self.params)
        blocks = [0 if bits == 32 else (p.numel() + 255) // 256 for p in self.params]
        if moments is None:
            moments = tuple([T.zeros(p.shape, device=dev).to(kind) for p in self.params] for _ in range(2)) + tuple(
                [T.zeros(b, device=dev) for b in blocks] for _ in range(2))
        self.m, self.v, self.m_scale, self.v_scale = (list(x) for x in moments)
        self.copies = [None] * n if copies is None else list(copies)
        _require(all(len(x) == n for x in (self.m, self.v, self.m_scale, self.v_scale, self.copies)),
                 "moments, scales and copies are as many as the parameters")
        self._table, used, self._held = np.zeros(n, _ADAMW_TENSOR), [], []
        for i, p in enumerate(self.params):
            held = [("p", p, p.shape, T.float32), ("m", self.m[i], p.shape, kind), ("v", self.v[i], p.shape, kind)]
            if bits == 8:
                held += [("ms", self.m_scale[i], (blocks[i],), T.float32), ("vs", self.v_scale[i], (blocks[i],), T.float32)]
            if self.copies[i] is not None:
                c = self.copies[i]
                _require(c.dtype in (T.bfloat16, T.float16), "copies are bfloat16 or float16")
                held.append(("copy", c, p.shape, c.dtype))
                self._table["copy_type"][i] = _ELEM[c.dtype]
            for name, t, shape, dtype in held:
                _require(t.is_cuda and t.device == dev and t.shape == shape and t.dtype == dtype and t.is_contiguous(),
                         f"{name} of parameter {i} must be a contiguous CUDA tensor {tuple(shape)} in {dtype} on {dev}")
                self._table[name][i] = t.data_ptr()
                self._held.append(t.detach())  # (while this holds it, its memory becomes nothing else's)
                if t.numel():
                    used.append((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()))
            self._table["n"][i] = p.numel()
        used.sort()
        _require(all(a[1] <= b[0] for a, b in zip(used, used[1:])), "parameters, moments, scales or copies overlap")
        self._shapes, self._at, self._table_at = [p.shape for p in self.params], self._addresses(), self._table.ctypes.data

    def _addresses(self):
        """Where all that a step writes lies now."""
        try:
            held = self.params + self.m + self.v
            if self.bits == 8:
                held += self.m_scale + self.v_scale
            return list(map(_T.Tensor.data_ptr, held)) + [0 if t is None else t.data_ptr() for t in self.copies]
        except (AttributeError, TypeError):  # something else than a tensor
            return None

    def step(self, grads, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, grad_scale=1.0, stream=None):
        """One step, in place: grads, one for each parameter (contiguous, float32 / bfloat16
        / float16, its shape; None leaves a parameter and its moments alone); step, counted from 1, a
        number or an int64 CUDA tensor of one element, which is read when the step
        runs (for captured steps)."""
        dev, table = self.device, self._table  # (the call reads it before it returns)
        _require(len(grads) == len(self._shapes), "grads are as many as the parameters")
        if self._addresses() != self._at:
            raise SnnError(1, "a parameter's, moment's, scale's or copy's memory is not what it was when this was made")
        at, kinds = [], []
        for g, shape in zip(grads, self._shapes):
            if g is None:
                at.append(0)
                kinds.append(0)
                continue
            if g.shape != shape or g.device != dev or not g.is_contiguous():
                raise SnnError(1, f"grads must be contiguous tensors of the parameters' shapes on {dev}")
            at.append(g.data_ptr())
            kinds.append(_elem(g.dtype))
        table["g"], table["g_type"] = at, kinds
        there = 0
        if isinstance(step, _T.Tensor):
            _cuda(step, "step", dev)
            _require(step.dtype == _T.int64 and step.numel() == 1, "step must be a number or one int64")
            there, step = step.data_ptr(), 0
        rule = _ADAMW_RULE.pack(lr, *betas, eps, weight_decay, grad_scale, step, there)
        _call(lib().snn_adamw, dev, stream, self._table_at, len(at), self.bits, rule)


def nccl_unique_id():
    """128-byte NCCL unique id (bytes) for snn_set_shard; make it on one rank
    and share it with the others."""
    buf = (C.c_uint8 * 128)()
    rc = lib().snn_nccl_unique_id(buf, 128)
    if rc:
        raise SnnError(rc, lib().snn_last_error(None).decode())
    return bytes(buf)


def shard_plan(spec, rank, world):
    """Host-only partition plan of a Stage 2e topology (no GPU needed)."""
    out = np.zeros(10, np.int64)
    rc = lib().snn_shard_plan(C.byref(spec), rank, world, out.ctypes.data, 10)
    if rc:
        raise SnnError(rc, lib().snn_last_error(None).decode())
    keys = ["n_local", "a0", "a1", "pf0", "pf1", "synapses", "groups_local", "groups_mirror",
            "mirror_pres", "remote_short_delay"]
    return {k: int(v) for k, v in zip(keys, out)}


def stream(n, seed=42, p_cjk=0.452, zipf_s=1.1):
    """Seeded synthetic UTF-8 byte stream (numpy uint8[n]).  p_cjk=0.452 is
    the `ref45` preset (about 47.5 % continuation bytes), 0.85 is `b85`."""
    out = np.zeros(n, np.uint8)
    rc = lib().snn_stream_generate(out.ctypes.data, n, seed, p_cjk, zipf_s)
    if rc:
        raise SnnError(rc, "snn_stream_generate")
    return out


def byte_classes(b):
    """Fractions of ASCII (< 0x80), UTF-8 lead (0xC0..0xF7) and continuation
    (0x80..0xBF) bytes (snn_byte_classes)."""
    a = np.ascontiguousarray(np.frombuffer(bytes(b), np.uint8))
    out = np.zeros(3, np.int64)
    rc = lib().snn_byte_classes(a.ctypes.data, a.size, out.ctypes.data, 3)
    if rc:
        raise SnnError(rc, "snn_byte_classes")
    n = max(a.size, 1)
    return {"ascii": float(out[0]) / n, "head": float(out[1]) / n,
            "continuation": float(out[2]) / n}


def topology(model=MODEL_STAGE2E, n_columns=50, **overrides):
    spec = TopologySpec()
    rc = lib().snn_topology_init(C.byref(spec), model, n_columns)
    if rc:
        raise SnnError(rc, "snn_topology_init")
    for k, v in overrides.items():
        setattr(spec, k, v)
    return spec


class Network:
    """One network on one GPU (one snn_ctx)."""

    def __init__(self, model=MODEL_STAGE2E, preset=PRESET_REF, device=0, e0=False,
                 phase_offset=0, raster_steps=1024, prop_mode=0, prop_rate=0.01, prop_w_max=0.0,
                 prop_push=0, refmath=False):
        """refmath=True runs the network on the core built with the
        reference's arithmetic (libsnn_b200_refmath.so)."""
        L = lib(refmath)
        self.L = L
        cfg = Config()
        self._check(L.snn_config_init(C.byref(cfg), model, preset), None)
        cfg.device, cfg.e0, cfg.phase_offset, cfg.raster_steps = device, int(e0), phase_offset, raster_steps
        if model == MODEL_PROP:
            cfg.prop_mode, cfg.prop_rate, cfg.prop_w_max = prop_mode, prop_rate, prop_w_max
            cfg.prop_push = prop_push
        h = C.c_void_p()
        rc = L.snn_create(C.byref(cfg), C.byref(h))
        if rc:
            raise SnnError(rc, L.snn_last_error(None).decode())
        self.h = h
        self.model = model
        self.N = self.S = 0

    def _check(self, rc, h="self"):
        if rc:
            msg = self.L.snn_last_error(self.h if h == "self" else None)
            raise SnnError(rc, msg.decode() if msg else "")

    def close(self):
        if getattr(self, "h", None):
            self.L.snn_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def build_columns(self, spec):
        self._check(self.L.snn_build_columns(self.h, C.byref(spec)))
        c = self.counters()
        self.N, self.S = c["n_neurons"], c["n_synapses"]
        self.words = (self.N + 31) // 32
        self.n_columns = spec.n_columns
        return self

    def set_corpus(self, data, text_filter=False):
        """The byte stream the network reads (one byte per inject step,
        wrapping).  text_filter=True applies the reference's corpus filter
        (NUL dropped, CR / LF / TAB -> space); returns the kept length."""
        b = np.ascontiguousarray(np.frombuffer(bytes(data), np.uint8))
        kept = C.c_int64(0)
        self._check(self.L.snn_set_corpus_ex(self.h, b.ctypes.data, b.size,
                                             CORPUS_TEXT_FILTER if text_filter else 0,
                                             C.byref(kept)))
        return kept.value

    def load_text_corpus(self, path):
        """Read a text file, filter it like the reference's load_text_corpus
        and make it the corpus; returns the kept length."""
        kept = C.c_int64(0)
        self._check(self.L.snn_load_text_corpus(self.h, os.fsencode(path), C.byref(kept)))
        return kept.value

    def step(self, step, inject_byte=-1, learn=True):
        self._check(self.L.snn_step(self.h, step, inject_byte, int(learn)))

    def run(self, n_steps, data=None, learn=True, raster=False, counts=False):
        """Run n_steps; returns (raster uint32[n_steps, words] or None,
        counts int32[n_steps] or None)."""
        r = np.zeros((n_steps, self.words), np.uint32) if raster else None
        c = np.zeros(n_steps, np.int32) if counts else None
        b = None
        if data is not None:
            b = np.ascontiguousarray(np.frombuffer(bytes(data), np.uint8))
        self._check(self.L.snn_run(self.h, n_steps, b.ctypes.data if b is not None else None,
                                   b.size if b is not None else 0, int(learn),
                                   r.ctypes.data if r is not None else None,
                                   c.ctypes.data if c is not None else None))
        return r, c

    def synchronize(self):
        self._check(self.L.snn_synchronize(self.h))

    def spikes(self):
        w = np.zeros(self.words, np.uint32)
        self._check(self.L.snn_get_spikes(self.h, w.ctypes.data, w.size))
        return np.unpackbits(w.view(np.uint8), bitorder="little")[: self.N]

    def state(self, name):
        which, dt, shape = STATE[name]
        if self.model == MODEL_PROP and name in ("R", "u"):
            shape = "N"  # per pre-synaptic neuron in the microbench
        n = {"N": self.N, "S": self.S, "N1": self.N + 1, "4": 4, "256": 256,
             "N256": self.N * 256, "G4": 4 * self.n_columns}[shape]
        out = np.zeros(n, dt)
        self._check(self.L.snn_get_state(self.h, which, out.ctypes.data, out.nbytes))
        return out.reshape(-1, 4) if shape == "G4" else out

    def counters(self):
        c = Counters()
        self._check(self.L.snn_get_counters(self.h, C.byref(c)))
        return c.as_dict()

    def semantic_eval(self, step=None):
        """Semantic evaluation of a Stage 2e network (snn_semantic_eval):
        dict of the scalars and per-layer lists, plus each column's cluster
        under "assign".  step defaults to the number of executed steps."""
        out = Semantic()
        n_col = max(int(getattr(self, "n_columns", 0) or 0), 1)
        asg = np.zeros(n_col, np.int32)
        st = self.counters()["step"] if step is None else int(step)
        self._check(self.L.snn_semantic_eval(self.h, st, C.byref(out), asg.ctypes.data, asg.size))
        d = out.as_dict()
        d["assign"] = asg[: d["n_columns"]]
        return d

    def set_profiling(self, enable=True):
        """True / 1: per-kernel device times; 2: whole-run device time only
        (Stage 2e); False / 0: off."""
        self._check(self.L.snn_set_profiling(self.h, int(enable)))

    def profile(self):
        p = Profile()
        self._check(self.L.snn_get_profile(self.h, C.byref(p)))
        return p.as_dict()

    def set_shard(self, rank, world, uid=None):
        """Column sharding (before build_columns): rank of world, NCCL id."""
        b = (C.c_uint8 * 128).from_buffer_copy(uid) if uid is not None else None
        self._check(self.L.snn_set_shard(self.h, rank, world, b, 128 if b is not None else 0))
        self.rank, self.world = rank, world

    def set_dopamine(self, level):
        self._check(self.L.snn_set_dopamine(self.h, level))

    def set_e0(self, enable):
        self._check(self.L.snn_set_e0(self.h, int(enable)))

    def save(self, path, fmt=FMT_NATIVE):
        self._check(self.L.snn_save(self.h, path.encode(), fmt))

    def load(self, path, fmt=FMT_NATIVE):
        self._check(self.L.snn_load(self.h, path.encode(), fmt))
