"""Layers of an acoustic network beside the decoder (include/psgpu.h, PSGPU_CAP_NET): a shared projection with a low-rank adapter per
utterance, group norm with an activation, and the senone scores of a network's outputs -- what the reference takes from a file
(ps_decode_senscr, reference src/pocketsphinx.c:1199-1218), made on the device for FwdtreeSearch.search.  Arithmetic in
csrc/psgpu_proj.hip, psgpu_gnorm.hip, psgpu_netscr.hip.

Tensors are torch's, on the device: rows [frames][width], rows of utterances back to back, with any row stride; float32, float16 or
bfloat16.  utt_off is an int32 tensor [n_utt + 1] of row offsets; rows of no utterance are left as they are in the output (in an
output that these functions make themselves they hold nothing defined).  Calls are queued on torch's current stream of the tensors' device and
can be captured into a graph; workspaces come from torch's allocator, call by call.  They compute forward alone: a tensor that asks for a
gradient is refused where torch records one, and so is one with a tangent of forward-mode differentiation."""
import ctypes as C

import numpy as np

from . import capi

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


_DTYPES = {}


def _dtypes():
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _DTYPES


class _On:
    """the device current in a scope, for calls that are made where it is already; gives torch's current stream there, as a handle"""
    __slots__ = ("index", "back")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        import torch
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        try:
            return torch._C._cuda_getCurrentRawStream(self.index)      # (a third of a small call's time less than the stream object)
        except AttributeError:
            return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.back != self.index:
            import torch
            torch.cuda.set_device(self.back)


def _no_gradient(t, name):
    import torch
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s asks for a gradient, and there is none here (torch.no_grad())" % name)
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError("%s has a tangent, and there is no forward-mode gradient here (detach())" % name)


def _rows(t, name, width=None, dtype=None, device=None, rows=None):
    """checks a 2-d device tensor of rows; returns its row stride in elements"""
    import torch
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError("%s: a tensor [frames][width] is needed" % name)
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device if device is not None else "a GPU"))
    if dtype is not None and t.dtype != dtype:
        raise ValueError("%s has type %s, not %s" % (name, t.dtype, dtype))
    if t.requires_grad or torch.autograd.forward_ad._current_level >= 0:       # (outside of a level nothing has a tangent)
        _no_gradient(t, name)
    (n, w), (stride, step) = t.shape, t.stride()
    if width is not None and w != width:
        raise ValueError("%s has rows of %d, not of %d" % (name, w, width))
    if rows is not None and n != rows:
        raise ValueError("%s has %d rows, not %d" % (name, n, rows))
    if n > 0x7fffffff:
        raise ValueError("%s has %d rows" % (name, n))
    if w > 1 and step != 1:
        raise ValueError("%s: a row's elements must lie side by side" % name)
    if n <= 1:
        return max(w, 1)
    if stride < w:
        raise ValueError("%s: rows overlap" % name)
    return stride


def _vector(t, name, n, dtype, device):
    import torch
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.dtype != dtype or t.device != device or (n is not None and t.shape[0] != n):
        raise ValueError("%s: a tensor %s of %s on %s is needed" % (name, "[%d]" % n if n is not None else "[n]", dtype, device))
    if dtype is not torch.int32 and (t.requires_grad or torch.autograd.forward_ad._current_level >= 0):
        _no_gradient(t, name)
    return t if t.is_contiguous() else t.contiguous()


def _offsets(utt_off, device):
    import torch
    utt_off = _vector(utt_off, "utt_off", None, torch.int32, device)
    if not utt_off.shape[0]:
        raise ValueError("utt_off: at least one offset")
    return utt_off, utt_off.shape[0] - 1


def _int32(v, name):
    """a whole number that the C calls can take (ctypes cuts off what 32 bits do not hold: 2^32 would be 0)"""
    if type(v) is int and -0x80000000 <= v <= 0x7fffffff:
        return v
    n = int(v)
    if n != v or not -0x80000000 <= n <= 0x7fffffff:
        raise ValueError("%s: %r is no whole number of 32 bits" % (name, v))
    return n


def _p(t):
    return None if t is None else t.data_ptr()


def _matrix(w, shape_name, dtype=None):
    """a weight as a contiguous tensor, where it lies"""
    import torch
    t = w if torch.is_tensor(w) else torch.from_numpy(np.ascontiguousarray(w))
    if t.dim() != 2 or t.dtype not in _dtypes() or (dtype is not None and t.dtype != dtype):
        raise ValueError("%s: a matrix of %s is needed" % (shape_name, dtype if dtype is not None else "float32, float16 or bfloat16"))
    return t.detach().contiguous()


class AdaptedProjection:
    """y[t] = bias + W x[t] + scale_a B_a (A_a x[t]): one projection for all, a low-rank adapter for each utterance (psgpu_proj_*).

    weight [d_out][d_in] (torch on the host or the device, or numpy; its type is the layer's), bias [d_out] or None; up to max_adapters adapters of ranks up to
    max_rank are loaded with set_adapter.  The object lives on the device that is current here."""

    def __init__(self, weight, bias=None, max_adapters=0, max_rank=64):
        import torch
        w = _matrix(weight, "weight [d_out][d_in]")
        self.dtype = w.dtype
        self.d_out, self.d_in = int(w.shape[0]), int(w.shape[1])
        self.max_adapters, self.max_rank = _int32(max_adapters, "max_adapters"), _int32(max_rank, "max_rank")
        b = None
        if bias is not None:
            b = (bias if torch.is_tensor(bias) else torch.from_numpy(np.ascontiguousarray(bias))).detach().float().contiguous()
            if tuple(b.shape) != (self.d_out,):
                raise ValueError("bias: [%d] is needed" % self.d_out)
        h = C.c_void_p()
        capi.check(capi.lib().psgpu_proj_create(C.byref(h), _dtypes()[self.dtype], self.d_in, self.d_out, _p(w), _p(b), self.max_adapters,
                                                self.max_rank), "psgpu_proj_create")
        self.h = h
        self.device = torch.device("cuda", torch.cuda.current_device())

    def set_adapter(self, slot, a, b, scale=1.0):
        """a [rank][d_in], b [d_out][rank] of the layer's type, on the host or the device, into a slot; a = b = None empties it.  Waits for the device."""
        import torch
        if (a is None) != (b is None):
            raise ValueError("an adapter is a and b")
        rank = 0
        if a is not None:
            a, b = _matrix(a, "a [rank][d_in]", self.dtype), _matrix(b, "b [d_out][rank]", self.dtype)
            rank = int(a.shape[0])
            if rank < 1 or tuple(a.shape) != (rank, self.d_in) or tuple(b.shape) != (self.d_out, rank):
                raise ValueError("a [rank][%d] and b [%d][rank] are needed" % (self.d_in, self.d_out))
        with torch.cuda.device(self.device):
            capi.check(capi.lib().psgpu_proj_set_adapter(self.h, _int32(slot, "slot"), rank, _p(a), _p(b), float(scale)), "psgpu_proj_set_adapter")

    def __call__(self, x, utt_off=None, adapter=None, out=None, out_dtype=None):
        """x [frames][d_in] of the layer's type -> [frames][d_out] of it or of out_dtype = torch.float32.  utt_off: int32 [n_utt + 1];
        adapter: int32 [n_utt], each utterance's slot (-1: none)."""
        import torch
        xs = _rows(x, "x", self.d_in, self.dtype, self.device)
        rows, n_utt = x.shape[0], 0
        if utt_off is not None:
            utt_off, n_utt = _offsets(utt_off, self.device)
        if adapter is not None:
            if utt_off is None:
                raise ValueError("adapter: utt_off is needed too")
            adapter = _vector(adapter, "adapter", n_utt, torch.int32, self.device)
        dt = out.dtype if out is not None else (out_dtype if out_dtype is not None else self.dtype)
        if dt not in (self.dtype, torch.float32) or (out is not None and out_dtype is not None and out_dtype != dt):
            raise ValueError("the output is of the layer's type or float32")
        L = capi.lib()
        with _On(self.device) as stream:
            if out is None:
                out = x.new_empty((rows, self.d_out), dtype=dt)
            ys = _rows(out, "out", self.d_out, dt, self.device, rows)
            need = int(L.psgpu_proj_work_bytes(self.h, rows)) if utt_off is not None else 0
            work = x.new_empty(need, dtype=torch.uint8) if need else None
            capi.check(L.psgpu_proj_run_dev(self.h, _p(x), xs, _p(utt_off), _p(adapter), n_utt, rows, _p(out), ys, _dtypes()[dt], _p(work),
                                            need, stream), "psgpu_proj_run_dev")
        return out

    def close(self):
        if getattr(self, "h", None):
            capi.lib().psgpu_proj_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def group_norm(x, utt_off, n_groups, weight=None, bias=None, eps=1e-5, act="none", out=None):
    """act((x - m) / sqrt(v + eps) * weight + bias), m and v over an utterance's frames x a group's channels (psgpu_group_norm_dev).
    x [frames][channels]; weight, bias: float32 [channels] or None; act: none, relu, silu, gelu; out may be x."""
    import torch
    xs = _rows(x, "x")
    if x.dtype not in _dtypes():
        raise ValueError("x has type %s" % x.dtype)
    if act not in ACTIVATIONS:
        raise ValueError("act: one of %s" % ", ".join(ACTIVATIONS))
    n_groups = _int32(n_groups, "n_groups")
    (rows, chan), dev = x.shape, x.device
    utt_off, n_utt = _offsets(utt_off, dev)
    weight = None if weight is None else _vector(weight, "weight", chan, torch.float32, dev)
    bias = None if bias is None else _vector(bias, "bias", chan, torch.float32, dev)
    L = capi.lib()
    with _On(dev) as stream:
        if out is None:
            out = x.new_empty((rows, chan))
        ys = _rows(out, "out", chan, x.dtype, dev, rows)
        need = int(L.psgpu_group_norm_work_bytes(n_utt, rows, n_groups))
        work = x.new_empty(need, dtype=torch.uint8) if need else None
        capi.check(L.psgpu_group_norm_dev(_dtypes()[x.dtype], _p(x), xs, _p(utt_off), n_utt, rows, chan, n_groups, _p(weight), _p(bias),
                                          float(eps), ACTIVATIONS[act], _p(out), ys, _p(work), need, stream), "psgpu_group_norm_dev")
    return out


def senone_scores(logits, log_prior=None, scale=1.0, logbase=1.0001, out=None, want_best=False):
    """The searches' scores of a network's outputs (psgpu_senone_scores_dev): logits [frames][n_sen] -> int16 [frames][n_sen], lower is
    better, the frame's best 0.  log_prior: float32 [n_sen] or None.  want_best: returns (scores, best float32 [frames]) with the best
    senone's log-likelihood, max(logits - log_prior) - log sum exp(logits)."""
    import torch
    zs = _rows(logits, "logits")
    if logits.dtype not in _dtypes():
        raise ValueError("logits have type %s" % logits.dtype)
    (rows, n_sen), dev = logits.shape, logits.device
    log_prior = None if log_prior is None else _vector(log_prior, "log_prior", n_sen, torch.float32, dev)
    with _On(dev) as stream:
        if out is None:
            out = logits.new_empty((rows, n_sen), dtype=torch.int16)
        ss = _rows(out, "out", n_sen, torch.int16, dev, rows)
        best = logits.new_empty(rows, dtype=torch.float32) if want_best else None
        capi.check(capi.lib().psgpu_senone_scores_dev(_dtypes()[logits.dtype], _p(logits), zs, rows, n_sen, _p(log_prior), float(scale),
                                                      float(logbase), _p(out), ss, _p(best), stream), "psgpu_senone_scores_dev")
    return (out, best) if want_best else out
