"""Host-side calls of the C ABI on torch CUDA tensors and on host (NumPy / pinned) buffers.

PyTorch is used for device memory and streams only; every computation is a cg_b200_* call.
bf16 host arrays travel as uint16 bit patterns.
"""
import ctypes as C
import math

import numpy as np
import torch

from . import capi
from .capi import BF16, F16, F32, check, lib

TORCH_DTYPE = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
DTYPE_OF_TORCH = {v: k for k, v in TORCH_DTYPE.items()}


def _stream(stream=None):
    s = torch.cuda.current_stream() if stream is None else stream
    return C.c_void_p(s.cuda_stream)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("cg_b200 ops take contiguous CUDA tensors")


def eltwise(desc, inputs, out, n=None, stream=None):
    _require_cuda(out, *inputs)
    n = out.numel() if n is None else n
    arr = (C.c_void_p * max(1, len(inputs)))(*[t.data_ptr() for t in inputs])
    check(lib().cg_b200_eltwise(C.byref(desc), arr, len(inputs), _ptr(out), n, _stream(stream)), "eltwise")
    return out


def softmax(x, out=None, stream=None):
    _require_cuda(x, out)
    out = torch.empty_like(x) if out is None else out
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    check(lib().cg_b200_softmax(DTYPE_OF_TORCH[x.dtype], _ptr(x), _ptr(out), rows, cols, _stream(stream)), "softmax")
    return out


def layernorm(x, gamma=None, beta=None, eps=1e-5, out=None, stream=None):
    _require_cuda(x, out, gamma, beta)
    out = torch.empty_like(x) if out is None else out
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    check(lib().cg_b200_layernorm(DTYPE_OF_TORCH[x.dtype], _ptr(x), _ptr(gamma), _ptr(beta), eps, _ptr(out),
                                  rows, cols, _stream(stream)), "layernorm")
    return out


def softmax_layernorm(x, gamma=None, beta=None, eps=1e-5, out=None, stream=None):
    _require_cuda(x, out, gamma, beta)
    out = torch.empty_like(x) if out is None else out
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    check(lib().cg_b200_softmax_layernorm(DTYPE_OF_TORCH[x.dtype], _ptr(x), _ptr(gamma), _ptr(beta), eps,
                                          _ptr(out), rows, cols, _stream(stream)), "softmax_layernorm")
    return out


def reduce_box(shape, axes):
    """(outer, reduce, inner) of a row-major tensor reduced over `axes`, or None when the axes are not a run of
    adjacent ones (no kernel then). Negative axes count from the end, as in the reference's shape inference."""
    rank = len(shape)
    ax = sorted({a + rank if a < 0 else a for a in axes})
    if not ax or ax[0] < 0 or ax[-1] >= rank or ax != list(range(ax[0], ax[-1] + 1)):
        return None
    outer = inner = red = 1
    for i, d in enumerate(shape):
        if i < ax[0]:
            outer *= d
        elif i > ax[-1]:
            inner *= d
        else:
            red *= d
    return outer, red, inner


def reduce(x, op, axes, keep_dims=False, out=None, stream=None):
    """reduce_sum / reduce_max / reduce_mean (op: "sum" | "max" | "mean") of a contiguous tensor over adjacent axes."""
    _require_cuda(x, out)
    box = reduce_box(tuple(x.shape), axes)
    if box is None or not x.is_contiguous():
        raise ValueError("reduce: the axes must be adjacent and the tensor contiguous")
    outer, red, inner = box
    rank = x.dim()
    ax = {a + rank if a < 0 else a for a in axes}
    shape = [1 if i in ax else d for i, d in enumerate(x.shape) if keep_dims or i not in ax]
    out = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
    check(lib().cg_b200_reduce(DTYPE_OF_TORCH[x.dtype], capi.REDUCE[op], _ptr(x), _ptr(out), outer, red, inner,
                               _stream(stream)), "reduce")
    return out


# ---- training operators ---------------------------------------------------------------------------
# These run on the device their tensors lie on (which need not be the current one) and on `stream` if one is given; what
# they allocate - results and workspaces, new ones for every call - then belongs to that stream. Inputs made on another
# stream are the caller's to order, as with every torch call.
def _call_context(stream, x):
    """None when the call can go ahead as it is, else the context that makes x's device (and `stream`) current."""
    index = x.device.index
    if stream is not None:
        if stream.device != x.device:
            raise ValueError(f"stream is on {stream.device}, tensors are on {x.device}")
        if index != torch.cuda.current_device() or stream != torch.cuda.current_stream():
            return torch.cuda.stream(stream)
    return torch.cuda.device(index) if index != torch.cuda.current_device() else None


def _require_one_device(x, *tensors):
    _require_cuda(x, *tensors)
    for t in tensors:
        if t is not None and t.device != x.device:
            raise ValueError(f"tensors are on {x.device} and {t.device}")


def _dtype_code(dtype):
    code = DTYPE_OF_TORCH.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}")
    return code


def _param_code(x, *params):
    """The type that gamma, beta and their gradients share: x's own or fp32."""
    kinds = {t.dtype for t in params if t is not None} or {x.dtype}
    if len(kinds) != 1 or not kinds <= {x.dtype, torch.float32}:
        raise ValueError(f"parameters must all have dtype {x.dtype} or float32")
    return DTYPE_OF_TORCH[kinds.pop()]


def _rows_cols(x):
    if x.dim() == 0:
        raise ValueError("a tensor of at least one dimension is needed")
    cols = x.shape[-1]
    return (x.numel() // cols if cols else math.prod(x.shape[:-1])), cols


def _check_like(t, shape, dtype, what):
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != dtype):
        raise ValueError(f"{what} must be {tuple(shape)} of {dtype}, got {tuple(t.shape)} of {t.dtype}")


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, out=None, mean=None, rstd=None, stream=None):
    """layernorm over the last axis that keeps its statistics: (y, mean, rstd), mean and rstd fp32 of shape x.shape[:-1].
    gamma, beta: [cols] of x's dtype or fp32, each may be None. `out` may be x."""
    _require_one_device(x, gamma, beta, out, mean, rstd)
    ctx = _call_context(stream, x)
    if ctx is not None:
        with ctx:
            return layernorm_forward(x, gamma, beta, eps, out, mean, rstd)
    dt, pt = _dtype_code(x.dtype), _param_code(x, gamma, beta)
    rows, cols = _rows_cols(x)
    for t, what in ((gamma, "gamma"), (beta, "beta")):
        if t is not None:
            _check_like(t, (cols,), t.dtype, what)
    _check_like(out, x.shape, x.dtype, "out")
    _check_like(mean, x.shape[:-1], torch.float32, "mean")
    _check_like(rstd, x.shape[:-1], torch.float32, "rstd")
    out = torch.empty_like(x) if out is None else out
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if mean is None else mean
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if rstd is None else rstd
    check(lib().cg_b200_layernorm_forward(dt, pt, _ptr(x), _ptr(gamma), _ptr(beta), eps, _ptr(out), _ptr(mean), _ptr(rstd),
                                          rows, cols, _stream()), "layernorm_forward")
    return out, mean, rstd


def layernorm_backward(dy, x, mean, rstd, gamma=None, bias=True, dx=None, dgamma=None, dbeta=None, stream=None):
    """Gradients of layernorm_forward: (dx, dgamma, dbeta). dgamma and dbeta are made when gamma is given (dbeta unless
    bias=False) and have gamma's dtype; buffers passed as dgamma / dbeta are filled in any case. `dx` may be dy or x."""
    _require_one_device(x, dy, mean, rstd, gamma, dx, dgamma, dbeta)
    ctx = _call_context(stream, x)
    if ctx is not None:
        with ctx:
            return layernorm_backward(dy, x, mean, rstd, gamma, bias, dx, dgamma, dbeta)
    dt, pt = _dtype_code(x.dtype), _param_code(x, gamma, dgamma, dbeta)
    rows, cols = _rows_cols(x)
    _check_like(dy, x.shape, x.dtype, "dy")
    _check_like(dx, x.shape, x.dtype, "dx")
    _check_like(mean, x.shape[:-1], torch.float32, "mean")
    _check_like(rstd, x.shape[:-1], torch.float32, "rstd")
    for t, what in ((gamma, "gamma"), (dgamma, "dgamma"), (dbeta, "dbeta")):
        if t is not None:
            _check_like(t, (cols,), t.dtype, what)
    dx = torch.empty_like(x) if dx is None else dx
    if gamma is not None:
        dgamma = torch.empty_like(gamma) if dgamma is None else dgamma
        dbeta = torch.empty_like(gamma) if dbeta is None and bias else dbeta
    ws, ws_bytes = None, 0
    if dgamma is not None or dbeta is not None:
        need = C.c_size_t(0)
        check(lib().cg_b200_layernorm_backward_workspace_bytes(rows, cols, C.byref(need)), "layernorm_backward_workspace_bytes")
        ws_bytes = need.value
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    check(lib().cg_b200_layernorm_backward(dt, pt, _ptr(dy), _ptr(x), _ptr(gamma), _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dgamma),
                                           _ptr(dbeta), rows, cols, _ptr(ws), ws_bytes, _stream()), "layernorm_backward")
    return dx, dgamma, dbeta


_ID_BYTES = {torch.int32: 4, torch.int64: 8}


def _id_bytes(ids):
    if ids.dtype not in _ID_BYTES:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    return _ID_BYTES[ids.dtype]


def embedding(table, ids, scale=1.0, dtype=None, out=None, stream=None):
    """scale * table[ids] of shape ids.shape + (cols,): the activations that a token sequence starts from. `dtype` (default:
    the table's) may be bf16 or f16 with an fp32 table. An id outside the table gives a row of zeros."""
    _require_one_device(table, ids, out)
    ctx = _call_context(stream, table)
    if ctx is not None:
        with ctx:
            return embedding(table, ids, scale, dtype, out)
    if table.dim() != 2:
        raise ValueError("table must be [vocab, cols]")
    dtype = (table.dtype if out is None else out.dtype) if dtype is None else dtype
    dt, tt, idb = _dtype_code(dtype), _dtype_code(table.dtype), _id_bytes(ids)
    vocab, cols = table.shape
    shape = (*ids.shape, cols)
    _check_like(out, shape, dtype, "out")
    out = torch.empty(shape, dtype=dtype, device=table.device) if out is None else out
    check(lib().cg_b200_embedding(dt, tt, _ptr(table), vocab, cols, _ptr(ids), idb, ids.numel(), scale, _ptr(out), _stream()),
          "embedding")
    return out


def embedding_backward(dy, ids, vocab, scale=1.0, padding_id=None, dtype=None, out=None, accumulate=False, stream=None):
    """Gradient of embedding's table, [vocab, cols] of `dtype` (dy's or fp32; default: dy's, or out's): row v is scale times the
    sum of dy over the places of ids that hold v, zero for ids that do not occur and for `padding_id`. accumulate=True adds
    to `out` instead. The same inputs give the same bits on every call."""
    _require_one_device(dy, ids, out)
    ctx = _call_context(stream, dy)
    if ctx is not None:
        with ctx:
            return embedding_backward(dy, ids, vocab, scale, padding_id, dtype, out, accumulate)
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape:
        raise ValueError(f"dy must be ids.shape + (cols,): got {tuple(dy.shape)} for ids {tuple(ids.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate=True needs the buffer to add to as `out`")
    dtype = (dy.dtype if out is None else out.dtype) if dtype is None else dtype
    dt, gt, idb = _dtype_code(dy.dtype), _dtype_code(dtype), _id_bytes(ids)
    n, cols = ids.numel(), dy.shape[-1]
    _check_like(out, (vocab, cols), dtype, "out")
    out = torch.empty((vocab, cols), dtype=dtype, device=dy.device) if out is None else out
    need = C.c_size_t(0)
    check(lib().cg_b200_embedding_backward_workspace_bytes(n, vocab, cols, C.byref(need)), "embedding_backward_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=dy.device)
    check(lib().cg_b200_embedding_backward(dt, gt, _ptr(dy), _ptr(ids), idb, n, scale, -1 if padding_id is None else padding_id,
                                           int(accumulate), _ptr(out), vocab, cols, _ptr(ws), need.value, _stream()),
          "embedding_backward")
    return out


def _grad_list(grads, outs):
    """The C ABI's table of a list of tensors. Empty tensors may be among them; no tensor may be written twice."""
    if len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients and {len(outs)} outputs")
    table = (capi.Grad * max(1, len(grads)))()
    device, written = None, set()
    for e, g, o in zip(table, grads, outs):
        if not g.is_cuda or not g.is_contiguous() or (o is not g and not (o.is_cuda and o.is_contiguous())):
            raise ValueError("cg_b200 ops take contiguous CUDA tensors")
        device = g.device if device is None else device
        if g.device != device or o.device != device:
            raise ValueError("the tensors of a list must be on one device")
        if o is not g and o.shape != g.shape:
            raise ValueError(f"output of shape {tuple(o.shape)} for a gradient of shape {tuple(g.shape)}")
        e.in_, e.out, e.n = g.data_ptr(), o.data_ptr(), g.numel()
        e.dtype, e.out_dtype = _dtype_code(g.dtype), _dtype_code(o.dtype)
        if e.n:
            if e.out in written:
                raise ValueError("a tensor is in the list twice")
            written.add(e.out)
    for e in table:
        if e.n and e.in_ != e.out and e.in_ in written:
            raise ValueError("an output is another gradient of the list")
    return table, device


def grad_norm(grads, norm=None, stream=None):
    """sqrt of the sum of squares over all tensors of `grads`: a 0-dim fp32 tensor on their device."""
    return _norm_of(list(grads), None, None, norm, stream)


def clip_grad_norm(grads, max_norm, out=None, norm=None, stream=None):
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)) and returns their norm before it (0-dim fp32, on the device;
    nothing waits for the GPU). In place, or into `out`: tensors of the same shapes, each of its gradient's dtype or fp32."""
    return _norm_of(list(grads), max_norm, out, norm, stream)


def _norm_of(grads, max_norm, out, norm, stream):
    if not grads:
        raise ValueError("the list of gradients is empty")
    outs = grads if out is None else list(out)
    if max_norm is None:
        table, device = _grad_list_norm(grads)
    else:
        table, device = _grad_list(grads, outs)
    if norm is not None:
        _require_one_device(grads[0], norm)
        _check_like(norm, (), torch.float32, "norm")
    ctx = _call_context(stream, grads[0])
    if ctx is not None:
        with ctx:
            return _norm_call(table, len(grads), max_norm, norm, device)
    return _norm_call(table, len(grads), max_norm, norm, device)


def _grad_list_norm(grads):
    """As _grad_list, for reading only: a tensor may be in the list more than once."""
    table = (capi.Grad * max(1, len(grads)))()
    device = grads[0].device
    for e, g in zip(table, grads):
        _require_one_device(grads[0], g)
        e.in_, e.n, e.dtype = g.data_ptr(), g.numel(), _dtype_code(g.dtype)
    return table, device


def _norm_call(table, count, max_norm, norm, device):
    norm = torch.empty((), dtype=torch.float32, device=device) if norm is None else norm
    need = C.c_size_t(0)
    check(lib().cg_b200_grad_norm_workspace_bytes(count, C.byref(need)), "grad_norm_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=device)
    if max_norm is None:
        check(lib().cg_b200_grad_norm(table, count, _ptr(norm), _ptr(ws), need.value, _stream()), "grad_norm")
    else:
        check(lib().cg_b200_clip_grad_norm(table, count, max_norm, _ptr(norm), _ptr(ws), need.value, _stream()), "clip_grad_norm")
    return norm


_workspaces = {}


def gemm_workspace(desc, device):
    need = C.c_size_t(0)
    check(lib().cg_b200_gemm_workspace_bytes(C.byref(desc), C.byref(need)), "gemm_workspace_bytes")
    if need.value == 0:
        return None, 0
    key = (device.index, torch.cuda.current_stream().cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws, ws.numel()


def gemm(desc, A, B, C_out, bias=None, residual=None, workspace=None, stream=None, tuning=None):
    """`tuning`: a capi.GemmTuning (an autotuner's tile choice) or None for the library's heuristic."""
    _require_cuda(A, B, C_out, bias, residual)
    if workspace is None:
        workspace, ws_bytes = gemm_workspace(desc, A.device)
    else:
        ws_bytes = workspace.numel() * workspace.element_size()
    if tuning is None:
        check(lib().cg_b200_gemm(C.byref(desc), _ptr(A), _ptr(B), _ptr(bias), _ptr(residual), _ptr(C_out),
                                 _ptr(workspace), ws_bytes, _stream(stream)), "gemm")
    else:
        check(lib().cg_b200_gemm_tuned(C.byref(desc), C.byref(tuning), _ptr(A), _ptr(B), _ptr(bias), _ptr(residual),
                                       _ptr(C_out), _ptr(workspace), ws_bytes, _stream(stream)), "gemm_tuned")
    return C_out


def last_device_error(stream=None):
    w = C.c_uint32(0)
    check(lib().cg_b200_last_device_error(_stream(stream), C.byref(w)), "last_device_error")
    return w.value


# ---- host-buffer entry (the call a user of the reference's Runtime would make) ------------------
class HostRunner:
    """Runs one op with HOST inputs and outputs: H2D copies, the kernel, D2H copy, sync.

    Device buffers and pinned staging are allocated once through the C ABI and reused, as a
    bound executable would hold them.
    """

    def __init__(self):
        self._dev = {}
        self.stream = C.c_void_p()
        check(lib().cg_b200_stream_create(C.byref(self.stream)), "stream_create")

    def dev(self, name, nbytes):
        cur = self._dev.get(name)
        if cur is None or cur[1] < nbytes:
            if cur is not None:
                check(lib().cg_b200_free(cur[0]), "free")
            p = C.c_void_p()
            check(lib().cg_b200_malloc(C.byref(p), nbytes), "malloc")
            cur = (p, nbytes)
            self._dev[name] = cur
        return cur[0]

    def h2d(self, name, host):
        """host: pinned torch tensor or numpy array."""
        nbytes = host.numel() * host.element_size() if hasattr(host, "numel") else host.nbytes
        src = host.data_ptr() if hasattr(host, "data_ptr") else host.ctypes.data
        d = self.dev(name, nbytes)
        check(lib().cg_b200_memcpy_h2d(d, C.c_void_p(src), nbytes, self.stream), "memcpy_h2d")
        return d

    def d2h(self, host, dev, nbytes=None):
        n = (host.numel() * host.element_size() if hasattr(host, "numel") else host.nbytes) if nbytes is None else nbytes
        dst = host.data_ptr() if hasattr(host, "data_ptr") else host.ctypes.data
        check(lib().cg_b200_memcpy_d2h(C.c_void_p(dst), dev, n, self.stream), "memcpy_d2h")

    def sync(self):
        check(lib().cg_b200_stream_sync(self.stream), "stream_sync")

    # ---- slab pipeline: copy in, compute, copy out on three streams ------------------------------
    # PCIe moves data in both directions at once and the copy engines run beside the SMs, so a step
    # whose input splits into independent slabs (row blocks of A, sequences of a batch, ranges of an
    # elementwise array) costs about max(copy in, compute, copy out) instead of their sum.
    def _pipeline_streams(self):
        if not hasattr(self, "_s_compute"):
            self._s_compute, self._s_out = C.c_void_p(), C.c_void_p()
            check(lib().cg_b200_stream_create(C.byref(self._s_compute)), "stream_create")
            check(lib().cg_b200_stream_create(C.byref(self._s_out)), "stream_create")
            self._events = []
        return self._s_compute, self._s_out

    def _event(self, i):
        while len(self._events) <= i:
            e = C.c_void_p()
            check(lib().cg_b200_event_create(C.byref(e)), "event_create")
            self._events.append(e)
        return self._events[i]

    def run_slabs(self, n_slabs, copy_in, compute, copy_out):
        """copy_in(i, stream), compute(i, stream), copy_out(i, stream) enqueue slab i's work on the
        stream they are given; anything all slabs share (weights, B) is copied on self.stream by the
        caller before this. Returns after everything has finished."""
        s_in = self.stream
        s_compute, s_out = self._pipeline_streams()
        for i in range(n_slabs):
            copy_in(i, s_in)
            ev_in = self._event(2 * i)
            check(lib().cg_b200_event_record(ev_in, s_in), "event_record")
            check(lib().cg_b200_stream_wait_event(s_compute, ev_in), "stream_wait_event")
            compute(i, s_compute)
            ev_done = self._event(2 * i + 1)
            check(lib().cg_b200_event_record(ev_done, s_compute), "event_record")
            check(lib().cg_b200_stream_wait_event(s_out, ev_done), "stream_wait_event")
            copy_out(i, s_out)
        check(lib().cg_b200_stream_sync(s_out), "stream_sync")
        check(lib().cg_b200_stream_sync(s_compute), "stream_sync")
        check(lib().cg_b200_stream_sync(s_in), "stream_sync")

    def close(self):
        for p, _ in self._dev.values():
            lib().cg_b200_free(p)
        self._dev = {}
        for e in getattr(self, "_events", []):
            lib().cg_b200_event_destroy(e)
        self._events = []
        for name in ("_s_compute", "_s_out"):
            if hasattr(self, name):
                lib().cg_b200_stream_destroy(getattr(self, name))
                delattr(self, name)
        if self.stream:
            lib().cg_b200_stream_destroy(self.stream)
            self.stream = C.c_void_p()
