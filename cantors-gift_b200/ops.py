"""Host-side calls of the C ABI on torch CUDA tensors and on host (NumPy / pinned) buffers.

PyTorch is used for device memory and streams only; every computation is a cg_b200_* call.
bf16 host arrays travel as uint16 bit patterns.
"""
import array
import ctypes as C
import functools
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
def _elsewhere(x, stream):
    """None when the call can go ahead as it is, else the context that makes x's device (and `stream`) current."""
    index = x.get_device()
    if stream is not None:
        if stream.device != x.device:
            raise ValueError(f"stream is on {stream.device}, tensors are on {x.device}")
        if index != torch.cuda.current_device() or stream != torch.cuda.current_stream():
            return torch.cuda.stream(stream)
    return torch.cuda.device(index) if index != torch.cuda.current_device() else None


def _require_one_device(x, *tensors):
    if not x.is_cuda or not x.is_contiguous():
        raise ValueError("cg_b200 ops take contiguous CUDA tensors")
    index = x.get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or not t.is_contiguous()):
            raise ValueError(f"cg_b200 ops take contiguous CUDA tensors on one device ({x.device})")


def _addr(t):
    return None if t is None else t.data_ptr()


def _raw_stream(index):
    """The current stream's handle: torch.cuda.current_stream(index).cuda_stream without building a Stream object (3.5 us)."""
    return torch._C._cuda_getCurrentRawStream(index)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(op, index, *sizes):
    """cg_b200_<op>_workspace_bytes(*sizes) on device `index`, the current one."""
    need = C.c_size_t(0)
    check(getattr(lib(), f"cg_b200_{op}_workspace_bytes")(*sizes, C.byref(need)), f"{op}_workspace_bytes")
    return need.value


def _dtype_code(dtype):
    code = DTYPE_OF_TORCH.get(dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {dtype}")
    return code


def _param_code(x, *params):
    """The type that gamma, beta and their gradients share: x's own or fp32. Their shape: [cols]."""
    kind, shape = None, x.shape[-1:]
    for t in params:
        if t is None:
            continue
        kind = t.dtype if kind is None else kind
        if t.dtype != kind or (kind != x.dtype and kind != torch.float32):
            raise ValueError(f"parameters must all have dtype {x.dtype} or all float32")
        if t.shape != shape:
            raise ValueError(f"parameters must be {tuple(shape)}, got {tuple(t.shape)}")
    return _dtype_code(x.dtype if kind is None else kind)


def _rows_cols(x):
    if x.dim() == 0:
        raise ValueError("a tensor of at least one dimension is needed")
    cols = x.shape[-1]
    return (x.numel() // cols if cols else math.prod(x.shape[:-1])), cols


def _check_like(t, shape, dtype, what):
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{what} must be {tuple(shape)} of {dtype}, got {tuple(t.shape)} of {t.dtype}")


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, out=None, mean=None, rstd=None, stream=None):
    """layernorm over the last axis that keeps its statistics: (y, mean, rstd), mean and rstd fp32 of shape x.shape[:-1].
    gamma, beta: [cols] of x's dtype or fp32, each may be None. `out` may be x. Rows without columns have NaN statistics, 0 / 0."""
    _require_one_device(x, gamma, beta, out, mean, rstd)
    ctx = _elsewhere(x, stream)
    if ctx is not None:
        with ctx:
            return layernorm_forward(x, gamma, beta, eps, out, mean, rstd)
    dt, pt = _dtype_code(x.dtype), _param_code(x, gamma, beta)
    rows, cols = _rows_cols(x)
    shape, lead = x.shape, x.shape[:-1]
    if out is None:
        out = torch.empty_like(x)
    else:
        _check_like(out, shape, x.dtype, "out")
    if mean is None:
        mean = x.new_empty(lead, dtype=torch.float32)
    else:
        _check_like(mean, lead, torch.float32, "mean")
    if rstd is None:
        rstd = torch.empty_like(mean)
    else:
        _check_like(rstd, lead, torch.float32, "rstd")
    check(lib().cg_b200_layernorm_forward(dt, pt, x.data_ptr(), _addr(gamma), _addr(beta), eps, out.data_ptr(), mean.data_ptr(),
                                          rstd.data_ptr(), rows, cols, _raw_stream(x.get_device())), "layernorm_forward")
    if cols == 0:   # the C entry does nothing then; bytes of 0xff are a NaN
        for t in (mean, rstd):
            check(lib().cg_b200_memset(t.data_ptr(), 0xff, 4 * rows, _raw_stream(x.get_device())), "memset")
    return out, mean, rstd


def layernorm_backward(dy, x, mean, rstd, gamma=None, bias=True, dx=None, dgamma=None, dbeta=None, stream=None):
    """Gradients of layernorm_forward: (dx, dgamma, dbeta). dgamma and dbeta are made when gamma is given (dbeta unless
    bias=False) and have gamma's dtype; buffers passed as dgamma / dbeta are filled in any case. `dx` may be dy or x."""
    _require_one_device(x, dy, mean, rstd, gamma, dx, dgamma, dbeta)
    ctx = _elsewhere(x, stream)
    if ctx is not None:
        with ctx:
            return layernorm_backward(dy, x, mean, rstd, gamma, bias, dx, dgamma, dbeta)
    dt, pt = _dtype_code(x.dtype), _param_code(x, gamma, dgamma, dbeta)
    rows, cols = _rows_cols(x)
    _check_like(dy, x.shape, x.dtype, "dy")
    _check_like(mean, x.shape[:-1], torch.float32, "mean")
    _check_like(rstd, x.shape[:-1], torch.float32, "rstd")
    if dx is None:
        dx = torch.empty_like(x)
    else:
        _check_like(dx, x.shape, x.dtype, "dx")
    if gamma is not None:
        dgamma = torch.empty_like(gamma) if dgamma is None else dgamma
        dbeta = torch.empty_like(gamma) if dbeta is None and bias else dbeta
    ws, ws_bytes = None, 0
    if dgamma is not None or dbeta is not None:
        ws_bytes = _workspace_bytes("layernorm_backward", x.get_device(), rows, cols)
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    check(lib().cg_b200_layernorm_backward(dt, pt, dy.data_ptr(), x.data_ptr(), _addr(gamma), mean.data_ptr(), rstd.data_ptr(),
                                           dx.data_ptr(), _addr(dgamma), _addr(dbeta), rows, cols, _addr(ws), ws_bytes,
                                           _raw_stream(x.get_device())), "layernorm_backward")
    return dx, dgamma, dbeta


_ID_BYTES = {torch.int32: 4, torch.int64: 8}


def _id_bytes(ids):
    width = _ID_BYTES.get(ids.dtype)
    if width is None:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    return width


def embedding(table, ids, scale=1.0, dtype=None, out=None, stream=None):
    """scale * table[ids] of shape ids.shape + (cols,): the activations that a token sequence starts from. `dtype` (default:
    the table's) may be bf16 or f16 with an fp32 table. An id outside the table gives a row of zeros."""
    _require_one_device(table, ids, out)
    ctx = _elsewhere(table, stream)
    if ctx is not None:
        with ctx:
            return embedding(table, ids, scale, dtype, out)
    if table.dim() != 2:
        raise ValueError("table must be [vocab, cols]")
    if dtype is None:
        dtype = table.dtype if out is None else out.dtype
    dt, tt, idb = _dtype_code(dtype), _dtype_code(table.dtype), _id_bytes(ids)
    vocab, cols = table.shape
    shape = (*ids.shape, cols)
    if out is None:
        out = table.new_empty(shape, dtype=dtype)
    else:
        _check_like(out, shape, dtype, "out")
    check(lib().cg_b200_embedding(dt, tt, table.data_ptr(), vocab, cols, ids.data_ptr(), idb, ids.numel(), scale, out.data_ptr(),
                                  _raw_stream(table.get_device())), "embedding")
    return out


def embedding_backward(dy, ids, vocab, scale=1.0, padding_id=None, dtype=None, out=None, accumulate=False, stream=None):
    """Gradient of embedding's table, [vocab, cols] of `dtype` (dy's or fp32; default: dy's, or out's): row v is scale times the
    sum of dy over the places of ids that hold v, zero for ids that do not occur and for `padding_id`. accumulate=True adds
    to `out` instead. The same inputs give the same bits on every call."""
    _require_one_device(dy, ids, out)
    ctx = _elsewhere(dy, stream)
    if ctx is not None:
        with ctx:
            return embedding_backward(dy, ids, vocab, scale, padding_id, dtype, out, accumulate)
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape:
        raise ValueError(f"dy must be ids.shape + (cols,): got {tuple(dy.shape)} for ids {tuple(ids.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate=True needs the buffer to add to as `out`")
    if dtype is None:
        dtype = dy.dtype if out is None else out.dtype
    dt, gt, idb = _dtype_code(dy.dtype), _dtype_code(dtype), _id_bytes(ids)
    n, cols = ids.numel(), dy.shape[-1]
    if out is None:
        out = dy.new_empty((vocab, cols), dtype=dtype)
    else:
        _check_like(out, (vocab, cols), dtype, "out")
    index = dy.get_device()
    need = _workspace_bytes("embedding_backward", index, n, vocab, cols)
    ws = dy.new_empty(need, dtype=torch.uint8)
    check(lib().cg_b200_embedding_backward(dt, gt, dy.data_ptr(), ids.data_ptr(), idb, n, scale,
                                           -1 if padding_id is None else padding_id, int(accumulate), out.data_ptr(), vocab, cols,
                                           ws.data_ptr(), need, _raw_stream(index)), "embedding_backward")
    return out


_contiguous, _device_index, _address, _numel = (torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.data_ptr,
                                                torch.Tensor.numel)


def _grad_words(tensors, index):
    """(addresses, sizes, type codes) of a list of contiguous tensors on CUDA device `index`."""
    if index < 0 or set(map(_device_index, tensors)) != {index} or not all(map(_contiguous, tensors)):
        raise ValueError("cg_b200 ops take contiguous CUDA tensors on one device")
    codes = [DTYPE_OF_TORCH.get(t.dtype) for t in tensors]
    if None in codes:
        raise ValueError("gradients are float32, bfloat16 or float16")
    return list(map(_address, tensors)), list(map(_numel, tensors)), codes


def _grad_table(grads, outs):
    """The C ABI's table of a list of tensors, four 64-bit words each (cg_b200_grad)."""
    index = grads[0].get_device()
    at, sizes, codes = _grad_words(grads, index)
    to, out_codes = at, codes
    if outs is not None:
        if len(outs) != len(grads):
            raise ValueError(f"{len(grads)} gradients and {len(outs)} outputs")
        to, out_sizes, out_codes = _grad_words(outs, index)
        if out_sizes != sizes:
            raise ValueError("each output must have as many elements as its gradient")
    words = [0] * (4 * len(grads))
    words[0::4], words[1::4], words[2::4] = at, to, sizes
    words[3::4] = [a | b << 32 for a, b in zip(codes, out_codes)]
    return array.array("q", words)


def grad_norm(grads, norm=None, stream=None):
    """sqrt of the sum of squares over all tensors of `grads`: a 0-dim fp32 tensor on their device."""
    return _norm_call(list(grads), None, None, norm, stream)


def clip_grad_norm(grads, max_norm, out=None, norm=None, stream=None):
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)) and returns their norm before it (0-dim fp32, on the device;
    nothing waits for the GPU). In place, or into `out`: one tensor for each, of as many elements, of its gradient's dtype or
    fp32, in memory of its own, as is `norm` if it is given. No tensor may be in the list twice."""
    return _norm_call(list(grads), max_norm, out, norm, stream)


def _norm_call(grads, max_norm, out, norm, stream):
    if not grads:
        raise ValueError("the list of gradients is empty")
    first = grads[0]
    ctx = _elsewhere(first, stream) if first.is_cuda else None
    if ctx is not None:
        with ctx:
            return _norm_call(grads, max_norm, out, norm, None)
    table = _grad_table(grads, None if out is None else list(out))
    if norm is None:
        norm = first.new_empty((), dtype=torch.float32)
    else:
        _require_one_device(first, norm)
        _check_like(norm, (), torch.float32, "norm")
    index, words = first.get_device(), table.buffer_info()[0]
    need = _workspace_bytes("grad_norm", index, len(grads))
    ws = first.new_empty(need, dtype=torch.uint8)
    if max_norm is None:
        check(lib().cg_b200_grad_norm(words, len(grads), norm.data_ptr(), ws.data_ptr(), need, _raw_stream(index)), "grad_norm")
    else:
        check(lib().cg_b200_clip_grad_norm(words, len(grads), max_norm, norm.data_ptr(), ws.data_ptr(), need, _raw_stream(index)),
              "clip_grad_norm")
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
