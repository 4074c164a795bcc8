"""Refusals of the training operators (layer norm with its backward pass, embedding with its gradient, gradient norm and clipping):
all of them are decided on the host, before a device is touched, so they run without a GPU."""
import ctypes as C

import pytest

P = C.c_void_p(4096)          # an aligned address that is never read
Q = C.c_void_p(8192)


def test_layernorm_forward_refusals(cgb):
    capi, L = cgb.capi, cgb.lib()

    def call(dtype=capi.BF16, pdtype=capi.F32, x=P, gamma=P, beta=P, eps=1e-5, y=Q, mean=P, rstd=P, rows=4, cols=8):
        return L.cg_b200_layernorm_forward(dtype, pdtype, x, gamma, beta, eps, y, mean, rstd, rows, cols, None)

    assert call(dtype=3) == capi.ERR_INVALID_ARG
    assert call(dtype=capi.F32, pdtype=capi.BF16) == capi.ERR_INVALID_ARG
    assert call(dtype=capi.F16, pdtype=capi.BF16) == capi.ERR_INVALID_ARG
    assert call(eps=-1.0) == capi.ERR_INVALID_ARG
    assert call(eps=float("nan")) == capi.ERR_INVALID_ARG
    assert call(rows=-1) == capi.ERR_INVALID_ARG
    assert call(cols=-8) == capi.ERR_INVALID_ARG
    assert call(rows=1 << 40, cols=1 << 30) == capi.ERR_INVALID_ARG
    assert call(x=None) == capi.ERR_NULL_POINTER
    assert call(y=None) == capi.ERR_NULL_POINTER
    assert call(x=C.c_void_p(4097)) == capi.ERR_MISALIGNED
    assert call(gamma=C.c_void_p(4098)) == capi.ERR_MISALIGNED
    assert call(rstd=C.c_void_p(4098)) == capi.ERR_MISALIGNED
    assert call(x=None, y=None, rows=0) == capi.OK
    assert call(x=None, y=None, cols=0) == capi.OK


def test_layernorm_backward_refusals(cgb):
    capi, L = cgb.capi, cgb.lib()
    need = C.c_size_t(0)
    assert L.cg_b200_layernorm_backward_workspace_bytes(100, 64, None) == capi.ERR_NULL_POINTER
    assert L.cg_b200_layernorm_backward_workspace_bytes(-1, 64, C.byref(need)) == capi.ERR_INVALID_ARG
    assert L.cg_b200_layernorm_backward_workspace_bytes(100, 64, C.byref(need)) == capi.OK and need.value > 0

    def call(dtype=capi.BF16, pdtype=capi.F32, dy=P, x=P, gamma=P, mean=P, rstd=P, dx=Q, dgamma=Q, dbeta=Q, rows=100, cols=64, ws=P,
             ws_bytes=need.value):
        return L.cg_b200_layernorm_backward(dtype, pdtype, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, ws, ws_bytes, None)

    assert call(dtype=-1) == capi.ERR_INVALID_ARG
    assert call(dtype=capi.F32, pdtype=capi.F16) == capi.ERR_INVALID_ARG
    assert call(dy=None) == capi.ERR_NULL_POINTER
    assert call(mean=None) == capi.ERR_NULL_POINTER
    assert call(dx=None, dgamma=None, dbeta=None) == capi.ERR_NULL_POINTER
    assert call(dgamma=C.c_void_p(8194)) == capi.ERR_MISALIGNED
    assert call(ws=C.c_void_p(4100)) == capi.ERR_MISALIGNED
    assert call(ws=None) == capi.ERR_WORKSPACE
    assert call(ws_bytes=need.value - 1) == capi.ERR_WORKSPACE
    assert call(cols=0) == capi.OK
    assert call(rows=0, dgamma=None, dbeta=None) == capi.OK


def test_embedding_refusals(cgb):
    capi, L = cgb.capi, cgb.lib()

    def fwd(dtype=capi.BF16, tdtype=capi.F32, table=P, vocab=10, cols=8, ids=P, idb=8, n=4, out=Q):
        return L.cg_b200_embedding(dtype, tdtype, table, vocab, cols, ids, idb, n, 1.0, out, None)

    assert fwd(dtype=capi.F32, tdtype=capi.BF16) == capi.ERR_INVALID_ARG
    assert fwd(idb=2) == capi.ERR_INVALID_ARG
    assert fwd(n=-1) == capi.ERR_INVALID_ARG
    assert fwd(n=1 << 31) == capi.ERR_INVALID_ARG
    assert fwd(vocab=0x7fffffff) == capi.ERR_INVALID_ARG
    assert fwd(table=None) == capi.ERR_NULL_POINTER
    assert fwd(ids=None) == capi.ERR_NULL_POINTER
    assert fwd(ids=C.c_void_p(4100)) == capi.ERR_MISALIGNED
    assert fwd(n=0, ids=None, out=None) == capi.OK

    need = C.c_size_t(0)
    assert L.cg_b200_embedding_backward_workspace_bytes(-4, 10, 8, C.byref(need)) == capi.ERR_INVALID_ARG
    assert L.cg_b200_embedding_backward_workspace_bytes(4, 10, 8, C.byref(need)) == capi.OK and need.value > 0

    def bwd(dtype=capi.BF16, gdtype=capi.F32, dy=P, ids=P, idb=4, n=4, acc=0, dtable=Q, vocab=10, cols=8, ws=P, ws_bytes=need.value):
        return L.cg_b200_embedding_backward(dtype, gdtype, dy, ids, idb, n, 1.0, -1, acc, dtable, vocab, cols, ws, ws_bytes, None)

    assert bwd(dtype=capi.F16, gdtype=capi.BF16) == capi.ERR_INVALID_ARG
    assert bwd(idb=1) == capi.ERR_INVALID_ARG
    assert bwd(dtable=None) == capi.ERR_NULL_POINTER
    assert bwd(dy=None) == capi.ERR_NULL_POINTER
    assert bwd(ws=C.c_void_p(4112)) == capi.ERR_MISALIGNED
    assert bwd(ws=None) == capi.ERR_WORKSPACE
    assert bwd(ws_bytes=need.value - 1) == capi.ERR_WORKSPACE
    assert bwd(vocab=0) == capi.OK
    assert bwd(n=0, acc=1, dy=None, ids=None) == capi.OK


def test_clip_refusals(cgb):
    capi, L = cgb.capi, cgb.lib()
    need = C.c_size_t(0)
    assert L.cg_b200_grad_norm_workspace_bytes(-1, C.byref(need)) == capi.ERR_INVALID_ARG
    assert L.cg_b200_grad_norm_workspace_bytes(2, C.byref(need)) == capi.OK and need.value > 0

    def table(**first):
        t = (capi.Grad * 2)()
        for e, at in zip(t, (1 << 16, 1 << 18)):
            e.in_, e.out, e.n, e.dtype, e.out_dtype = at, at, 100, capi.BF16, capi.BF16
        for k, v in first.items():
            setattr(t[0], k, v)
        return t

    def clip(t, count=2, max_norm=1.0, norm=P, ws=P, ws_bytes=need.value):
        return L.cg_b200_clip_grad_norm(t, count, max_norm, norm, ws, ws_bytes, None)

    assert clip(table(), max_norm=-1.0) == capi.ERR_INVALID_ARG
    assert clip(table(), max_norm=float("nan")) == capi.ERR_INVALID_ARG
    assert clip(table(), count=-1) == capi.ERR_INVALID_ARG
    assert clip(None) == capi.ERR_NULL_POINTER
    assert clip(table(), norm=None) == capi.ERR_NULL_POINTER
    assert clip(table(), norm=C.c_void_p(4098)) == capi.ERR_MISALIGNED
    assert clip(table(in_=None)) == capi.ERR_NULL_POINTER
    assert clip(table(out=None)) == capi.ERR_NULL_POINTER
    assert clip(table(in_=(1 << 16) + 1)) == capi.ERR_MISALIGNED
    assert clip(table(n=-1)) == capi.ERR_INVALID_ARG
    assert clip(table(dtype=9)) == capi.ERR_INVALID_ARG
    assert clip(table(out_dtype=capi.F16)) == capi.ERR_INVALID_ARG
    assert clip(table(out_dtype=capi.F32)) == capi.ERR_INVALID_ARG               # widened over its own input
    assert clip(table(out=(1 << 16) + 2)) == capi.ERR_INVALID_ARG                # shifted over its own input
    assert clip(table(in_=1 << 18, out=1 << 18)) == capi.ERR_INVALID_ARG         # the same tensor twice
    assert clip(table(out=(1 << 18) + 100)) == capi.ERR_INVALID_ARG              # into the other gradient
    assert clip(table(out=(1 << 18) + 198)) == capi.ERR_INVALID_ARG              # by its last element
    assert clip(table(out=(1 << 18) + 200), ws=None) == capi.ERR_WORKSPACE       # beside it is fine
    assert clip(table(), ws=None) == capi.ERR_WORKSPACE
    assert clip(table(), ws_bytes=need.value - 1) == capi.ERR_WORKSPACE
    t = table(out_dtype=77, out=None)
    assert L.cg_b200_grad_norm(t, 2, None, P, need.value, None) == capi.ERR_NULL_POINTER   # outputs are not looked at, norm is


@pytest.mark.parametrize("count", [2, 100])   # with the address ranges on the stack, and allocated
def test_clip_norm_apart_from_the_list(cgb, count):
    """The norm is written while the list is still being read, so it may be no part of a gradient or of an output."""
    capi, L = cgb.capi, cgb.lib()
    t = (capi.Grad * count)()
    for i, e in enumerate(t):
        e.in_, e.out, e.n, e.dtype, e.out_dtype = (1 << 16) + i * 1024, (1 << 20) + i * 1024, 100, capi.F32, capi.F32
    last = count - 1
    # a call that gets past this check is refused for its missing workspace
    for at, status in (((1 << 16) - 4, capi.ERR_WORKSPACE), (1 << 16, capi.ERR_INVALID_ARG),
                       ((1 << 16) + last * 1024 + 396, capi.ERR_INVALID_ARG), ((1 << 16) + last * 1024 + 400, capi.ERR_WORKSPACE),
                       ((1 << 20) - 4, capi.ERR_WORKSPACE), (1 << 20, capi.ERR_INVALID_ARG),
                       ((1 << 20) + last * 1024 + 396, capi.ERR_INVALID_ARG), ((1 << 20) + last * 1024 + 400, capi.ERR_WORKSPACE)):
        assert L.cg_b200_clip_grad_norm(t, count, 1.0, C.c_void_p(at), None, 0, None) == status, hex(at)


def test_python_entry_points_take_cuda_tensors(cgb):
    import torch
    from cantors_gift_b200 import ops
    x, v = torch.zeros(4, 8), torch.zeros(4)
    with pytest.raises(ValueError):
        ops.layernorm_forward(x)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x, x, v, v)
    with pytest.raises(ValueError):
        ops.embedding(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.embedding_backward(x, torch.zeros(4, dtype=torch.int64), 10)
    with pytest.raises(ValueError):
        ops.clip_grad_norm([x], 1.0)
    with pytest.raises(ValueError):
        ops.grad_norm([])


def test_calls_go_to_their_tensors_device(cgb, monkeypatch):
    """A tensor on another device than the current one is worked on there, and a stream of a third one is refused (no GPU is touched)."""
    import torch
    from cantors_gift_b200 import ops

    class Fake:
        def __init__(self, index):
            self.index, self.device = index, torch.device("cuda", index)

        def get_device(self):
            return self.index

    class FakeStream:
        def __init__(self, index):
            self.device = torch.device("cuda", index)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "device", lambda index: ("device", index))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: ("stream", s))
    assert ops._elsewhere(Fake(0), None) is None
    assert ops._elsewhere(Fake(1), None) == ("device", 1)
    s = FakeStream(1)
    assert ops._elsewhere(Fake(1), s) == ("stream", s)
    with pytest.raises(ValueError):
        ops._elsewhere(Fake(0), s)
