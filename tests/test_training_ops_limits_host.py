"""Calls of the training operators that their documentation rules out, decided on the host before a device is touched."""
import ctypes as C
import subprocess
import sys

from conftest import ROOT

AT = 1 << 20   # an address that is never read


def test_layernorm_forward_overlaps(cgb):
    """4 x 8 bf16 rows (64 bytes), fp32 parameters (32 bytes), statistics of 16 bytes."""
    capi, L = cgb.capi, cgb.lib()
    place = dict(x=AT, gamma=AT + 256, beta=AT + 512, y=AT + 768, mean=AT + 1024, rstd=AT + 1280)

    def call(**moved):
        a = {**place, **moved}
        return L.cg_b200_layernorm_forward(capi.BF16, capi.F32, *(C.c_void_p(a[k]) for k in ("x", "gamma", "beta")), 1e-5,
                                           *(C.c_void_p(a[k]) for k in ("y", "mean", "rstd")), 4, 8, None)

    bad = [dict(y=AT + 2), dict(y=AT - 2), dict(y=AT + 62), dict(y=AT - 62), dict(y=AT + 256), dict(y=AT + 286), dict(y=AT + 512 - 62),
           dict(y=AT + 1024), dict(y=AT + 1280 + 14), dict(mean=AT), dict(mean=AT + 60), dict(mean=AT + 256), dict(mean=AT + 512 + 28),
           dict(mean=AT + 1280), dict(rstd=AT), dict(rstd=AT + 256 - 12), dict(rstd=AT + 512), dict(rstd=AT + 1024 + 12), dict(rstd=AT + 768)]
    for moved in bad:
        assert call(**moved) == capi.ERR_INVALID_ARG, moved


def test_layernorm_backward_overlaps(cgb):
    capi, L = cgb.capi, cgb.lib()
    need = C.c_size_t(0)
    assert L.cg_b200_layernorm_backward_workspace_bytes(4, 8, C.byref(need)) == capi.OK
    names = ("dy", "x", "gamma", "mean", "rstd", "dx", "dgamma", "dbeta")
    place = {k: AT + 256 * i for i, k in enumerate(names)}
    place["ws"] = AT + 4096

    def call(**moved):
        a = {**place, **moved}
        return L.cg_b200_layernorm_backward(capi.BF16, capi.F32, *(C.c_void_p(a[k]) for k in names), 4, 8, C.c_void_p(a["ws"]), need, None)

    bad = [dict(dx=place[k] + d) for k, d in (("dy", 2), ("dy", -62), ("x", -2), ("x", 62), ("gamma", 0), ("gamma", 30), ("mean", 0), ("rstd", 14),
                                              ("dgamma", -62), ("dbeta", 0), ("ws", 0))]
    bad += [dict(dgamma=place["dbeta"] + 28), dict(dbeta=place["dgamma"]), dict(dbeta=place["dx"] + 60)]
    bad += [dict(ws=place[k] // 16 * 16) for k in names] + [dict(ws=AT + 16 - need.value // 16 * 16)]
    for moved in bad:
        assert call(**moved) == capi.ERR_INVALID_ARG, moved


def test_embedding_overlaps(cgb):
    """A table of 10 rows of 8 fp32 (320 bytes), 4 ids of 8 bytes, 4 rows of 8 bf16 (64 bytes)."""
    capi, L = cgb.capi, cgb.lib()
    table, ids, rows = AT, AT + 512, AT + 768

    def lookup(out):
        return L.cg_b200_embedding(capi.BF16, capi.F32, C.c_void_p(table), 10, 8, C.c_void_p(ids), 8, 4, 1.0, C.c_void_p(out), None)

    for out in (table, table - 62, table + 318, ids, ids - 62, ids + 30):
        assert lookup(out) == capi.ERR_INVALID_ARG, out - AT

    need = C.c_size_t(0)
    assert L.cg_b200_embedding_backward_workspace_bytes(4, 10, 8, C.byref(need)) == capi.OK
    place = dict(dy=rows, ids=ids, dtable=table, ws=AT + 4096)

    def gradient(accumulate=0, **moved):
        a = {k: C.c_void_p(v) for k, v in {**place, **moved}.items()}
        return L.cg_b200_embedding_backward(capi.BF16, capi.F32, a["dy"], a["ids"], 8, 4, 1.0, -1, accumulate, a["dtable"], 10, 8, a["ws"], need, None)

    for moved in (dict(dy=table), dict(dy=table + 318), dict(dy=table - 62), dict(ids=table + 312), dict(dtable=rows + 60), dict(dtable=ids - 316),
                  dict(ws=AT), dict(ws=AT + 512), dict(ws=AT + 768), dict(dtable=AT + 4096 + need.value - 4), dict(dy=AT + 4096 - 62)):
        for accumulate in (0, 1):
            assert gradient(accumulate, **moved) == capi.ERR_INVALID_ARG, moved


def test_embedding_gradient_of_too_many_pieces(cgb):
    """More blocks than a grid has are refused before anything is launched: 2^26 chunks of 32 ids, 32 or more tiles of 512 bytes."""
    capi, L = cgb.capi, cgb.lib()

    def call(dtype, cols, n=(1 << 31) - 1, ws=1 << 62):
        need = C.c_size_t(0)
        assert L.cg_b200_embedding_backward_workspace_bytes(n, 10, cols, C.byref(need)) == capi.OK
        return L.cg_b200_embedding_backward(dtype, capi.F32, C.c_void_p(1 << 60), C.c_void_p(1 << 59), 8, n, 1.0, -1, 0, C.c_void_p(1 << 58), 10, cols,
                                            C.c_void_p(ws), need, None)

    for dtype, tile in ((capi.F32, 128), (capi.BF16, 256), (capi.F16, 256)):
        assert call(dtype, 32 * tile) == capi.ERR_UNSUPPORTED
        assert call(dtype, 1 << 30) == capi.ERR_UNSUPPORTED
        assert call(dtype, 31 * tile, ws=None) == capi.ERR_WORKSPACE           # fits
        assert call(dtype, 31 * tile + 1) == capi.ERR_UNSUPPORTED


def test_clip_workspace_apart_from_the_list(cgb):
    capi, L = cgb.capi, cgb.lib()
    need = C.c_size_t(0)
    assert L.cg_b200_grad_norm_workspace_bytes(2, C.byref(need)) == capi.OK
    t = (capi.Grad * 2)()
    for i, e in enumerate(t):
        e.in_, e.out, e.n, e.dtype, e.out_dtype = AT + i * 4096, AT + 16384 + i * 4096, 100, capi.BF16, capi.F32
    far = AT + (1 << 20)

    def clip(ws, norm=far):
        return L.cg_b200_clip_grad_norm(t, 2, 1.0, C.c_void_p(norm), C.c_void_p(ws), need, None)

    def norm_only(ws, norm=far):
        return L.cg_b200_grad_norm(t, 2, C.c_void_p(norm), C.c_void_p(ws), need, None)

    before = need.value // 16 * 16
    for at in (AT, AT + 192, AT + 4096 + 192, AT - before + 16):
        assert clip(at) == norm_only(at) == capi.ERR_INVALID_ARG, at - AT
    for at in (AT + 16384 + 384, AT + 20480 + 384, AT + 20480):
        assert clip(at) == capi.ERR_INVALID_ARG, at - AT
    for at in (far, far + need.value - 4):
        assert clip(far, norm=at) == norm_only(far, norm=at) == capi.ERR_INVALID_ARG


def test_clip_without_host_memory(cgb):
    """A list of 2^20 tensors takes 48 MB on the host for its address ranges; a process that may not have them is told so."""
    code = """
import ctypes as C, resource
from cantors_gift_b200 import capi
L = capi.lib()
count = 1 << 20
t = (capi.Grad * count)()
for i, e in enumerate(t):
    e.in_ = e.out = (1 << 30) + i * 64
    e.n, e.dtype, e.out_dtype = 16, capi.F32, capi.F32
clip = lambda: L.cg_b200_clip_grad_norm(t, count, 1.0, C.c_void_p(1 << 20), None, 0, None)
assert clip() == capi.ERR_WORKSPACE, "with memory"
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (16 << 20),) * 2)
assert clip() == capi.ERR_NO_MEMORY, "without"
assert L.cg_b200_status_string(capi.ERR_NO_MEMORY) == b"out of host memory"
print("refused")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout + r.stderr
