"""The training operators at the limits of what their documentation allows. Definitions and bounds as in test_training_ops_gpu.py."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_training_ops_gpu import normal

pytestmark = pytest.mark.gpu


# ---- calls from several host threads ------------------------------------------------------------------------
def ln_sets():
    """fp32 rows of 1024 columns: 77 and 4096 of them go to one and the same kernel with different amounts of shared memory."""
    out = []
    for rows in (77, 4096):
        x, dy = normal(rows, 1024, seed=rows), normal(rows, 1024, seed=rows + 1)
        out.append((x, dy, normal(1024, seed=2, offset=1.0), normal(1024, seed=3)))
    return out


def ln_both(ops, x, dy, gamma, beta, stream=None):
    y, mean, rstd = ops.layernorm_forward(x, gamma, beta, stream=stream)
    return (y, mean, rstd, *ops.layernorm_backward(dy, x, mean, rstd, gamma, stream=stream))


def test_layernorm_from_host_threads(ops, cgb):
    """Four threads, each on a stream of its own and with buffers of its own, two to each size, call the entry points over and over with nothing
    between the calls: every call goes through, and every result has the bits that one thread alone gets."""
    L, sets = cgb.lib(), ln_sets() * 2
    wants = [ln_both(ops, *s) for s in sets]
    bufs = [[torch.full_like(t, -1.0) for t in w] for w in wants]
    need = max(ops._workspace_bytes("layernorm_backward", 0, s[0].shape[0], 1024) for s in sets)
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    start, status = threading.Barrier(len(sets)), [{} for _ in sets]

    def work(k):
        (x, dy, gamma, beta), (y, mean, rstd, dx, dgamma, dbeta) = ([t.data_ptr() for t in ts] for ts in (sets[k], bufs[k]))
        rows, f32, stream = sets[k][0].shape[0], cgb.capi.F32, streams[k].cuda_stream
        forward = (f32, f32, x, gamma, beta, 1e-5, y, mean, rstd, rows, 1024, stream)
        backward = (f32, f32, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, rows, 1024, ws[k].data_ptr(), need, stream)
        start.wait()
        for _ in range(3000):
            for st in (L.cg_b200_layernorm_forward(*forward), L.cg_b200_layernorm_backward(*backward)):
                status[k][st] = status[k].get(st, 0) + 1

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [{cgb.capi.OK: 6000}] * len(sets), status
    for got, want in zip(bufs, wants):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_layernorm_graph_of_two_sizes_replays(ops):
    sets = ln_sets()
    wants = [ln_both(ops, *s) for s in sets]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gots = [ln_both(ops, *s) for s in sets]
    ln_both(ops, *sets[1])   # a call between the capture and its replays
    for got in gots:
        for t in got:
            t.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
