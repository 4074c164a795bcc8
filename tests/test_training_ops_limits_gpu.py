"""The training operators at the limits of what their documentation allows. Definitions and bounds as in test_training_ops_gpu.py."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_training_ops_gpu import CHAIN, DTYPES, assert_within, check_ln_backward, check_ln_forward, guarded, ln_backward_reference, normal, embedding_grad_reference

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


def test_embedding_and_clipping_from_host_threads(ops):
    """The same for the embedding, its gradient (sorts by one CTA, by clusters of two and sixteen, and by launches over all ids) and clipping."""
    sizes = [(900, 300, 64), (2000, 5000, 40), (70000, 700, 24), (140000, 3000, 8)]
    g = torch.Generator(device="cuda").manual_seed(1)
    sets = [(normal(v, c, seed=n), torch.randint(-1, v, (n,), device="cuda", generator=g), normal(n, c, seed=n + 1)) for n, v, c in sizes]

    def once(table, ids, dy, stream=None):
        out = ops.embedding(table, ids, scale=2.0, stream=stream)
        grad = ops.embedding_backward(dy, ids, table.shape[0], scale=2.0, stream=stream)
        return out, grad, ops.clip_grad_norm([grad, out], 1.0, stream=stream)

    wants = [once(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    start, faults = threading.Barrier(len(sets)), []

    def work(k):
        try:
            start.wait()
            for i in range(100):
                got = once(*sets[k], stream=streams[k])
                if i % 10 == 9:
                    streams[k].synchronize()
                    for a, b in zip(got, wants[k]):
                        assert torch.equal(a, b), f"call {i}"
        except Exception as e:
            faults.append(f"thread {k}: {e!r}")

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not faults, faults


# ---- long sums ----------------------------------------------------------------------------------------------
def steady_rows(rows, cols, dtype, shift):
    """x and dy with the same values in every row: the sums over rows are rows times one term, and the rounding errors of a running sum,
    all of one sign between two powers of two, add up instead of cancelling. Mean 0 and rstd 1 are given, so that h is x."""
    # 16-bit values, so that x * dy is exact in fp32
    u, v = normal(cols, seed=1, dtype=torch.bfloat16), normal(cols, seed=2, dtype=torch.bfloat16)
    _, x = guarded((rows, cols), dtype, 0)
    _, dy = guarded((rows, cols), dtype, shift)
    x.copy_(u)
    dy.copy_(v)
    return x, dy, u.double(), v.double()


def check_weight_gradients(ops, rows, cols, dtype, shift, chain):
    x, dy, u, v = steady_rows(rows, cols, dtype, shift)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    gamma = torch.ones(cols, device="cuda")
    _, dgamma, dbeta = ops.layernorm_backward(dy, x, mean, rstd, gamma, dx=x)
    assert_within(dgamma, rows * u * v, rows * (u * v).abs(), "dgamma", chain=chain)
    assert_within(dbeta, rows * v, rows * v.abs(), "dbeta", chain=chain)


@pytest.mark.parametrize("rows,cols,shift", [(400000, 1024, 1), (40000, 16400, 0), (60000, 40000, 0)])
def test_layernorm_streaming_weight_gradients_of_many_rows(ops, rows, cols, shift):
    """Bases off by different amounts, and rows above 16384 columns: a thread adds 64 terms in fp32 and such sums in fp64, then eight
    threads' sums and those of at most 152 slices in 16 strands follow: below CHAIN's 128 steps."""
    check_weight_gradients(ops, rows, cols, torch.bfloat16, shift, CHAIN)


@pytest.mark.parametrize("rows,cols", [(200000, 512), (30000, 16384)])
def test_layernorm_weight_gradients_of_many_rows(ops, rows, cols):
    """The register kernels: a group's threads add the rows of their group one after another. 512 columns of 16 bits have 16 groups to each of
    148 CTAs, 16384 columns one group; 64 steps are left for the joins of 16 groups and of 148 CTAs in 16 strands."""
    groups = 16 if cols == 512 else 1
    chain = (-(-rows // (148 * groups)) + 64) * 2.0 ** -24
    check_weight_gradients(ops, rows, cols, torch.bfloat16, 0, chain)


def test_layernorm_weight_gradients_of_many_random_rows(ops):
    rows, cols = 200000, 512
    x, dy = normal(rows, cols, seed=3, dtype=torch.bfloat16), normal(rows, cols, seed=4, dtype=torch.bfloat16)
    gamma, beta = normal(cols, seed=5, offset=1.0), normal(cols, seed=6)
    _, mean, rstd = check_ln_forward(ops, x, gamma, beta)
    check_ln_backward(ops, dy, x, mean, rstd, gamma)


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_layernorm_of_a_million_columns(ops, dtype):
    """Two values in turn, so that a thread's running sum adds one and the same value every time."""
    dt, cols = DTYPES[dtype], 1 << 20
    x = torch.empty(2, cols, device="cuda", dtype=dt)
    x[:, ::2], x[:, 1::2] = 0.1, 0.9
    dy = torch.empty_like(x)
    dy[:, ::2], dy[:, 1::2] = 0.7, 0.3
    _, mean, rstd = check_ln_forward(ops, x, None, None)
    check_ln_backward(ops, dy, x, mean, rstd, None)


# ---- tensors without columns ----------------------------------------------------------------------------------
def test_layernorm_without_columns_gives_no_number(ops):
    """The mean of nothing is 0 / 0: the statistics of such rows are NaN, in new tensors and in given ones."""
    x = torch.empty(5, 0, device="cuda")
    mean, rstd = torch.full((5,), 3.0, device="cuda"), torch.full((5,), 4.0, device="cuda")
    y, m, r = ops.layernorm_forward(x, mean=mean, rstd=rstd)
    assert m is mean and r is rstd and y.shape == (5, 0)
    assert bool(torch.isnan(mean).all()) and bool(torch.isnan(rstd).all())
    junk = torch.full((4096,), 7.0, device="cuda")   # what the allocator hands out next
    del junk
    _, m, r = ops.layernorm_forward(torch.empty(64, 64, 0, device="cuda"))
    assert m.shape == r.shape == (64, 64) and bool(torch.isnan(m).all()) and bool(torch.isnan(r).all())


# ---- tensors beside and over one another ------------------------------------------------------------------------
def adjacent(*shapes):
    """fp32 tensors one behind another in one buffer."""
    sizes = [torch.Size(s).numel() for s in shapes]
    buf = torch.zeros(sum(sizes), device="cuda")
    return [t.view(s) for t, s in zip(buf.split(sizes), shapes)]


def test_layernorm_of_tensors_side_by_side(ops):
    """Nothing lies between the tensors, and every call is right. Moved by one element, it is refused."""
    from cantors_gift_b200 import CgB200Error
    rows, cols = 29, 100
    x, dy, gamma, beta = normal(rows, cols, seed=1), normal(rows, cols, seed=2), normal(cols, seed=3), normal(cols, seed=4)
    want = check_ln_forward(ops, x, gamma, beta)
    check_ln_backward(ops, dy, x, want[1], want[2], gamma)
    out, x2, mean, g2, rstd, b2 = adjacent((rows, cols), (rows, cols), (rows,), (cols,), (rows,), (cols,))
    x2.copy_(x), g2.copy_(gamma), b2.copy_(beta)
    for a, b in zip(ops.layernorm_forward(x2, g2, b2, out=out, mean=mean, rstd=rstd), want):
        assert torch.equal(a, b)   # a row's sums do not depend on where the parameters lie
    dx, dy2, dg, x2, db, m2, g2, r2 = adjacent((rows, cols), (rows, cols), (cols,), (rows, cols), (cols,), (rows,), (cols,), (rows,))
    x2.copy_(x), dy2.copy_(dy), g2.copy_(gamma), m2.copy_(want[1]), r2.copy_(want[2])
    ops.layernorm_backward(dy2, x2, m2, r2, g2, dx=dx, dgamma=dg, dbeta=db)
    for t, v in ((x2, x), (dy2, dy), (g2, gamma), (m2, want[1]), (r2, want[2])):
        assert torch.equal(t, v)
    # where gamma lies decides how many CTAs take the rows and so the order of the sums over them: held to the definition
    wx, wg, wb = ln_backward_reference(dy, x, want[1], want[2], gamma)
    h, g = (x.double() - want[1].double()[:, None]).abs() * want[2].double()[:, None], dy.double().abs() * gamma.double().abs()
    size = x.double().abs() * want[2].double()[:, None] + h
    assert_within(dg, wg, (dy.double().abs() * size).sum(0), "dgamma")
    assert_within(db, wb, dy.double().abs().sum(0), "dbeta")
    assert_within(dx, wx, want[2].double()[:, None] * (g + g.mean(1, keepdim=True) + size * (g * size).mean(1, keepdim=True)), "dx")
    buf = torch.zeros(2 * rows * cols, device="cuda")
    at = lambda i: buf[i:i + rows * cols].view(rows, cols)
    for bad in (lambda: ops.layernorm_forward(at(0), out=at(1)), lambda: ops.layernorm_forward(at(5), out=at(0)),
                lambda: ops.layernorm_backward(at(0), x, mean, rstd, dx=at(cols)), lambda: ops.layernorm_backward(dy, at(4), mean, rstd, dx=at(0)),
                lambda: ops.layernorm_backward(dy, x, want[1], want[2], gamma, dgamma=g2, dbeta=g2)):
        with pytest.raises(CgB200Error):
            bad()


def test_embedding_of_tensors_side_by_side(ops):
    from cantors_gift_b200 import CgB200Error
    n, vocab, cols = 40, 30, 33
    table, dy = normal(vocab, cols, seed=1), normal(n, cols, seed=2)
    ids = torch.arange(n, device="cuda") % vocab
    out, t2, grad, dy2 = adjacent((n, cols), (vocab, cols), (vocab, cols), (n, cols))
    t2.copy_(table), dy2.copy_(dy)
    assert torch.equal(ops.embedding(t2, ids, out=out), table[ids])
    got = ops.embedding_backward(dy2, ids, vocab, out=grad)
    assert torch.equal(t2, table) and torch.equal(dy2, dy) and torch.equal(out, table[ids])
    want, size, count = embedding_grad_reference(dy, ids, vocab, 1.0)
    assert_within(got, want, size, "gradient", chain=64 * 2.0 ** -24)
    square = torch.zeros(n * cols + 1, device="cuda")
    at = lambda i: square[i:i + n * cols].view(n, cols)
    for bad in (lambda: ops.embedding(at(0), ids, out=at(0)), lambda: ops.embedding(at(0), ids, out=at(1)),
                lambda: ops.embedding_backward(at(0), ids, n, out=at(0)), lambda: ops.embedding_backward(at(1), ids, n, out=at(0), accumulate=True)):
        with pytest.raises(CgB200Error):
            bad()
