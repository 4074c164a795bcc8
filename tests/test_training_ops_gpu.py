"""Layer norm with its backward pass, embedding with its gradient, gradient norm and clipping, against the definitions in 64 bits.

Tolerances. Every result is rounded once to its type: off by at most eps / 2 of its value (plus half the smallest step near zero). Before
that, fp32 arithmetic: each term of a sum is off by a few 2^-24 of its magnitude, and a sum adds one 2^-24 of the running magnitude per
addition in its longest chain. The kernels' chains are short (at most 64 terms in a thread, 10 levels of a tree, a few hundred partial sums
in eight strands), so CHAIN = 128 steps of 2^-24 times the sum of the terms' magnitudes bounds them; `scale` in each test is that sum,
written out per element."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

CHAIN = 128 * 2.0 ** -24
DTYPES = {"F32": torch.float32, "BF16": torch.bfloat16, "F16": torch.float16}


def assert_within(got, want, scale, what, chain=CHAIN):
    """|got - want| <= half a step of got's type at want + chain * scale."""
    info = torch.finfo(got.dtype)
    got64 = got.double()
    bound = info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2 + chain * (1 + info.eps) * scale
    over = (got64 - want).abs() - bound
    assert bool(torch.isfinite(got64).all()), f"{what}: not finite"
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} over the bound at {int(over.argmax())}"


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + offset).to(dtype)


def guarded(shape, dtype, shift=0, margin=64):
    """A tensor of `shape` inside a buffer of sentinels, its base `shift` elements from a 16-byte boundary."""
    n = 1
    for d in shape:
        n *= d
    buf = torch.full((margin + shift + n + margin,), -77.0, dtype=dtype, device="cuda")
    return buf, buf[margin + shift:margin + shift + n].view(shape)


def assert_guards(buf, view, what):
    lo = view.storage_offset()
    hi = lo + view.numel()
    assert bool((buf[:lo] == -77.0).all()) and bool((buf[hi:] == -77.0).all()), f"{what}: written outside its tensor"


# ---- layer norm ------------------------------------------------------------------------------------------
def ln_reference(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1)
    var = ((x - mean[:, None]) ** 2).mean(1)
    rstd = 1 / torch.sqrt(var + eps)
    y = (x - mean[:, None]) * rstd[:, None]
    y = y if gamma is None else y * gamma.double()
    return (y if beta is None else y + beta.double()), mean, rstd


def check_ln_forward(ops, x, gamma, beta, eps=1e-5, out=None):
    y, mean, rstd = ops.layernorm_forward(x, gamma, beta, eps=eps, out=out)
    wy, wm, wr = ln_reference(x, gamma, beta, eps)
    g = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if gamma is None else gamma.double().abs()
    size = x.double().abs().mean(1)
    # x - mean is off by the mean's error and its own rounding; rstd by half the variance's relative error
    scale = g * ((x.double().abs() + size[:, None] + wm.abs()[:, None]) * wr[:, None])
    scale = scale if beta is None else scale + beta.double().abs()
    assert_within(y, wy, scale, "y")
    assert_within(mean, wm, size, "mean")
    # variance: the squared deviations are off by 2 |d| times an error of 2^-24 (|x| + |mean|) each; d itself is CHAIN-accurate
    assert_within(rstd, wr, wr * (1 + size * wr), "rstd")
    return y, mean, rstd


def ln_backward_reference(dy, x, mean, rstd, gamma):
    dy, x, m, r = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    h = (x - m) * r
    g = dy if gamma is None else dy * gamma.double()
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def check_ln_backward(ops, dy, x, mean, rstd, gamma, dx=None, bias=True):
    wx, wg, wb = ln_backward_reference(dy, x, mean, rstd, gamma)
    r = rstd.double()[:, None]
    hs = (x.double().abs() + mean.double().abs()[:, None]) * r     # the magnitudes that h is a difference of
    gs = dy.double().abs() * (1 if gamma is None else gamma.double().abs())
    scale = r * (gs + gs.mean(1, keepdim=True) + hs * (gs * hs).mean(1, keepdim=True))
    scale_g, scale_b = (dy.double().abs() * hs).sum(0), dy.double().abs().sum(0)
    dx, dgamma, dbeta = ops.layernorm_backward(dy, x, mean, rstd, gamma, bias=bias, dx=dx)
    assert_within(dx, wx, scale, "dx")
    if gamma is None:
        assert dgamma is None and dbeta is None
    else:
        assert_within(dgamma, wg, scale_g, "dgamma")
        assert (dbeta is None) == (not bias)
        if bias:
            assert_within(dbeta, wb, scale_b, "dbeta")
    return dx, dgamma, dbeta


# one column, fewer columns than a packet, widths on and beside every variant's border, widths that no packet divides, long rows
LN_SHAPES = [(1, 1), (5, 3), (1, 8), (3, 64), (700, 64), (9, 65), (17, 100), (33, 256), (4, 257), (600, 512), (13, 513), (77, 1024),
             (1300, 1001), (2, 1025), (31, 2048), (6, 2047), (9, 4096), (40, 4099), (3, 8192), (5, 8200), (2, 16384), (3, 16385),
             (2, 20001), (5000, 130), (7, 9001), (3, 16383), (1500, 72), (2000, 250), (301, 12001)]


@pytest.mark.parametrize("params", ["own", "F32"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layernorm_forward_and_backward(ops, dtype, params, rows, cols):
    dt = DTYPES[dtype]
    pt = dt if params == "own" else torch.float32
    x = normal(rows, cols, seed=rows + cols, dtype=dt, offset=0.7)
    dy = normal(rows, cols, seed=rows + cols + 1, dtype=dt)
    gamma, beta = normal(cols, seed=2, dtype=pt, offset=1.0), normal(cols, seed=3, dtype=pt)
    _, mean, rstd = check_ln_forward(ops, x, gamma, beta, eps=1e-2 if cols == 1 else 1e-5)
    check_ln_backward(ops, dy, x, mean, rstd, gamma)


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("cols", [96, 1000, 2049, 9000])
@pytest.mark.parametrize("shifts", [(3, 3, 3), (0, 1, 0), (1, 0, 2)])
def test_layernorm_any_alignment_and_no_write_outside(ops, dtype, cols, shifts):
    """Tensors whose bases lie off the 16-byte boundary, by the same and by different offsets."""
    dt, rows = DTYPES[dtype], 19
    _, x = guarded((rows, cols), dt, shifts[0])
    _, dy = guarded((rows, cols), dt, shifts[1])
    obuf, out = guarded((rows, cols), dt, shifts[2])
    x.copy_(normal(rows, cols, seed=5, dtype=dt))
    dy.copy_(normal(rows, cols, seed=6, dtype=dt))
    _, gamma = guarded((cols,), dt, 1)
    _, beta = guarded((cols,), dt, 3)
    gamma.copy_(normal(cols, seed=7, dtype=dt))
    beta.copy_(normal(cols, seed=8, dtype=dt))
    _, mean, rstd = check_ln_forward(ops, x, gamma, beta, out=out)
    assert_guards(obuf, out, "forward")
    check_ln_backward(ops, dy, x, mean, rstd, gamma, dx=out)
    assert_guards(obuf, out, "backward")


@pytest.mark.parametrize("cols", [72, 1024, 1003, 18000])
def test_layernorm_without_parameters_and_in_place(ops, cols):
    x = normal(37, cols, seed=1, dtype=torch.bfloat16)
    dy = normal(37, cols, seed=2, dtype=torch.bfloat16)
    y, mean, rstd = check_ln_forward(ops, x, None, None)
    dx, _, _ = check_ln_backward(ops, dy, x, mean, rstd, None)
    gamma = normal(cols, seed=3)
    want = check_ln_backward(ops, dy, x, mean, rstd, gamma, bias=False)
    for where in ("dy", "x"):
        a, b = dy.clone(), x.clone()
        got = ops.layernorm_backward(a, b, mean, rstd, gamma, bias=False, dx=a if where == "dy" else b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), where
    z = x.clone()
    assert ops.layernorm_forward(z, out=z)[0] is z and torch.equal(z, y)
    beta_only = ops.layernorm_forward(x, None, gamma)[0]
    assert_within(beta_only, ln_reference(x, None, gamma, 1e-5)[0], gamma.double().abs() + 4 * rstd.double()[:, None] + 8, "beta alone")


def test_layernorm_forward_agrees_with_the_inference_kernel(ops):
    x = normal(500, 1024, seed=4, dtype=torch.bfloat16)
    g, b = normal(1024, seed=5, dtype=torch.bfloat16), normal(1024, seed=6, dtype=torch.bfloat16)
    y, mean, rstd = ops.layernorm_forward(x, g, b)
    wy = ln_reference(x, g, b, 1e-5)[0]
    scale = g.double().abs() * (x.double().abs() + 2) * rstd.double()[:, None] + b.double().abs()
    assert_within(ops.layernorm(x, g, b), wy, scale, "layernorm")
    assert_within(y, wy, scale, "layernorm_forward")


def test_layernorm_statistics_survive_a_large_offset(ops):
    """Deviations of 1 around 4096: a one-pass variance would lose them in fp32."""
    x = normal(64, 1500, seed=9, offset=4096.0)
    y, mean, rstd = ops.layernorm_forward(x)
    _, wm, wr = ln_reference(x, None, None, 1e-5)
    assert_within(mean, wm, wm.abs(), "mean")
    # each deviation is off by at most CHAIN * 4096 = 0.031 and all of a row by the same amount, which the centred square sees squared
    assert float((rstd.double() / wr - 1).abs().max()) < 0.5 * (CHAIN * 4096) ** 2 + CHAIN


@pytest.mark.parametrize("cols", [40, 1024, 1001, 17000])
def test_layernorm_infinities_stay_in_their_rows(ops, cols):
    x = normal(12, cols, seed=1)
    dy = normal(12, cols, seed=2)
    clean = ops.layernorm_forward(x)
    cdx = ops.layernorm_backward(dy, x, clean[1], clean[2])[0]
    x2 = x.clone()
    x2[3, cols // 2] = float("inf")
    x2[7, cols - 1] = float("nan")
    y, mean, rstd = ops.layernorm_forward(x2)
    dx = ops.layernorm_backward(dy, x2, mean, rstd)[0]
    rows = [r for r in range(12) if r not in (3, 7)]
    for got, want in ((y, clean[0]), (mean, clean[1]), (rstd, clean[2]), (dx, cdx)):
        assert torch.equal(got[rows], want[rows])
    assert bool(torch.isnan(y[3]).any()) and bool(torch.isnan(y[7]).all()) and bool(torch.isnan(dx[7]).all())
    same = torch.full((4, cols), 2.5, device="cuda")   # no variance: eps keeps it finite
    assert float(ops.layernorm_forward(same)[0].abs().max()) == 0.0


def test_layernorm_no_rows_and_no_columns(ops):
    gamma = normal(300, seed=1)
    x = torch.empty(0, 300, device="cuda")
    y, mean, rstd = ops.layernorm_forward(x, gamma)
    assert y.shape == (0, 300) and mean.shape == (0,)
    dx, dg, db = ops.layernorm_backward(x, x, mean, rstd, gamma)
    assert dx.shape == (0, 300) and float(dg.abs().max()) == 0 and float(db.abs().max()) == 0
    e = torch.empty(4, 0, device="cuda")
    y, mean, rstd = ops.layernorm_forward(e)
    assert y.shape == (4, 0) and mean.shape == (4,)


def test_layernorm_gradient_against_differences(ops):
    """d/dt of <w, layernorm(x + t u)> by central differences of the fp32 forward pass. At t = 1/64 the difference quotient is off by
    t^2 / 6 times the third derivative (of the order of rstd^3 |u|^3 |w|: 1e-4 of the sums' scale here) and by the rounding of y,
    2^-24 sqrt(n) / t of it (4e-6)."""
    rows, cols, t = 6, 120, 1 / 64
    x, w, u = (normal(rows, cols, seed=s) for s in (1, 2, 3))
    gamma, beta, v = (normal(cols, seed=s) for s in (4, 5, 6))
    y, mean, rstd = ops.layernorm_forward(x, gamma, beta)
    dx, dg, db = ops.layernorm_backward(w, x, mean, rstd, gamma)

    def f(x, gamma, beta):
        return float((ops.layernorm_forward(x, gamma, beta)[0].double() * w.double()).sum())

    size = float((w.double() * gamma.double()).norm()) * float(u.double().norm()) / cols ** 0.5
    assert abs((f(x + t * u, gamma, beta) - f(x - t * u, gamma, beta)) / (2 * t) - float((dx.double() * u).sum())) < 2e-3 * size
    size = float(w.double().norm()) * float(v.double().norm())
    assert abs((f(x, gamma + t * v, beta) - f(x, gamma - t * v, beta)) / (2 * t) - float((dg.double() * v).sum())) < 1e-4 * size
    assert abs((f(x, gamma, beta + t * v) - f(x, gamma, beta - t * v)) / (2 * t) - float((db.double() * v).sum())) < 1e-4 * size


def test_layernorm_refusals(ops):
    x = normal(4, 16, dtype=torch.bfloat16)
    m = torch.zeros(4, device="cuda")
    for bad in (lambda: ops.layernorm_forward(x.t()), lambda: ops.layernorm_forward(x, normal(15)),
                lambda: ops.layernorm_forward(x, normal(16, dtype=torch.float16)), lambda: ops.layernorm_forward(x.double()),
                lambda: ops.layernorm_forward(x, normal(16), normal(16, dtype=torch.bfloat16)),
                lambda: ops.layernorm_forward(x, out=torch.empty(4, 16, device="cuda")),
                lambda: ops.layernorm_backward(x.float(), x, m, m), lambda: ops.layernorm_backward(x, x, m[:3].contiguous(), m),
                lambda: ops.layernorm_backward(x, x, m.double(), m), lambda: ops.layernorm_forward(torch.zeros((), device="cuda"))):
        with pytest.raises(ValueError):
            bad()


# ---- embedding ---------------------------------------------------------------------------------------------
def embedding_reference(table, ids, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    rows = table.double()[ids.long().clamp(0, max(0, table.shape[0] - 1))]
    return rows * scale * ok.unsqueeze(-1)


def embedding_grad_reference(dy, ids, vocab, scale, padding_id=None):
    keep = (ids >= 0) & (ids < vocab)
    if padding_id is not None:
        keep &= ids != padding_id
    total = torch.zeros(vocab, dy.shape[-1], device="cuda", dtype=torch.float64)
    size, count = torch.zeros_like(total), torch.zeros(vocab, device="cuda", dtype=torch.float64)
    d = dy.double().reshape(-1, dy.shape[-1])[keep.reshape(-1)]
    i = ids.reshape(-1)[keep.reshape(-1)].long()
    total.index_add_(0, i, d)
    size.index_add_(0, i, d.abs())
    count.index_add_(0, i, torch.ones_like(i, dtype=torch.float64))
    return total * scale, size * abs(scale), count


@pytest.mark.parametrize("types", [("F32", "F32"), ("BF16", "BF16"), ("BF16", "F32"), ("F16", "F16"), ("F16", "F32")])
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (7, 5, 3), (130, 50, 64), (33, 4000, 520), (300, 7, 1024), (5, 9, 1100), (64, 33, 777)])
def test_embedding_forward(ops, types, n, vocab, cols):
    dt, tt = DTYPES[types[0]], DTYPES[types[1]]
    table = normal(vocab, cols, seed=n, dtype=tt)
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(-2, vocab + 2, (n,), device="cuda", generator=g)
    for kind in (torch.int32, torch.int64):
        obuf, out = guarded((n, cols), dt, shift=8 if n != 33 else 1)
        got = ops.embedding(table, ids.to(kind), scale=1.7, dtype=dt, out=out)
        want = embedding_reference(table, ids, 1.7)
        # the factor is rounded to fp32 and so is the product: two roundings
        assert_within(got, want, want.abs(), "embedding", chain=2 * 2.0 ** -24)
        assert_guards(obuf, out, "embedding")
    assert ops.embedding(table, ids.view(n, 1)).shape == (n, 1, cols)


GRAD_CASES = [(1, 1, 1), (2, 1, 5), (31, 7, 64), (32, 3, 100), (33, 2, 256), (200, 100000, 40), (2048, 600, 264), (2049, 1, 128),
              (5000, 300, 1032), (9999, 1000, 33), (4100, 300000, 16), (20000, 90, 16), (40000, 3000, 20), (70000, 50000, 24),
              (140000, 700, 12), (150000, 300000, 5)]


@pytest.mark.parametrize("types", [("F32", "F32"), ("BF16", "BF16"), ("BF16", "F32"), ("F16", "F16"), ("F16", "F32")])
@pytest.mark.parametrize("n,vocab,cols", GRAD_CASES)
def test_embedding_gradient(ops, types, n, vocab, cols):
    dt, gt = DTYPES[types[0]], DTYPES[types[1]]
    dy = normal(n, cols, seed=n, dtype=dt, scale=0.1)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    ids = (torch.rand(n, device="cuda", generator=g) ** 3 * (vocab + 1)).long() - int(n > 40)   # some ids fall outside on both sides
    for kind, padding in ((torch.int64, None), (torch.int32, vocab // 2)):
        want, size, count = embedding_grad_reference(dy, ids, vocab, 0.3, padding)
        obuf, out = guarded((vocab, cols), gt, shift=8 if cols != 40 else 3)
        got = ops.embedding_backward(dy, ids.to(kind), vocab, scale=0.3, padding_id=padding, dtype=gt, out=out)
        # a chunk adds 32 rows, eight strands add the chunks' sums: at most 64 + count / 256 additions in a chain
        chain = (64 + count.max() / 256) * 2.0 ** -24
        assert_within(got, want, size, "gradient", chain=float(chain))
        assert_guards(obuf, out, "gradient")
        assert bool((got[count == 0] == 0).all())
        again = ops.embedding_backward(dy, ids.to(kind), vocab, scale=0.3, padding_id=padding, dtype=gt)
        assert torch.equal(again, got)


@pytest.mark.parametrize("types", [("F32", "F32"), ("BF16", "BF16"), ("BF16", "F32")])
@pytest.mark.parametrize("n,vocab,cols", [(3, 10, 16), (700, 90, 256), (700, 9000, 33)])
def test_embedding_gradient_accumulates(ops, types, n, vocab, cols):
    dt, gt = DTYPES[types[0]], DTYPES[types[1]]
    dy = normal(n, cols, seed=1, dtype=dt)
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(-1, vocab, (n,), device="cuda", generator=g)
    old = normal(vocab, cols, seed=3, dtype=gt)
    want, size, count = embedding_grad_reference(dy, ids, vocab, 2.0)
    got = ops.embedding_backward(dy, ids, vocab, scale=2.0, out=old.clone(), accumulate=True)
    assert_within(got, want + old.double(), size + old.double().abs(), "accumulated")
    assert torch.equal(got[count == 0], old[count == 0])


@pytest.mark.parametrize("n,vocab,cols", [(131072, 32000, 4), (131073, 3, 8), (600011, 32000, 5), (1048583, 3, 4), (1048583, 1 << 20, 4)])
def test_embedding_gradient_of_many_ids(ops, n, vocab, cols):
    """Sorts of one to three passes with hundreds of tiles. Integers whose sums stay below 2^24: exact in any order of additions."""
    g = torch.Generator(device="cuda").manual_seed(n)
    dy = torch.randint(-4, 5, (n, cols), device="cuda", generator=g).float()
    ids = (torch.rand(n, device="cuda", generator=g) ** 2 * (vocab + 1)).long() - 1
    inside = ids >= 0
    want = torch.zeros(vocab, cols, device="cuda", dtype=torch.float64).index_add_(0, ids[inside], dy[inside].double())
    obuf, out = guarded((vocab, cols), torch.float32)
    got = ops.embedding_backward(dy, ids, vocab, out=out)
    assert torch.equal(got.double(), want)
    assert_guards(obuf, out, "gradient")


def test_embedding_gradient_of_one_id_everywhere(ops):
    """Every pair names one row: the sums of all chunks are joined (1250 of them)."""
    n, vocab, cols = 40000, 1000, 72
    dy = normal(n, cols, seed=1)
    ids = torch.full((n,), 613, device="cuda")
    want, size, count = embedding_grad_reference(dy, ids, vocab, 1.0)
    got = ops.embedding_backward(dy, ids, vocab)
    assert_within(got, want, size, "one id", chain=(64 + n / 256) * 2.0 ** -24)
    nothing = ops.embedding_backward(dy, ids, vocab, padding_id=613)
    assert float(nothing.abs().max()) == 0


def test_embedding_gradient_keeps_infinities_to_their_rows(ops):
    dy = normal(300, 64, seed=1)
    ids = torch.arange(300, device="cuda") % 50
    clean = ops.embedding_backward(dy, ids, 60)
    dy[17, 3] = float("inf")     # id 17
    dy[120, 5] = float("nan")    # id 20
    got = ops.embedding_backward(dy, ids, 60)
    bad = [17, 20]
    rest = [i for i in range(60) if i not in bad]
    assert torch.equal(got[rest], clean[rest])
    assert float(got[17, 3]) == float("inf") and bool(torch.isnan(got[20, 5]))
    dropped = ids.clone()
    dropped[17] = dropped[120] = -100
    assert bool(torch.isfinite(ops.embedding_backward(dy, dropped, 60)).all())


def test_embedding_empty(ops):
    table = normal(10, 16)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops.embedding(table, none).shape == (0, 16)
    got = ops.embedding_backward(torch.empty(0, 16, device="cuda"), none, 10, out=torch.ones(10, 16, device="cuda"))
    assert float(got.abs().max()) == 0
    kept = ops.embedding_backward(torch.empty(0, 16, device="cuda"), none, 10, out=torch.ones(10, 16, device="cuda"), accumulate=True)
    assert float(kept.min()) == 1
    empty = ops.embedding(torch.empty(0, 16, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert empty.shape == (3, 16) and float(empty.abs().max()) == 0


def test_embedding_refusals(ops):
    table, ids = normal(10, 16), torch.zeros(4, dtype=torch.int64, device="cuda")
    dy = normal(4, 16)
    for bad in (lambda: ops.embedding(table.view(-1), ids), lambda: ops.embedding(table, ids.float()),
                lambda: ops.embedding(table, ids.short()), lambda: ops.embedding(table.t(), ids),
                lambda: ops.embedding(table, ids, out=torch.empty(5, 16, device="cuda")),
                lambda: ops.embedding_backward(dy, ids[:3], 10), lambda: ops.embedding_backward(dy.half(), ids, 10, dtype=torch.float64),
                lambda: ops.embedding_backward(dy, ids, 10, accumulate=True),
                lambda: ops.embedding_backward(dy, ids, 10, out=torch.empty(9, 16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    from cantors_gift_b200 import CgB200Error
    with pytest.raises(CgB200Error):
        ops.embedding(table.bfloat16(), ids, dtype=torch.float32)   # 16-bit table, fp32 output: no such kernel
    with pytest.raises(CgB200Error):
        ops.embedding_backward(dy, ids, 10, dtype=torch.bfloat16)


# ---- gradient norm and clipping -----------------------------------------------------------------------------
LISTS = {
    "one": [(1,)],
    "odd": [(3,), (17, 5), (1,), (0,), (1000,), (16384,), (16385,), (33, 333)],
    "many": [(i * 37 % 501,) for i in range(1000)],
    "large": [(1 << 22,), (777, 1001), (5,)],
}


def gradient_list(name, dtype, shift=0):
    out = []
    for i, shape in enumerate(LISTS[name]):
        dt = DTYPES[dtype] if dtype != "mixed" else list(DTYPES.values())[i % 3]
        _, t = guarded(shape, dt, shift=(i % 8 if shift else 0))
        t.copy_(normal(*shape, seed=i, dtype=dt, scale=0.1))
        out.append(t)
    return out


def check_clip(got_norm, got, grads, max_norm):
    norm = sum(float((t.double() ** 2).sum()) for t in grads) ** 0.5
    # a packet adds up to 8 squares in fp32 (8 roundings of the square, halved by the root), the result is rounded once
    assert abs(float(got_norm) - norm) <= 6 * 2.0 ** -24 * norm
    factor = min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(got, grads):
        want = g.double() * factor
        # the factor carries the norm's error and its own rounding, the product one more
        if g.numel():
            assert_within(o, want, want.abs(), "clipped", chain=8 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("shift", [0, 1])
def test_clip(ops, name, dtype, shift):
    grads = gradient_list(name, dtype, shift)
    norm = float(ops.grad_norm(grads))
    for max_norm in (norm / 3, norm * 2, 0.0):
        wide = [torch.full_like(t, 9.0, dtype=torch.float32) for t in grads]
        check_clip(ops.clip_grad_norm(grads, max_norm, out=wide), wide, grads, max_norm)
        same = [torch.full_like(t, 9.0) for t in grads]
        check_clip(ops.clip_grad_norm(grads, max_norm, out=same), same, grads, max_norm)
        place = [t.clone() for t in grads]
        n = ops.clip_grad_norm(place, max_norm)
        check_clip(n, place, grads, max_norm)
        for a, b in zip(place, same):
            assert torch.equal(a, b)
    assert float(ops.grad_norm(grads)) == norm


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("size", [1e25, 1e-25])
def test_norm_beyond_the_range_of_fp32_squares(ops, dtype, size):
    g = normal(5000, seed=1, scale=size).to(DTYPES[dtype])
    check_clip(ops.grad_norm([g, g]), [], [g, g], 1.0)


def test_clip_infinities_and_zeros(ops):
    z = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=torch.float16)]
    assert float(ops.clip_grad_norm(z, 1.0)) == 0 and float(z[0].abs().max()) == 0
    g = [normal(100), normal(50, seed=2)]
    g[0][3] = float("inf")
    assert float(ops.clip_grad_norm(g, 1.0)) == float("inf")
    assert bool(torch.isnan(g[0][3])) and float(g[1].abs().max()) == 0
    g = [normal(100), normal(50, seed=2)]
    g[0][3] = float("nan")
    assert bool(torch.isnan(ops.clip_grad_norm(g, 1.0)))
    assert bool(torch.isnan(g[0]).all()) and bool(torch.isnan(g[1]).all())


def test_clip_no_write_outside(ops):
    bufs = [guarded((1003,), torch.bfloat16, 3), guarded((40001,), torch.float32, 1)]
    for b, v in bufs:
        v.copy_(normal(*v.shape, seed=3, dtype=v.dtype))
    ops.clip_grad_norm([v for _, v in bufs], 0.01)
    for b, v in bufs:
        assert_guards(b, v, "clip")


def test_clip_refusals(ops):
    g = normal(64)
    for bad in (lambda: ops.clip_grad_norm([], 1.0), lambda: ops.clip_grad_norm([g], 1.0, out=[]),
                lambda: ops.clip_grad_norm([g], 1.0, out=[normal(63)]), lambda: ops.clip_grad_norm([g.view(8, 8).t()], 1.0),
                lambda: ops.clip_grad_norm([g.double()], 1.0), lambda: ops.clip_grad_norm([g, g.cpu()], 1.0)):
        with pytest.raises(ValueError):
            bad()
    from cantors_gift_b200 import CgB200Error
    other, half = normal(64, seed=1), torch.empty(64, dtype=torch.float16, device="cuda")
    for bad in (lambda: ops.clip_grad_norm([g], -1.0), lambda: ops.clip_grad_norm([g], 1.0, out=[half]),
                lambda: ops.clip_grad_norm([g, g], 1.0),                                          # scaled twice
                lambda: ops.clip_grad_norm([g, g[8:16]], 1.0),                                     # in part
                lambda: ops.clip_grad_norm([g, other], 1.0, out=[torch.empty_like(g), g]),         # over another gradient
                lambda: ops.clip_grad_norm([g, other], 1.0, out=[half.float()] * 2)):
        with pytest.raises(CgB200Error):
            bad()
    assert float(ops.grad_norm([g, g])) > 0   # reading one twice is no harm


# ---- streams, graphs, and the operators one after another ----------------------------------------------------
def one_step(ops, table, ids, gamma, beta, dout, max_norm):
    """ids -> embedding -> layer norm, and back: the gradients of <layernorm(embedding), dout>, clipped."""
    x = ops.embedding(table, ids, scale=3.0)
    y, mean, rstd = ops.layernorm_forward(x, gamma, beta)
    dx, dgamma, dbeta = ops.layernorm_backward(dout, x, mean, rstd, gamma)
    dtable = ops.embedding_backward(dx, ids, table.shape[0], scale=3.0, padding_id=0)
    grads = [dtable, dgamma, dbeta]
    norm = ops.clip_grad_norm(grads, max_norm)
    return y, norm, grads


def step_inputs(seed=0, n=(5, 41), vocab=97, cols=200):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, n, device="cuda", generator=g)
    return normal(vocab, cols, seed=seed), ids, normal(cols, seed=seed + 1, offset=1.0), normal(cols, seed=seed + 2), normal(*n, cols, seed=seed + 3)


def test_a_training_step_against_autograd_in_64_bits(ops):
    table, ids, gamma, beta, dout = step_inputs()
    y, norm, grads = one_step(ops, table, ids, gamma, beta, dout, 5.0)
    leaves = [t.double().requires_grad_() for t in (table, gamma, beta)]
    wy = torch.nn.functional.layer_norm(leaves[0][ids] * 3.0, (table.shape[1],), leaves[1], leaves[2], 1e-5)
    (wy * dout.double()).sum().backward()
    wy = wy.detach()
    want = [t.grad for t in leaves]
    want[0][0] = 0
    wnorm = sum(float((t ** 2).sum()) for t in want) ** 0.5
    # the chain of roundings from end to end is below 256 steps of 2^-24 of each tensor's size
    tol = 256 * 2.0 ** -24
    assert abs(float(norm) / wnorm - 1) < tol
    assert float((y.double() - wy).norm() / wy.norm()) < tol
    for g, w in zip(grads, want):
        w = w * min(1.0, 5.0 / (wnorm + 1e-6))
        assert float((g.double() - w).norm() / w.norm()) < tol


def test_another_stream_gives_the_same(ops):
    args = step_inputs(seed=3)
    y, norm, grads = one_step(ops, *args, 1.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    x = ops.embedding(args[0], args[1], scale=3.0, stream=s)
    y2, mean, rstd = ops.layernorm_forward(x, args[2], args[3], stream=s)
    dx, dg, db = ops.layernorm_backward(args[4], x, mean, rstd, args[2], stream=s)
    dt = ops.embedding_backward(dx, args[1], args[0].shape[0], scale=3.0, padding_id=0, stream=s)
    norm2 = ops.clip_grad_norm([dt, dg, db], 1.0, stream=s)
    plain = ops.grad_norm([y], stream=s)
    s.synchronize()
    assert torch.equal(y, y2) and torch.equal(norm, norm2)
    assert float(plain) == float(ops.grad_norm([y]))
    for a, b in zip(grads, (dt, dg, db)):
        assert torch.equal(a, b)


def test_captured_graphs_replay_side_by_side(ops):
    """Two captured steps of different sizes, replayed at once on two streams, over new values in the same tensors: each has its own
    workspaces, and an eager step between them disturbs neither."""
    sets = [step_inputs(seed=5), step_inputs(seed=6, n=(3000,), vocab=50, cols=333)]
    graphs, results = [], []
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        for a in sets:
            one_step(ops, *a, 1.0)
    torch.cuda.synchronize()
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(one_step(ops, *a, 1.0))
        graphs.append(g)
    fresh = [step_inputs(seed=15), step_inputs(seed=16, n=(3000,), vocab=50, cols=333)]
    for a, f in zip(sets, fresh):
        for t, v in zip(a, f):
            t.copy_(v)
    wants = [one_step(ops, *f, 1.0) for f in fresh]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    one_step(ops, *fresh[1], 1.0)
    torch.cuda.synchronize()
    for (y, norm, grads), (wy, wnorm, wgrads) in zip(results, wants):
        assert torch.equal(y, wy) and torch.equal(norm, wnorm)
        for a, b in zip(grads, wgrads):
            assert torch.equal(a, b)


def test_the_same_inputs_give_the_same_bits(ops):
    args = step_inputs(seed=8, n=(4097,), vocab=20, cols=1024)
    first = one_step(ops, *args, 1.0)
    for _ in range(3):
        again = one_step(ops, *args, 1.0)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        for a, b in zip(first[2], again[2]):
            assert torch.equal(a, b)


def test_two_calls_at_once_on_two_streams(ops):
    """The same operators on two streams, neither waiting for the other: each call has workspaces of its own."""
    sets = [step_inputs(seed=21, n=(6000,), vocab=300, cols=513), step_inputs(seed=22, n=(9000,), vocab=40, cols=264)]
    wants = [one_step(ops, *a, 1.0) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    gots = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                gots[k].append(one_step(ops, *sets[k], 1.0))
    torch.cuda.synchronize()
    for (wy, wnorm, wgrads), got in zip(wants, gots):
        for y, norm, grads in got:
            assert torch.equal(y, wy) and torch.equal(norm, wnorm)
            for a, b in zip(grads, wgrads):
                assert torch.equal(a, b)


def test_a_first_call_can_be_captured():
    """The operators set nothing up that a capture would refuse: in a new process, the first call of each is a captured one."""
    import subprocess
    import sys
    from conftest import ROOT
    code = """
import torch
from cantors_gift_b200 import ops
x = torch.randn(40, 300, device="cuda"); gamma = torch.randn(300, device="cuda")
ids = torch.randint(0, 90, (40,), device="cuda"); table = torch.randn(90, 300, device="cuda")
torch.cuda.synchronize()
def step():
    e = ops.embedding(table, ids)
    y, m, r = ops.layernorm_forward(e, gamma, gamma)
    dx, dg, db = ops.layernorm_backward(x, e, m, r, gamma)
    dt = ops.embedding_backward(dx, ids, 90)
    n = ops.grad_norm([dt, dg, db])
    ops.clip_grad_norm([dt, dg, db], 0.5)
    return y, dt, dg, db, n
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay(); torch.cuda.synchronize()
for a, b in zip(out, step()):
    assert torch.equal(a, b)
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


# ---- offsets that pass 32 bits ---------------------------------------------------------------------------------
def test_layernorm_beyond_32_bit_offsets(ops):
    """2.3e9 elements; all rows alike but the last three, which must come out as they do by themselves."""
    rows, cols = 140001, 16384
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[:, ::2] = 1.0
    tail = normal(3, cols, seed=1, dtype=torch.bfloat16)
    x[-3:] = tail
    gamma = normal(cols, seed=2)
    y, mean, rstd = ops.layernorm_forward(x, gamma, gamma, out=torch.empty_like(x))
    wy, wm, wr = ops.layernorm_forward(tail, gamma, gamma)
    assert torch.equal(y[-3:], wy) and torch.equal(mean[-3:], wm) and torch.equal(rstd[-3:], wr)
    assert torch.equal(y[0], y[rows // 2]) and float(mean[7]) == 0.5
    dx, dg, db = ops.layernorm_backward(x, x, mean, rstd, gamma, dx=y)
    wdx = ops.layernorm_backward(tail, tail, wm, wr, gamma)[0]
    assert torch.equal(dx[-3:], wdx)
    # dbeta: half of the columns add 1 in every row but the last three
    want = (rows - 3) * (torch.arange(cols, device="cuda") % 2 == 0).double() + tail.double().sum(0)
    assert_within(db, want, want.abs() + tail.double().abs().sum(0), "dbeta")


def test_embedding_beyond_32_bit_offsets(ops):
    vocab, cols = 1100000, 2048     # 2.25e9 elements
    table = torch.zeros(vocab, cols, device="cuda", dtype=torch.bfloat16)
    table[-2:] = normal(2, cols, seed=1, dtype=torch.bfloat16)
    ids = torch.tensor([0, vocab - 1, vocab - 2, vocab], device="cuda")
    out = ops.embedding(table, ids)
    assert torch.equal(out[1], table[-1]) and torch.equal(out[2], table[-2]) and float(out[0].abs().max()) == 0 and float(out[3].abs().max()) == 0
    dy = normal(4, cols, seed=2, dtype=torch.bfloat16)
    grad = ops.embedding_backward(dy, ids, vocab, out=table)
    assert torch.equal(grad[-1], dy[1]) and torch.equal(grad[-2], dy[2]) and torch.equal(grad[0], dy[0])
    assert float(grad[1:-2].abs().amax()) == 0
    del table, grad
    n = 1100000
    ids = torch.arange(n, device="cuda") % 7
    dy = torch.ones(n, cols, device="cuda", dtype=torch.bfloat16)
    grad = ops.embedding_backward(dy, ids, 9, dtype=torch.float32)
    count = torch.bincount(ids, minlength=9).float()
    assert torch.equal(grad, count[:, None].expand(9, cols))    # whole numbers below 2^24: exact in fp32
    assert float(ops.embedding(grad.bfloat16(), ids, out=dy)[-1, -1]) == float(count[int(ids[-1])].bfloat16())


def test_clip_beyond_32_bit_offsets(ops):
    n = (1 << 31) + 1001
    g = torch.full((n,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    norm = ops.clip_grad_norm([g], 2.0)
    want = (n * 2.0 ** -20) ** 0.5
    assert abs(float(norm) - want) <= 6 * 2.0 ** -24 * want
    value = torch.tensor(2.0 ** -10 * 2.0 / (want + 1e-6), dtype=torch.float64).to(torch.bfloat16)
    assert float(g.min()) == float(value) == float(g.max())
