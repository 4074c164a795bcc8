"""Training operators around the transformer block, as measured cases: layer norm with its backward pass, token embedding with
its gradient, and clipping of a gradient list by its global norm.

Each case is a dict of plain values. `prepare` makes its inputs on the GPU from a seed, `run` is one pass through the operator
(`own` chooses between elementary torch operations in 32 bits and this repository's kernels), `exact` is the same result from the
definition in 64 bits, `work` the bytes and operations that one pass cannot do without."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5
PADDING_ID = 1


def listed():
    return [
        # the encoder block's layer norm at its full batch: 32 sequences of 2048 tokens, d_model 1024
        dict(name="ln_fwd block", op="ln_fwd", rows=65536, cols=1024, dtype="bf16", params="bf16"),
        # wide rows of an fp32 model with a width that no vector load divides
        dict(name="ln_fwd odd f32", op="ln_fwd", rows=4099, cols=4097, dtype="f32", params="f32"),
        # a short fine-tuning sequence: the launch counts
        dict(name="ln_fwd small", op="ln_fwd", rows=77, cols=1024, dtype="f16", params="f16"),
        # the row-kernel configuration's 32768 x 4096, 16-bit activations with fp32 parameters
        dict(name="ln_bwd wide", op="ln_bwd", rows=32768, cols=4096, dtype="bf16", params="f32"),
        # ragged token count and width, everything in fp32
        dict(name="ln_bwd odd f32", op="ln_bwd", rows=9001, cols=1001, dtype="f32", params="f32"),
        dict(name="ln_bwd small", op="ln_bwd", rows=77, cols=1024, dtype="f16", params="f16"),
        # the block's batch looked up in a 32000-word table, ids by a natural frequency law
        dict(name="emb_fwd block", op="emb_fwd", n=65536, vocab=32000, cols=1024, dtype="bf16", table="bf16", ids=8, pad=0),
        # an fp32 master table read into 16-bit activations by one short ragged batch
        dict(name="emb_fwd small", op="emb_fwd", n=509, vocab=5003, cols=520, dtype="f16", table="f32", ids=4, pad=8),
        # the same batch's gradient into an fp32 table, an eighth of each sequence padding
        dict(name="emb_bwd block", op="emb_bwd", n=65536, vocab=32000, cols=1024, dtype="bf16", table="f32", ids=8, pad=8),
        # a large vocabulary against few tokens: the untouched rows are most of the work
        dict(name="emb_bwd large table", op="emb_bwd", n=8191, vocab=128000, cols=2048, dtype="bf16", table="bf16", ids=8, pad=0),
        # ten layers of width 1024 (16-bit matrices, fp32 norm parameters), with an output table, clipped into the fp32 gradients an optimizer takes
        dict(name="clip blocks", op="clip", layers=10, width=1024, dtype="bf16", out="f32", norm=0.25),
        # a small fp32 model with odd sizes
        dict(name="clip small", op="clip", layers=2, width=129, dtype="f32", out="f32", norm=4.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):
        w = spread(lo, hi)
        return max(lo, w // 64 * 64) if rng.random() < 0.6 else w

    op = rng.choice(["ln_fwd", "ln_bwd", "emb_fwd", "emb_bwd", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("ln_fwd", "ln_bwd"):
        cols = width(64, 12288)
        rows = spread(1, max(2, min(65536, 50_000_000 // cols)))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, params=rng.choice([dtype, "f32"]))
    if op in ("emb_fwd", "emb_bwd"):
        cols = width(64, 8192)
        vocab = spread(1000, min(200000, (1 << 27) // cols))
        n = spread(1, max(2, min(131072, (1 << 25) // cols)))
        return dict(op=op, n=n, vocab=vocab, cols=cols, dtype=dtype, table=rng.choice([dtype, "f32"]), ids=rng.choice([4, 8]), pad=rng.choice([0, 8]))
    return dict(op=op, layers=rng.randint(1, 10), width=spread(48, 700 if dtype == "f32" else 1024), dtype=dtype, out=rng.choice([dtype, "f32"]), norm=rng.choice([0.25, 1.0, 1e6]))


def _shapes(case):
    """The gradient list: an embedding table, and for each layer two vectors of the norm (fp32) and the block's matrices and a bias."""
    w = case["width"]
    layer = [(w,), (w,), (2 * w, w), (4 * w, w), (w, 4 * w), (4 * w,)]
    return [(8 * w, w)] + layer * case["layers"]


def _list_dtypes(case):
    return [torch.float32 if len(s) == 1 and s[0] == case["width"] else DTYPES[case["dtype"]] for s in _shapes(case)]


def _id_probabilities(vocab):
    """Frequency law of the ids: id v has probability ln((v+2)/(v+1)) / ln(vocab+1)."""
    v = np.arange(vocab, dtype=np.float64)
    return np.log((v + 2) / (v + 1)) / math.log(vocab + 1)


def _distinct(case):
    """Expected number of different ids in a batch."""
    p, n = _id_probabilities(case["vocab"]), case["n"]
    live = n - (n // case["pad"] if case["pad"] else 0)
    return float(np.sum(-np.expm1(live * np.log1p(-np.minimum(p, 1 - 1e-12))))) + (1 if case["pad"] else 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    op, dt = case["op"], DTYPES[case["dtype"]]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, pt = case["rows"], case["cols"], DTYPES[case["params"]]
        # a residual stream: rows of different size, channels with an offset
        x = ((normal(rows, cols) * (0.5 + normal(rows, 1).abs())) + normal(1, cols)).to(dt)
        gamma, beta = (1 + 0.2 * normal(cols)).to(pt), (0.1 * normal(cols)).to(pt)
        s = dict(case=case, x=x, gamma=gamma, beta=beta)
        if op == "ln_bwd":
            s["dy"] = (0.05 * normal(rows, cols)).to(dt)
            xf = x.float()
            s["mean"] = xf.mean(dim=1)
            s["rstd"] = (xf.var(dim=1, unbiased=False) + EPS).rsqrt()
        return s
    if op in ("emb_fwd", "emb_bwd"):
        n, vocab, cols = case["n"], case["vocab"], case["cols"]
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        ids = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)
        if case["pad"]:
            ids[n - n // case["pad"]:] = PADDING_ID
        s = dict(case=case, ids=ids.to(torch.int32 if case["ids"] == 4 else torch.int64), scale=math.sqrt(cols))
        if op == "emb_fwd":
            s["table"] = (0.02 * normal(vocab, cols)).to(DTYPES[case["table"]])
        else:
            s["dy"] = (0.01 * normal(n, cols)).to(dt)
        return s
    grads = [(0.01 * normal(*shape)).to(t) for shape, t in zip(_shapes(case), _list_dtypes(case))]
    out = [torch.empty_like(t, dtype=DTYPES[case["out"]] if len(t.shape) == 2 else t.dtype) for t in grads]
    return dict(case=case, grads=grads, out=out)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from cantors_gift_b200 import ops
        if op == "ln_fwd":
            return ops.layernorm_forward(state["x"], state["gamma"], state["beta"], eps=EPS)
        if op == "ln_bwd":
            return ops.layernorm_backward(state["dy"], state["x"], state["mean"], state["rstd"], state["gamma"])
        if op == "emb_fwd":
            return ops.embedding(state["table"], state["ids"], scale=state["scale"], dtype=DTYPES[case["dtype"]])
        if op == "emb_bwd":
            return ops.embedding_backward(state["dy"], state["ids"], case["vocab"], scale=state["scale"],
                                          padding_id=PADDING_ID if case["pad"] else None, dtype=DTYPES[case["table"]])
        norm = ops.clip_grad_norm(state["grads"], case["norm"], out=state["out"])
        return [norm] + state["out"]

    if op == "ln_fwd":
        x = state["x"].float()
        mean = x.mean(dim=1, keepdim=True)
        d = x - mean
        rstd = ((d * d).mean(dim=1, keepdim=True) + EPS).rsqrt()
        y = d * rstd * state["gamma"].float() + state["beta"].float()
        return y.to(state["x"].dtype), mean.squeeze(1), rstd.squeeze(1)
    if op == "ln_bwd":
        rstd = state["rstd"].unsqueeze(1)
        dy = state["dy"].float()
        xhat = (state["x"].float() - state["mean"].unsqueeze(1)) * rstd
        gy = dy * state["gamma"].float()
        dx = rstd * (gy - gy.mean(dim=1, keepdim=True) - xhat * (gy * xhat).mean(dim=1, keepdim=True))
        pt = state["gamma"].dtype
        return dx.to(state["x"].dtype), (dy * xhat).sum(dim=0).to(pt), dy.sum(dim=0).to(pt)
    if op == "emb_fwd":
        return (state["table"][state["ids"].long()].float() * state["scale"]).to(DTYPES[case["dtype"]])
    if op == "emb_bwd":
        dy, ids = state["dy"].float(), state["ids"].long()
        if case["pad"]:
            dy = dy * (ids != PADDING_ID).unsqueeze(1)
        total = torch.zeros(case["vocab"], case["cols"], device="cuda").index_add_(0, ids, dy)
        return (total * state["scale"]).to(DTYPES[case["table"]])
    squares = torch.stack([(t.float() * t.float()).sum() for t in state["grads"]])
    norm = squares.double().sum().sqrt()
    factor = (case["norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return [norm.float()] + [(t.float() * factor).to(o.dtype) for t, o in zip(state["grads"], state["out"])]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        y, mean, rstd = [], [], []
        for x in s["x"].split(4096):
            x = x.double()
            m = x.sum(1) / case["cols"]
            var = ((x - m[:, None]) ** 2).sum(1) / case["cols"]
            r = 1 / torch.sqrt(var + EPS)
            y.append((x - m[:, None]) * r[:, None] * s["gamma"].double() + s["beta"].double())
            mean.append(m)
            rstd.append(r)
        return torch.cat(y), torch.cat(mean), torch.cat(rstd)
    if op == "ln_bwd":
        # with h = (x - mean) rstd: dx = J^T (gamma dy), J = rstd (I - 1 1^T / C - h h^T / C)
        cols = case["cols"]
        dx, dgamma, dbeta = [], 0, 0
        for x, dy, m, r in zip(*(s[k].split(4096) for k in ("x", "dy", "mean", "rstd"))):
            h = (x.double() - m.double()[:, None]) * r.double()[:, None]
            dy = dy.double()
            dgamma = dgamma + torch.einsum("rc,rc->c", dy, h)
            dbeta = dbeta + dy.sum(0)
            t = dy * s["gamma"].double()
            along = torch.einsum("rc,rc->r", t, h) / cols
            dx.append((t - t.sum(1, keepdim=True) / cols - h * along[:, None]) * r.double()[:, None])
        return torch.cat(dx), dgamma, dbeta
    if op == "emb_fwd":
        return torch.nn.functional.one_hot(s["ids"].long(), case["vocab"]).double() @ (s["table"].double() * s["scale"]) \
            if case["n"] * case["vocab"] < 1 << 24 else s["table"].double().index_select(0, s["ids"].long()) * s["scale"]
    if op == "emb_bwd":
        keep = s["ids"].long() != (PADDING_ID if case["pad"] else -1)
        total = torch.zeros(case["vocab"], case["cols"], device="cuda", dtype=torch.float64)
        total.index_put_((s["ids"].long()[keep],), s["dy"][keep].double() * s["scale"], accumulate=True)
        return total
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.double())) ** 2 for t in s["grads"]))
    factor = min(1.0, case["norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64)] + [t.double() * factor for t in s["grads"]]


def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op in ("ln_fwd", "ln_bwd"):
        r, c, pe = case["rows"], case["cols"], BYTES[case["params"]]
        if op == "ln_fwd":   # x, gamma, beta in; y, mean, rstd out
            return dict(bytes=2 * r * c * e + 2 * c * pe + 8 * r, flops=8 * r * c)
        return dict(bytes=3 * r * c * e + 3 * c * pe + 8 * r, flops=14 * r * c)   # x, dy, gamma, mean, rstd in; dx, dgamma, dbeta out
    if op in ("emb_fwd", "emb_bwd"):
        n, c, te = case["n"], case["cols"], BYTES[case["table"]]
        if op == "emb_fwd":   # the rows that occur, once each
            return dict(bytes=_distinct(case) * c * te + n * c * e + n * case["ids"], flops=n * c)
        live = n - (n // case["pad"] if case["pad"] else 0)
        return dict(bytes=live * c * e + n * case["ids"] + case["vocab"] * c * te, flops=live * c + case["vocab"] * c)
    total = flops = 0
    for shape, t in zip(_shapes(case), _list_dtypes(case)):
        size = 4 if t == torch.float32 else 2
        total += math.prod(shape) * (size + (BYTES[case["out"]] if len(shape) == 2 else size))
        flops += 3 * math.prod(shape)   # square, add, scale
    return dict(bytes=total, flops=flops)
