"""The operators of a full-catalogue softmax model and their plain forms: embedding lookup with its gradient by sorted
tokens, layer norm with its weight gradients, log probabilities of given items with entropy and top alternatives, and the
global gradient norm with clipping. `run` computes a case with the framework's kernels where `own` is true and with
elementary torch operations in 32 bits elsewhere; `exact` computes it in 64 bits."""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5             # layer norm
CLIP_EPS = 1e-6        # in the clipping coefficient's denominator
MAX_NORM = 1.0
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the user rows of one training batch out of the user table (35 598 users, batch 1024): pure latency
        dict(name="embed batch users", op="embed", rows=35598, d=64, n=1024, dtype="float32", grad=False),
        # one training batch of item histories, 50 items each, with the item table's gradient
        dict(name="embed histories train", op="embed", rows=18357, d=64, n=51200, dtype="float32", grad=True),
        # a million-item table at width 128, as many tokens as items: the largest gradient
        dict(name="embed million train", op="embed", rows=1000000, d=128, n=1000003, dtype="bfloat16", grad=True),
        # the norm of one batch of user vectors before scoring, serving: pure latency
        dict(name="norm batch users", op="norm", rows=1024, d=64, dtype="float32", grad=False),
        # histories through a norm in training, an odd number of rows
        dict(name="norm histories train", op="norm", rows=51197, d=256, dtype="float32", grad=True),
        # raw image features (width 4096) of a large batch, training
        dict(name="norm features train", op="norm", rows=65536, d=4096, dtype="bfloat16", grad=True),
        # one user against a million items, with the alternatives an answer shows: one long row
        dict(name="logprobs one user", op="logprobs", rows=1, cols=1000000, k=20, dtype="float32", masked=0.0, grad=False),
        # evaluation of a batch: seen items at -inf, 50 alternatives
        dict(name="logprobs evaluation", op="logprobs", rows=1024, cols=18357, k=50, dtype="float32", masked=0.01, grad=False),
        # training on the full catalogue: loss, entropy and the scores' gradient
        dict(name="logprobs train", op="logprobs", rows=8192, cols=35598, k=0, dtype="bfloat16", masked=0.0, grad=True),
        # clipping the gradients of a small model: 24 tensors
        dict(name="clip small", op="clip", tensors=24, numel=300000, dtype="float32"),
        # clipping many small half-precision tensors of odd sizes
        dict(name="clip many", op="clip", tensors=600, numel=60000000, dtype="bfloat16"),
        # clipping the gradients of 2 M user and 1 M item rows at width 128
        dict(name="clip tables", op="clip", tensors=9, numel=384000000, dtype="float32"),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "norm", "logprobs", "clip"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "embed":
        d = rng.choice([32, 64, 65, 100, 128, 256, 1000, 1024])
        n = _between(rng, 1, 60000000 // d)
        rows = _between(rng, 100, min(1000000, 120000000 // d))
        return dict(op=op, rows=rows, d=d, n=n, dtype=dtype, grad=rng.random() < 0.7)
    if op == "norm":
        d = _between(rng, 16, 16384)
        if rng.random() < 0.6:
            d = max(16, d // 64 * 64)
        rows = _between(rng, 1, min(200000, 130000000 // d))
        return dict(op=op, rows=rows, d=d, dtype=dtype, grad=rng.random() < 0.6)
    if op == "logprobs":
        cols = _between(rng, 1000, 1000000)
        rows = _between(rng, 1, min(8192, 100000000 // cols))
        return dict(op=op, rows=rows, cols=cols, k=rng.choice([0, 1, 5, 10, 20, 50]), dtype=dtype,
                    masked=rng.choice([0.0, 0.01, 0.5]), grad=rng.random() < 0.5)
    return dict(op=op, tensors=_between(rng, 1, 800), numel=_between(rng, 10000, 100000000), dtype=dtype)


def _sizes(case):
    """Numbers of elements of a gradient list: a few large tensors, many small ones, odd sizes among them."""
    k, total = case["tensors"], case["numel"]
    w = [1.0 / (1 + i) ** 1.2 for i in range(k)]
    s = sum(w)
    return [max(1, int(total * x / s) - (i % 3)) for i, x in enumerate(w)]


def _bucket(case, t):
    """One flat buffer that holds the clipped gradients, each from a 16-byte boundary on, and its pieces."""
    sizes = _sizes(case)
    step = [-(-m // 8) * 8 for m in sizes]
    flat = torch.zeros(sum(step), dtype=t, device=DEVICE)
    return flat, [p[:m] for p, m in zip(flat.split(step), sizes)]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _popular(n, rows, g):
    """Row numbers whose popularity falls with rank^-0.8 (the synthetic graphs' item popularity), ranks shuffled."""
    cdf = torch.arange(1, rows + 1, dtype=torch.float64, device=DEVICE).pow_(-0.8).cumsum_(0)
    u = torch.rand(n, generator=g, dtype=torch.float64, device=DEVICE) * cdf[-1]
    r = torch.searchsorted(cdf, u).clamp_(max=rows - 1)
    return torch.randperm(rows, generator=g, device=DEVICE)[r]


def prepare(case, seed):
    g, t = _gen(seed), TYPES[case["dtype"]]
    s = {"case": case}
    normal = lambda *shape: torch.randn(shape, generator=g, dtype=torch.float32, device=DEVICE)  # noqa: E731
    if case["op"] == "embed":
        n, rows, d = case["n"], case["rows"], case["d"]
        s["table"] = (normal(rows, d) * 0.1).to(t).requires_grad_(case["grad"])
        s["idx"] = _popular(n, rows, g)
        s["scale"] = math.sqrt(d)
        if case["grad"]:
            s["gout"] = (normal(n, d) * 0.01).to(t)
    elif case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        s["x"] = (normal(rows, d) * 2 + 0.5).to(t).requires_grad_(case["grad"])
        s["w"] = (1 + 0.1 * normal(d)).to(t).requires_grad_(case["grad"])
        s["b"] = (0.1 * normal(d)).to(t).requires_grad_(case["grad"])
        if case["grad"]:
            s["gout"] = (normal(rows, d) * 0.01).to(t)
    elif case["op"] == "logprobs":
        rows, cols = case["rows"], case["cols"]
        x = normal(rows, cols) * 3
        s["target"] = torch.randint(cols, (rows,), generator=g, device=DEVICE)
        if case["masked"]:
            out = torch.rand((rows, cols), generator=g, device=DEVICE) < case["masked"]
            out.scatter_(1, s["target"].unsqueeze(1), False)          # the asked item is among those that are left
            x.masked_fill_(out, -math.inf)
        s["x"] = x.to(t).requires_grad_(case["grad"])
        if case["grad"]:
            # the mean over the rows; with half precision the loss is scaled up, as its range demands
            scale = 1000.0 if case["dtype"] == "float16" else 1.0 / rows
            s["glogp"] = normal(rows) * scale
            s["gentropy"] = normal(rows) * (0.01 * scale)
    else:
        s["grads"] = [(normal(m) * 0.01).to(t) for m in _sizes(case)]
        s["bucket"], s["out"] = _bucket(case, t)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from mmssl_amd import ops, optim
    case = s["case"]
    if case["op"] == "embed":
        out = ops.embed_rows(s["table"], s["idx"], scale=s["scale"])
        if not case["grad"]:
            return out
        return (out,) + torch.autograd.grad(out, (s["table"],), s["gout"])
    if case["op"] == "norm":
        y = ops.layernorm_rows(s["x"], s["w"], s["b"], eps=EPS)
        if not case["grad"]:
            return y
        return (y,) + torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gout"])
    if case["op"] == "logprobs":
        logp, entropy, top_logp, top_idx = ops.logprobs_rows(s["x"], s["target"], k=case["k"])
        grads = torch.autograd.grad((logp, entropy), (s["x"],), (s["glogp"], s["gentropy"])) if case["grad"] else ()
        return [logp, entropy] + ([top_logp, top_idx] if case["k"] else []) + list(grads)
    total = optim.clip_grads(s["grads"], MAX_NORM, out=s["out"])
    return total, s["bucket"]


@torch.no_grad()
def _plain(s):
    case = s["case"]
    if case["op"] == "embed":
        table, idx = s["table"], s["idx"]
        out = (table[idx].float() * s["scale"]).to(table.dtype)
        if not case["grad"]:
            return out
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        grad.index_add_(0, idx, s["gout"].float() * s["scale"])
        return out, grad.to(table.dtype)
    if case["op"] == "norm":
        t = s["x"].dtype
        x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
        x = x - x.mean(1, keepdim=True)
        r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        h = x * r
        y = (h * w + b).to(t)
        if not case["grad"]:
            return y
        g = s["gout"].float()
        gw, gb = (g * h).sum(0), g.sum(0)
        g = g * w
        gx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        return y, gx.to(t), gw.to(t), gb.to(t)
    if case["op"] == "logprobs":
        raw, target = s["x"], s["target"].unsqueeze(1)
        x = raw.float()
        u = x - x.max(1, keepdim=True).values
        p = torch.exp(u)
        total = p.sum(1, keepdim=True)
        lp = u - torch.log(total)
        p = p / total
        logp = lp.gather(1, target).squeeze(1)
        held = lp.masked_fill(p == 0, 0.0)                             # 0 log 0 = 0
        entropy = -(p * held).sum(1, keepdim=True)
        outs = [logp, entropy.squeeze(1)]
        if case["k"]:
            top = _top(x, case["k"])
            outs += [lp.gather(1, top), top]
        if case["grad"]:
            g = -p * (s["glogp"].unsqueeze(1) + s["gentropy"].unsqueeze(1) * (held + entropy))
            g.scatter_add_(1, target, s["glogp"].unsqueeze(1))
            outs.append(g.to(raw.dtype))
        return outs
    total = torch.stack([x.float().square().sum() for x in s["grads"]]).sum().sqrt()
    c = (MAX_NORM / (total + CLIP_EPS)).clamp(max=1.0)
    for x, o in zip(s["grads"], s["out"]):
        torch.mul(x.float(), c, out=o)
    return total, s["bucket"]


def _top(x, k):
    """Columns of the k largest values of each row, ties to the lowest column: the value's bits in an order of whole
    numbers above the column's complement."""
    key = x.view(torch.int32).to(torch.int64)
    key = torch.where(key < 0, -(key & 0x7FFFFFFF), key)
    key = key * (1 << 31) + (x.shape[1] - torch.arange(x.shape[1], device=x.device))
    return key.topk(k, dim=1).indices


# ---------------------------------------------------------------------------------------------------------------------
# work and the values in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations that a pass cannot do without: inputs read once, outputs written once."""
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "embed":
        n, rows, d = case["n"], case["rows"], case["d"]
        # rows that are looked up: at most all, at most one for each token
        size, flops = 8 * n + min(n, rows) * d * e + n * d * e, n * d
        if case["grad"]:
            size, flops = size + n * d * e + rows * d * e, flops + 2 * n * d
        return {"bytes": size, "flops": flops}
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        # forward: x in, y out; backward: the gradient in, gx out (x counts once for both)
        if case["grad"]:
            return {"bytes": 4 * n * d * e + 4 * d * e, "flops": 20 * n * d}
        return {"bytes": 2 * n * d * e + 2 * d * e, "flops": 8 * n * d}
    if case["op"] == "logprobs":
        n, c, k = case["rows"], case["cols"], case["k"]
        size, flops = n * c * e + n * (16 + 12 * k), 6 * n * c
        if case["grad"]:
            size, flops = size + n * c * e + 8 * n, flops + 8 * n * c
        return {"bytes": size, "flops": flops}
    total = sum(_sizes(case))
    return {"bytes": 2 * total * e + 4, "flops": 3 * total}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        n, rows, d = case["n"], case["rows"], case["d"]
        w = s["table"].detach().to(torch.float64)
        out = torch.index_select(w, 0, s["idx"]).mul_(s["scale"])
        if not case["grad"]:
            return out
        # a row's tokens stand together once they are sorted
        order = torch.sort(s["idx"], stable=True)
        seen, count = torch.unique_consecutive(order.values, return_counts=True)
        grad = torch.zeros((rows, d), dtype=torch.float64, device=w.device)
        g = s["gout"].to(torch.float64)[order.indices]
        grad[seen] = torch.segment_reduce(g, "sum", lengths=count, axis=0).mul_(s["scale"])
        return out, grad
    if case["op"] == "norm":
        x, w, b = (s[k].detach().to(torch.float64) for k in ("x", "w", "b"))
        d = x.shape[1]
        mean = x.sum(1, keepdim=True) / d
        var = ((x - mean) ** 2).sum(1, keepdim=True) / d
        inv = 1.0 / torch.sqrt(var + EPS)
        hat = (x - mean) * inv
        y = w * hat + b
        if not case["grad"]:
            return y
        g = s["gout"].to(torch.float64)
        gh = g * w
        gx = inv / d * (d * gh - gh.sum(1, keepdim=True) - hat * (gh * hat).sum(1, keepdim=True))
        return y, gx, (g * hat).sum(0), g.sum(0)
    if case["op"] == "logprobs":
        parts = []
        step = max(1, 64000000 // case["cols"])
        for a in range(0, case["rows"], step):
            x = s["x"].detach()[a:a + step].to(torch.float64)
            t = s["target"][a:a + step]
            lse = torch.logsumexp(x, 1)
            lp = x - lse[:, None]
            p = torch.exp(lp)
            h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
            row = torch.arange(len(t), device=t.device)
            outs = [lp[row, t], h]
            if case["k"]:
                # a stable descending sort keeps equal values in the order of their columns
                o = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
                outs += [torch.gather(lp, 1, o), o]
            if case["grad"]:
                gl, gh = s["glogp"][a:a + step].double(), s["gentropy"][a:a + step].double()
                gx = -p * gl[:, None] - gh[:, None] * torch.where(p > 0, p * (lp + h[:, None]), torch.zeros_like(p))
                gx[row, t] += gl
                outs.append(gx)
            parts.append(outs)
        return [torch.cat(c) for c in zip(*parts)]
    total = math.sqrt(sum(float(torch.linalg.vector_norm(x.to(torch.float64))) ** 2 for x in s["grads"]))
    c = min(1.0, MAX_NORM / (total + CLIP_EPS))
    flat, pieces = _bucket(case, torch.float64)
    for x, o in zip(s["grads"], pieces):
        o.copy_(x).mul_(c)
    return torch.tensor(total, dtype=torch.float64), flat
