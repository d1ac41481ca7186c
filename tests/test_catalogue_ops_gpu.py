"""Row lookup, layer norm, item log probabilities and gradient clipping (the operators of a full-catalogue softmax model)
against plain implementations in 64 bits.

Tolerances. An output in type t is its value in 32 bits rounded once: off by eps(t) / 2 of itself (bf16 2^-8 .. of a value
with 8 significant bits, fp16 2^-11, fp32 2^-24). A sum of n numbers in 32 bits is off by at most (n - 1) 2^-24 of the sum of
their magnitudes, whatever its order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, bound, what):
    """|got - want| <= bound, elementwise, with equal infinities and NaN in the same places."""
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(off[bad][0]), float(bound[bad][0]), bad.nonzero()[0].tolist())


# ---- embed_rows -------------------------------------------------------------------------------------------------------
def embed_exact(table, idx, scale, pad, g):
    """(out, grad, sum of magnitudes and number of terms of each gradient entry) in 64 bits."""
    rows, d = table.shape
    t, flat = table.double(), idx.reshape(-1).long()
    ok = (flat >= 0) & (flat < rows)
    padded = torch.zeros_like(ok) if pad is None else flat == pad
    out = t[flat.clamp(0, max(rows - 1, 0))] * scale if rows else torch.zeros(flat.numel(), d, dtype=torch.float64)
    out[~ok] = float("nan")
    out[padded] = 0.0
    use = ok & ~padded
    gg = g.double().reshape(-1, d)[use]
    grad, mag, cnt = (torch.zeros(rows, d, dtype=torch.float64) for _ in range(3))
    grad.index_add_(0, flat[use], gg * scale)
    mag.index_add_(0, flat[use], gg.abs() * abs(scale))
    cnt.index_add_(0, flat[use], torch.ones_like(gg))
    return out.reshape(idx.shape + (d,)), grad, mag, cnt


def check_embed(rows, d, idx, t, scale=1.0, pad=None, seed=0, g=None, table=None):
    from mmssl_amd import ops
    table = torch.randn(rows, d, generator=gen(seed)).to(t) if table is None else table
    g = torch.randn(tuple(idx.shape) + (d,), generator=gen(seed + 1)).to(t) if g is None else g
    want, grad, mag, cnt = embed_exact(table, idx, scale, pad, g)
    w = table.to(DEV).requires_grad_(True)
    out = ops.embed_rows(w, idx.to(DEV), scale=scale, padding_idx=pad)
    h = half_step(t)
    s = torch.finfo(t).smallest_normal * torch.finfo(t).eps          # half a step of the smallest numbers, and more
    # the product is rounded to 32 bits first, and the scale with it
    within(out, want, want.abs().nan_to_num() * (h + 2 ** -23) + s, "out")
    (got,) = torch.autograd.grad(out, w, g.to(DEV))
    within(got, grad, grad.abs() * h + mag * (cnt + 3) * 2 ** -24 + s, "grad")
    with torch.no_grad():
        assert torch.equal(ops.embed_rows(w, idx.to(DEV), scale=scale, padding_idx=pad).nan_to_num(7.0),
                           out.detach().nan_to_num(7.0))
    return got


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,d,n", [(1, 1, 1), (5, 3, 7), (50, 64, 200), (300, 65, 1000), (33, 128, 4097), (1000, 100, 1024),
                                      (7, 257, 500), (40, 1000, 64), (3, 2049, 40), (5000, 32, 16384)])
def test_embed_rows_and_gradient(rows, d, n, t):
    idx = torch.randint(rows, (n,), generator=gen(d + n))
    check_embed(rows, d, idx, t, scale=1.7, seed=n)


@pytest.mark.parametrize("n", [16385, 40000, 262144 + 5000])
@pytest.mark.parametrize("rows", [1, 200, 300, 70000])
def test_embed_gradient_of_long_lists_is_sorted_by_radix(rows, n):
    """More places than are ranked by counting: one to three passes, whole and partial tiles, all places of one token."""
    g = gen(rows + n)
    idx = torch.randint(rows, (n,), generator=g)
    check_embed(rows, 8, idx, torch.float32, scale=0.5, seed=3)
    got = check_embed(rows, 8, idx, torch.bfloat16, seed=4)
    assert torch.equal(got, check_embed(rows, 8, idx, torch.bfloat16, seed=4)), "the same call, the same bits"


@pytest.mark.parametrize("n", [8191, 8192, 8193, 9216, 9217])
def test_embed_gradient_where_ranking_ends(n):
    for rows in (1, 255, 256, 65537):
        check_embed(rows, 12, torch.randint(rows, (n,), generator=gen(n + rows)), torch.float32, seed=n)


def test_embed_popular_tokens_cross_many_chunks():
    """Tokens whose places fill one chunk, several, more than one lane group joins alone, and the whole list."""
    for counts in ([1, 7, 8, 9, 64, 65, 200, 1000, 0, 3], [5000], [1, 0, 0, 4000, 1], [8, 8, 8, 8], [16, 0, 128, 129, 127]):
        idx = torch.cat([torch.full((c,), v) for v, c in enumerate(counts)])
        idx = idx[torch.randperm(idx.numel(), generator=gen(1))]
        for t, d in ((torch.float32, 64), (torch.bfloat16, 64), (torch.float32, 30), (torch.float16, 520)):
            check_embed(len(counts), d, idx, t, seed=9)
    idx = torch.randint(3, (70000,), generator=gen(5))
    check_embed(4, 16, idx, torch.float32, seed=2)


@pytest.mark.parametrize("n", [600, 20000])
def test_embed_padding_and_tokens_outside_the_table(n):
    from mmssl_amd import ops
    rows, d = 40, 24
    idx = torch.randint(-3, rows + 3, (n,), generator=gen(1))
    for pad in (None, -1, 5, rows + 1, 1 << 40):
        check_embed(rows, d, idx, torch.float32, scale=2.0, pad=pad)
    check_embed(rows, d, idx.int(), torch.float16, pad=0)
    big = idx.clone()
    big[::7] = 1 << 40                                     # does not fit 32 bits: outside, not wrapped into the table
    big[1::7] = -(1 << 40)
    check_embed(rows, d, big, torch.float32)
    none = torch.full((n,), -1)
    got = check_embed(rows, d, none, torch.float32, pad=-1)
    assert not bool(got.any())
    w = torch.randn(rows, d, device=DEV)
    assert bool(ops.embed_rows(w, none.to(DEV)).isnan().all())


def test_embed_shapes_strides_and_empty_inputs():
    from mmssl_amd import ops
    g = gen(2)
    base = torch.randn(30, 40, generator=g)
    idx = torch.randint(30, (4, 3, 5), generator=g)
    for t in TYPES:
        wide = base.to(t).to(DEV)
        table = wide[:, 3:20]                               # odd width, odd pitch, odd start
        got = ops.embed_rows(table, idx.to(DEV), scale=3.0)
        assert got.shape == (4, 3, 5, 17)
        assert torch.equal(got, (table.double() * 3.0).to(t)[idx.to(DEV)])
        w = table.detach().clone().requires_grad_(True)
        out = ops.embed_rows(w, idx.to(DEV).transpose(0, 2), scale=3.0)
        assert out.shape == (5, 3, 4, 17)
        row = torch.randn(17, generator=g).to(t).to(DEV)
        (a,) = torch.autograd.grad(out, w, row.expand(5, 3, 4, 17), retain_graph=True)      # one row for all places
        (b,) = torch.autograd.grad(out, w, row.expand(5, 3, 4, 17).contiguous(), retain_graph=True)
        (c,) = torch.autograd.grad(out, w, row.expand(5, 3, 4, 17).permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3))
        assert torch.equal(a, b) and torch.equal(a, c)
    for idx in (torch.empty(0, dtype=torch.int64), torch.empty(3, 0, dtype=torch.int32)):
        got = check_embed(11, 7, idx, torch.float32)
        assert not bool(got.any())
    w = torch.zeros(0, 8, device=DEV, requires_grad=True)
    out = ops.embed_rows(w, torch.tensor([0, 1], device=DEV))
    assert bool(out.isnan().all())
    assert torch.autograd.grad(out, w, torch.ones_like(out))[0].shape == (0, 8)
    assert ops.embed_rows(torch.ones(3, 2, device=DEV), [2, 0]).tolist() == [[1, 1], [1, 1]]


def test_embed_gradient_where_places_times_width_pass_32_bits():
    from mmssl_amd import ops
    n, d, rows = 2200000, 1024, 50                           # 2.25e9 elements of g, bf16: 4.5 GB
    idx = torch.full((n,), 7, device=DEV)
    idx[-3:] = torch.tensor([9, 49, 9], device=DEV)
    g = torch.zeros(n, d, dtype=torch.bfloat16, device=DEV)
    g[-3:] = torch.tensor([1.0, 2.0, 4.0], device=DEV, dtype=torch.bfloat16)[:, None]
    g[0] = 8.0
    w = torch.zeros(rows, d, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    out = ops.embed_rows(w, idx)
    assert out.shape == (n, d) and not bool(out[-1].any())
    (got,) = torch.autograd.grad(out, w, g)
    want = torch.zeros(rows, dtype=torch.float32)
    want[7], want[9], want[49] = 8.0, 5.0, 2.0
    assert torch.equal(got.float().cpu(), want[:, None].expand(rows, d))


# ---- layernorm_rows ---------------------------------------------------------------------------------------------------
def norm_exact(x, w, b, eps, g):
    """y, gx, gw, gb in 64 bits, and the sums of magnitudes behind the last two."""
    x, g = x.double(), g.double()
    d = x.shape[-1]
    w1 = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    mu = x.mean(-1, keepdim=True)
    var = ((x - mu) ** 2).mean(-1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    h = (x - mu) * r
    y = h * w1 + (0 if b is None else b.double())
    q = g * w1
    gx = r * (q - q.mean(-1, keepdim=True) - h * (q * h).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, d)      # noqa: E731
    # how far the 32-bit statistics let h be off: the mean by (d + 2) 2^-24 of the magnitudes' mean, the deviation's square by
    # the same share again, and six roundings
    e = (6 + d) * 2.0 ** -24
    eh = e * (1 + 2 * x.abs().mean(-1, keepdim=True) * r) + h.abs() * e
    qa = q.abs()
    egx = r * (e * (qa + qa.mean(-1, keepdim=True) + h.abs() * (qa * h.abs()).mean(-1, keepdim=True)) * 3
               + eh * (qa * h.abs()).mean(-1, keepdim=True) + h.abs() * (qa * eh).mean(-1, keepdim=True))
    n = max(1, flat(x).shape[0])
    gw, gb = flat(g * h).sum(0), flat(g).sum(0)
    egw = flat(g.abs() * eh).sum(0) + flat((g * h).abs()).sum(0) * (n + 3) * 2.0 ** -24
    egb = flat(g.abs()).sum(0) * (n + 3) * 2.0 ** -24
    ey = eh * w1.abs() + y.abs() * 2.0 ** -23 + (h * w1).abs() * 2.0 ** -23
    return (y, gx, gw, gb), (ey, egx, egw, egb)


def check_norm(shape, t, pt=None, eps=1e-5, affine=(True, True), seed=0, x=None, offset=0.5):
    from mmssl_amd import ops
    pt = t if pt is None else pt
    g0 = gen(seed)
    x = (torch.randn(shape, generator=g0) * 2 + offset).to(t) if x is None else x
    d = shape[-1]
    w = (1 + 0.3 * torch.randn(d, generator=g0)).to(pt) if affine[0] else None
    b = (0.3 * torch.randn(d, generator=g0)).to(pt) if affine[1] else None
    g = torch.randn(shape, generator=g0).to(t)
    want, off = norm_exact(x, w, b, eps, g)
    leaves = [v.to(DEV).requires_grad_(True) if v is not None else None for v in (x, w, b)]
    y = ops.layernorm_rows(*leaves, eps=eps)
    ins = [v for v in leaves if v is not None]
    grads = iter(torch.autograd.grad(y, ins, g.to(DEV)))
    got = [y] + [next(grads) if v is not None else None for v in leaves]
    for name, a, v, o, ty in zip(("y", "gx", "gw", "gb"), got, want, off, (t, t, pt, pt)):
        if a is not None:
            assert a.dtype == ty, name
            tiny = torch.finfo(ty).smallest_normal * torch.finfo(ty).eps
            within(a, v, v.abs() * half_step(ty) + o * (1 + half_step(ty)) + tiny, name)
    with torch.no_grad():
        assert torch.equal(ops.layernorm_rows(*leaves, eps=eps), y)
    return got


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 8), (5, 31), (17, 32), (64, 64), (33, 65), (7, 128), (9, 200), (5, 256),
                                    (3, 257), (11, 512), (4, 513), (5, 1000), (3, 1024), (2, 1500), (3, 2048), (2, 2047),
                                    (3, 4096), (2, 4100), (1, 5001), (2, 8192), (2, 12345), (2, 16384), (3, 16385),
                                    (2, 20000)])
def test_layernorm_rows_and_gradients(rows, d, t):
    check_norm((rows, d), t, seed=d)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,d", [(5000, 16), (1025, 64), (2100, 130), (3001, 384), (1300, 1028), (600, 4608), (530, 16500)])
def test_layernorm_gradients_of_many_rows(rows, d, t):
    """More rows than blocks: the weights' sums add up over a block's rows, then over the blocks."""
    a = check_norm((rows, d), t, seed=rows)
    b = check_norm((rows, d), t, seed=rows)
    assert all(torch.equal(x, y) for x, y in zip(a, b)), "the same call, the same bits"


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,d", [(2100, 5), (2100, 9), (1500, 77), (1300, 131), (1100, 257), (700, 513), (600, 1001),
                                    (560, 2051), (530, 4097), (520, 8193)])
def test_layernorm_rows_that_end_inside_a_vector(rows, d, t):
    """One to seven columns behind the last whole vector, at every lane group and number of vectors a lane."""
    check_norm((rows, d), t, seed=d)


def test_layernorm_parameters_types_and_absence():
    for affine in ((True, False), (False, True), (False, False)):
        for t in TYPES:
            check_norm((37, 96), t, affine=affine, seed=3)
            check_norm((3, 17000), t, affine=affine, seed=3)
    for t in (torch.bfloat16, torch.float16):
        check_norm((29, 100), t, pt=torch.float32, seed=4)
        check_norm((2, 16400), t, pt=torch.float32, seed=4)
    check_norm((4, 64), torch.float32, eps=0.0)
    check_norm((2, 3, 5, 24), torch.float32)
    check_norm((40,), torch.float32)


def test_layernorm_values_far_from_zero_and_constant_rows():
    """The variance is taken around the mean: a row far from zero keeps its digits, a constant row gives the bias."""
    from mmssl_amd import ops
    x = torch.randn(40, 256, generator=gen(1)) + 4096.0
    check_norm((40, 256), torch.float32, x=x)
    c = torch.full((3, 100), 7.0, device=DEV)
    b = torch.randn(100, device=DEV)
    assert torch.equal(ops.layernorm_rows(c, None, b), b.expand(3, 100))
    for bad in (float("nan"), float("inf")):
        x = torch.randn(5, 300, generator=gen(2))
        x[3, 17] = bad
        y = ops.layernorm_rows(x.to(DEV)).cpu()
        assert bool(y[3].isnan().all()) and bool(y[[0, 1, 2, 4]].isfinite().all())


def test_layernorm_strides_and_empty_inputs():
    from mmssl_amd import ops
    for t in TYPES:
        wide = torch.randn(50, 91, generator=gen(4)).to(t).to(DEV)
        g = torch.randn(50, 33, generator=gen(5)).to(t).to(DEV)
        for x in (wide[:, 5:38], wide[::3, 1:34], wide.t()[:33].t(), wide[:1, :33].expand(50, 33)):
            a = x.detach().requires_grad_(True)
            c = x.detach().contiguous().requires_grad_(True)
            ya, yc = ops.layernorm_rows(a), ops.layernorm_rows(c)
            gg = g[:x.shape[0]]
            assert torch.equal(ya, yc)
            assert torch.equal(torch.autograd.grad(ya, a, gg)[0], torch.autograd.grad(yc, c, gg)[0])
        one = torch.randn(33, generator=gen(6)).to(t).to(DEV).expand(50, 33)
        y = ops.layernorm_rows(c)
        assert torch.equal(torch.autograd.grad(y, c, one, retain_graph=True)[0],
                           torch.autograd.grad(y, c, one.contiguous())[0])
        w = torch.ones(8, dtype=t, device=DEV, requires_grad=True)
        x = torch.zeros(0, 8, dtype=t, device=DEV, requires_grad=True)
        y = ops.layernorm_rows(x, w, w)
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == gx.shape == (0, 8) and not bool(gw.any())


def test_layernorm_gradient_against_differences():
    """The gradient of a weighted sum against central differences of the 64-bit formula along a random direction."""
    from mmssl_amd import ops
    g0 = gen(8)
    x, w, b, c = (torch.randn(s, generator=g0, dtype=torch.float64) for s in ((6, 40), (40,), (40,), (6, 40)))
    f = lambda x, w, b: (norm_exact(x, w, b, 1e-5, x)[0][0] * c).sum()        # noqa: E731
    leaves = [v.float().to(DEV).requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad((ops.layernorm_rows(*leaves) * c.float().to(DEV)).sum(), leaves)
    x, w, b = (v.detach().cpu().double() for v in leaves)
    for k, v in enumerate((x, w, b)):
        u = torch.randn(v.shape, generator=g0, dtype=torch.float64)
        e = 1e-5
        args = [x, w, b]
        hi, lo = list(args), list(args)
        hi[k], lo[k] = v + e * u, v - e * u
        slope = float((f(*hi) - f(*lo)) / (2 * e))
        mine = float((grads[k].cpu().double() * u).sum())
        # differences: e^2 of the third derivative and 1e-16 / e of rounding, both far below the 32-bit sums' share
        assert abs(mine - slope) <= 1e-5 * float((grads[k].cpu().double().abs() * u.abs()).sum()) + 1e-6, (k, mine, slope)


# ---- logprobs_rows ----------------------------------------------------------------------------------------------------
def logprobs_exact(x, target, k, temperature, ignore, grads=None):
    """(logp, entropy, top_logp, top_idx[, gx]) in 64 bits."""
    z = x.double() / temperature
    n, cols = z.shape
    empty = torch.isneginf(z).all(1)
    top = z.amax(1, keepdim=True)
    u = z - torch.where(empty[:, None], torch.zeros_like(top), top)       # off first: a row of the type's lowest value is even
    lp = u - torch.log(torch.exp(u).sum(1, keepdim=True))
    lp[empty] = float("-inf")
    p = lp.exp()
    held = torch.where(p > 0, lp, torch.zeros_like(lp))            # 0 log 0 = 0
    h = -(p * held).sum(1)
    row = torch.arange(n)
    ok = (target >= 0) & (target < cols)
    logp = torch.where(ok, lp[row, target.clamp(0, cols - 1).long()], torch.full((n,), float("nan"), dtype=torch.float64))
    logp[target == ignore] = 0.0
    # descending value, ties by ascending column; torch sorts NaN above +inf
    idx = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
    held32 = lambda v: torch.where(v < torch.finfo(torch.float32).min, float("-inf"), v)      # noqa: E731  (fp32 outputs)
    outs = [held32(logp), h, held32(lp.gather(1, idx)), idx]
    if grads is not None:
        gl, gh, gt = (g.double() for g in grads)
        asked = ok & (target != ignore)
        gl = torch.where(asked, gl, torch.zeros_like(gl))
        named = torch.zeros_like(z)
        named[row[asked], target[asked].long()] += gl[asked]
        named.scatter_add_(1, idx, gt)
        gx = named - p * (gl + gt.sum(1))[:, None] - gh[:, None] * p * (held + h[:, None])
        gx[empty] = 0.0
        outs.append(gx / temperature)
    return outs


def check_logprobs(x, k=0, temperature=1.0, target=None, ignore=-100, grad=True, seed=0):
    from mmssl_amd import ops
    n, cols = x.shape
    g0 = gen(seed + 77)
    if target is None:
        target = torch.randint(cols, (n,), generator=g0)
    grads = [torch.randn(n, generator=g0), torch.randn(n, generator=g0), torch.randn(n, k, generator=g0)]
    want = logprobs_exact(x, target, k, temperature, ignore, grads)
    xd = x.to(DEV).requires_grad_(True)
    got = ops.logprobs_rows(xd, target.to(DEV), k=k, temperature=temperature, ignore_index=ignore)
    # exp2 of y log2 e / T: two roundings of y and one unit of the instruction let a term be off by 2^-23 (1 + |y|) of itself,
    # and |y| e^y <= 1; a sum of `cols` terms by 2^-24 of itself for each level of its tree and each of a thread's 64 adds
    # in a row, the joins of slices more
    rel = (64 + 20 + cols / 16384) * 2.0 ** -24 + 3 * 2.0 ** -23
    # (x - m) / T - log S: |x - m| / T <= |logp|, three roundings of it
    within(got[0], want[0], want[0].abs().nan_to_num(posinf=0.0) * 2.0 ** -22 + rel, "logp")
    eh = rel * (2 + 2 * want[1].abs().nan_to_num())
    within(got[1], want[1], eh, "entropy")
    if k:
        assert torch.equal(got[3].cpu(), want[3]), ("top_idx", (got[3].cpu() != want[3]).nonzero()[:3])
        within(got[2], want[2], want[2].abs().nan_to_num(posinf=0.0) * 2.0 ** -22 + rel, "top_logp")
    else:
        assert got[2] is None and got[3] is None
    if grad:
        outs, gs = list(got[:2]), grads[:2]
        if k:
            outs.append(got[2])
            gs.append(grads[2])
        (gx,) = torch.autograd.grad(outs, xd, [g.to(DEV) for g in gs])
        t = x.dtype
        gl, gh, gt = (g.double().abs() for g in grads)
        # p is off by the sum's share and by |log p| roundings of the exponent; the entropy's factor by the same again
        size = gl + gt.sum(1) + gh * (2 + want[1].abs().nan_to_num())
        bound = want[4].abs() * half_step(t) * 2 + (size * (rel * 6 + 40 * 2.0 ** -23) / temperature)[:, None]
        bound = bound + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        within(gx, want[4], bound.nan_to_num(), "gx")
    with torch.no_grad():
        again = ops.logprobs_rows(xd, target.to(DEV), k=k, temperature=temperature, ignore_index=ignore)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
    return got


def scores(n, cols, t, seed, masked=0.0, scale=3.0):
    g0 = gen(seed)
    x = torch.randn(n, cols, generator=g0) * scale
    if masked:
        x[torch.rand(n, cols, generator=g0) < masked] = float("-inf")
    return x.to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,cols,k", [(1, 1, 1), (3, 2, 2), (2, 7, 5), (5, 64, 10), (4, 65, 64), (3, 255, 100), (2, 500, 128),
                                      (7, 1000, 20), (3, 1025, 128), (2, 1500, 128), (5, 2048, 50), (2, 2500, 128),
                                      (1, 4099, 1), (3, 16384, 20), (3, 16385, 50), (2, 40001, 128), (1, 100000, 20)])
def test_logprobs_rows(n, cols, k, t):
    check_logprobs(scores(n, cols, t, cols), k=k, seed=k)
    check_logprobs(scores(n, cols, t, cols + 1, masked=0.3), k=0, seed=k)


@pytest.mark.parametrize("t", TYPES)
def test_logprobs_many_rows_whole_slices_and_one_launch(t):
    """From 512 blocks on the slices are as long as the registers hold; short rows are done in one launch."""
    check_logprobs(scores(1100, 1300, t, 1), k=10)
    check_logprobs(scores(530, 9000, t, 2, masked=0.1), k=50)
    check_logprobs(scores(300, 33001, t, 3), k=0)
    check_logprobs(scores(260, 17000, t, 4), k=3)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(2048, 1), (2050, 100), (2049, 511), (2051, 1000), (3001, 1025), (2048, 2048),
                                       (2047, 700), (2048, 2049)])
def test_logprobs_many_short_rows(rows, cols, t):
    """Rows that a wave takes alone, forward and backward, and their neighbours that a block takes; a masked row, an empty one,
    one with a NaN among them."""
    x = scores(rows, cols, t, rows + cols, masked=0.2)
    x[5] = float("-inf")
    x[7] = torch.finfo(t).min
    check_logprobs(x, k=0, temperature=1.7)
    check_logprobs(x[:, :cols], k=min(3, cols))
    from mmssl_amd import ops
    x[rows - 1, cols // 2] = float("nan")
    o = ops.logprobs_rows(x.to(DEV), torch.zeros(rows, dtype=torch.int64, device=DEV))
    assert bool(o[0][-1].isnan()) and bool(o[1][-1].isnan()) and not bool(o[1][:-1].isnan().any())


@pytest.mark.parametrize("cols", [100, 900, 3000, 70000])
def test_logprobs_rows_of_equal_and_masked_values(cols):
    """Ties go to the lowest column, whatever their number; rows that the mask leaves little or nothing of; masks of the
    type's lowest value."""
    inf = float("inf")
    for t in TYPES:
        low = torch.finfo(t).min
        x = torch.zeros(12, cols)
        g0 = gen(cols)
        x[1] = 2.0
        x[1, cols // 2] = 3.0
        x[2] = -inf
        x[3] = -inf
        x[3, cols - 1] = 1.0
        x[4] = -inf
        x[4, [5, cols // 3, cols - 2]] = torch.tensor([0.5, 0.5, 4.0])
        x[5] = torch.randint(0, 3, (cols,), generator=g0).float()
        x[6] = low
        x[7] = low
        x[7, 3] = 0.0
        x[8] = torch.where(torch.rand(cols, generator=g0) < 0.99, -inf, 0.0)
        x[9, ::2] = -0.0
        x[10] = torch.randn(cols, generator=g0).round()
        x[11] = -inf
        x[11, :cols // 2] = low
        x = x.to(t)
        for k in (0, 1, 20, 100):
            target = torch.randint(cols, (12,), generator=g0)
            check_logprobs(x, k=k, target=target)
            check_logprobs(x, k=k, target=target, temperature=0.7, grad=False)


def test_logprobs_of_nan_and_infinite_scores():
    from mmssl_amd import ops
    for cols in (50, 5000):
        x = torch.randn(6, cols, generator=gen(3))
        x[0, 7] = float("nan")
        x[1, 8] = float("inf")
        x[2] = float("nan")
        x[3] = float("-inf")
        x[3, 4] = float("nan")
        x[4, 9] = float("nan")
        x[4, 3] = float("inf")
        for t in TYPES:
            v = x.to(t)
            logp, h, tl, ti = ops.logprobs_rows(v.to(DEV), torch.zeros(6, dtype=torch.int32, device=DEV), k=5)
            assert bool(logp[:5].isnan().all()) and bool(h[:5].isnan().all()) and bool(logp[5].isfinite())
            want = torch.sort(v.double(), dim=1, descending=True, stable=True).indices[:, :5]
            assert torch.equal(ti.cpu(), want)
            assert bool(tl[:3].isnan().all())


def test_logprobs_targets_that_name_no_column():
    x = scores(9, 1234, torch.float32, 5)
    target = torch.tensor([0, 1233, -100, 1234, -1, 1 << 40, 5, -(1 << 40), -100])
    check_logprobs(x, k=4, target=target)
    check_logprobs(x, k=4, target=target, ignore=-1)
    check_logprobs(x, k=0, target=target[[0, 1, 2, 3, 4, 6, 6, 2, 2]].int())


def test_logprobs_temperature_and_large_scores():
    for temperature in (0.05, 0.5, 1.0, 3.0, 100.0):
        for t in TYPES:
            check_logprobs(scores(4, 3001, t, 9), k=7, temperature=temperature)
    x = scores(4, 5000, torch.float32, 10) + 10000.0               # far from zero: the maximum is taken off first
    check_logprobs(x, k=5)
    check_logprobs(scores(3, 2000, torch.float32, 11, scale=200.0), k=5)
    x = scores(3, 2000, torch.float32, 11)
    x[0] = x[0] * 1e37
    x[1, 5] = 3e38
    x[1, 6] = -3e38
    check_logprobs(x, k=5, grad=False)


def test_logprobs_shapes_strides_and_empty_inputs():
    from mmssl_amd import ops
    wide = scores(24, 701, torch.float32, 12)
    target = torch.randint(600, (24,), generator=gen(1))
    for t in TYPES:
        w = wide.to(t).to(DEV)
        for x in (w[:, 7:650], w[:, :643], w[:1, :643].expand(24, 643), w[:, :643].t().contiguous().t()):
            tg = target.to(DEV)
            a = x.detach().requires_grad_(True)
            b = x.detach().contiguous().requires_grad_(True)
            oa, ob = ops.logprobs_rows(a, tg, k=6), ops.logprobs_rows(b, tg, k=6)
            assert all(torch.equal(u, v) for u, v in zip(oa, ob))
            ga = torch.autograd.grad(oa[0].sum() + oa[1].mean(), a)[0]
            gb = torch.autograd.grad(ob[0].sum() + ob[1].mean(), b)[0]
            assert torch.equal(ga, gb)
        c = w[:, :640].reshape(2, 3, 4, 640)
        o3 = ops.logprobs_rows(c, tg.reshape(2, 3, 4), k=3)
        o2 = ops.logprobs_rows(c.reshape(24, 640), tg, k=3)
        assert o3[0].shape == (2, 3, 4) and o3[3].shape == (2, 3, 4, 3)
        assert all(torch.equal(u.reshape(v.shape), v) for u, v in zip(o3, o2))
    one = ops.logprobs_rows(wide[0].to(DEV), torch.tensor(5, device=DEV), k=2)
    assert one[0].shape == () and one[3].shape == (2,)
    e = torch.zeros(0, 40, device=DEV, requires_grad=True)
    o = ops.logprobs_rows(e, torch.zeros(0, dtype=torch.int64, device=DEV), k=3)
    assert o[0].shape == (0,) and o[2].shape == (0, 3)
    assert torch.autograd.grad(o[0].sum(), e)[0].shape == (0, 40)
    # each output by itself, and the gradient of a sum where all of them meet
    x = scores(5, 333, torch.float32, 13).to(DEV).requires_grad_(True)
    tg = torch.arange(5, device=DEV)
    o = ops.logprobs_rows(x, tg, k=4)
    parts = [torch.autograd.grad(o[i].sum(), x, retain_graph=True)[0] for i in range(3)]
    whole = torch.autograd.grad(o[0].sum() + o[1].sum() + o[2].sum(), x)[0]
    assert float((sum(parts) - whole).abs().max()) <= 1e-5


def test_logprobs_gradient_against_differences():
    from mmssl_amd import ops
    g0 = gen(21)
    x = torch.randn(4, 50, generator=g0) * 2
    target = torch.tensor([3, 49, 0, -100])
    c = [torch.randn(4, generator=g0).double(), torch.randn(4, generator=g0).double(), torch.randn(4, 6, generator=g0).double()]

    def f(v):
        o = logprobs_exact(v, target, 6, 1.3, -100)
        return float(sum((a * b).sum() for a, b in zip(o[:3], c)))

    xd = x.to(DEV).requires_grad_(True)
    o = ops.logprobs_rows(xd, target.to(DEV), k=6, temperature=1.3)
    (gx,) = torch.autograd.grad(sum((a * b.float().to(DEV)).sum() for a, b in zip(o[:3], c)), xd)
    for seed in range(4):
        u = torch.randn(4, 50, generator=gen(seed)).double()
        e = 1e-6
        slope = (f(x.double() + e * u) - f(x.double() - e * u)) / (2 * e)
        mine = float((gx.cpu().double() * u).sum())
        assert abs(mine - slope) <= 2e-5 * float((gx.cpu().double().abs() * u.abs()).sum()) + 1e-5, (mine, slope)


def test_logprobs_row_offsets_past_32_bits():
    from mmssl_amd import ops
    cols = 1 << 20
    rows = 2100                                              # 2.2e9 columns of bf16: 4.4 GB
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-1, 77] = 3.0
    x[-1, -1] = 2.0
    x.requires_grad_(True)
    target = torch.full((rows,), cols - 1, device=DEV)
    o = ops.logprobs_rows(x, target, k=3)
    assert o[3][-1].tolist() == [77, cols - 1, 0] and o[3][0].tolist() == [0, 1, 2]
    lse = torch.logsumexp(x.detach()[-1].double(), 0)
    assert abs(float(o[0][-1].double() - (2.0 - lse))) < 1e-5
    (gx,) = torch.autograd.grad(o[0][-1], x)
    assert not bool(gx[:-1].any()) and abs(float(gx[-1, -1]) - 1.0) < 2 ** -8 and float(gx[-1, 77]) < 0


# ---- gradient norm and clipping ---------------------------------------------------------------------------------------
def grad_lists():
    g0 = gen(31)
    sizes = [1, 2, 3, 8, 17, 255, 256, 8191, 8192, 8193, 100000, 0, 65536, 33333]
    yield "one", [torch.randn(5, generator=g0)]
    yield "fp32", [torch.randn(n, generator=g0) for n in sizes]
    yield "mixed", [torch.randn(n, generator=g0).to(TYPES[i % 3]) for i, n in enumerate(sizes)]
    yield "many", [(torch.randn(n % 700 + 1, generator=g0) * 0.01).to(TYPES[n % 2]) for n in range(300)]
    yield "96", [torch.randn(40, generator=g0) for _ in range(96)]
    yield "shapes", [torch.randn(30, 20, 7, generator=g0), torch.randn((), generator=g0), torch.randn(1000, 64, generator=g0)]
    yield "large", [torch.randn(3000001, generator=g0).bfloat16(), torch.randn(9000000, generator=g0)]


@pytest.mark.parametrize("name,grads", list(grad_lists()), ids=lambda v: v if isinstance(v, str) else "")
def test_grad_norm_and_clipping(name, grads):
    from mmssl_amd import optim
    total = sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5
    dev = [g.to(DEV) for g in grads]
    assert abs(float(optim.grad_norm(dev)) - total) <= total * (2.0 ** -24 + 1e-12)
    for max_norm in (total * 0.3, total * 7, 0.0):
        c = min(1.0, max_norm / (total + 1e-6))
        out = [torch.full_like(g, 5.0) for g in dev]
        n1 = optim.clip_grads(dev, max_norm, out=out)
        mine = [g.clone() for g in dev]
        n2 = optim.clip_grads(mine, max_norm)
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in dev]
        for p, g in zip(params, dev):
            p.grad = g.clone()
        n3 = optim.clip_grad_norm(params + [torch.nn.Parameter(torch.zeros(3, device=DEV))], max_norm)
        for n in (n1, n2, n3):
            assert n.shape == () and abs(float(n) - total) <= total * (2.0 ** -24 + 1e-12)
        for g, a, b, p, d in zip(grads, out, mine, params, dev):
            t = g.dtype
            tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
            # the factor is rounded to 32 bits, so is the product, then the type
            within(a, g.double() * c, (g.double() * c).abs() * (half_step(t) + 2.0 ** -22) + tiny, name)
            assert torch.equal(a, b) and torch.equal(a, p.grad) and torch.equal(d.cpu(), g)
            if c == 1.0:
                assert torch.equal(a, d)


def test_grad_norm_keeps_range_and_reports_what_is_not_finite():
    from mmssl_amd import optim
    for v in (1e-30, 1e30, 3e38):                            # squares that fp32 does not hold
        g = [torch.full((1000,), v, device=DEV), torch.full((24,), v, device=DEV)]
        want = 32.0 * float(torch.tensor(v)) if v < 1e37 else float("inf")
        got = float(optim.grad_norm(g))
        assert got == want or abs(got - want) <= want * 1e-7
    g = [torch.full((10,), 3e38, device=DEV)]                # the norm passes fp32, the factor does not
    optim.clip_grads(g, 1.0)
    assert float((g[0] - 10 ** -0.5).abs().max()) < 1e-6
    z = [torch.zeros(100, device=DEV)]
    assert float(optim.clip_grads(z, 1.0)) == 0.0 and not bool(z[0].any())
    a = [torch.ones(5, device=DEV), torch.tensor([1.0, float("inf")], device=DEV)]
    assert float(optim.clip_grads(a, 1.0)) == float("inf")
    assert not bool(a[0].any()) and bool(a[1][1].isnan())
    b = [torch.ones(5, device=DEV), torch.tensor([1.0, float("nan")], device=DEV)]
    n = optim.clip_grads(b, 1.0)
    assert bool(n.isnan()) and bool(b[0].isnan().all())


def test_clipping_unaligned_pieces_and_neighbours():
    """Pieces of a flat buffer that begin anywhere: what lies between them is left as it was."""
    from mmssl_amd import optim
    g0 = gen(41)
    for t in TYPES:
        flat = torch.randn(60000, generator=g0).to(t)
        cuts = [(1, 4), (7, 20), (33, 8192), (9001, 20000), (30003, 29997)]
        dev = flat.to(DEV)
        pieces = [dev[a:a + n] for a, n in cuts]
        want = flat.double().clone()
        total = sum(float((flat[a:a + n].double() ** 2).sum()) for a, n in cuts) ** 0.5
        for a, n in cuts:
            want[a:a + n] *= 0.5 * total / (total + 1e-6)
        optim.clip_grads(pieces, 0.5 * total)
        within(dev, want, want.abs() * (half_step(t) + 2.0 ** -22) + 1e-7, "flat")
        keep = torch.ones(60000, dtype=torch.bool)
        for a, n in cuts:
            keep[a:a + n] = False
        assert torch.equal(dev.cpu()[keep], flat[keep])
    p = torch.nn.Parameter(torch.zeros(30, 50, device=DEV))
    p.grad = torch.randn(50, 30, device=DEV).t()
    was = p.grad.clone()
    n = optim.clip_grad_norm([p], 1.0)
    assert abs(float(n) - float(was.double().norm())) < 1e-4
    assert float((p.grad - was / (n + 1e-6)).abs().max()) < 1e-6


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_a_full_catalogue_model_trains_a_step(t):
    """Histories -> rows -> norm -> scores against the item table -> log probabilities -> backward -> clipping -> AdamW, twice,
    against the same in 64 bits on the host: losses, clipped gradients, weights."""
    from mmssl_amd import ops, optim
    g0 = gen(51)
    items, d, b, length = 500, 64, 32, 20
    table = (torch.randn(items, d, generator=g0) * 0.05).to(t)
    w, bias = torch.ones(d).to(t), torch.zeros(d).to(t)
    hist = torch.randint(-1, items, (b, length), generator=g0)            # -1: shorter histories
    hist[3] = -1                                                          # one user without any
    pos = torch.randint(items, (b,), generator=g0)
    seen = torch.zeros(b, items, dtype=torch.bool)
    seen.scatter_(1, hist.clamp(min=0), True)
    seen[torch.arange(b), pos] = False
    leaves = [torch.nn.Parameter(v.float().to(DEV)) for v in (table, w, bias)]      # fp32 master weights
    opt = optim.FusedAdamW(leaves, lr=0.01, weight_decay=0.0)
    ref = [v.double().clone().requires_grad_(True) for v in (table, w, bias)]
    ropt = torch.optim.AdamW(ref, lr=0.01, weight_decay=0.0)
    scale = d ** 0.5
    tol = 2e-5 if t == torch.float32 else 4e-2
    for step in range(2):
        opt.zero_grad()
        tab, ww, bb = (p.to(t) for p in leaves)
        rows = ops.embed_rows(tab, hist.to(DEV), scale=scale, padding_idx=-1)
        user = ops.layernorm_rows(rows.float().mean(1).to(t), ww, bb)
        s = (user.float() @ tab.float().t()).masked_fill(seen.to(DEV), float("-inf"))
        logp, entropy, _, top = ops.logprobs_rows(s, pos.to(DEV), k=5, temperature=0.5)
        loss = -logp.mean() - 0.01 * entropy.mean()
        loss.backward()
        norm = optim.clip_grad_norm(leaves, 0.1)

        ropt.zero_grad()
        ok = (hist >= 0)[..., None]
        rr = torch.where(ok, ref[0][hist.clamp(min=0)] * scale, torch.zeros((), dtype=torch.float64)).mean(1)
        hu = (rr - rr.mean(1, keepdim=True)) / (rr.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * ref[1] + ref[2]
        z = (hu @ ref[0].t()).masked_fill(seen, float("-inf")) / 0.5
        lp = torch.log_softmax(z, 1)
        h = -(lp.exp() * lp.masked_fill(seen, 0.0)).sum(1)
        rloss = -lp[torch.arange(b), pos].mean() - 0.01 * h.mean()
        rloss.backward()
        rnorm = torch.nn.utils.clip_grad_norm_(ref, 0.1)
        assert abs(float(loss.detach()) - float(rloss.detach())) <= tol * abs(float(rloss.detach()))
        assert abs(float(norm) - float(rnorm)) <= tol * float(rnorm)
        for p, r in zip(leaves, ref):
            assert float((p.grad.cpu().double() - r.grad).norm()) <= tol * float(r.grad.norm())
        assert torch.equal(top, ops.topk_rows(s.detach(), 5))
        opt.step()
        ropt.step()
        with torch.no_grad():
            for p, r in zip(leaves, ref):                     # the next step starts from the same weights
                if t == torch.float32:
                    assert float((p.cpu().double() - r).abs().max()) <= 2e-3
                r.copy_(p.cpu().double() if t == torch.float32 else p.cpu().to(t).double())


def test_catalogue_operators_in_a_captured_graph():
    """The whole chain with its backward forms captured and replayed on new inputs, the program's own eager work between the
    replays, two graphs and an eager call side by side: every replay gives the eager bits."""
    from mmssl_amd import ops, optim
    g0 = gen(61)
    items, d, n = 700, 64, 300

    def inputs(seed):
        q = gen(seed)
        return [torch.randn(items, d, generator=q), torch.randint(items, (n,), generator=q),
                torch.randn(d, generator=q), torch.randint(items, (n,), generator=q)]

    def chain(table, idx, w, pos):
        with torch.enable_grad():
            leaves = [v.detach().requires_grad_(True) for v in (table, w)]
            rows = ops.embed_rows(leaves[0], idx, scale=2.0)
            user = ops.layernorm_rows(rows, leaves[1])
            s = user @ leaves[0].t()
            logp, entropy, top_logp, top = ops.logprobs_rows(s, pos, k=5)
            grads = list(torch.autograd.grad((logp, entropy, top_logp), leaves,
                                             (torch.ones_like(logp), torch.ones_like(entropy), torch.ones_like(top_logp))))
        norm = optim.clip_grads(grads, 1.0)
        return [logp.detach(), entropy.detach(), top_logp.detach(), top, norm] + grads

    stream = torch.cuda.Stream()
    graphs = []
    for seed in (1, 2):
        static = [v.to(DEV) for v in inputs(seed)]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            chain(*static)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            outs = chain(*static)
        graphs.append((g, static, outs))
    for turn in range(4):
        for k, (g, static, outs) in enumerate(graphs):
            fresh = [v.to(DEV) for v in inputs(10 + 2 * turn + k)]
            for a, b in zip(static, fresh):
                a.copy_(b)
            g.replay()
            want = chain(*fresh)                              # eager, between the replays
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), (turn, k, i)


@pytest.mark.parametrize("d", [8, 20, 64, 300])
@pytest.mark.parametrize("kind", ["one", "half", "steep", "two"])
def test_embed_gradient_of_popular_tokens(kind, d):
    """Tokens that hold a large part of 300 001 places: their chunks are counted by a search, their partial rows joined by a whole
    block, and the rows without a place among them found by a search. fp32 sums: chunks of up to 64 places, then the chunks' sums
    over 4 to 32 groups, so no entry passes through more than 64 + 4688 / 4 + 32 additions; the same call gives the same bits."""
    from mmssl_amd import ops
    n, rows = 300001, 3001
    q = gen(d)
    u = torch.rand(n, generator=q)
    idx = {"one": torch.full((n,), 1500), "half": torch.where(u < 0.5, 7, (u * 3000).long()),
           "steep": (rows * u ** 6).long().clamp_(0, rows - 1), "two": torch.where(u < 0.4, 0, 3000)}[kind].long()
    g = torch.randn(n, d, generator=q)
    w = torch.zeros(rows, d, device=DEV, requires_grad=True)
    out = ops.embed_rows(w, idx.to(DEV))
    (a,) = torch.autograd.grad(out, w, g.to(DEV), retain_graph=True)
    (b,) = torch.autograd.grad(out, w, g.to(DEV))
    assert torch.equal(a, b)
    want = torch.zeros(rows, d, dtype=torch.float64).index_add_(0, idx, g.double())
    size = torch.zeros(rows, d, dtype=torch.float64).index_add_(0, idx, g.double().abs())
    err = (a.cpu().double() - want).abs()
    assert bool((err <= 1300 * 2.0 ** -24 * size).all()), float((err / size.clamp_min(1e-30)).max())
    assert bool((a.cpu()[size[:, 0] == 0] == 0).all())


def test_capture_refuses_what_the_capture_could_not_hold():
    """A leaf of a live eager graph of the default stream, a producer of one, numbers on the host: an error before anything is
    recorded; the same calls are captured once the eager graph is gone, or without gradients."""
    from mmssl_amd import ops
    from mmssl_amd._lib import MmsslError
    w = torch.randn(50, 64, device=DEV, requires_grad=True)
    v = torch.randn(64, device=DEV, requires_grad=True)
    idx = torch.arange(20, device=DEV)
    rows = w.detach()[:20]
    eager = ops.layernorm_rows(ops.embed_rows(w, idx), v)                # kept: holds the accumulators of w and v
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def captured(fn):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            out = fn()
        return g, out

    for name, fn in (("leaf", lambda: ops.embed_rows(w, idx)), ("parameter", lambda: ops.layernorm_rows(rows, v)),
                     ("producer", lambda: ops.layernorm_rows(eager)), ("scores", lambda: ops.logprobs_rows(eager, idx)),
                     ("tokens", lambda: ops.embed_rows(w.detach(), [1, 2, 3])),
                     ("target", lambda: ops.logprobs_rows(rows, torch.zeros(20, dtype=torch.int64)))):
        print(name, flush=True)
        with pytest.raises(MmsslError):
            captured(fn)
    with torch.no_grad():
        g, out = captured(lambda: ops.layernorm_rows(ops.embed_rows(w, idx), v))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager.detach())
    want = torch.autograd.grad(eager, (w, v), torch.ones_like(eager))
    one = torch.ones_like(eager).detach()
    del eager
    g, got = captured(lambda: torch.autograd.grad(ops.layernorm_rows(ops.embed_rows(w, idx), v), (w, v), one))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_catalogue_operators_on_two_streams_at_once():
    from mmssl_amd import ops, optim
    g0 = gen(71)
    table = torch.randn(5000, 64, generator=g0).to(DEV)
    idx = torch.randint(5000, (20000,), generator=g0).to(DEV)
    g = torch.randn(20000, 64, generator=g0).to(DEV)
    x = torch.randn(200, 20000, generator=g0).to(DEV)
    tg = torch.randint(20000, (200,), generator=g0).to(DEV)

    def work():
        w = table.detach().requires_grad_(True)
        out = ops.embed_rows(w, idx)
        (gw,) = torch.autograd.grad(out, w, g)
        y = ops.layernorm_rows(out.detach())
        o = ops.logprobs_rows(x, tg, k=30)
        c = [gw.clone(), y.clone()]
        return [gw, y, o[0], o[1], o[2], o[3], optim.clip_grads(c, 1.0)] + c

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(work())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_catalogue_operators_refuse():
    from mmssl_amd import ops, optim
    from mmssl_amd._lib import MmsslError
    x = torch.randn(6, 40, device=DEV)
    idx = torch.zeros(6, dtype=torch.int64, device=DEV)
    w = torch.ones(40, device=DEV)
    half = x.half()
    refused = [
        lambda: ops.embed_rows(x.double(), idx), lambda: ops.embed_rows(x[0], idx), lambda: ops.embed_rows(x.t(), idx),
        lambda: ops.embed_rows(x, idx.float()), lambda: ops.embed_rows(x, idx.bool()), lambda: ops.embed_rows([1.0], idx),
        lambda: ops.embed_rows(x[:, :0], idx), lambda: ops.embed_rows(x.to_sparse(), idx),
        lambda: ops.layernorm_rows(x.double()), lambda: ops.layernorm_rows(x.int()), lambda: ops.layernorm_rows(x[:, :0]),
        lambda: ops.layernorm_rows(x, w[:39]), lambda: ops.layernorm_rows(x, w[None]), lambda: ops.layernorm_rows(x, w.half()),
        lambda: ops.layernorm_rows(half, w, w.half()), lambda: ops.layernorm_rows(x, w.cpu()),
        lambda: ops.layernorm_rows(x, eps=-1.0), lambda: ops.layernorm_rows(x, eps=float("nan")),
        lambda: ops.layernorm_rows(x, eps=float("inf")), lambda: ops.layernorm_rows(torch.tensor(1.0, device=DEV)),
        lambda: ops.logprobs_rows(x, idx, k=41), lambda: ops.logprobs_rows(x, idx, k=-1),
        lambda: ops.logprobs_rows(torch.randn(6, 400, device=DEV), idx, k=129), lambda: ops.logprobs_rows(x, idx[:5]),
        lambda: ops.logprobs_rows(x, idx[None]), lambda: ops.logprobs_rows(x, idx.float()),
        lambda: ops.logprobs_rows(x, idx, temperature=0.0), lambda: ops.logprobs_rows(x, idx, temperature=-1.0),
        lambda: ops.logprobs_rows(x, idx, temperature=float("nan")), lambda: ops.logprobs_rows(x, idx, temperature=float("inf")),
        lambda: ops.logprobs_rows(x.double(), idx), lambda: ops.logprobs_rows(x[:, :0], idx),
        lambda: optim.clip_grads([x], 1.0, out=[half]), lambda: optim.clip_grads([x], 1.0, out=[x[:5].clone()]),
        lambda: optim.clip_grads([x, w], 1.0, out=[x]), lambda: optim.clip_grads([x, x.cpu()], 1.0),
        lambda: optim.clip_grads([x, x], 1.0), lambda: optim.clip_grads([x[:4], x[2:]], 1.0),
        lambda: optim.clip_grads([x[0], x[1]], 1.0, out=[x[1], x[2]]), lambda: optim.clip_grads([x.t()], 1.0),
        lambda: optim.clip_grads([x.double()], 1.0), lambda: optim.clip_grads([x], float("nan")),
        lambda: optim.grad_norm([x, x.cpu()]), lambda: optim.grad_norm([x.t()]), lambda: optim.grad_norm([]),
    ]
    before = x.clone()
    for i, fn in enumerate(refused):
        try:
            fn()
        except MmsslError:
            continue
        raise AssertionError("case %d was not refused" % i)
    assert torch.equal(x, before)
    # read-only lists may name a tensor twice, and an empty tensor is no overlap
    assert abs(float(optim.grad_norm([x, x])) - 2 ** 0.5 * float(x.norm())) < 1e-4
    e = torch.empty(0, device=DEV)
    optim.clip_grads([e, x.clone(), e], 1.0)


def test_gradients_are_not_differentiable_again():
    from mmssl_amd import ops
    x = torch.randn(6, 40, device=DEV, requires_grad=True)
    idx = torch.zeros(6, dtype=torch.int64, device=DEV)
    for out in (ops.embed_rows(x, idx), ops.layernorm_rows(x), ops.logprobs_rows(x, idx)[0]):
        with pytest.raises(RuntimeError, match="not differentiable again"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_modes_without_gradients_and_changed_inputs():
    from mmssl_amd import ops, optim
    x = torch.randn(6, 40, device=DEV, requires_grad=True)
    idx = torch.arange(6, device=DEV)
    want = ops.layernorm_rows(x).detach()
    with torch.inference_mode():
        got = ops.layernorm_rows(x)
        assert torch.equal(got, want) and not got.requires_grad
        g = torch.ones(5, device=DEV)
        optim.clip_grads([g], 1.0)
    with torch.no_grad():
        assert not ops.embed_rows(x, idx).requires_grad and not ops.logprobs_rows(x, idx)[0].requires_grad
    y = x * 1.0
    out = ops.logprobs_rows(y, idx)[0]
    optim.clip_grads([y.detach()], 0.5)                       # changes what the backward pass needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # only some of the inputs want gradients
    w = torch.ones(40, device=DEV, requires_grad=True)
    b = torch.zeros(40, device=DEV)
    a = x.detach()
    (gw,) = torch.autograd.grad(ops.layernorm_rows(a, w, b).sum(), w)
    assert torch.allclose(gw, torch.nn.functional.layer_norm(a, (40,)).sum(0), atol=1e-4)
    b.requires_grad_(True)
    (gb,) = torch.autograd.grad(ops.layernorm_rows(a, None, b).sum(), b)
    assert torch.equal(gb, torch.full_like(gb, 6.0))
    (gx,) = torch.autograd.grad(ops.layernorm_rows(x, w.detach(), b.detach()).sum(), x)
    assert float(gx.abs().max()) < 1e-4                       # the rows' gradients of a plain sum cancel


def test_long_gradient_lists_of_more_chunks_than_a_block_looks_ahead():
    """97 tensors of 560 M elements: a block has more chunks than it works out at once. The squares are whole numbers, so the norm
    is exact up to its last rounding, and the factor 2^-8 is as well."""
    from mmssl_amd import optim
    sizes = [5_770_000 + 37 * i for i in range(96)] + [1_000_003]
    grads = [torch.full((n,), 1.0 + i % 3, device=DEV, dtype=torch.bfloat16) for i, n in enumerate(sizes)]
    for i, g in enumerate(grads):
        g[-1] = 200.0 + i                                                 # (rounded by the type)
    total = sum(int(g[-1]) ** 2 + (n - 1) * (1 + i % 3) ** 2 for i, (n, g) in enumerate(zip(sizes, grads)))
    norm = total ** 0.5
    out = [torch.empty_like(g) for g in grads]
    got = optim.clip_grads(grads, norm / 256, out=out)
    assert abs(float(got) - norm) <= 2 ** -23 * norm
    for g, o in zip(grads, out):
        # the factor is 2^-8 up to a few half steps of 32 bits, far below one of bf16
        assert bool((o.float() - g.float() / 256).abs().max() <= float(g.max()) / 256 * 2 ** -8)
        assert torch.equal(o[0].float() * 256, g[0].float()) and torch.equal(o[-1].float() * 256, g[-1].float())


def test_long_gradient_lists_in_captured_graphs():
    """Lists past the kernel arguments' go through a table in the workspace: two graphs with their own, replayed in turn with
    eager calls between them."""
    from mmssl_amd import optim
    g0 = gen(81)
    sizes = [int(v) for v in torch.randint(1, 20000, (250,), generator=g0)]
    stream = torch.cuda.Stream()
    graphs = []
    for k in range(2):
        grads = [torch.randn(n, generator=g0).to(TYPES[(i + k) % 3]).to(DEV) for i, n in enumerate(sizes)]
        out = [torch.empty_like(g) for g in grads]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            norm = optim.clip_grads(grads, 2.0, out=out)
        graphs.append((graph, grads, out, norm))
    for turn in range(4):
        for graph, grads, out, norm in graphs:
            for g in grads:
                g.mul_(0.5 if turn % 2 else 3.0)
            graph.replay()
            want = [torch.empty_like(g) for g in grads]
            eager = optim.clip_grads(grads, 2.0, out=want)
            torch.cuda.synchronize()
            assert torch.equal(norm, eager)
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_forward_mode_tangents_are_refused():
    """An operand or an incoming gradient with a tangent: there is no such derivative, and none may come out as zero."""
    from torch.autograd import forward_ad as fw
    from mmssl_amd import ops, optim
    from mmssl_amd._lib import MmsslError
    x = torch.randn(6, 40, device=DEV)
    idx = torch.arange(6, device=DEV)
    w = torch.ones(40, device=DEV)
    with fw.dual_level():
        def dual(v):
            return fw.make_dual(v, torch.ones_like(v))
        for base in (x, x.clone().requires_grad_(True)):
            for fn in (lambda: ops.embed_rows(dual(base), idx), lambda: ops.layernorm_rows(dual(base)),
                       lambda: ops.layernorm_rows(base, dual(w)), lambda: ops.layernorm_rows(base, None, dual(w)),
                       lambda: ops.layernorm_rows(base, w, dual(w)), lambda: ops.logprobs_rows(dual(base), idx),
                       lambda: ops.logprobs_rows(dual(base), idx, k=3)):
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(MmsslError, match="forward-mode"):
                        fn()
        y = x.clone()
        for fn in (lambda: optim.grad_norm([y, dual(y)]), lambda: optim.clip_grads([dual(y)], 0.1),
                   lambda: optim.clip_grads([y], 0.1, out=[dual(torch.zeros_like(y))])):
            with pytest.raises(MmsslError, match="forward-mode"):
                fn()
        assert torch.equal(y, x)
        leaf = x.clone().requires_grad_(True)
        for fn in (lambda: ops.embed_rows(leaf, idx), lambda: ops.layernorm_rows(leaf),
                   lambda: ops.logprobs_rows(leaf, idx)[0], lambda: ops.logprobs_rows(leaf, idx)[1],
                   lambda: ops.logprobs_rows(leaf, idx, k=3)[2]):
            out = fn()
            one = torch.ones_like(out)
            want = torch.autograd.grad(out, leaf, one, retain_graph=True)[0]
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaf, dual(one), retain_graph=True)
            assert torch.equal(torch.autograd.grad(out, leaf, one)[0], want)
        held = dual(x)
        want = ops.layernorm_rows(x)
        assert torch.equal(ops.layernorm_rows(fw.unpack_dual(held).primal), want)
    assert torch.equal(ops.layernorm_rows(held), want)                    # the level is gone, and the tangent with it


def test_capture_refuses_eager_leaves_behind_recorded_operations():
    """The leaf of a live eager graph of the default stream, reached through operations that the capture itself records: refused
    by the forward call (no backward pass is made here). Once the eager graph is gone the same chains are captured, and replay
    the eager bits."""
    from mmssl_amd import ops
    from mmssl_amd._lib import MmsslError
    q = gen(91)
    w = torch.randn(50, 64, generator=q).to(DEV).requires_grad_(True)
    v = torch.randn(64, generator=q).to(DEV).requires_grad_(True)
    rows = torch.randn(20, 64, generator=q).to(DEV)
    idx = torch.arange(20, device=DEV)
    chains = [("one operation", lambda: ops.embed_rows(w.to(torch.bfloat16), idx)),
              ("a parameter", lambda: ops.layernorm_rows(rows, v * 2.0)),
              ("a product", lambda: ops.logprobs_rows(rows @ w.t(), idx)[0]),
              ("several", lambda: ops.layernorm_rows(((rows + 1.0) * (w[:20] - 2.0)).exp().tanh())),
              ("an operator of this package", lambda: ops.layernorm_rows(ops.embed_rows(w * 1.0, idx)))]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(stream):        # a library's first product sets the library up, which no capture holds
        for _, fn in chains:
            fn()
    torch.cuda.synchronize()
    eager = ops.layernorm_rows(ops.embed_rows(w, idx), v)                # kept: holds the accumulators of w and v

    def captured(fn):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            out = fn()
        return g, out

    for name, fn in chains:
        print(name, flush=True)
        with pytest.raises(MmsslError, match="eager graph of the default stream"):
            captured(fn)
    del eager
    for name, fn in chains:
        print(name, flush=True)
        with torch.no_grad():
            want = fn()
        g, out = captured(lambda: fn().detach())
        for _ in range(3):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), name
    # eagerly, also on a stream of its own, nothing is refused
    keep = [fn() for _, fn in chains]
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        keep += [fn() for _, fn in chains]
    torch.cuda.synchronize()
    for a, b in zip(keep[:5], keep[5:]):
        assert torch.equal(a, b)


def test_lazily_negated_views_count_as_what_they_show():
    """The imaginary part of a conjugate holds its values with the other sign in memory: one column (whose strides need no copy),
    several, as an operand, as a parameter, as an incoming gradient, in lists."""
    from mmssl_amd import ops, optim
    from mmssl_amd._lib import MmsslError
    q = gen(95)
    idx = torch.arange(6, device=DEV)

    def both(*shape):
        v = torch.randn(shape, dtype=torch.complex64, generator=q).to(DEV).conj().imag
        assert v.is_neg()
        return v, v.resolve_neg().contiguous()

    for d in (1, 5):
        (x, y), (g, h), (w, u) = both(6, d), both(6, d), both(d)
        for fn in (lambda v, w: ops.embed_rows(v if d == 1 else v.contiguous(), idx), lambda v, w: ops.layernorm_rows(v, w, w),
                   lambda v, w: ops.layernorm_rows(y, w), lambda v, w: ops.logprobs_rows(v, idx.clamp(max=d - 1), k=1)[2]):
            assert torch.equal(fn(x, w), fn(y, u)), d
        for fn in (lambda v, w: ops.embed_rows(v, idx), lambda v, w: ops.layernorm_rows(v, w)):
            leaf, lw = y.clone().requires_grad_(True), u.clone().requires_grad_(True)
            out = fn(leaf, lw)
            for a, b in zip(torch.autograd.grad(out, (leaf, lw), g, allow_unused=True, retain_graph=True),
                            torch.autograd.grad(out, (leaf, lw), h, allow_unused=True)):
                assert (a is None and b is None) or torch.equal(a, b), d
    (x, y), (g, h) = both(6, 300), both(6)
    leaf = y.clone().requires_grad_(True)
    out = ops.logprobs_rows(leaf, idx)[0]
    assert torch.equal(torch.autograd.grad(out, leaf, g, retain_graph=True)[0], torch.autograd.grad(out, leaf, h)[0])
    (a, b) = both(1)
    assert a.is_contiguous()
    assert torch.equal(optim.grad_norm([a]), optim.grad_norm([b]))
    with pytest.raises(MmsslError):
        optim.clip_grads([a], 0.25, out=[torch.zeros_like(b)])
    optim.clip_grads([a], 0.25)
    optim.clip_grads([b], 0.25)
    assert torch.equal(a, b)


def test_gradient_lists_that_require_grad():
    """Norms and clipping are not recorded: what requires grad is refused while a graph is recorded, before anything is written.
    Without recording, and for the .grad of a create_graph=True pass, they run."""
    from mmssl_amd import optim
    from mmssl_amd._lib import MmsslError
    p = torch.nn.Parameter(torch.full((16,), 2.0, device=DEV))
    h = p * 3.0
    plain = torch.ones(16, device=DEV)
    for fn in (lambda: optim.grad_norm([p]), lambda: optim.grad_norm([plain, h]), lambda: optim.clip_grads([p], 1.0),
               lambda: optim.clip_grads([plain, h], 1.0), lambda: optim.clip_grads([plain], 1.0, out=[p]),
               lambda: optim.clip_grads([h], 1.0, out=[plain])):
        with pytest.raises(MmsslError, match="not differentiable"):
            fn()
    assert bool((p == 2.0).all()) and bool((h == 6.0).all()) and bool((plain == 1.0).all())
    with torch.no_grad():
        want = (16 * 4.0 + 16 * 36.0) ** 0.5        # no fp32 number: the result is rounded once, half a step off at most
        assert abs(float(optim.grad_norm([p, h])) - want) <= want * 2.0 ** -24
        assert float(optim.clip_grads([p], 4.0)) == 8.0
    assert float((p.detach() - 1.0).abs().max()) <= 1e-6
    loss = (p ** 3).sum()
    loss.backward(create_graph=True)
    assert p.grad.requires_grad
    want = p.grad.detach() / 12.0                                          # gradients of 3, sixteen of them: norm 12
    norm = optim.clip_grad_norm([p], 1.0)
    assert not norm.requires_grad and abs(float(norm) - 12.0) <= 1e-4
    assert float((p.grad.detach() - want).abs().max()) <= 1e-5
    p.grad = None


def test_parameters_that_share_a_gradient():
    """Two parameters with one .grad, contiguous and not, and the same parameter twice: counted each time, scaled once."""
    from mmssl_amd import optim
    from mmssl_amd._lib import MmsslError
    q = gen(97)
    for make in (lambda: torch.randn(30, 50, generator=q).to(DEV), lambda: torch.randn(50, 30, generator=q).to(DEV).t()):
        a, b, c = (torch.nn.Parameter(torch.zeros(30, 50, device=DEV)) for _ in range(3))
        a.grad, c.grad = make(), torch.randn(30, 50, generator=q).to(DEV)
        b.grad = a.grad
        was, other = a.grad.double(), c.grad.double()
        for given, times in (([a, b, c], 2), ([a, c, a, b], 3)):
            assert b.grad is a.grad
            total = float((times * (was ** 2).sum() + (other ** 2).sum()) ** 0.5)
            norm = optim.clip_grad_norm(given, total / 2)
            assert abs(float(norm) - total) <= total * (2.0 ** -24 + 1e-12)
            factor = total / 2 / (total + 1e-6)
            for p, w in ((a, was), (c, other)):
                # the factor is rounded to 32 bits, so is the product
                within(p.grad, w * factor, (w * factor).abs().cpu() * 2.0 ** -22 + 1e-30, "grad")
            was, other = a.grad.double(), c.grad.double()
    whole = torch.randn(40, device=DEV)
    a, b = (torch.nn.Parameter(torch.zeros(30, device=DEV)) for _ in range(2))
    a.grad, b.grad = whole[:30], whole[10:]
    with pytest.raises(MmsslError, match="overlap"):
        optim.clip_grad_norm([a, b], 1.0)


def test_factors_that_require_grad_are_refused():
    from mmssl_amd import ops
    from mmssl_amd._lib import MmsslError
    x = torch.randn(6, 40, generator=gen(99)).to(DEV)
    idx = torch.arange(6, device=DEV)
    two = torch.tensor(2.0, device=DEV, requires_grad=True)
    calls = [lambda v: ops.embed_rows(x, idx, scale=v), lambda v: ops.layernorm_rows(x, eps=v),
             lambda v: ops.logprobs_rows(x, idx, temperature=v)[0]]
    for fn in calls:
        want = fn(2.0)
        for v in (two, two * 1.0):
            with pytest.raises(MmsslError, match="plain number"):
                fn(v)
            with torch.no_grad():
                assert torch.equal(fn(v), want)
        assert torch.equal(fn(two.detach()), want)


def popular_places(kind, n, rows, q):
    """Tokens of n places: evenly spread, one with all or half of them, steeply falling, the first and the last."""
    u = torch.rand(n, generator=q, device=DEV)
    return {"even": lambda: (rows * u).long().clamp_(max=rows - 1), "one": lambda: torch.full((n,), rows // 2, device=DEV),
            "half": lambda: torch.where(u < 0.5, torch.full_like(u, 7), rows * u).long().clamp_(max=rows - 1),
            "steep": lambda: (rows * u ** 6).long().clamp_(max=rows - 1),
            "two": lambda: torch.where(u < 0.4, 0, rows - 1)}[kind]().long()


def whole_sums(idx, whole, rows):
    """Sums of whole numbers (int64) over the places of each token, exactly: differences of running sums along the sorted list."""
    key, order = torch.sort(idx)
    run = torch.cat([torch.zeros_like(whole[:1]), whole[order].cumsum(0)])
    at = torch.searchsorted(key, torch.arange(rows + 1, device=DEV))
    return run[at[1:]] - run[at[:-1]]


@pytest.mark.parametrize("kind", ["even", "one", "half", "steep", "two"])
@pytest.mark.parametrize("n", [32767, 32768, 524287, 524288, 600011])
def test_embed_gradient_where_chunks_change_length(n, kind):
    """Lists around the lengths at which a chunk goes from 8 to 16 and from 16 to 64 places. Whole numbers: every sum stays below 2^24
    (at most 600011 terms of at most 8), so fp32 holds it and each sum on the way exactly, in any order, and the results
    are equal; a half type rounds that once."""
    from mmssl_amd import ops
    rows = 3001
    q = torch.Generator(device=DEV).manual_seed(n)
    idx = popular_places(kind, n, rows, q)
    for d, t in ((8, torch.float32), (64, torch.bfloat16), (300, torch.float32), (65, torch.float16)):
        whole = torch.randint(-8, 9, (n, d), generator=q, device=DEV)
        w = torch.zeros(rows, d, device=DEV, dtype=t, requires_grad=True)
        (a,) = torch.autograd.grad(ops.embed_rows(w, idx, scale=0.5), w, whole.to(t))
        assert torch.equal(a, (whole_sums(idx, whole, rows).double() * 0.5).to(t)), (d, t)


@pytest.mark.parametrize("kind", ["even", "one", "half", "steep", "two"])
@pytest.mark.parametrize("n", [300001, 524287, 524288])
def test_embed_gradient_of_long_lists_within_the_chain_of_its_sums(n, kind):
    """Numbers with 20 bits behind the point, whose sums fp32 has to round. A term passes the sum of its chunk (16 places below
    2^19 of them, 64 from there on), then, over more than 16 chunks, the sum of one of the block's lane groups (each takes
    every so-manyth chunk), the groups' sum and the first chunk's part: off by 2^-24 of the magnitudes for each."""
    from mmssl_amd import ops
    rows = 3001
    q = torch.Generator(device=DEV).manual_seed(n + 1)
    idx = popular_places(kind, n, rows, q)
    chunk = 64 if n >= 1 << 19 else 16
    chunks = -(-n // chunk)
    for d, lanes in ((20, 8), (64, 16), (300, 64)):
        groups = 256 // lanes
        chain = chunk + max(16, -(-chunks // groups)) + groups + 1
        whole = (torch.randn(n, d, generator=q, device=DEV) * 2 ** 20).round().clamp_(-(2 ** 23), 2 ** 23).long()
        w = torch.zeros(rows, d, device=DEV, requires_grad=True)
        (a,) = torch.autograd.grad(ops.embed_rows(w, idx), w, whole.float() / 2 ** 20)
        want, size = whole_sums(idx, whole, rows).double() / 2 ** 20, whole_sums(idx, whole.abs(), rows).double() / 2 ** 20
        assert bool(((a.double() - want).abs() <= chain * 2.0 ** -24 * size).all()), d


def test_long_gradient_lists_clip_every_element():
    """Lists of more chunks than a block looks ahead, as above, every element against its own value, into outputs that hold
    something else before."""
    from mmssl_amd import optim
    sizes = [5_770_000 + 37 * i for i in range(96)] + [1_000_003]
    grads = [torch.full((n,), 1.0 + i % 3, device=DEV, dtype=torch.bfloat16) for i, n in enumerate(sizes)]
    for i, g in enumerate(grads):
        g[-1] = 200.0 + i                                                 # (rounded by the type)
    norm = sum(int(g[-1]) ** 2 + (n - 1) * (1 + i % 3) ** 2 for i, (n, g) in enumerate(zip(sizes, grads))) ** 0.5
    out = [torch.full_like(g, float("nan")) for g in grads]
    optim.clip_grads(grads, norm / 256, out=out)
    for i, (g, o) in enumerate(zip(grads, out)):
        # the factor is 2^-8 up to a few half steps of 32 bits, and the product's nearest bf16 number is the value's 2^-8 fold,
        # which bf16 holds: no element is off at all
        assert torch.equal(o.float() * 256, g.float()), i
