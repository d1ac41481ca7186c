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
