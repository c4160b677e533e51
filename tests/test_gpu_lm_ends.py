"""Layer norm, token embedding, top logits and the distillation loss against plain statements in 64 bits.

Tolerances are error bounds of the arithmetic, not fits: `u = 2^-24` is half a step of fp32, a sum of n terms in order is
off by at most n u times the sum of its terms' sizes, a stored bf16 value by half a step (2^-8 of its size).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
bf, f32 = torch.bfloat16, torch.float32
U = 2.0**-24


@pytest.fixture(scope="module")
def nv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from param_decomp_b200.ops import native

    native.lib()  # must load: nothing falls back to another path where there is a GPU
    return native


def _done(nv):
    torch.cuda.synchronize()
    nv.check_status()


def _within(got, want, bound, what):
    """`got` is `want` (64 bits) to within `bound` and the rounding to the type that it is stored in."""
    half_step = 2.0**-8 if got.dtype == bf else U
    got, want = got.detach().double().cpu(), want.cpu()
    limit = bound.cpu() * (1 + 2.0**-7) + want.abs() * half_step + 1e-300
    off = (got - want).abs()
    assert bool((off <= limit).all()), f"{what}: {float((off / limit).max()):.3f} of its bound"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- layer norm -------------------------------------------------------------------------------------------------------


def _norm_reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    # a row's sum: at most 24 terms a thread, 5 halvings in a warp, 16 warps; the mean's error is relative to mean |x|
    n = 64
    spread = xh.abs() + rstd * x.abs().mean(1, keepdim=True)
    bounds = dict(
        y=2 * n * U * (spread * w.abs() + b.abs()),
        dx=4 * n * U * rstd * (g.abs() + g.abs().mean(1, keepdim=True) + spread * (g.abs() * spread).mean(1, keepdim=True)),
        dw=(x.shape[0] + 2 * n) * U * (dy.abs() * spread).sum(0),
        db=(x.shape[0] + n) * U * dy.abs().sum(0))
    return dict(y=xh * w + b, dx=dx, dw=(dy * xh).sum(0), db=dy.sum(0)), bounds


@pytest.mark.parametrize("p_type", [bf, f32])
@pytest.mark.parametrize("x_type", [bf, f32])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 8), (700, 33), (33, 256), (2500, 768), (257, 769), (64, 1000), (129, 1032),
                                    (41, 2047), (300, 4096), (7, 8192), (9, 8193), (4, 12288)])
def test_layer_norm_and_its_gradients(nv, rows, d, x_type, p_type):
    from param_decomp_b200.ops.elementwise import layer_norm

    g = _gen(rows * d)
    x = (torch.randn(rows, d, generator=g) * 2 + 1).to(x_type)
    w, b = (1 + 0.3 * torch.randn(d, generator=g)).to(p_type), torch.randn(d, generator=g).to(p_type)
    dy = torch.randn(rows, d, generator=g).to(x_type)
    want, bounds = _norm_reference(x, w, b, dy, 1e-5)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, 1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    _done(nv)
    assert y.dtype == x_type and dx.dtype == x_type and dw.dtype == p_type and db.dtype == p_type
    for name, got in dict(y=y, dx=dx, dw=dw, db=db).items():
        _within(got, want[name], bounds[name], name)


def test_layer_norm_options(nv):
    """No parameters, one of them, frozen ones, only parameters trained, no gradient at all, empty batches, leading axes,
    strided inputs and upstream gradients, and inputs at addresses that allow no 16-byte access."""
    from param_decomp_b200.ops.elementwise import layer_norm

    g = _gen(1)
    x, dy = torch.randn(6, 10, 264, generator=g), torch.randn(6, 10, 264, generator=g)
    w, b = torch.randn(264, generator=g), torch.randn(264, generator=g)
    for use_w, use_b, train in [(False, False, "x"), (True, False, "xw"), (False, True, "xb"), (True, True, "x"), (True, True, "w"),
                                (True, True, "b"), (True, True, "")]:
        want, bounds = _norm_reference(x.view(60, 264), w if use_w else None, b if use_b else None, dy.view(60, 264), 1e-6)
        leaf = {"x": x.cuda().requires_grad_("x" in train), "w": w.cuda().requires_grad_("w" in train) if use_w else None,
                "b": b.cuda().requires_grad_("b" in train) if use_b else None}
        y = layer_norm(leaf["x"], leaf["w"], leaf["b"], 1e-6)
        assert y.shape == x.shape and y.requires_grad == bool(train)
        _within(y.view(60, 264), want["y"], bounds["y"], "y")
        if train:
            for k, grad in zip(train, torch.autograd.grad(y, [leaf[k] for k in train], dy.cuda())):
                _within(grad.reshape(want["d" + k].shape), want["d" + k], bounds["d" + k], "d" + k)
    # a row of a wider tensor, an expanded upstream gradient, a tensor that starts 4 bytes into its storage
    wide = torch.randn(40, 600, generator=g)
    xs = wide.cuda()[:, 5:269].requires_grad_(True)
    y = layer_norm(xs, w.cuda(), b.cuda(), 1e-6)
    (dx,) = torch.autograd.grad(y.sum(), (xs,))
    want, bounds = _norm_reference(wide[:, 5:269], w, b, torch.ones(40, 264), 1e-6)
    _within(y, want["y"], bounds["y"], "y")
    _within(dx, want["dx"], bounds["dx"], "dx")
    flat = torch.randn(40 * 264 + 1, generator=g)
    odd = flat.cuda()[1:].view(40, 264)
    want, bounds = _norm_reference(flat[1:].view(40, 264), w, b, torch.ones(40, 264), 1e-6)
    _within(layer_norm(odd, w.cuda(), b.cuda(), 1e-6), want["y"], bounds["y"], "y")
    # nothing to norm
    none = torch.zeros(0, 264, device="cuda", requires_grad=True)
    wg, bg = w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    grads = torch.autograd.grad(layer_norm(none, wg, bg, 1e-6).sum(), (none, wg, bg))
    assert grads[0].shape == (0, 264) and not bool(grads[1].any()) and not bool(grads[2].any())
    _done(nv)


def test_layer_norm_far_means_and_special_rows(nv):
    """Rows far from zero keep their variance (it is summed around the mean), a constant row has the gradient of its eps, a
    row with an infinity or NaN stays its own affair."""
    from param_decomp_b200.ops.elementwise import layer_norm

    g = _gen(2)
    x = torch.randn(50, 768, generator=g) + 1000.0
    x[7] = 3.0
    w, b = torch.randn(768, generator=g), torch.randn(768, generator=g)
    dy = torch.randn(50, 768, generator=g)
    want, bounds = _norm_reference(x, w, b, dy, 1e-5)
    xs = x.cuda().requires_grad_(True)
    y = layer_norm(xs, w.cuda(), b.cuda(), 1e-5)
    (dx,) = torch.autograd.grad(y, (xs,), dy.cuda())
    _within(y, want["y"], bounds["y"], "y")
    _within(dx, want["dx"], bounds["dx"], "dx")
    bad = x.clone()
    bad[3, 5], bad[9, 700] = float("nan"), float("inf")
    yb = layer_norm(bad.cuda(), w.cuda(), b.cuda(), 1e-5)
    keep = [i for i in range(50) if i not in (3, 9)]
    assert torch.equal(yb[keep], y.detach()[keep]) and bool(yb[3].isnan().all()) and bool(yb[9].isnan().any())
    _done(nv)


def test_layer_norm_gradient_against_differences(nv):
    from param_decomp_b200.ops.elementwise import layer_norm

    g = _gen(3)
    x, w, b = torch.randn(3, 40, generator=g), torch.randn(40, generator=g), torch.randn(40, generator=g)
    dy = torch.randn(3, 40, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves, 1e-5), leaves, dy.cuda())

    def loss(x, w, b):
        m = x.mean(1, keepdim=True)
        return float((((x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-5) * w + b) * dy.double()).sum())

    args = [t.double() for t in (x, w, b)]
    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        plus, minus = ([a + s * h * way if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = (loss(*plus) - loss(*minus)) / (2 * h)
        size = float((grad.cpu().double().abs() * way.abs()).sum())
        # differences: h^2 times the third derivative (order one here) and 2^-52 / h; the kernel: 512 u
        assert abs(float((grad.cpu().double() * way).sum()) - slope) <= size * 512 * U + 1e-6


# ---- embedding --------------------------------------------------------------------------------------------------------


def _zipf(n, V, g):
    p = 1.0 / torch.arange(1, V + 1, dtype=torch.float64)
    return torch.multinomial(p, n, replacement=True, generator=g)


@pytest.mark.parametrize("table_type,out_type", [(bf, bf), (f32, bf), (f32, f32), (bf, f32)])
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 50, 8), (33, 1, 24), (32, 7, 8), (2500, 3, 40), (1000, 2000, 264), (5000, 300, 33),
                                   (4097, 50277, 16), (300, 400000, 8), (20000, 1000, 768), (777, 151936, 5), (2048, 147, 1032)])
def test_embedding_and_its_gradient(nv, n, V, d, table_type, out_type):
    """Rows seen never, once, up to a slab of tokens, and by more than a slab (one token fills a slab row exactly, runs that
    start and end inside slabs, one id for all tokens)."""
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(n + V + d)
    tokens = _zipf(n, V, g) if V > 1 else torch.zeros(n, dtype=torch.int64)
    table, dy = torch.randn(V, d, generator=g).to(table_type), torch.randn(n, d, generator=g).to(out_type)
    scale = math.sqrt(d)
    for ids in (tokens.cuda(), tokens.to(torch.int32).cuda()):
        leaf = table.cuda().requires_grad_(True)
        y = embedding(ids, leaf, scale, out_dtype=out_type)
        (dE,) = torch.autograd.grad(y, (leaf,), dy.cuda())
        _done(nv)
        assert y.dtype == out_type and dE.dtype == table_type and y.shape == (n, d) and dE.shape == (V, d)
        s = float(torch.tensor(scale, dtype=f32))
        want = table.double()[tokens] * s
        _within(y, want, 2 * U * want.abs(), "y")
        wantE = torch.zeros(V, d, dtype=torch.float64).index_add_(0, tokens, dy.double()) * s
        sizes = torch.zeros(V, d, dtype=torch.float64).index_add_(0, tokens, dy.double().abs()) * s
        counts = torch.bincount(tokens, minlength=V).double()[:, None]
        _within(dE, wantE, (counts + 2) * U * sizes, "dE")


def test_embedding_gradient_is_the_same_every_time(nv):
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(5)
    tokens, table, dy = _zipf(30000, 500, g).cuda(), torch.randn(500, 136, generator=g).cuda().requires_grad_(True), torch.randn(
        30000, 136, generator=g).cuda()
    first = torch.autograd.grad(embedding(tokens, table), (table,), dy)[0]
    for _ in range(10):
        assert torch.equal(first, torch.autograd.grad(embedding(tokens, table), (table,), dy)[0])


def test_embedding_options_and_refused_tokens(nv):
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(6)
    table = torch.randn(30, 24, generator=g).cuda().requires_grad_(True)
    # leading axes, strided ids, ids of an odd storage offset, a transposed table, an expanded upstream gradient
    ids = torch.randint(0, 30, (4, 9), generator=g).cuda()
    want = table.detach()[ids.T]
    y = embedding(ids.T, table)
    assert torch.equal(y.detach(), want) and y.shape == (9, 4, 24)
    (dE,) = torch.autograd.grad(y.sum(), (table,))
    assert torch.equal(dE, torch.bincount(ids.view(-1), minlength=30)[:, None].expand(30, 24).float())
    square = torch.randn(24, 30, generator=g).cuda()
    assert torch.equal(embedding(ids.view(-1)[1:], square.T), square.T[ids.view(-1)[1:]])
    # none
    y = embedding(ids[:0], table)
    assert y.shape == (0, 9, 24) and not bool(torch.autograd.grad(y.sum(), (table,))[0].any())
    _done(nv)
    # unknown ids: zero rows, no part in the gradient, reported to the next call and by the status word
    bad = ids.view(-1).clone()
    bad[3], bad[7], bad[20] = -1, 30, 2**40
    y = embedding(bad, table)
    (dE,) = torch.autograd.grad(y, (table,), torch.ones_like(y))
    torch.cuda.synchronize()
    good = torch.ones(36, dtype=torch.bool)
    good[[3, 7, 20]] = False
    assert torch.equal(y.detach().cpu()[good], table.detach().cpu()[bad.cpu()[good]]) and not bool(y.detach().cpu()[~good].any())
    assert torch.equal(dE[:, 0].cpu(), torch.bincount(bad.cpu()[good], minlength=30).float())
    with pytest.raises(nv.NativeError, match="token"):
        embedding(ids, table)
    embedding(bad, table)
    with pytest.raises(nv.NativeError, match="token"):
        nv.check_status()
    embedding(ids, table)
    _done(nv)


# ---- top logits -------------------------------------------------------------------------------------------------------


def _top_reference(z, k, T):
    idx = torch.sort(z.double(), dim=1, descending=True, stable=True)[1][:, :k]
    rest = (z.double() / T).scatter(1, idx, -math.inf)
    return torch.gather(z, 1, idx), idx.to(torch.int32), torch.logsumexp(rest, 1)


def _check_top(z, k, T=1.0):
    from param_decomp_b200.ops.top_logits import top_logits

    values, indices, tail = top_logits(z, k, T)
    want = _top_reference(z.cpu(), k, T)
    assert torch.equal(indices.cpu(), want[1])
    assert torch.equal(values.cpu().view(torch.int16 if z.dtype == bf else torch.int32),
                       want[0].view(torch.int16 if z.dtype == bf else torch.int32))
    fine = want[2].isfinite()
    assert torch.equal(tail.cpu()[~fine].double(), want[2][~fine])
    # a thread adds V / 256 terms at most, each off by its argument's rounding (under 128 u) and the exponential's (4 u)
    bound = (z.shape[1] / 256 + 64 + 132) * U + 4 * U * want[2][fine].abs()
    assert bool(((tail.cpu()[fine].double() - want[2][fine]).abs() <= bound).all())


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (3, 5, 5), (2, 8, 3), (5, 100, 99), (4, 1000, 256), (9, 2000, 8), (700, 2003, 40),
                                   (3, 4096, 128), (5, 4099, 1), (7, 50277, 64), (2, 151936, 256), (1, 300001, 200)])
def test_top_logits_against_a_stable_sort(nv, n, V, k, kind):
    z = (torch.randn(n, V, generator=_gen(n + V)) * 2.5).to(kind).cuda()
    _check_top(z, k)
    _check_top(z, k, 2.0)
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("n,V,k,steep", [(40, 50277, 64, 1.0), (40, 50277, 256, 1.0), (40, 50277, 256, 2.0), (9, 151936, 64, 2.0),
                                         (9, 151936, 256, 2.0), (6, 9000, 256, 4.0), (5, 3000, 100, 3.0), (3, 400001, 256, 1.5)])
def test_top_logits_of_columns_in_order_of_frequency(nv, n, V, k, steep, kind):
    """Logits about a mean that falls with the logarithm of the column, above and below zero: the largest are neighbours, more
    reach the first bound than there is room for. The same in every run."""
    from param_decomp_b200.ops.top_logits import top_logits

    z = torch.randn(n, V, generator=_gen(V + k)) * 1.5 - steep * torch.log(torch.arange(1, V + 1).float()) + 2.0
    z[0] -= 40.0
    z = z.to(kind)
    _check_top(z.cuda(), k)
    _check_top(z.cuda(), k, 3.0)
    first = top_logits(z.cuda(), k)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, top_logits(z.cuda(), k)))
    _done(nv)


@pytest.mark.parametrize("kind,n,V,k", [(f32, 900, 5003, 20), (bf, 900, 5003, 200), (f32, 300, 151936, 64)])
def test_top_logits_do_not_change_from_run_to_run(nv, kind, n, V, k):
    """Logits are collected in the order in which threads come to them; nothing of that is left in the tails."""
    from param_decomp_b200.ops.top_logits import top_logits

    z = torch.randn(n, V, generator=_gen(3)).to(kind).cuda()
    first = top_logits(z, k)
    for _ in range(30):
        again = top_logits(z, k)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("V,k", [(2003, 40), (50277, 64), (9000, 256)])
def test_top_logits_of_awkward_rows(nv, V, k, kind):
    """Equal logits in masses, few logits above -inf, infinities, zeros of both signs, values that rise or fall along the
    row, one column far above the rest, all candidates in one block's columns, rows at odd addresses."""
    g = _gen(V)
    z = torch.randn(14, V, generator=g)
    z[0] = 1.0
    z[1] = (z[1] * 2).round()
    z[2] = -math.inf
    z[2, V // 2:V // 2 + k // 2] = 1.0
    z[3] = -math.inf
    z[4, 5:9] = math.inf
    z[5, :k + 3] = math.inf
    z[6] = torch.where(torch.arange(V) % 3 == 0, 0.0, -0.0)
    z[7] = torch.linspace(-5, 5, V)
    z[8] = torch.linspace(5, -5, V)
    z[9] -= 200.0
    z[9, :k] = 0.0
    z[10, 17:17 + 2 * k] += 50.0
    z[11] = torch.finfo(kind).min
    z[11, 3::7] = -1.0
    z[12] = torch.finfo(kind).min
    z[13, 64:80] = 30.0
    z = z.to(kind)
    _check_top(z.cuda(), k)
    wide = torch.full((14, V + 11), 99.0, dtype=kind)
    wide[:, 3:3 + V] = z
    _check_top(wide.cuda()[:, 3:3 + V], k)
    _done(nv)


def test_top_logits_shapes_and_nan(nv):
    from param_decomp_b200.ops.top_logits import top_logits

    g = _gen(9)
    z = torch.randn(2, 3, 5000, generator=g)
    z[0, 1, 77] = float("nan")
    z[1, 2, 4000:4010] = float("nan")
    out = top_logits(z.cuda(), 4)
    assert out.values.shape == (2, 3, 4) and out.indices.shape == (2, 3, 4) and out.tail.shape == (2, 3)
    assert int(out.indices[0, 1, 0]) == 77 and bool(out.values[0, 1, 0].isnan()) and bool(out.tail[0, 1].isfinite())
    assert out.indices[1, 2].tolist() == [4000, 4001, 4002, 4003] and bool(out.tail[1, 2].isnan())
    t = torch.randn(5000, 6, generator=g).cuda()
    assert torch.equal(top_logits(t.T, 4).indices, top_logits(t.T.contiguous(), 4).indices)
    e = top_logits(t[:, 0].expand(3, 5000), 4)
    assert torch.equal(e.indices[0], e.indices[2])
    assert top_logits(t.T[:0], 4).values.shape == (0, 4)
    assert torch.equal(top_logits(t[:, 0], 4).indices, e.indices[0])
    _done(nv)


# ---- distillation loss ------------------------------------------------------------------------------------------------


def _kl_reference(z, idx, t, tail, T):
    """Loss, gradient and their error bounds, in 64 bits."""
    n, V = z.shape
    x = z.double() / T
    used = (idx >= 0) & (idx < V)
    col = torch.where(used, idx, 0).long()
    low = torch.full((n, 1), -math.inf, dtype=torch.float64)
    events = torch.cat([torch.where(used, t.double() / T, -math.inf), low if tail is None else tail.double()[:, None]], 1)
    live = (events > -math.inf).any(1, keepdim=True)
    logp = torch.log_softmax(torch.where(live, events, 0.0), 1)
    p = torch.where(live, logp.exp(), 0.0)
    named = torch.zeros(n, V, dtype=torch.float64).scatter_add_(1, col, used.double()) > 0
    p_col = torch.zeros(n, V, dtype=torch.float64).scatter_add_(1, col, torch.where(used, p[:, :-1], 0.0))
    q = torch.softmax(x, 1)
    lse = torch.logsumexp(x, 1, keepdim=True)
    others = x.masked_fill(named, -math.inf)
    some = (others > -math.inf).any(1, keepdim=True)
    lse_rest = torch.where(some, torch.logsumexp(torch.where(some, others, 0.0), 1, keepdim=True), low)
    r = p[:, -1:]
    logq = torch.cat([torch.gather(x, 1, col) - lse, lse_rest - lse], 1)
    terms = torch.where(p > 0, p * (torch.where(p > 0, logp, 0.0) - torch.where(p > 0, logq, 0.0)), 0.0)
    share = torch.where(some, (others - torch.where(some, lse_rest, 0.0)).exp(), 0.0)
    dz = torch.where(named, q - p_col, q - r * share) / T
    dz = torch.where(live, dz, 0.0)
    # a sum of exponentials: V / 256 terms a thread, arguments' rounding under 128 u, 4 u an exponential, merges
    lost = (V / 256 + 256) * U
    loss_bound = 4 * lost + 16 * U * terms.abs().sum(1)
    dz_bound = (4 * lost + 256 * U) * (q + r * share + p_col) / T
    return terms.sum(1), dz, loss_bound, torch.where(live, dz_bound, 0.0)


def _check_kl(z, idx, t, tail=None, T=1.0, scale=None):
    from param_decomp_b200.ops.top_logits import top_kl, top_kl_rows

    cpu = lambda a: None if a is None else a.cpu()  # noqa: E731
    loss, dz, lb, db = _kl_reference(cpu(z), cpu(idx), cpu(t), cpu(tail), T)
    got, grad = top_kl_rows(z, idx, t, tail, T)
    assert grad.shape == z.shape and grad.dtype == z.dtype and got.dtype == f32
    _within(got, loss, lb, "loss")
    _within(grad, dz, db, "dz")
    assert torch.equal(top_kl_rows(z, idx, t, tail, T, want_grad=False)[0], got)
    leaf = z.detach().requires_grad_(True)
    up = torch.rand(z.shape[0], generator=_gen(3)) + 0.5
    auto = top_kl(leaf, idx, t, tail, T)
    assert torch.equal(auto.detach(), got)
    (grad,) = torch.autograd.grad(auto, (leaf,), up.cuda())
    _within(grad, dz * up.double()[:, None], (db + 4 * U * dz.abs()) * up.double()[:, None], "dz")


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (2, 2, 1), (3, 7, 7), (4, 8, 3), (5, 9, 2), (6, 1000, 256), (900, 2003, 9), (5, 8195, 64),
                                   (310, 50277, 64), (3, 151936, 130), (40, 300001, 5)])
def test_top_kl_and_its_gradient(nv, n, V, K, kind):
    """Clusters of 1 to 8 blocks, several rows a cluster, rows at every address modulo 16, both index types."""
    g = _gen(n + V + K)
    z = (torch.randn(n, V, generator=g) * 2).to(kind)
    teacher = z.float() + torch.randn(n, V, generator=g)
    t, idx = torch.topk(teacher, K, dim=1)
    tail = torch.logsumexp(teacher.scatter(1, idx, -math.inf) / 2.0, 1)
    _check_kl(z.cuda(), idx.cuda(), t.to(kind).cuda(), None)
    if tail.isfinite().all():
        _check_kl(z.cuda(), idx.to(torch.int32).cuda(), t.cuda(), tail.cuda(), 2.0)
    wide = torch.full((n, V + 11), 77.0, dtype=kind)
    wide[:, 3:3 + V] = z
    _check_kl(wide.cuda()[:, 3:3 + V], idx.cuda(), t.cuda(), None)
    _done(nv)


@pytest.mark.parametrize("kind,n,V,K", [(bf, 2000, 50277, 3), (bf, 900, 120001, 40), (f32, 700, 60000, 200), (f32, 700, 151936, 1)])
def test_top_kl_backward_from_kept_sums(nv, kind, n, V, K):
    """Many rows a cluster of 1 to 8 blocks: the gradient that a backward forms from the sums that the forward kept is, bit for
    bit, that of one pass, and the losses too."""
    from param_decomp_b200.ops.top_logits import top_kl, top_kl_rows

    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(n, V, generator=g, device="cuda").to(kind)
    idx = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t, tail = torch.randn(n, K, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda") + 8.0
    loss, dz = top_kl_rows(z, idx, t, tail, 2.0)
    leaf = z.requires_grad_(True)
    auto = top_kl(leaf, idx, t, tail, 2.0)
    (grad,) = torch.autograd.grad(auto, (leaf,), torch.ones(n, device="cuda"))
    _done(nv)
    assert torch.equal(auto.detach(), loss) and torch.equal(grad, dz)


@pytest.mark.parametrize("kind,V", [(bf, 470001), (bf, 884720), (f32, 225001), (f32, 442352)])
def test_top_kl_of_the_longest_rows(nv, kind, V):
    g = _gen(V)
    z = (torch.randn(2, V, generator=g) * 2).to(kind)
    teacher = z.float() + torch.randn(2, V, generator=g)
    t, idx = torch.topk(teacher, 17, dim=1)
    tail = torch.logsumexp(teacher.scatter(1, idx, -math.inf), 1)
    _check_kl(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("V", [1003, 50277, 200003])
def test_top_kl_of_awkward_rows(nv, V, kind):
    """Unused slots (with NaN in them), a column named several times, rows without any slot or any mass, masked student
    logits (-inf and the type's lowest) beside and under the named ones, a rest far below the named logits and the other
    way round, a teacher of one certain column."""
    g = _gen(V)
    n, K = 12, 6
    z = torch.randn(n, V, generator=g) * 2
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    t = torch.randn(n, K, generator=g)
    tail = torch.randn(n, generator=g)
    idx[0, 2:4], t[0, 2:4] = -1, float("nan")
    idx[1, 1] = idx[1, 4] = idx[1, 5] = idx[1, 0]
    idx[2, 3] = idx[2, 2]
    idx[3], tail[3] = -1, -math.inf
    t[4], tail[4] = -math.inf, -math.inf
    idx[5] = -1
    keep = z[6, idx[6]].clone()
    z[6] = -math.inf
    z[6, idx[6]] = keep
    z[6, (int(idx[6, 0]) + 1) % V] = 0.5
    z[7, 100:] = torch.finfo(kind).min
    z[7, idx[7]] = 0.25
    z[8] -= 150.0
    z[8, idx[8]] = 3.0
    z[9, idx[9]] = -100.0
    t[10, 1:], tail[10] = -math.inf, -math.inf
    z[11] = torch.finfo(kind).min
    z[11, 5::3] = 1.0
    z[11, idx[11]] = 2.0
    z, t = z.to(kind), t.to(kind)
    _check_kl(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    some = [i for i in range(n) if i != 5]
    _check_kl(z[some].cuda(), idx[some].cuda(), t[some].cuda(), None, 3.0)
    _done(nv)


def test_top_kl_where_the_loss_is_infinite(nv):
    """A named column that the student has masked, or a rest that it has masked while the teacher has a tail: the loss is
    infinite, the gradient is not, and the rows beside it are as without it."""
    from param_decomp_b200.ops.top_logits import top_kl_rows

    g = _gen(4)
    z = torch.randn(3, 2000, generator=g)
    idx, t, tail = torch.tensor([[4, 9], [4, 9], [4, 9]]), torch.randn(3, 2, generator=g), torch.zeros(3)
    base = top_kl_rows(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    z[0, 4] = -math.inf
    z[2] = -math.inf
    z[2, 4:10] = 1.0
    z[2, 5:9] = -math.inf
    loss, dz = top_kl_rows(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    assert loss[0].item() == math.inf and loss[2].item() == math.inf and bool(dz.isfinite().all())
    assert torch.equal(loss[1], base[0][1]) and torch.equal(dz[1], base[1][1])
    p = torch.softmax(torch.cat([t, tail[:, None]], 1), 1)
    assert abs(float(dz[0, 4]) + float(p[0, 0])) < 1e-6 and abs(float(dz[2, 9]) - (0.5 - float(p[2, 1]))) < 1e-6
    assert abs(float(dz[0].double().sum())) < 2000 * U * 4  # a softmax's gradient sums to nothing
    _done(nv)


def test_top_kl_refused_columns_and_empty_batches(nv):
    from param_decomp_b200.ops.top_logits import next_token_loss, top_kl, top_kl_rows

    g = _gen(8)
    z, t = torch.randn(5, 600, generator=g).cuda(), torch.randn(5, 3, generator=g).cuda()
    idx = torch.randint(0, 600, (5, 3), generator=g).cuda()
    bad, unused = idx.clone(), idx.clone()
    bad[1, 2], bad[3, 0], unused[1, 2], unused[3, 0] = 600, 2**40, -1, -1
    want = top_kl_rows(z, unused, t)
    got = top_kl_rows(z, bad, t)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    torch.cuda.synchronize()
    with pytest.raises(nv.NativeError, match="column"):
        top_kl(z, idx, t)
    top_kl(z, idx, t)
    loss, dz = top_kl_rows(z[:0], idx[:0], t[:0])
    assert loss.shape == (0,) and dz.shape == (0, 600)
    # the mean over the positions that have a target, and its gradient
    targets = torch.tensor([[3, -1, 599], [-1, 0, 3]])
    logits = torch.randn(2, 3, 600, generator=g)
    leaf = logits.cuda().requires_grad_(True)
    ce = next_token_loss(leaf, targets.cuda())
    (grad,) = torch.autograd.grad(ce, (leaf,))
    ref = logits.double().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(ref.view(-1, 600), targets.view(-1), ignore_index=-1)
    (want_grad,) = torch.autograd.grad(want, (ref,))
    assert abs(float(ce) - float(want)) < 600 * U * 8
    assert float((grad.cpu().double() - want_grad).abs().max()) < 600 * U
    _done(nv)


def test_top_kl_of_top_logits_is_the_whole_divergence(nv):
    """The two together: at k one short of the row and at the whole row the loss is the divergence over all columns, between
    it grows with k; and the gradient is that of differences."""
    from param_decomp_b200.ops.top_logits import top_kl, top_logits

    g = _gen(11)
    teacher, z = torch.randn(6, 200, generator=g), torch.randn(6, 200, generator=g)
    p = torch.log_softmax(teacher.double(), 1)
    whole = (p.exp() * (p - torch.log_softmax(z.double(), 1))).sum(1)
    before = torch.zeros(6)
    for k in (1, 10, 100, 199, 200):
        loss = top_kl(z.cuda(), top_logits(teacher.cuda(), k).indices, top_logits(teacher.cuda(), k).values,
                      top_logits(teacher.cuda(), k).tail).cpu()
        assert bool((loss >= before - 1e-6).all())
        before = loss
        if k >= 199:
            assert float((loss.double() - whole).abs().max()) < 600 * U
    leaf = z.cuda().requires_grad_(True)
    top = top_logits(teacher.cuda(), 10)
    (grad,) = torch.autograd.grad(top_kl(leaf, top.indices, top.values, top.tail).sum(), (leaf,))
    way = torch.randn(6, 200, generator=g, dtype=torch.float64)
    h = 1e-5
    args = (top.indices.cpu(), top.values.cpu(), top.tail.cpu(), 1.0)
    slope = sum(s * _kl_reference(z.double() + s * h * way, *args)[0].sum() for s in (1, -1)) / (2 * h)
    assert abs(float((grad.cpu().double() * way).sum() - slope)) < 1e-5


# ---- a run of them together ---------------------------------------------------------------------------------------------


def test_output_edge_of_top_logits_on_the_fused_backend(nv):
    """Clean top logits and the masked side's loss as a decomposition step takes them, over several chunks of positions: the
    loss and the hidden state's gradient against 64 bits, and against the whole vocabulary's where k is all but one of it."""
    from param_decomp_b200.ops import vocab_kl

    g = _gen(21)
    n, d, V, k = 700, 128, 1003, 64
    head = (torch.randn(V, d, generator=g) / d**0.5).to(bf).cuda()
    hc = torch.randn(n, d, generator=g).to(bf).cuda()
    hm = (hc.float().cpu() + 0.3 * torch.randn(n, d, generator=g)).to(bf).cuda()
    top = vocab_kl.top_logits_from_hidden(hc, head, k, 256)
    leaf = hm.clone().requires_grad_(True)
    loss = vocab_kl.top_kl_from_hidden(top, leaf, head, 256)
    (grad,) = torch.autograd.grad(loss * 3.0, (leaf,))
    _done(nv)
    # the same from the logits that the kernels saw, which were rounded to bf16
    lc, lm = vocab_kl.padded_logits(hc, head), vocab_kl.padded_logits(hm, head)
    want = _top_reference(lc.cpu(), k, 1.0)
    assert torch.equal(top.indices.cpu(), want[1]) and torch.equal(top.values.cpu(), want[0])
    rows, dz, bound, _ = _kl_reference(lm.cpu(), want[1], want[0], want[2].float(), 1.0)
    assert abs(float(loss) - float(rows.mean())) <= float(bound.mean()) + (n + 8) * U * float(rows.abs().mean())
    dh = 3.0 / n * dz @ head.cpu().double()
    # dz and dh are rounded to bf16 (2^-8 of each), and 3 dh again; the sums of the product in fp32
    size = 3.0 / n * dz.abs() @ head.cpu().double().abs()
    assert bool(((grad.cpu().double() - dh).abs() <= (2.0**-8 * 1.01 + V * U) * size + 2.01 * 2.0**-8 * dh.abs()).all())


def test_pretraining_step_on_native_kernels(nv, tmp_path):
    """The pretrainer's model with `kernels: native` against library ops: loss and every weight's gradient of one batch, for
    the model that has all of them (learned positions, LayerNorm, tied head); then the command's loop, to its snapshot."""
    from param_decomp_b200.models import transformer as tf
    from param_decomp_b200.ops.top_logits import next_token_loss
    from param_decomp_b200.pretrain.train import PretrainConfig, pretrain

    cfg = PretrainConfig.model_validate(dict(
        run_name="t", seed=1, dtype="float32", global_batch=4, num_iterations=3, learning_rate=1e-3, kernels="native", log_every=1,
        val_every=3, val_steps=1, save_every=3, model=dict(model_type="GPT2Simple", vocab_size=211, n_layer=2, n_head=2, n_embd=48, n_ctx=16)))
    arch = cfg.model.arch()
    w = tf.random_init_weights(arch, 0, f32)
    g = _gen(5)
    w = {k: (v + 0.1 * torch.randn(v.shape, generator=g) if "norm" in k else v).cuda().requires_grad_(True) for k, v in w.items()}
    toks = torch.randint(0, 211, (4, 17), generator=g).cuda()
    results = []
    for native in (False, True):
        model = tf.TransformerDecomposedModel(arch, w, {}, attention="xla", train_kernels=native)
        logits = model.logits(model._run(tf.LMBatch(toks[:, :-1]), None, None, (), want_taps=False).output)
        loss = (next_token_loss(logits, toks[:, 1:]) if native
                else torch.nn.functional.cross_entropy(logits.reshape(-1, 211), toks[:, 1:].reshape(-1)))
        results.append((loss.detach(), torch.autograd.grad(loss, list(w.values()))))
    _done(nv)
    assert abs(float(results[0][0]) - float(results[1][0])) < 1e-5
    for name, a, b in zip(w, results[0][1], results[1][1]):
        # fp32 on both sides; library products may be taken in another order
        assert float((a - b).norm()) <= 1e-4 * float(a.norm()) + 1e-7, name
    entry = pretrain(cfg, tmp_path, run_id="t-00000007", device="cuda:0")
    _done(nv)
    assert "\"val_loss\"" in (entry / "metrics.jsonl").read_text() and list(entry.glob("model_step_3.safetensors"))


def test_two_decomposition_steps_with_the_top_logits_edge(nv, tmp_path):
    """Through the engine on the fused backend, step by step and recorded into a graph: the edge's kernels are captured."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).parent))
    from test_lm_ends_cpu import _lm_config

    from param_decomp_b200.config.experiments import LMExperimentConfig
    from param_decomp_b200.experiments.lm.training import train_lm

    losses = []
    for recording in ("off", "cuda_graph"):
        c = _lm_config({"kind": "top_logits", "k": 32}, "fused_sm100", "bfloat16")
        c["runtime"]["step_recording"] = recording
        c["pd"]["steps"] = 6
        c["cadence"] = {"train_log_every": 1, "checkpointing": {"kind": "none"}}
        c["eval"] = None
        res = train_lm(LMExperimentConfig.model_validate(c), tmp_path, run_id=f"p-0000ee0{len(losses)}", device="cuda:0")
        _done(nv)
        assert res.final_step == 6 and math.isfinite(res.last_metrics["train/loss/total"])
        losses.append(res.last_metrics["train/loss/total"])
    assert abs(losses[0] - losses[1]) < 0.05 * abs(losses[0])


def test_graphs_and_streams(nv):
    """Forward and backward of all four captured into two graphs that are replayed in turn with new contents, and run on two
    streams at once: each result as without."""
    from param_decomp_b200.ops.elementwise import layer_norm
    from param_decomp_b200.ops.embedding import embedding
    from param_decomp_b200.ops.top_logits import top_kl, top_logits

    def inputs(seed):
        g = _gen(seed)
        return dict(tokens=torch.randint(0, 300, (900,), generator=g).cuda(), table=torch.randn(300, 64, generator=g).cuda(),
                    w=torch.randn(64, generator=g).cuda(), b=torch.randn(64, generator=g).cuda(),
                    head=torch.randn(64, 5003, generator=g).cuda(), teacher=torch.randn(900, 5003, generator=g).cuda())

    def work(s):
        leaves = [s[k].detach().requires_grad_(True) for k in ("table", "w", "b")]
        h = layer_norm(embedding(s["tokens"], leaves[0], 8.0), leaves[1], leaves[2], 1e-5)
        top = top_logits(s["teacher"], 20)
        loss = top_kl(h @ s["head"], top.indices, top.values, top.tail)
        return [loss.detach(), *torch.autograd.grad(loss.sum(), leaves)]

    sets = [inputs(i) for i in range(4)]
    want = [[t.clone() for t in work(s)] for s in sets]
    _done(nv)
    held = [{k: v.clone() for k, v in sets[0].items()} for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in held:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(work(s))
        graphs.append(graph)
    for first, second in ((1, 2), (3, 1)):
        for s, i in zip(held, (first, second)):
            for k in s:
                s[k].copy_(sets[i][k])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, i in zip(outs, (first, second)):
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got: list = [None, None]
    for _ in range(5):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[j] = work(sets[j + 1])
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[j], want[j + 1]))
    _done(nv)


def _differentiable():
    """(name, leaves, function of the leaves) of every operator with a gradient."""
    from param_decomp_b200.ops.elementwise import layer_norm
    from param_decomp_b200.ops.embedding import embedding
    from param_decomp_b200.ops.top_logits import top_kl

    g = _gen(6)
    leaf = lambda *shape: torch.randn(*shape, generator=g).cuda().requires_grad_(True)  # noqa: E731
    tokens, idx, t = (torch.randint(0, 50, (40,), generator=g).cuda(), torch.randint(0, 50, (7, 3), generator=g).cuda(),
                      torch.randn(7, 3, generator=g).cuda())
    return [("layer_norm", (leaf(5, 24), leaf(24), leaf(24)), lambda x, w, b: layer_norm(x, w, b, 1e-5)),
            ("embedding", (leaf(50, 8),), lambda table: embedding(tokens, table, 2.0)),
            ("top_kl", (leaf(7, 50),), lambda z: top_kl(z, idx, t))]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_backwards(nv, which):
    """A kept graph gives the same gradients again, a freed one raises, and a gradient that is differentiated again raises
    (alone or beside a path that is differentiable twice) where it would otherwise count as a constant."""
    name, leaves, f = _differentiable()[which]
    y = f(*leaves)
    up = torch.rand(y.shape, generator=_gen(1)).cuda()
    first = torch.autograd.grad(y, leaves, up, retain_graph=True)
    again = torch.autograd.grad(y, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(y, leaves, up)
    y = f(*leaves)
    mixed = (y * y.detach()).sum() + sum((p ** 3).sum() for p in leaves)
    grads = torch.autograd.grad(mixed, leaves, create_graph=True)
    with pytest.raises(RuntimeError, match=f"{name} is not differentiable twice"):
        torch.autograd.grad(sum(g.sum() for g in grads), leaves)
    _done(nv)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_some_gradients_and_accumulated_ones(nv, which):
    """Each leaf's gradient asked for alone; `.grad` added up over two backwards; gradients that come broadcast."""
    _, leaves, f = _differentiable()[which]
    y = f(*leaves)
    whole = torch.autograd.grad(y.sum(), leaves)
    for i, leaf in enumerate(leaves):
        (alone,) = torch.autograd.grad(f(*(p if j == i else p.detach() for j, p in enumerate(leaves))).sum(), (leaf,))
        assert torch.equal(alone, whole[i])
    for _ in range(2):
        f(*leaves).sum().backward()
    assert all(torch.equal(p.grad, 2 * g) for p, g in zip(leaves, whole))
    with torch.no_grad():
        assert not f(*leaves).requires_grad and torch.equal(f(*leaves), y)
    _done(nv)


def test_values_changed_between_the_passes_are_noticed(nv):
    """What a backward reads must be what its forward read."""
    for _, leaves, f in _differentiable()[::2]:
        x = leaves[0] * 1.0
        y = f(x, *leaves[1:])
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("V,d,n", [(700, 1, 60), (5000, 2, 40), (1201, 3, 900), (900, 5, 1), (40000, 7, 300), (2000, 9, 0), (3001, 515, 77),
                                   (600, 8, 500), (160000, 24, 1000)])
def test_every_row_of_an_embedding_gradient_is_written(nv, V, d, n, kind):
    """Rows at every alignment between rows of zeros: whole numbers, so the sums are exact; memory held other values before."""
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(V + d)
    tokens, dy = torch.randint(0, V, (n,), generator=g), torch.randint(-2, 3, (n, d), generator=g).float()
    want = torch.zeros(V, d).index_add_(0, tokens, dy)
    table = torch.zeros(V, d, dtype=kind).cuda().requires_grad_(True)
    for _ in range(2):
        (grad,) = torch.autograd.grad(embedding(tokens.cuda(), table), (table,), dy.to(kind).cuda())
        assert torch.equal(grad.float().cpu(), want)
        grad.fill_(5.0)
        del grad
    _done(nv)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_is_refused(nv, which):
    import torch.autograd.forward_ad as fwd

    _, leaves, f = _differentiable()[which]
    with fwd.dual_level():
        dual = fwd.make_dual(leaves[0].detach(), torch.ones_like(leaves[0]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(dual, *leaves[1:])
    _done(nv)


@pytest.mark.parametrize("kind,V", [(f32, 60000), (bf, 151936), (f32, 300007)])
def test_clusters_on_two_streams_at_once(nv, kind, V):
    """Rows spread over 4 and 8 blocks, two calls of each kernel at a time: each result as alone."""
    from param_decomp_b200.ops.top_logits import top_kl, top_logits

    def work(z, idx, t):
        leaf = z.detach().requires_grad_(True)
        loss = top_kl(leaf, idx, t, None, 1.5)
        return [*top_logits(z, 50), loss.detach(), *torch.autograd.grad(loss.sum(), (leaf,))]

    sets = []
    for i in range(2):
        g = torch.Generator(device="cuda").manual_seed(i)
        sets.append((torch.randn(90, V, generator=g, device="cuda").to(kind),
                     torch.randint(0, V, (90, 33), generator=g, device="cuda"), torch.randn(90, 33, generator=g, device="cuda")))
    want = [work(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(work(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    _done(nv)


@pytest.mark.parametrize("V,n,d", [(50277, 20000, 64), (2000, 3000, 33), (400000, 5000, 16), (149, 700, 8), (148, 40, 24)])
def test_embedding_gradient_of_ids_in_order_of_frequency(nv, V, n, d):
    """Low ids hold most of the tokens, up to thousands each: whole numbers, so the sums are exact."""
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(V)
    tokens = (V ** torch.rand(n, generator=g, dtype=torch.float64)).long() - 1
    dy = torch.randint(-2, 3, (n, d), generator=g).float()
    want = torch.zeros(V, d).index_add_(0, tokens, dy)
    table = torch.zeros(V, d).cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(embedding(tokens.cuda(), table), (table,), dy.cuda())
    assert torch.equal(grad.cpu(), want)
    _done(nv)


@pytest.mark.parametrize("kind,V,k", [(bf, 120001, 40), (f32, 60000, 7), (f32, 151936, 64), (bf, 400001, 20)])
def test_top_logits_of_the_last_rows_of_a_cluster(nv, kind, V, k):
    """Clusters of 2 to 8 blocks that have one to a few rows each, some of them rows that the readers pass over at once and the
    selection takes long for: the last two rows of every cluster are handed over as all others are."""
    from param_decomp_b200.ops.top_logits import top_logits

    g = _gen(k)
    z = torch.randn(161, V, generator=g)
    z[1::5] = -math.inf
    z[1::5, 3:3 + 2 * k:2] = 1.0
    z = z.to(kind)
    want = _top_reference(z, k, 1.0)
    z = z.cuda()
    for n in (2, 19, 37, 75, 76, 110, 149, 161):
        first = top_logits(z[:n], k)
        assert torch.equal(first.indices.cpu(), want[1][:n]) and torch.equal(first.values.cpu(), want[0][:n])
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(first, top_logits(z[:n], k)))
    _done(nv)


@pytest.mark.parametrize("n,V", [(1, 1003), (257, 1003), (513, 2001), (2, 50277), (1, 50277)])
def test_output_edge_with_a_chunk_of_one_position(nv, n, V):
    """The last chunk has one row, of a width that is no whole number of 16 bytes: loss and gradient as in one chunk, whose
    products add up in the same order for every row; and the gradient's rows lie like the logits'."""
    from param_decomp_b200.ops import vocab_kl
    from param_decomp_b200.ops.top_logits import top_kl_rows

    g = _gen(n + V)
    d, k, rows = 128, 16, 256 if n > 2 else 1
    head = (torch.randn(V, d, generator=g) / d**0.5).to(bf).cuda()
    hc, hm = (torch.randn(n, d, generator=g).to(bf).cuda() for _ in range(2))
    results = []
    for chunk in (rows, 1024):
        top = vocab_kl.top_logits_from_hidden(hc, head, k, chunk)
        leaf = hm.clone().requires_grad_(True)
        loss = vocab_kl.top_kl_from_hidden(top, leaf, head, chunk)
        results.append((loss.detach(), torch.autograd.grad(loss, (leaf,))[0]))
    _done(nv)
    lm = vocab_kl.padded_logits(hm, head)
    # the two sums of n losses are in another order
    assert abs(float(results[0][0]) - float(results[1][0])) <= 2 * (n + 2) * U * float(results[1][0].abs())
    loss, dz = top_kl_rows(lm[n - 1:], top.indices[n - 1:], top.values[n - 1:], top.tail[n - 1:])
    assert dz.stride(0) % 8 == lm.stride(0) % 8 == 0
    want = dz.double().cpu() @ head.double().cpu() / n
    size = dz.double().abs().cpu() @ head.double().abs().cpu() / n
    for _, grad in results:  # sums of V products in fp32, rounded to bf16 once as the product is stored, once times the upstream 1
        off = (grad[n - 1].double().cpu() - want[0]).abs()
        assert bool((off <= V * U * size[0] + 1.01 * 2.0**-8 * want[0].abs()).all())


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("V", [1, 7, 1001, 2001, 50277, 300001])
def test_top_kl_of_rows_with_nan(nv, V, kind):
    """One NaN among a row's logits (named, not named, the last column, beside nothing but -inf) makes the row's loss and all of
    its gradient NaN, in every form, and no other row's."""
    from param_decomp_b200.ops.top_logits import top_kl, top_kl_rows

    g = _gen(V)
    n, K, nan = 8, min(3, V), float("nan")
    z = torch.randn(n, V, generator=g).to(kind)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    idx[1, 0] = 0
    t, tail = torch.randn(n, K, generator=g), torch.randn(n, generator=g)
    bad = z.clone()
    bad[1, 0] = nan  # named
    bad[3, V - 1] = nan
    bad[4] = -math.inf
    bad[4, V // 2] = nan
    bad[5] = -math.inf
    bad[5, V - 1] = nan
    bad[6] = torch.finfo(kind).min
    bad[6, V // 3] = nan
    rows, rest = [1, 3, 4, 5, 6], [0, 2, 7]
    at_odd = lambda a: torch.nn.functional.pad(a, (1, 2), value=9.0).cuda()[:, 1:V + 1]  # noqa: E731
    for x, clean in ((bad.cuda(), z.cuda()), (at_odd(bad), at_odd(z))):  # addresses decide the order of sums
        for tails in (tail.cuda(), None):
            want, dz = top_kl_rows(clean, idx.cuda(), t.cuda(), tails)
            loss, grad = top_kl_rows(x, idx.cuda(), t.cuda(), tails)
            leaf = x.detach().requires_grad_(True)
            auto = top_kl(leaf, idx.cuda(), t.cuda(), tails)
            (auto_grad,) = torch.autograd.grad(auto.sum(), (leaf,))
            for got, got_grad in ((loss, grad), (auto.detach(), auto_grad)):
                assert bool(got[rows].isnan().all()) and bool(got_grad[rows].isnan().all())
                assert torch.equal(got[rest], want[rest]) and torch.equal(got_grad[rest], dz[rest])
                assert not bool(got[rest].isnan().any()) and not bool(got_grad[rest].isnan().any())
            assert bool(top_kl_rows(x, idx.cuda(), t.cuda(), tails, want_grad=False)[0][rows].isnan().all())
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("V", [1003, 50277, 120001])
def test_top_kl_of_logits_far_from_zero(nv, V, kind):
    """A large offset common to a row, or a small temperature, on either side: many logits share the largest values (two bf16
    numbers that differ are hundreds apart there), and each one's gradient is as exact as around zero."""
    from param_decomp_b200.ops.top_logits import top_kl, top_kl_rows

    g = _gen(V)
    n, K = 8, 5
    z = torch.randint(-2, 1, (n, V), generator=g) * 1024.0
    z += torch.tensor([99840.0, -99840.0, 45056.0, 300032.0, 0.0, -3e6, 6000.0, 500.0])[:, None]
    z = z.to(kind)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    t, tail = torch.randn(n, K, generator=g), torch.randn(n, generator=g)
    small = (torch.randint(-8, 1, (n, V), generator=g) * 0.25 + 45.0).to(kind)
    for x, tails, T in ((z, tail, 1.0), (z, None, 1.0), (small, tail, 0.001), (-small, None, 0.01)):
        loss, dz, lb, db = _kl_reference(x, idx, t, tails, T)
        # an exponential below 2^-126 is zero; a gradient is at most 1 / T times its row's exponentials
        db = db + 2.0**-126 / T
        tails = None if tails is None else tails.cuda()
        got, grad = top_kl_rows(x.cuda(), idx.cuda(), t.cuda(), tails, T)
        _within(got, loss, lb, "loss")
        _within(grad, dz, db, "dz")
        leaf = x.cuda().requires_grad_(True)
        _within(torch.autograd.grad(top_kl(leaf, idx.cuda(), t.cuda(), tails, T).sum(), (leaf,))[0], dz, db, "dz")
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("K,T", [(3, 0.7), (40, 0.001), (130, 0.5), (5, 2.0**-120), (5, 2.0**120)])
def test_top_kl_of_a_teacher_past_the_range_of_fp32(nv, K, T, kind):
    """A teacher's logits over the temperature leave fp32 on either side (all of them masked with the type's lowest value, among
    others): the row counts like any other, with the same probabilities as around zero."""
    from param_decomp_b200.ops.top_logits import top_kl_rows

    g = _gen(K)
    n, V = 7, 1003
    most = torch.finfo(kind).max
    z = (torch.randn(n, V, generator=g) * min(T, 1.0)).to(kind)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    t = torch.randn(n, K, generator=g)
    t[1], t[2] = -most, most
    t[3], t[3, 1:] = most, -most
    t[4, 1:], t[5] = -most, most / 2
    t[5, 0] = most
    t, tail = t.to(kind), torch.randn(n, generator=g)
    tail[1], tail[2] = -math.inf, -math.inf
    for tails in (None, tail):
        loss, dz, lb, db = _kl_reference(z, idx, t, tails, T)
        got, grad = top_kl_rows(z.cuda(), idx.cuda(), t.cuda(), None if tails is None else tails.cuda(), T)
        # what the reference's own 64 bits lose of a log probability of 1e38 and more beside one of zero is nothing here
        fine = loss.isfinite() & (loss.abs() < 1e30)
        assert bool(fine[1:3].all()) and bool(fine.any())
        _within(got[fine.cuda()], loss[fine], lb[fine], "loss")
        # an exponential below 2^-126, or a gradient, may be zero
        _within(grad, dz, db + 2.0**-126 * (1.0 + 1.0 / T), "dz")
    _done(nv)


def test_top_kl_of_a_teacher_with_nan(nv):
    """A NaN in a used slot or in the tail makes the row's loss and all of its gradient NaN, one in an unused slot nothing."""
    from param_decomp_b200.ops.top_logits import top_kl_rows

    g = _gen(12)
    z, t, tail = torch.randn(5, 600, generator=g), torch.randn(5, 3, generator=g), torch.randn(5, generator=g)
    idx = torch.stack([torch.randperm(600, generator=g)[:3] for _ in range(5)])
    idx[3, 1] = -1
    want, dz = top_kl_rows(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    t[1, 2], t[3, 1], t[4], tail[2], tail[4] = float("nan"), float("nan"), -math.inf, float("nan"), float("nan")
    loss, grad = top_kl_rows(z.cuda(), idx.cuda(), t.cuda(), tail.cuda())
    assert bool(loss[[1, 2, 4]].isnan().all()) and bool(grad[[1, 2, 4]].isnan().all())
    assert torch.equal(loss[[0, 3]], want[[0, 3]]) and torch.equal(grad[[0, 3]], dz[[0, 3]])
    _done(nv)


@pytest.mark.parametrize("n", [700, 257, 1])
def test_evaluated_divergence_with_the_top_logits_edge_on_the_fused_backend(nv, n):
    """The divergence over the whole vocabulary, in chunks, is that of the materialised edge; the edge's loss is not above it."""
    from types import SimpleNamespace

    from param_decomp_b200.config.experiments import TransformerArchConfig
    from param_decomp_b200.models import transformer as tf

    arch = TransformerArchConfig(family="glu_transformer", n_layer=1, d_model=128, n_head=2, d_ff=128, vocab_size=1003, max_seq_len=n)
    w = {k: v.to(bf).cuda() for k, v in tf.random_init_weights(arch, 0, f32).items()}
    g = _gen(n)
    hc, hm = ((torch.randn(1, n, 128, generator=g) * 4).to(bf).cuda() for _ in range(2))
    values = []
    for n_top in (None, 16):
        model = tf.TransformerDecomposedModel(arch, w, {}, backend="fused_sm100", n_top_logits=n_top, kl_token_chunk=256)
        clean, masked = SimpleNamespace(output=hc, aux={"clean_stats": model._clean_logit_stats(hc)}), SimpleNamespace(output=hm)
        with torch.no_grad():
            values.append((float(model.output_kl(clean, masked)), float(model.recon_loss(clean, masked))))
    _done(nv)
    assert values[0][0] == values[0][1]
    # the same rows' values, added in another order
    assert abs(values[1][0] - values[0][0]) <= 2 * (n + 2) * U * values[0][0]
    assert 0 < values[1][1] <= values[1][0]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_hooks_on_the_nodes(nv, which):
    """Tensors saved on the host, or given back in another layout; recomputation of a checkpoint; hooks that see and change
    gradients: each with the gradients that the formula gives."""
    from torch.utils.checkpoint import checkpoint

    _, leaves, f = _differentiable()[which]
    up = torch.rand(f(*leaves).shape, generator=_gen(2)).cuda()
    want = torch.autograd.grad(f(*leaves), leaves, up)
    turned = lambda t: t if t.dim() < 2 else t.t().contiguous().t()  # noqa: E731  (the same values by columns)
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned)):
        with hooks:
            y = f(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, up), want))
    y = checkpoint(f, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, up), want))
    seen = []
    y = f(*leaves)
    y.register_hook(lambda g: 2.0 * g)
    mids = [p * 1.0 for p in leaves]
    z = f(*mids)
    for m in mids:
        m.register_hook(lambda g: seen.append(g.clone()))
    assert all(torch.equal(a, 2.0 * b) for a, b in zip(torch.autograd.grad(y, leaves, up), want))
    grads = torch.autograd.grad(z, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    assert len(seen) == len(leaves) and all(any(torch.equal(a, b) for a in seen if a.shape == b.shape) for b in want)
    with torch.autograd.detect_anomaly():
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(f(*leaves), leaves, up), want))
    _done(nv)


@pytest.mark.parametrize("table_type,out_type", [(bf, bf), (f32, f32), (f32, bf)])
@pytest.mark.parametrize("n,V,d", [(30000, 1, 24), (30000, 3, 33), (70000, 100, 40), (40000, 300, 264), (200000, 450, 8), (25000, 700, 515),
                                   (50000, 189441, 16)])
def test_embedding_gradient_of_blocks_with_many_tokens(nv, n, V, d, table_type, out_type):
    """More tokens of one block's ids than it sorts on chip (4096), more in a warp's part than it notes (128), beside ids of the
    same block with one token, a few and a slab's worth of them: against whole numbers, whose sums are exact."""
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(n + V)
    blocks = -(-V // -(-V // max(148, -(-V // 1280))))  # ids v, v + blocks, .. belong to block v % blocks
    tokens = torch.zeros(n, dtype=torch.int64)
    tokens[torch.rand(n, generator=g) < 0.4] = min(1, V - 1)
    where = torch.randperm(n, generator=g)
    at = 0
    for first in (0, 1):  # the two full blocks: neighbours of their id with 1, 2, 31, 32, 33 and 100 tokens
        for i, count in enumerate((1, 2, 31, 32, 33, 100), start=1):
            if first + i * blocks < V:
                tokens[where[at:at + count]] = first + i * blocks
                at += count
    some = where[at:at + n // 8]
    tokens[some] = torch.randint(0, V, (len(some),), generator=g)
    assert int(torch.bincount(tokens % blocks).max()) > 4096
    dy = torch.randint(-2, 3, (n, d), generator=g).float()
    want = torch.zeros(V, d, dtype=torch.float64).index_add_(0, tokens, dy.double())
    table = torch.zeros(V, d, dtype=table_type).cuda().requires_grad_(True)
    for ids in (tokens, torch.sort(tokens)[0], torch.sort(tokens, descending=True)[0]):
        order = torch.sort(tokens, stable=True, descending=bool(ids[0] > ids[-1]))[1] if ids is not tokens else torch.arange(n)
        y = embedding(ids.cuda(), table, 1.0, out_dtype=out_type)
        (grad,) = torch.autograd.grad(y, (table,), dy[order].to(out_type).cuda())
        # sums of whole numbers below 2^24 are exact; the result is rounded once
        assert torch.equal(grad.cpu(), want.to(table_type))
    _done(nv)


def test_embedding_gradient_of_a_full_block_in_64_bits(nv):
    """The same paths with values that round: each row's sum to within the roundings of as many additions."""
    from param_decomp_b200.ops.embedding import embedding

    g = _gen(31)
    n, V, d = 30000, 500, 136
    tokens, dy = _zipf(n, V, g), torch.randn(n, d, generator=g)
    tokens[::3] = 7
    table = torch.zeros(V, d).cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(embedding(tokens.cuda(), table), (table,), dy.cuda())
    want = torch.zeros(V, d, dtype=torch.float64).index_add_(0, tokens, dy.double())
    sizes = torch.zeros(V, d, dtype=torch.float64).index_add_(0, tokens, dy.double().abs())
    _within(grad, want, (torch.bincount(tokens, minlength=V).double()[:, None] + 2) * U * sizes, "dE")
    _done(nv)


@pytest.mark.parametrize("kind", [bf, f32])
@pytest.mark.parametrize("rows,d", [(32771, 768), (70001, 256), (5003, 4096), (2003, 8192), (2005, 12288), (9001, 2048), (33003, 264),
                                    (20001, 500), (4001, 2047)])
def test_layer_norm_over_many_handfuls(nv, rows, d, kind):
    """Every group of warps walks more handfuls of rows than shared memory holds at a time, up to about twenty (the last ragged): its
    places are filled anew, the weights' sums run on over all of them."""
    from param_decomp_b200.ops.elementwise import layer_norm

    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 2 + 1).to(kind)
    x[rows // 2:] *= 3.0  # rows differ: one that is read in another's place shows
    w, b = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(kind), torch.randn(d, generator=g, device="cuda").to(kind)
    dy = torch.randn(rows, d, generator=g, device="cuda").to(kind)
    want, bounds = _norm_reference(x, w, b, dy, 1e-5)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    _done(nv)
    for name, got in zip(("y", "dx", "dw", "db"), (y, *grads)):
        _within(got, want[name], bounds[name], name)
    assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(layer_norm(*leaves, 1e-5), leaves, dy)))
    (alone,) = torch.autograd.grad(layer_norm(leaves[0], leaves[1].detach(), leaves[2].detach(), 1e-5), (leaves[0],), dy)
    assert torch.equal(alone, grads[0])


def test_hybrid_target_with_the_top_logits_edge_fused_against_eager(nv):
    """Gated delta rule, attention and routed experts through three steps with the edge, on both backends; and what evaluations
    call the divergence, with chunks."""
    from types import SimpleNamespace

    from param_decomp_b200.config.experiments import LMExperimentConfig
    from param_decomp_b200.core.objective import build_objective
    from param_decomp_b200.core.run import init_train_state
    from param_decomp_b200.core.train import StepContext, train_step
    from param_decomp_b200.experiments.lm.build import build_lm_run
    from param_decomp_b200.models import qwen35

    arch = dict(family="qwen35_moe", n_layer=2, d_model=64, n_head=4, n_kv_head=2, head_dim=64, d_ff=64, vocab_size=509,
                max_seq_len=64, n_experts=4, experts_per_token=2, full_attention_interval=2, partial_rotary_factor=0.5,
                linear_num_key_heads=2, linear_key_head_dim=64, linear_num_value_heads=4, linear_value_head_dim=64,
                linear_conv_kernel_dim=4, shared_expert_intermediate=64)
    raw = LMExperimentConfig.from_file("param_decomp_b200/experiments/configs/lm_moe4l_e42.yaml").model_dump(mode="json")
    raw["target"]["spec"]["arch"] = arch
    raw["target"]["output_edge"] = {"kind": "top_logits", "k": 32}
    raw["decomposition"]["sites"] = {"kind": "qwen36_moe", "layers": {"kind": "all"},
                                     "cs": {k: (128 if k.startswith("experts_") else 64) for k in qwen35.KIND_ORDER}}
    raw["decomposition"]["ci"] = {"type": "layerwise_mlp", "hidden_dims": [64]}
    raw["data"]["seq_len"] = 64
    raw["pd"]["batch_size"] = 4
    dev = torch.device("cuda", 0)
    res = {}
    for backend in ("eager_torch", "fused_sm100"):
        raw["runtime"]["backend"] = backend
        cfg = LMExperimentConfig.model_validate(raw)
        run = build_lm_run(cfg, None, dev)
        assert run.model.n_top_logits == 32
        run.model.kl_token_chunk = 255  # the last chunk has one position
        obj = build_objective(cfg.pd)
        fused = backend == "fused_sm100"
        ctx = StepContext.build(run.model, obj, cfg.pd, lazy_masks=fused)
        st = init_train_state(run.model, run.ci_fn, cfg.pd, obj, dev, cfg.pd.batch_size, cfg.data.seq_len, use_fused_optim=fused)
        for s in range(3):
            m = train_step(ctx, st, run.sample_train(s))
        with torch.no_grad():
            clean = run.model.clean_forward(run.sample_eval(0))
            whole = run.model.output_kl(clean, SimpleNamespace(output=clean.output * 0.5))
        _done(nv)
        res[backend] = {k: float(v) for k, v in m.items()} | {"kl": float(whole)}
    # bf16 weights and activations on both sides, through three updates: a few roundings of 2^-8 each
    for k in ("loss/total", "loss/FaithfulnessLoss", "loss/StochasticReconLoss", "loss/ImportanceMinimalityLoss", "kl"):
        a, b = res["eager_torch"][k], res["fused_sm100"][k]
        assert abs(a - b) <= 5e-2 * abs(a) + 1e-6, (k, a, b)


def test_a_first_call_that_is_captured(nv):
    """In a process whose first calls are captured into a graph: results as without, and replays leave alone what other kernels
    have reported."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from param_decomp_b200.ops import native
from param_decomp_b200.ops.elementwise import layer_norm
from param_decomp_b200.ops.embedding import embedding
from param_decomp_b200.ops.top_logits import top_kl, top_logits

g = torch.Generator(device="cuda").manual_seed(0)
tokens, table = torch.arange(100, device="cuda"), torch.randn(200, 600, device="cuda", generator=g, requires_grad=True)
w = torch.ones(600, device="cuda")

def work():
    logits = layer_norm(embedding(tokens, table), w, None, 1e-5)
    top = top_logits(logits.detach() * 1.5, 8)
    loss = top_kl(logits, top.indices, top.values, top.tail)
    return [loss.detach(), *torch.autograd.grad(loss.sum(), (table,))]

torch.cuda.synchronize()
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    out = work()
graph.replay()
torch.cuda.synchronize()
native.check_status()
assert all(torch.equal(a, b) for a, b in zip(out, work()))
embedding(tokens + 150, table)  # ids outside the table: reported
graph.replay()
torch.cuda.synchronize()
try:
    native.check_status()
    raise SystemExit("the report is lost")
except native.NativeError as e:
    assert "token" in str(e)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parents[1], capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stdout + done.stderr


def test_offsets_past_32_bits(nv):
    """More than 2^32 elements of rows, of a table and of logits: rows on both sides of 2^31 and 2^32 as alone."""
    from param_decomp_b200.ops.elementwise import layer_norm
    from param_decomp_b200.ops.embedding import embedding
    from param_decomp_b200.ops.top_logits import top_kl_rows, top_logits

    g = torch.Generator(device="cuda").manual_seed(0)
    rows, d = (1 << 22) + 5, 1040
    places = lambda n, d: (0, (1 << 31) // d - 3, (1 << 32) // d - 3, n - 7)  # noqa: E731
    x = torch.randn(rows, d, device="cuda", generator=g, dtype=bf).requires_grad_(True)
    w, b = torch.randn(d, device="cuda", generator=g), torch.randn(d, device="cuda", generator=g)
    y = layer_norm(x, w, b, 1e-5)
    (dx,) = torch.autograd.grad(y, (x,), x.detach())
    for s in places(rows, d):
        part = x.detach()[s:s + 7].clone().requires_grad_(True)
        alone = layer_norm(part, w, b, 1e-5)
        assert torch.equal(alone, y[s:s + 7]) and torch.equal(torch.autograd.grad(alone, (part,), part.detach())[0], dx[s:s + 7])
    del x, y, dx, part, alone
    V, d, n = (1 << 22) + 3, 1032, (1 << 22) + 9
    table = torch.randn(V, d, device="cuda", generator=g, dtype=bf).requires_grad_(True)
    tokens = torch.randint(0, V, (n,), device="cuda", generator=g)
    tokens[-100:], tokens[1000:1100] = V - 1, V - 2
    y = embedding(tokens, table)
    for s in places(n, d):
        assert torch.equal(y.detach()[s:s + 7], table.detach()[tokens[s:s + 7]])
    dy = torch.randint(-1, 2, (1, d), device="cuda", generator=g).to(bf)  # a row's gradient is its count times this, exactly
    (grad,) = torch.autograd.grad(y, (table,), dy.expand(n, d))
    counts = torch.bincount(tokens, minlength=V)
    for s in range(0, V, 1 << 18):
        assert torch.equal(grad[s:s + (1 << 18)].float(), counts[s:s + (1 << 18), None].float() * dy.float())
    del table, y, grad
    n, V = 90001, 50277
    z = torch.randn(n, V, device="cuda", generator=g, dtype=bf)
    top = top_logits(z, 64)
    loss, dz = top_kl_rows(z, top.indices, top.values * 0.5, top.tail)
    for s in places(n, V):
        s = s // 8 * 8  # rows at the same addresses modulo 16 bytes
        part = [t[s:s + 7] for t in (z, *top)]
        assert all(torch.equal(a, b) for a, b in zip(part[1:], top_logits(part[0], 64)))
        alone = top_kl_rows(part[0], part[2], part[1] * 0.5, part[3])
        assert torch.equal(alone[0], loss[s:s + 7]) and torch.equal(alone[1], dz[s:s + 7])
    far = z.view(-1).as_strided((3, 2000), (2_100_000_000, 1))  # by the pitch alone
    assert all(torch.equal(a, b) for a, b in zip(top_logits(far, 10), top_logits(far.contiguous(), 10)))
    _done(nv)
    del z, dz, far
    torch.cuda.empty_cache()
