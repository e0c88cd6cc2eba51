"""The head with its cross entropy (mindxsoup_amd/fused_ce.py on csrc/head_ce.hip) against its
definition in 64 bits.

Tolerances, u = 2^-24 and r half a step of the element type (fp16 2^-11, bf16 2^-8), both relative:
- a logit sums D products in fp32: e_z = D u max_v sum_d |h_d w_vd| per row;
- a loss: e_z twice (the label's and the sum's), the exponentials' and the logarithm's own (4 u
  |z|), and sums of at most 128 terms in a chain (128 u): e_l = 2 e_z + u (4 max |z| + 128);
- without the table's gradient fp16 exponentials keep 29 binades below a row's largest but the
  label's, p'; each smaller one is off by at most 2^-29 p';
- a weight p of dz is off by e_p = 2 e_l relative; dz is rounded twice on its way (2 r), and below
  fp16's normal range (times 2^14) by 2^-39; products sum in fp32 over n terms (n u), so a
  gradient is within (2 r + e_p + n u + 8 u) sum |dz| |other factor|, plus 2^-39 sum |other factor|,
  plus its own rounding r (2^-25 below fp16's normal range)."""

import pytest
import torch

from mindxsoup_amd import fused_ce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def _case(rows, vocab, cols, dtype, ignored=0, seed=0, spread=2.0):
    g = torch.Generator("cuda").manual_seed(seed)
    h = torch.randn(rows, cols, device="cuda", generator=g) * spread
    w = torch.randn(vocab, cols, device="cuda", generator=g) / cols ** 0.5
    y = torch.randint(vocab, (rows,), device="cuda", generator=g)
    gone = torch.randperm(rows, device="cuda", generator=g)[:ignored]
    h = h + torch.rand(rows, 1, device="cuda", generator=g) * 8 * w[y]  # some are predicted well
    y[gone] = -100
    return h.to(dtype), w.to(dtype), y


def _exact(h, w, y, reduction, g, ignore=-100):
    """Losses and gradients in 64 bits, and their bounds, in slices of the rows."""
    r, cols, vocab = R[h.dtype], h.shape[1], w.shape[0]
    rows = (y != ignore).nonzero()[:, 0]
    w64 = w.double()
    loss = torch.zeros(len(y), dtype=torch.float64, device=h.device)
    loss_tol = torch.zeros_like(loss)
    dh, dh_tol = torch.zeros_like(h, dtype=torch.float64), torch.zeros_like(h, dtype=torch.float64)
    dw, dw_tol = torch.zeros_like(w64), torch.zeros_like(w64)
    per = g if reduction == "none" else g / (max(1, len(rows)) if reduction == "mean" else 1)
    per = per.double().expand(len(y))
    big = per[rows].abs().max() if len(rows) else 0.0
    for some in rows.split(512):
        x = h[some].double()
        z = x @ w64.t()
        lse = z.logsumexp(1)
        at = torch.arange(len(some), device=h.device)
        loss[some] = lse - z[at, y[some]]
        e_l = 2 * cols * U * (x.abs() @ w64.abs().t()).amax(1) + U * (4 * z.abs().amax(1) + 128)
        loss_tol[some] = e_l
        dz = (z - lse[:, None]).exp()
        dz[at, y[some]] -= 1
        dz *= per[some][:, None]
        dh[some] = dz @ w64
        dw += dz.t() @ x
        e_p = 2 * e_l[:, None]
        p = (z - lse[:, None]).exp() * per[some].abs()[:, None]  # what carries e_p
        rel = 2 * r + (vocab + 8) * U
        small = 2.0 ** -39 * big
        other = p.clone()
        other[at, y[some]] = 0
        cut = 2.0 ** -29 * other.amax(1, keepdim=True) if h.dtype == F16 else 0.0
        dh_tol[some] = cut * w64.abs().sum(0) + rel * (dz.abs() @ w64.abs()) + e_p * (p @ w64.abs()) + \
            small * w64.abs().sum(0)
        rel = 2 * r + (len(rows) + 8) * U
        dw_tol += rel * (dz.abs().t() @ x.abs()) + (e_p * p).t() @ x.abs() + \
            small * x.abs().sum(0)
    low = 2.0 ** -25 if h.dtype == F16 else 0.0
    dh_tol += r * dh.abs() + low
    dw_tol += r * dw.abs() + low
    if reduction != "none":
        n = len(rows) if reduction == "mean" else 1
        loss_tol = loss_tol.sum() / n + 4 * U * loss.sum().abs() / n
        loss = loss.sum() / n
    return (loss, loss_tol), (dh, dh_tol), (dw, dw_tol)


def _within(got, want, what):
    value, tol = want
    off = (got.double() - value).abs()
    assert got.shape == value.shape
    assert bool((off <= tol).all()), \
        f"{what}: {float((off / tol.clamp_min(1e-300)).max()):.3g} of the bound"


def _check(h, w, y, reduction="mean", trained=True, scale=3.0, ignore=-100):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(trained)
    g = torch.tensor(scale, device="cuda")
    if reduction == "none":
        g = torch.randn(len(y), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    loss = fused_ce.head_cross_entropy(h, w, y, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32
    got = torch.autograd.grad(loss, (h, w) if trained else (h,), g)
    want = _exact(h.detach(), w.detach(), y, reduction, g, ignore)
    _within(loss, want[0], "loss")
    assert got[0].dtype == h.dtype
    _within(got[0], want[1], "dh")
    if trained:
        assert got[1].dtype == w.dtype
        _within(got[1], want[2], "dw")
    with torch.no_grad():
        again = fused_ce.head_cross_entropy(h, w, y, ignore_index=ignore, reduction=reduction)
    _within(again, want[0], "loss without gradients")
    return loss, got


# ---- values -----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 64, 65, 128, 129, 160, 161, 192, 193, 255,
                                  257, 320, 321, 384, 385, 513, 576, 577])
def test_rows(cuda, rows, dtype):
    print(f"case rows={rows} {dtype}", flush=True)
    _check(*_case(rows, 1000, 128, dtype, ignored=rows // 3))
    _check(*_case(rows, 1000, 128, dtype), trained=False)


@pytest.mark.parametrize("trained", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 31, 63, 64, 65, 255, 256, 257, 1003, 5000])
def test_vocabularies(cuda, vocab, trained):
    print(f"case vocab={vocab}", flush=True)
    _check(*_case(70, vocab, 192, F16), trained=trained)
    _check(*_case(300, vocab, 192, BF16), trained=trained)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 33, 64, 65, 128])
@pytest.mark.parametrize("vocab", [5023, 16384, 16385, 70001])
def test_few_rows_of_tables(cuda, vocab, rows, dtype):
    """Tables of 64 columns a compute unit and fewer, and larger ones: each has tiles of its own."""
    print(f"case vocab={vocab} rows={rows} {dtype}", flush=True)
    _check(*_case(rows, vocab, 192, dtype, ignored=rows // 3), trained=False)


@pytest.mark.parametrize("cols", [64, 128, 192, 256, 320, 448, 1536, 4096])
def test_widths(cuda, cols):
    print(f"case cols={cols}", flush=True)
    _check(*_case(40, 700, cols, BF16, ignored=3))
    _check(*_case(270, 700, cols, F16, ignored=3))


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("trained", [False, True])
@pytest.mark.parametrize("rows", [50, 400])
def test_reductions(cuda, reduction, trained, rows):
    _check(*_case(rows, 900, 256, F16, ignored=17), reduction=reduction, trained=trained)


def test_loss_scale_reaches_the_gradients_in_fp32(cuda):
    """A half-precision loss scale multiplies gradients whose unscaled values lie below fp16."""
    h, w, y = _case(1000, 2000, 128, F16)
    _check(h, w * 0.001, y, scale=65536.0)


def test_long_and_in_pieces(cuda):
    """More rows than one piece of exponentials holds at this vocabulary, an odd count of them."""
    _check(*_case(2501, 151936, 64, F16, ignored=77), trained=True)


def test_gradient_by_differences(cuda):
    """The loss along a direction, central difference: loss(h + t d) - loss(h - t d) over 2 t against
    <dh, d>, in the kernel's own losses.  Step t = 1/4 of exactly representable moves; the third
    derivative of a log-sum of D = 64 products with |d| <= 1/8 and |w| < 1 leaves t^2 (64/8)^3 / 6
    / 64 < 1/2 percent of it, the losses' rounding far less."""
    h, w, y = _case(40, 300, 64, BF16, spread=0.5)
    d = (torch.randint(-1, 2, h.shape, device="cuda") / 128).to(BF16)
    base = (h * 64).round() / 64  # so that h +- d / 4 ... stay exact in bf16 for |h| < 2
    base = base.clamp(-0.9, 0.9).to(BF16)
    d = (torch.randint(-1, 2, h.shape, device="cuda") / 64).to(BF16)
    hi, lo = base.float() + d.float(), base.float() - d.float()
    assert torch.equal(hi, hi.to(BF16).float()) and torch.equal(lo, lo.to(BF16).float())
    f = lambda x: fused_ce.head_cross_entropy(x.to(BF16), w, y, reduction="sum").item()  # noqa: E731
    x = base.clone().requires_grad_(True)
    (dh,) = torch.autograd.grad(fused_ce.head_cross_entropy(x, w, y, reduction="sum"), x)
    want = (f(hi) - f(lo)) / 2
    got = (dh.double() * d.double()).sum().item()
    size = (dh.double() * d.double()).abs().sum().item()
    assert abs(got - want) <= size * 2.0 ** -7


# ---- masks, infinities, labels ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [40, 300])
def test_ignored_rows_may_hold_anything(cuda, dtype, rows):
    h, w, y = _case(rows, 600, 128, dtype, ignored=rows // 4)
    clean = _check(h, w, y)
    gone = (y == -100).nonzero()[:, 0]
    h = h.clone()
    h[gone[0]], h[gone[1]], h[gone[2:]] = float("nan"), float("inf"), torch.finfo(dtype).min
    loss, got = _check(h, w, y)
    assert torch.equal(loss, clean[0]) and all(map(torch.equal, got, clean[1]))
    assert not got[0][gone].any()


def test_own_ignore_index_and_no_row_left(cuda):
    h, w, y = _case(50, 600, 128, F16)
    y[10:20] = 7
    _check(h, w, y, ignore=7)
    y[:] = -100
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    for reduction in ("mean", "sum", "none"):
        loss = fused_ce.head_cross_entropy(h, w, y, reduction=reduction)
        if reduction == "mean":
            assert torch.isnan(loss)
        else:
            assert not loss.any()
        for g in torch.autograd.grad(loss.sum(), (h, w)):
            assert not g.any()


def test_no_rows(cuda):
    h = torch.empty(0, 64, device="cuda", dtype=F16, requires_grad=True)
    w = torch.randn(10, 64, device="cuda").half().requires_grad_(True)
    y = torch.empty(0, device="cuda", dtype=torch.int64)
    for reduction in ("mean", "sum", "none"):
        loss = fused_ce.head_cross_entropy(h, w, y, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert dh.shape == h.shape and not dw.any()


def test_labels_outside_the_vocabulary_are_nan(cuda):
    h, w, y = _case(40, 300, 64, F16)
    y[3], y[5] = 300, -1
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = fused_ce.head_cross_entropy(h, w, y, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.equal(torch.isnan(loss), bad)
    (dh,) = torch.autograd.grad(
        fused_ce.head_cross_entropy(h, w.detach(), y, reduction="none").sum(), h)
    assert torch.equal(torch.isnan(dh).any(1), bad) and torch.isnan(dh[bad]).all()
    mean = fused_ce.head_cross_entropy(h, w, y)
    assert torch.isnan(mean)
    _, dw = torch.autograd.grad(mean, (h, w))
    assert torch.isnan(dw).all()


def test_lowest_value_and_infinite_logits(cuda):
    """A column of the type's lowest value, whose logits are -inf, has no weight; a logit of +inf
    makes its row NaN, as log-sum-exp does."""
    h, w, y = _case(40, 300, 64, BF16)
    h = h.abs() + 1
    w[7] = torch.finfo(BF16).min
    y[y == 7] = 8
    y[2] = 7
    hh, ww = h.requires_grad_(True), w.requires_grad_(True)
    loss = fused_ce.head_cross_entropy(hh, ww, y, reduction="none")
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[2] = False
    assert loss[2].item() == float("inf") and torch.isfinite(loss[keep]).all()
    want = torch.nn.functional.cross_entropy(
        h[keep].detach().double() @ w.detach().double()[:300].t(), y[keep], reduction="none")
    assert (loss[keep].double() - want).abs().max() <= 1e-4
    y[2] = -100
    dh, dw = torch.autograd.grad(fused_ce.head_cross_entropy(hh, ww, y), (hh, ww))
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all() and not dw[7].any()
    w2 = w.detach().clone()
    w2[7] = torch.finfo(BF16).max
    assert torch.isnan(fused_ce.head_cross_entropy(h.detach(), w2, y, reduction="none")[0])


def test_large_logits(cuda):
    """Logits in the thousands: the sum is relative to the largest, so nothing overflows."""
    h, w, y = _case(300, 1000, 128, F16)
    _check(h * 20, w * 40, y)


# ---- layouts ----------------------------------------------------------------------------------


def test_strides_and_alignment(cuda):
    h, w, y = _case(140, 500, 128, F16, ignored=9)
    want = _check(h, w, y)
    wide = torch.zeros(140, 300, device="cuda", dtype=F16)
    table = torch.zeros(500, 264, device="cuda", dtype=F16)
    for at, wat in ((0, 0), (8, 8), (1, 3), (5, 136)):
        wide[:, at:at + 128], table[:, wat:wat + 128] = h, w
        got = _check(wide[:, at:at + 128], table[:, wat:wat + 128], y)
        assert torch.equal(got[0], want[0]) and all(map(torch.equal, got[1], want[1]))
    got = _check(h.t().contiguous().t(), w.t().contiguous().t(), y)
    assert torch.equal(got[0], want[0]) and all(map(torch.equal, got[1], want[1]))
    every = torch.stack([y, y], 1)[:, 0]
    assert not every.is_contiguous()
    assert torch.equal(_check(h, w, every)[0], want[0])


def test_leading_shapes_and_label_types(cuda):
    h, w, y = _case(60, 500, 128, F16, ignored=9)
    flat = fused_ce.head_cross_entropy(h, w, y, reduction="none")
    got = fused_ce.head_cross_entropy(h.view(3, 20, 128), w, y.view(3, 20).int(),
                                      reduction="none")
    assert got.shape == (3, 20) and torch.equal(got.view(-1), flat)
    one = fused_ce.head_cross_entropy(h[0], w, y[0], reduction="none")
    assert one.shape == ()
    for x in (h.expand(2, 60, 128)[:, :1].reshape(2, 1, 128), h[:1].expand(4, 128)):
        fused_ce.head_cross_entropy(x, w, torch.zeros(x.shape[:-1], device="cuda").long())


def test_autocast(cuda):
    h, w, y = _case(60, 500, 128, F16)
    want = fused_ce.head_cross_entropy(h, w, y)
    a, b = h.float().requires_grad_(True), w.float().requires_grad_(True)
    with torch.autocast("cuda", dtype=F16):
        loss = fused_ce.head_cross_entropy(a, b, y)
    assert torch.equal(loss, want)
    da, db = torch.autograd.grad(loss, (a, b))
    assert da.dtype == db.dtype == torch.float32 and da.any() and db.any()


@pytest.mark.parametrize("trained", [False, True])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_both_routes_give_the_same_bits(cuda, monkeypatch, reduction, trained):
    """The compiled operator and the Python Function over ctypes."""
    from mindxsoup_amd import direct, ops

    case = _case(150, 700, 128, F16, ignored=20)
    assert ops.ENABLED
    a = _check(*case, reduction=reduction, trained=trained)
    leaf = case[0].clone().requires_grad_(True)
    node = fused_ce.head_cross_entropy(leaf, case[1], case[2]).grad_fn
    assert "FusedHeadCE" in node.name() and type(node).__name__ == "CppFunction"
    monkeypatch.setattr(ops, "ENABLED", False)
    for nograd in (False, True):
        monkeypatch.setattr(direct, "enabled", nograd)
        b = _check(*case, reduction=reduction, trained=trained)
        assert torch.equal(a[0], b[0]) and all(map(torch.equal, a[1], b[1]))


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("vocab", [700, 151936])  # at 2100 rows: one piece, two pieces
def test_one_of_two_gradients(cuda, monkeypatch, reduction, vocab, compiled):
    """Of a trained table either gradient alone is what it is beside the other, whether the other
    input needs none or is only not asked for: the same bits, but for the hidden states' alone
    under per-row losses, which then takes the route of a frozen table."""
    from mindxsoup_amd import ops

    monkeypatch.setattr(ops, "ENABLED", compiled)
    h, w, y = _case(2100, vocab, 64, BF16, ignored=50)
    g = torch.ones((), device="cuda") if reduction == "mean" else torch.rand(2100, device="cuda")

    def grads(a, b, leaves):
        loss = fused_ce.head_cross_entropy(a, b, y, reduction=reduction)
        return torch.autograd.grad(loss, leaves, g, retain_graph=True)

    hh, ww = h.requires_grad_(True), w.requires_grad_(True)
    dh, dw = grads(hh, ww, (hh, ww))
    assert torch.equal(grads(hh, ww, (ww,))[0], dw)
    alone = grads(hh, ww, (hh,))[0]
    if reduction == "mean":
        assert torch.equal(alone, dh)
    else:
        _within(alone, _exact(hh.detach(), ww.detach(), y, reduction, g)[1], "dh alone")
    assert torch.equal(grads(hh.detach(), ww, (ww,))[0], dw)


def test_inference_and_no_grad(cuda):
    h, w, y = _case(300, 700, 128, F16, ignored=20)
    want = fused_ce.head_cross_entropy(h, w, y, reduction="none")
    w.requires_grad_(True)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = fused_ce.head_cross_entropy(h, w, y, reduction="none")
        assert torch.equal(got, want) and not got.requires_grad


def test_more_rows_than_a_grid_side_and_than_a_piece(cuda):
    """70001 rows of a small vocabulary, in pieces of the row limit; against the losses and gradients
    of the same rows in two calls, which are independent of one another row by row."""
    h, w, y = _case(70001, 300, 64, F16, ignored=1000)
    g = torch.rand(70001, device="cuda")

    def run(a, b, f):
        a = a.detach().requires_grad_(True)
        loss = fused_ce.head_cross_entropy(a, w, b, reduction="none")
        return loss.detach(), torch.autograd.grad(loss, a, f)[0]

    loss, dh = run(h, y, g)
    for part in (slice(0, 40000), slice(40000, 70001)):
        l, d = run(h[part], y[part], g[part])
        assert torch.equal(l, loss[part])
        # the same dz; the shares of the vocabulary may differ with the rows, and with them the
        # order of fp32 sums, of at most 300 terms, before the one rounding to fp16
        off = (d.float() - dh[part].float()).abs()
        assert bool((off <= 2.0 ** -10 * d.float().abs() + 300 * U * 8 + 2.0 ** -24).all())


def test_no_second_derivative(cuda):
    h, w, y = _case(20, 100, 64, F16)
    h = h.requires_grad_(True)
    loss = fused_ce.head_cross_entropy(h, w, y)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, h, create_graph=True)


@pytest.mark.parametrize("compiled", [True, False])
def test_refusals(cuda, monkeypatch, compiled):
    from mindxsoup_amd import ops

    monkeypatch.setattr(ops, "ENABLED", compiled)
    h, w, y = _case(4, 20, 64, F16)
    run = fused_ce.head_cross_entropy
    for bad in (dict(reduction="max"),):
        with pytest.raises(ValueError):
            run(h, w, y, **bad)
    for args in ((h.float(), w.float(), y), (h, w.bfloat16(), y), (h, w, y.float()),
                 (h, w, y[:3]), (h, w[:, :32], y), (h[:, :32], w[:, :32], y), (h, w[:0], y),
                 (h.cpu(), w, y), (h, w.cpu(), y), (h, w, y.cpu()), (h, w[0], y),
                 (h, w, y.bool()), (h.double(), w.double(), y)):
        with pytest.raises(ValueError):
            run(*args)


# ---- order, streams, graphs -------------------------------------------------------------------


def test_the_same_twice(cuda):
    """No result depends on the order in which workgroups run: sums of shares have an order."""
    for rows in (40, 600):
        case = _case(rows, 3000, 256, BF16, ignored=11)
        a, b = _check(*case), _check(*case)
        assert torch.equal(a[0], b[0]) and all(map(torch.equal, a[1], b[1]))


@pytest.mark.parametrize("trained", [False, True])
def test_captured_forward_and_backward(cuda, trained):
    rows, static = 200, [x.clone() for x in _case(200, 1500, 128, F16, ignored=20)]
    h, w, y = static[0].requires_grad_(True), static[1].requires_grad_(trained), static[2]
    leaves = (h, w) if trained else (h,)

    def run():
        loss = fused_ce.head_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(1, 5):
        new = _case(rows, 1500, 128, F16, ignored=40 * seed, seed=seed)
        with torch.no_grad():
            for x, v in zip((h, w, y), new):
                x.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in out]
        eager = run()
        assert all(map(torch.equal, kept, eager)), seed


@pytest.mark.parametrize("leaf", ["hidden", "weight"])
def test_capture_beside_a_living_graph_is_refused(cuda, leaf):
    """On the default stream: the captured backward would end the process.  Nothing is captured."""
    h, w, y = _case(60, 300, 64, F16)
    (h if leaf == "hidden" else w).requires_grad_(True)
    alive = fused_ce.head_cross_entropy(h, w, y)
    with pytest.raises(RuntimeError, match=leaf + " is used by an autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fused_ce.head_cross_entropy(h, w, y)
    value = alive.item()
    alive.backward()  # the living one goes on
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_ce.head_cross_entropy(h, w, y)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert out.item() == value


def test_two_streams_at_once(cuda):
    cases = [_case(300, 2000, 128, F16, seed=i) for i in range(4)]
    want = [_check(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None] * 4
    for _ in range(3):
        for i, (c, s) in enumerate(zip(cases, streams)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                h, w = c[0].detach().requires_grad_(True), c[1].detach().requires_grad_(True)
                loss = fused_ce.head_cross_entropy(h, w, c[2])
                got[i] = (loss, torch.autograd.grad(loss, (h, w),
                                                    torch.tensor(3.0, device="cuda")))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and all(map(torch.equal, a[1], b[1]))


def test_backward_twice(cuda):
    h, w, y = _case(60, 500, 128, F16)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = fused_ce.head_cross_entropy(h, w, y)
    a = torch.autograd.grad(loss, (h, w), torch.tensor(2.0, device="cuda"), retain_graph=True)
    b = torch.autograd.grad(loss, (h, w), torch.tensor(4.0, device="cuda"))
    for x, z in zip(a, b):
        assert torch.allclose(x.float() * 2, z.float(), rtol=2.0 ** -10, atol=2.0 ** -24)


# ---- the model's patch, and the operators together --------------------------------------------


def _tiny_model(dtype):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(0)
    cfg = transformers.Qwen2Config(vocab_size=1000, hidden_size=128, intermediate_size=256,
                                   num_hidden_layers=2, num_attention_heads=2,
                                   num_key_value_heads=1, max_position_embeddings=128,
                                   tie_word_embeddings=True)
    return transformers.Qwen2ForCausalLM(cfg).cuda().to(dtype)


@pytest.fixture
def patched(monkeypatch):
    modeling = pytest.importorskip("transformers.models.qwen2.modeling_qwen2")
    cls = modeling.Qwen2ForCausalLM
    original = cls.forward
    assert fused_ce.patch_qwen2_head_ce() and fused_ce.patch_qwen2_head_ce()
    yield original
    cls.forward = original
    cls._mindx_head_ce = False


def test_qwen2_training_loss_without_logits(cuda, patched):
    model = _tiny_model(BF16).train()
    ids = torch.randint(1000, (2, 50), device="cuda")
    labels = ids.clone()
    labels[:, :10] = -100
    out = model(input_ids=ids, labels=labels)
    assert out.logits is None
    out.loss.backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    want = patched(model, input_ids=ids, labels=labels)
    # the model's own logits are rounded to bf16 (2^-8 of values below 2 here)
    assert abs(out.loss.item() - want.loss.item()) <= 2.0 ** -7
    want.loss.backward()
    for n, p in model.named_parameters():
        a, b = grads[n].float(), p.grad.float()
        # bf16 chains of about ten roundings, of either side
        assert (a - b).norm() <= 20 * 2.0 ** -8 * b.norm(), n
    summed = model(input_ids=ids, labels=labels, num_items_in_batch=torch.tensor(160)).loss
    assert abs(summed.item() - out.loss.item() * 80 / 160) <= 1e-4  # 40 labels a row
    model.eval()
    assert model(input_ids=ids, labels=labels).logits is not None


def test_qwen2_calls_that_ask_for_more_run_the_original(cuda, patched):
    """A loss function of the model's own, a hook on the head, and tuples instead of outputs."""
    model = _tiny_model(BF16).train()
    ids = torch.randint(1000, (2, 20), device="cuda")
    assert model(input_ids=ids, labels=ids).logits is None
    seen = []
    hook = model.lm_head.register_forward_hook(lambda *a: seen.append(a[2].shape))
    assert model(input_ids=ids, labels=ids).logits is not None
    assert len(seen) == 1 and seen[0][:2] == ids.shape
    hook.remove()
    out = model(input_ids=ids, labels=ids, return_dict=False)
    assert isinstance(out, tuple) and out[1].shape[:2] == ids.shape
    assert model(input_ids=ids, labels=ids, return_dict=None).logits is None  # as configured
    model.loss_function = lambda logits, labels, **kw: logits.float().sum() * 0 + 7
    assert model(input_ids=ids, labels=ids).loss.item() == 7.0


def test_training_step_end_to_end(cuda, patched):
    """The step's end as a program runs it, all operators in a row: head and loss, gradients,
    their norm, clipping and AdamW with 8-bit states; every matrix moves and stays finite,
    and the loss is that of an unpatched forward of the same weights."""
    from mindxsoup_amd import optim

    model = _tiny_model(BF16).train()
    opt = optim.AdamW(model.parameters(), lr=1e-3, state_bits=8, max_grad_norm=1.0)
    ids = torch.randint(1000, (2, 50), device="cuda")
    for _ in range(3):
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        loss = model(input_ids=ids, labels=ids).loss
        with torch.no_grad():
            want = patched(model, input_ids=ids, labels=ids).loss
        assert abs(loss.item() - want.item()) <= 2.0 ** -6
        loss.backward()
        grads = torch.cat([p.grad.double().flatten() for p in model.parameters()])
        opt.step()
        norm = opt.grad_norm.item()
        assert abs(norm - grads.norm().item()) <= 2 * U * norm
        for n, p in model.named_parameters():
            assert torch.isfinite(p).all()
            # the norms' ones stay: a step of at most lr = 1e-3 is under half of bf16's 2^-8 below 1
            if p.dim() == 2 and p.grad.any():
                assert not torch.equal(p, before[n]), n
        opt.zero_grad()
