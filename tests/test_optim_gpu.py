"""Gradient norm and AdamW step over many tensors (mindxsoup_amd/optim.py on csrc/optim.hip)
against the formulas in 64 bits.

Tolerances: u = 2^-24 is half a step of fp32 relative to the value.  A new parameter is
fl(fl(p k) - s m / (sqrt(v) r + eps)): p k carries the rounding of k, of the product and of the
difference (4 u |p| with a margin); the update's factors carry at most 24 roundings of half a
step (gradient times factor 2, m 5, v 7 of which the root halves, root, scale, sum, quotient and
product 2 each for a division and a root within one step), on the sum of the magnitudes that m is
made of.  16-bit parameters add their own rounding.  m and v: 8 u of the sum of magnitudes."""

import copy
import io

import numpy as np
import pytest
import torch

from mindxsoup_amd import optim
from mindxsoup_amd.quant import dynamic_map

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SIZES = [1, 7, 0, 8, 255, 256, 257, 2047, 2048, 2049, 8191, 8192, 8193, 30000]
ARGS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(n, std, seed, dtype=torch.float32):
    return (torch.randn(n, device="cuda", generator=_gen(seed)) * std).to(dtype)


def _books():
    signed = dynamic_map().astype(np.float64)
    unsigned = [0.0, 1.0]
    for i in range(7):
        n = 2 << i
        edge = np.array([np.float32(0.1 + 0.9 * j / n) for j in range(n + 1)], np.float32)
        unsigned += [float(np.float32(10.0 ** (i - 6) * float(m)))
                     for m in (edge[:-1] + edge[1:]) / np.float32(2)]
    return [torch.tensor(b, dtype=torch.float64, device="cuda")
            for b in (signed, sorted(unsigned))]


def _nearest(x, book):
    """Index of the nearest value, the lower of two as near, by all the distances."""
    return (x[:, None] - book[None, :]).abs().argmin(1)


def _exact(p, g, m, v, t, lr, betas, eps, weight_decay, c=1.0):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    b1, b2 = betas
    g = g * c
    new_m, new_v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * (g * g)
    den = (new_v / (1 - b2 ** t)).sqrt() + eps
    size = lr / (1 - b1 ** t)
    bound = 4 * U * p.abs() + 24 * U * size * (b1 * m.abs() + (1 - b1) * g.abs()) / den
    return p * (1 - lr * weight_decay) - size * new_m / den, new_m, new_v, bound


def _case(dtype, sizes=SIZES, offset=0):
    """Tensors of these sizes, each a view `offset` values into a buffer of its own."""
    out = []
    for k, (std, dt) in enumerate(((0.02, dtype), (1e-2, dtype), (1e-2, torch.float32),
                                   (1e-2, torch.float32))):
        out.append([_randn(n + offset, std, 10 * i + k, dt)[offset:]
                    for i, n in enumerate(sizes)])
    p, g, m, v = out
    return p, g, m, [x.square() if offset == 0 else x.square_() for x in v]


# ---- gradient norm ----------------------------------------------------------------------------


@pytest.mark.parametrize("offset", [0, 1])
def test_norm_of_mixed_tensors(cuda, offset):
    gs = []
    for i, n in enumerate(SIZES):
        dt = (torch.float32, torch.float16, torch.bfloat16)[i % 3]
        gs.append(_randn(n + offset, 10.0 ** (i % 4), i, dt)[offset:])
    want = torch.cat([g.double() for g in gs]).norm().item()
    got = optim.grad_norm(gs)
    assert got.shape == () and got.dtype == torch.float32 and got.device == cuda
    assert abs(got.item() - want) <= 2 * U * want  # one rounding to fp32, sums in fp64
    scale = torch.tensor(1024.0, device=cuda)
    assert abs(optim.grad_norm(gs, scale).item() - want / 1024) <= 2 * U * want / 1024


@pytest.mark.parametrize("count,size", [(1, 1), (450, 33), (3, 0), (2, 20_000_001)])
def test_norm_of_few_and_many(cuda, count, size):
    gs = [_randn(size, 1.0, i) for i in range(count)]
    want = sum(float(g.double().square().sum()) for g in gs) ** 0.5
    assert abs(optim.grad_norm(gs).item() - want) <= 2 * U * want


def test_norm_range_and_nonfinite(cuda):
    big, small = torch.full((5000,), 3e38, device=cuda), torch.full((5000,), 1e-40, device=cuda)
    assert optim.grad_norm([big]).item() == float("inf")  # past fp32's range once rounded
    want = small.double().norm().item()
    assert abs(optim.grad_norm([small]).item() - want) <= 2.0 ** -149
    x = _randn(5000, 1.0, 0)
    x[4999] = float("nan")
    assert torch.isnan(optim.grad_norm([big * 0, x]))
    x[4999] = float("-inf")
    assert optim.grad_norm([x]).item() == float("inf")


def test_norm_layouts(cuda):
    x = _randn(600, 1.0, 3).view(20, 30)
    for y in (x.t(), x[:, ::2], x[1:2].expand(7, 30), x.view(2, 10, 30).permute(2, 0, 1)):
        want = y.double().norm().item()
        assert abs(optim.grad_norm([y]).item() - want) <= 2 * U * want


# ---- the step, states in 32 bits --------------------------------------------------------------


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_step32(cuda, dtype, offset):
    p, g, m, v = _case(dtype, offset=offset)
    step = torch.tensor(4.0, device=cuda)
    want = [_exact(*x, 5, **ARGS) for x in zip(p, g, m, v)]
    old = [(b1 * x.abs().double() + (1 - b1) * y.abs().double())
           for b1 in (ARGS["betas"][0],) for x, y in zip(m, g)]
    optim.adamw_step(p, g, m, v, step, **ARGS)
    assert step.item() == 5.0
    for i, (wp, wm, wv, bound) in enumerate(want):
        tol = bound + HALF[dtype] * wp.abs() * (dtype != torch.float32)
        if dtype == torch.float16:  # below its normal range half a step is 2^-25
            tol += 2.0 ** -25
        assert ((p[i].double() - wp).abs() <= tol).all(), (SIZES[i], dtype)
        assert ((m[i].double() - wm).abs() <= 8 * U * old[i]).all()
        assert ((v[i].double() - wv).abs() <= 8 * U * wv).all()


def test_step32_clip_scale_and_device_lr(cuda):
    p, g, m, v = _case(torch.float32)
    g = [x * 512.0 for x in g]
    scale = torch.tensor(512.0, device=cuda)
    norm = optim.grad_norm(g, scale)
    c = min(1.0, 0.25 / (norm.item() + 1e-6)) / 512.0
    assert c < 1 / 512
    args = dict(ARGS, lr=torch.tensor(ARGS["lr"], device=cuda))
    lr32 = float(args["lr"])  # the number the device holds
    want = [_exact(*x, 1, **dict(ARGS, lr=lr32), c=c) for x in zip(p, g, m, v)]
    step = torch.zeros((), device=cuda)
    optim.adamw_step(p, g, m, v, step, norm=norm, max_norm=0.25, grad_scale=scale, **args)
    for i, (wp, wm, wv, bound) in enumerate(want):
        assert ((p[i].double() - wp).abs() <= bound).all()


def test_norm_below_the_bound_does_not_clip(cuda):
    p, g, m, v = _case(torch.float32, [1000])
    q, n, w = p[0].clone(), m[0].clone(), v[0].clone()
    optim.adamw_step(p, g, m, v, torch.zeros((), device=cuda), norm=optim.grad_norm(g),
                     max_norm=1e9, **ARGS)
    optim.adamw_step([q], g, [n], [w], torch.zeros((), device=cuda), **ARGS)
    assert torch.equal(p[0], q) and torch.equal(m[0], n) and torch.equal(v[0], w)


@pytest.mark.parametrize("bits", [32, 8])
def test_found_inf_leaves_everything(cuda, bits):
    p, g, m, v = _case(torch.float32, [1000, 3])
    kw = {}
    if bits == 8:
        st = [optim.zero_state8(x) for x in p]
        m, v, sm, sv = map(list, zip(*st))
        kw["scales"] = (sm, sv)
    step = torch.tensor(7.0, device=cuda)
    before = copy.deepcopy((p, m, v, step))
    g[1][2] = float("inf")
    flag = torch.ones((), device=cuda)
    optim.adamw_step(p, g, m, v, step, found_inf=flag, **ARGS, **kw)
    for a, b in zip((*p, *m, *v, step), (*before[0], *before[1], *before[2], before[3])):
        assert torch.equal(a, b)
    optim.adamw_step(p, g, m, v, step, found_inf=flag.zero_(), **ARGS, **kw)
    assert step.item() == 8.0 and not torch.equal(p[0], before[0][0])


def test_layouts_and_many_tensors(cuda):
    """Transposed parameters with gradients laid out otherwise, and more tensors than a launch's
    table holds."""
    n = 300
    p = [_randn(6 * (i % 5 + 1), 0.02, i).view(-1, 6).t() for i in range(n)]
    g = [_randn(x.numel(), 0.1, 1000 + i).view(x.shape) for i, x in enumerate(p)]
    m = [torch.zeros_like(x) for x in p]
    v = [torch.zeros_like(x) for x in p]
    assert m[1].stride() == p[1].stride() != g[1].stride()
    want = [_exact(*x, 1, **ARGS) for x in zip(p, g, m, v)]
    optim.adamw_step(p, g, m, v, torch.zeros((), device=cuda), **ARGS)
    for i, (wp, wm, wv, bound) in enumerate(want):
        assert ((p[i].double() - wp).abs() <= bound).all()


# ---- the step, states in 8 bits ---------------------------------------------------------------


def _step8_want(books, p, g, m, v, sm, sv, t):
    rep = lambda s, n: s.double().repeat_interleave(256)[:n]  # noqa: E731
    n = p.numel()
    om, ov = books[0][m.long()] * rep(sm, n), books[1][v.long()] * rep(sv, n)
    wp, wm, wv, bound = _exact(p, g, om, ov, t, **ARGS)
    out = []
    for x, book in ((wm, books[0]), (wv, books[1])):
        pad = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
        top = pad.amax(1).float()
        t64 = rep(top, n)
        rel = torch.where(t64 > 0, x / t64, torch.zeros_like(x))
        out += [_nearest(rel, book).to(torch.uint8), top]
    return wp, bound, out


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_step8(cuda, dtype, offset):
    """Three steps: codes and scales as the formulas in 64 bits give them, every one."""
    books = _books()
    p, _, _, _ = _case(dtype, offset=offset)
    st = [optim.zero_state8(x) for x in p]
    if offset:  # codes off their alignment too
        st = [(torch.cat([m, m])[len(m):] if len(m) % 2 else m, v, a, b) for m, v, a, b in st]
    m, v, sm, sv = map(list, zip(*st))
    step = torch.zeros((), device=cuda)
    for t in (1, 2, 3):
        g = [_randn(n, 10.0 ** -(i % 5), 100 * t + i, dtype) for i, n in enumerate(SIZES)]
        want = [_step8_want(books, *x, t) for x in zip(p, g, m, v, sm, sv)]
        optim.adamw_step(p, g, m, v, step, scales=(sm, sv), **ARGS)
        for i, (wp, bound, (cm, tm, cv, tv)) in enumerate(want):
            assert torch.equal(sm[i], tm) and torch.equal(sv[i], tv), (t, SIZES[i])
            assert torch.equal(m[i], cm) and torch.equal(v[i], cv), (t, SIZES[i])
            tol = bound + HALF[dtype] * wp.abs() * (dtype != torch.float32)
            if dtype == torch.float16:
                tol += 2.0 ** -25
            assert ((p[i].double() - wp).abs() <= tol).all()
            for codes, scale, book, signed in ((m[i], sm[i], books[0], True),
                                               (v[i], sv[i], books[1], False)):
                val = optim.state_values(codes, scale, signed)
                full = book[codes.long()] * scale.double().repeat_interleave(256)[:codes.numel()]
                assert torch.equal(val, full.float())


def test_code_search_takes_the_nearest_everywhere(cuda):
    """Every code's own value, the values next to every border on both sides, and the borders
    themselves (the lower code): beta 0 makes the new state the gradient itself."""
    for book, signed in zip(_books(), (True, False)):
        border = (book[1:] + book[:-1]) / 2
        f = border.float()
        xs = [book.float(), f, torch.nextafter(f, f + 1), torch.nextafter(f, f - 1)]
        lo, hi = (-1.0, 1.0) if signed else (0.0, 1.0)
        xs = torch.cat(xs).clamp(lo, hi)
        blocks = torch.nn.functional.pad(xs, (0, -len(xs) % 255)).view(-1, 255)
        g = torch.cat([torch.ones(len(blocks), 1, device=cuda), blocks], 1).view(-1)
        if not signed:  # v takes squares: give it roots, and judge by the squares it gets
            g = g.sqrt()
        p = torch.zeros_like(g)
        m, v, sm, sv = optim.zero_state8(p)
        optim.adamw_step([p], [g], [m], [v], torch.zeros((), device=cuda), lr=0.0,
                         betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, scales=([sm], [sv]))
        x = g.double() if signed else g.double().square()
        got, scale = (m, sm) if signed else (v, sv)
        top = scale.double().repeat_interleave(256)
        assert torch.equal(got.long(), _nearest(x / top, book))


def test_state8_nonfinite_and_zero_blocks(cuda):
    p = torch.zeros(256 * 4 + 10, device=cuda)
    m, v, sm, sv = optim.zero_state8(p)
    g = _randn(p.numel(), 1.0, 0)
    g[300], g[1030] = float("nan"), float("inf")
    g[512:768] = 0.0
    optim.adamw_step([p], [g], [m], [v], torch.zeros((), device=cuda), scales=([sm], [sv]),
                     **ARGS)
    for codes, scale, signed in ((m, sm, True), (v, sv, False)):
        assert torch.isnan(scale).tolist() == [False, True, False, False, True]
        assert scale[2] == 0.0
        val = optim.state_values(codes, scale, signed)
        assert torch.isnan(val[256:512]).all() and torch.isnan(val[1024:]).all()
        assert (val[512:768] == 0).all() and torch.isfinite(val[768:1024]).all()


# ---- refusals ---------------------------------------------------------------------------------


def test_refusals(cuda):
    x = lambda n=8, dt=torch.float32: torch.zeros(n, device=cuda, dtype=dt)  # noqa: E731
    step = torch.zeros((), device=cuda)
    run = optim.adamw_step
    with pytest.raises(RuntimeError, match="as many"):
        run([x()], [], [x()], [x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="must be \\[8\\]"):
        run([x()], [x(9)], [x()], [x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="grads"):
        run([x()], [x(dt=torch.float16)], [x()], [x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="states"):
        run([x(dt=torch.float16)], [x(dt=torch.float16)], [x(dt=torch.float16)], [x()], step,
            lr=0.1)
    with pytest.raises(RuntimeError, match="fp32, fp16 or bf16"):
        run([x(dt=torch.float64)], [x(dt=torch.float64)], [x()], [x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="one fp32 value"):
        run([x()], [x()], [x()], [x()], torch.zeros((), device=cuda, dtype=torch.int64), lr=0.1)
    with pytest.raises(RuntimeError, match="scales"):
        u = x(dt=torch.uint8)
        run([x()], [x()], [u], [u.clone()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="must be fp32 \\[1\\]"):
        u = x(dt=torch.uint8)
        run([x()], [x()], [u], [u.clone()], step, lr=0.1, scales=([x(2)], [x(1)]))
    with pytest.raises(RuntimeError, match="strides"):
        run([x(64).view(8, 8)], [x(64).view(8, 8)], [x(64).view(8, 8).t()],
            [x(64).view(8, 8)], step, lr=0.1)
    with pytest.raises(RuntimeError, match="one piece"):
        run([x(16)[::2]], [x()], [x()], [x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        p = x(12)
        run([p[:8], p[4:]], [x(), x()], [x(), x()], [x(), x()], step, lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        p = x()
        run([p, p], [x(), x()], [x(), x()], [x(), x()], step, lr=0.1)
    with pytest.raises(ValueError, match="GPU tensor"):
        run([x()], [torch.zeros(8)], [x()], [x()], step, lr=0.1)
    for kw in (dict(norm=step), dict(max_norm=1.0), dict(betas=(1.0, 0.5)), dict(eps=-1.0),
               dict(weight_decay=-1.0), dict(norm=step, max_norm=0.0)):
        with pytest.raises(ValueError):
            run([x()], [x()], [x()], [x()], step, lr=0.1, **kw)
    assert step.item() == 0.0
    run([], [], [], [], step, lr=0.1)  # nothing to do but to count
    assert step.item() == 1.0


def test_tensors_whose_memory_is_not_their_values_are_refused(cuda):
    """Negated views and zeros without memory: the kernels would take what lies there."""
    x = torch.ones(8, device=cuda)
    step = torch.zeros((), device=cuda)
    for odd in (torch._neg_view(x), torch._efficientzerotensor((8,), device=cuda)):
        with pytest.raises(ValueError, match="holds its values"):
            optim.grad_norm([x, odd])
        with pytest.raises(ValueError, match="holds its values"):
            optim.adamw_step([x.clone()], [odd], [x.clone()], [x.clone()], step, lr=0.1)
    with pytest.raises(ValueError, match="norm must be a tensor that holds"):
        optim.adamw_step([x.clone()], [x], [x.clone()], [x.clone()], step, lr=0.1,
                         norm=torch._neg_view(step), max_norm=1.0)
    assert step.item() == 0.0


# ---- streams, graphs, versions ----------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays_like_eager(cuda, bits):
    def fresh():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(n, device=cuda)) for n in (5000, 37, 4096)]
        return ps, optim.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=0.5)

    grads = [[_randn(n, 1.0, 10 * t + i) for i, n in enumerate((5000, 37, 4096))]
             for t in range(6)]
    eager, opt = fresh()
    for gs in grads:
        for p, g in zip(eager, gs):
            p.grad = g.clone()
        opt.step()
    ps, opt2 = fresh()
    for p, g in zip(ps, grads[0]):
        p.grad = g.clone()
    opt2.step()  # makes the states
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt2.step()
    for gs in grads[1:]:
        for p, g in zip(ps, gs):
            p.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        _randn(100, 1.0, 0).sum()  # eager work between the replays
    for a, b in zip(eager, ps):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_captured_after_a_first_step(cuda, bits):
    """Replays go on where eager steps would; what a replay would start anew is refused."""
    def make():
        ps = [torch.nn.Parameter(torch.linspace(-1, 1, n, device=cuda)) for n in (5000, 300)]
        for i, p in enumerate(ps):
            p.grad = torch.full_like(p, 0.25 + i)
        return ps, optim.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=1.0)

    ps, opt = make()
    with pytest.raises(RuntimeError, match="first step cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert not any(opt.state[p] for p in ps)
    want, eager = make()
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 4):
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(map(torch.equal, ps, want))
        assert opt.state[ps[0]]["step"].item() == 1 + k
    some, opt = make()
    opt.param_groups[0]["state_bits"] = 32  # both share a step count
    opt.step()
    some[1].grad = None
    with pytest.raises(RuntimeError, match="stepped together"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    assert [opt.state[p]["step"].item() for p in some] == [2.0, 1.0]


def test_side_stream(cuda):
    p, g, m, v = _case(torch.float32, [50000])
    q, n, w = p[0].clone(), m[0].clone(), v[0].clone()
    optim.adamw_step([q], g, [n], [w], torch.zeros((), device=cuda), norm=optim.grad_norm(g),
                     max_norm=0.1, **ARGS)
    s = torch.cuda.Stream()
    step = torch.zeros((), device=cuda)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        optim.adamw_step(p, g, m, v, step, norm=optim.grad_norm(g), max_norm=0.1, **ARGS)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(p[0], q) and torch.equal(m[0], n) and torch.equal(v[0], w)


def test_a_saved_parameter_is_seen_to_change(cuda):
    p = torch.nn.Parameter(torch.ones(8, device=cuda))
    loss = (p * p).sum()
    z = lambda: torch.zeros(8, device=cuda)  # noqa: E731
    optim.adamw_step([p], [z()], [z()], [z()], torch.zeros((), device=cuda), lr=0.1)
    assert p.is_leaf and p.grad_fn is None
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- the optimizer ----------------------------------------------------------------------------


def test_optimizer_follows_torchs(cuda):
    """20 steps beside torch.optim.AdamW on fp32 parameters: both are fp32 recurrences of the same
    formula; a step's rounding of a parameter of size 1 is 2^-24 and the update's is far smaller,
    so 20 steps stay within 20 * 4 * 2^-24 of each other."""
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.rand(n, device=cuda) * 0.5 + 0.25) for n in (300, 5000)]
    b = [torch.nn.Parameter(x.detach().clone()) for x in a]
    mine = optim.AdamW(a, lr=1e-3, weight_decay=0.1)
    theirs = torch.optim.AdamW(b, lr=1e-3, weight_decay=0.1)
    for t in range(20):
        for i, (x, y) in enumerate(zip(a, b)):
            x.grad = _randn(x.numel(), 1.0, 10 * t + i)
            y.grad = x.grad.clone()
        mine.step()
        theirs.step()
    for x, y in zip(a, b):
        assert (x - y).abs().max().item() <= 80 * U


def test_parameters_without_gradient_keep_their_count(cuda):
    ps = [torch.nn.Parameter(torch.ones(8, device=cuda)) for _ in range(3)]
    opt = optim.AdamW(ps, lr=0.1)
    for live in ((0, 1), (0, 1, 2), (1,), (0, 2)):
        for i, p in enumerate(ps):
            p.grad = torch.ones_like(p) if i in live else None
        opt.step()
    assert [float(opt.state[p]["step"]) for p in ps] == [3.0, 3.0, 2.0]


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(cuda, bits):
    def params():
        torch.manual_seed(1)
        return [torch.nn.Parameter(torch.randn(n, device=cuda).bfloat16()) for n in (5000, 30)]

    def steps(ps, opt, ts):
        for t in ts:
            for i, p in enumerate(ps):
                p.grad = _randn(p.numel(), 1.0, 10 * t + i, torch.bfloat16)
            opt.step()

    a = params()
    opt = optim.AdamW(a, lr=1e-2, state_bits=bits)
    steps(a, opt, range(3))
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf)
    buf.seek(0)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = optim.AdamW(b, lr=1e-2, state_bits=bits)
    other.load_state_dict(torch.load(buf, weights_only=True))
    kinds = {k: v.dtype for k, v in other.state[b[0]].items()}
    assert kinds["exp_avg"] == (torch.uint8 if bits == 8 else torch.float32)
    steps(a, opt, range(3, 6))
    steps(b, other, range(3, 6))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_grad_scaler_hands_over_scale_and_overflow(cuda):
    p = torch.nn.Parameter(torch.ones(5000, device=cuda))
    q = torch.nn.Parameter(torch.ones(5000, device=cuda))
    a, b = optim.AdamW([p], lr=0.1), optim.AdamW([q], lr=0.1)
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0, growth_interval=1000)
    x = _randn(5000, 1.0, 0)
    scaler.scale((p * x).sum()).backward()
    scaler.step(a)
    scaler.update()
    q.grad = x.clone()
    b.step()
    assert torch.equal(p, q)  # the scale is a power of two
    before = p.detach().clone()
    p.grad = torch.full_like(p, float("inf"))
    scaler.scale(torch.zeros((), device=cuda))
    scaler.step(a)
    scaler.update()
    assert torch.equal(p, before) and scaler.get_scale() == 128.0
    assert float(a.state[p]["step"]) == 1.0


def test_checkpoint_of_torchs_adamw(cuda):
    """States of torch's optimizer, in the parameters' type and with a step count each, carry on."""
    torch.manual_seed(2)
    a = torch.nn.Parameter(torch.randn(500, device=cuda).bfloat16())
    theirs = torch.optim.AdamW([a], lr=1e-2)
    for t in range(2):
        a.grad = _randn(500, 1.0, t, torch.bfloat16)
        theirs.step()
    b, c = (torch.nn.Parameter(a.detach().clone()) for _ in range(2))
    mine = optim.AdamW([b], lr=1e-2)
    mine.load_state_dict(copy.deepcopy(theirs.state_dict()))
    st = theirs.state[a]
    assert mine.state[b]["exp_avg"].dtype == torch.float32
    assert torch.equal(mine.state[b]["exp_avg"], st["exp_avg"].float())
    assert float(mine.state[b]["step"]) == 2.0
    want = _exact(b.detach(), _randn(500, 1.0, 9, torch.bfloat16), st["exp_avg"], st["exp_avg_sq"],
                  3, 1e-2, (0.9, 0.999), 1e-8, 1e-2)
    b.grad = _randn(500, 1.0, 9, torch.bfloat16)
    mine.step()
    assert ((b.double() - want[0]).abs() <= want[3] + 2.0 ** -8 * want[0].abs()).all()


def test_scaled_gradients_are_clipped_by_their_true_norm(cuda):
    """GradScaler's factor with max_grad_norm: as the unscaled gradients clipped; the scale is a
    power of two, so the two differ only where fp32 rounds the coefficient's products."""
    x = _randn(3000, 1.0, 4)
    ps = [torch.nn.Parameter(torch.ones(3000, device=cuda)) for _ in range(2)]
    a, b = (optim.AdamW([p], lr=0.1, eps=1e-3, max_grad_norm=0.5) for p in ps)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    scaler.scale((ps[0] * x).sum()).backward()
    scaler.step(a)
    ps[1].grad = x.clone()
    b.step()
    assert torch.equal(a.grad_norm, b.grad_norm)
    assert (ps[0] - ps[1]).abs().max().item() <= 8 * U


def test_more_than_2_to_the_31_values(cuda):
    """One tensor of 2^31 + 300 values: past 32 bits of offsets and into a second table entry."""
    n = (1 << 31) + 300
    g = torch.zeros(n, device=cuda, dtype=torch.bfloat16)
    at = [0, 5, (1 << 31) - 1, 1 << 31, n - 1]
    for k, i in enumerate(at):
        g[i] = 2.0 ** k
    want = sum(4.0 ** k for k in range(5)) ** 0.5
    assert abs(optim.grad_norm([g]).item() - want) <= 2 * U * want
    p = torch.ones(n, device=cuda, dtype=torch.bfloat16)
    m, v, sm, sv = optim.zero_state8(p)
    optim.adamw_step([p], [g], [m], [v], torch.zeros((), device=cuda), lr=0.5, eps=1e-6,
                     betas=(0.9, 0.99), weight_decay=0.0, scales=([sm], [sv]))
    # a first step moves a parameter by lr wherever there is a gradient: 1 -> 0.5
    assert torch.equal(p[at].float().cpu(), torch.full((5,), 0.5))
    p[at] = 1.0
    assert bool((p == 1.0).all())
    tail = optim.state_values(m[-300:].clone(), sm[-2:], True)
    full = optim.state_values(m, sm, True)
    assert torch.equal(full[-300:], tail) and full[n - 1] == sm[-1] and sm[-1] > 1.0


def test_norm_and_step_of_two_calls_at_once(cuda):
    """Calls on two streams keep their workspaces apart."""
    cases = [_case(torch.float32, [70000, 11]) for _ in range(2)]
    want = copy.deepcopy(cases)
    for p, g, m, v in want:
        optim.adamw_step(p, g, m, v, torch.zeros((), device=cuda), norm=optim.grad_norm(g),
                         max_norm=0.1, **ARGS)
    steps = [torch.zeros((), device=cuda) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s, (p, g, m, v), step in zip(streams, cases, steps):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            optim.adamw_step(p, g, m, v, step, norm=optim.grad_norm(g), max_norm=0.1, **ARGS)
    torch.cuda.synchronize()
    for a, b in zip(cases, want):
        for x, y in zip(a, b):
            assert all(map(torch.equal, x, y))
