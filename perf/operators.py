"""The operators at the end of a training step, as they are timed: the language-model head with
its cross entropy (loss, and the gradients of the hidden states and, for a trained head, of the
table), the global norm of a step's gradients, and the AdamW step over many tensors with states
in 32 or in 8 bits.

`run` computes each in its plain form, elementary torch operations, or with `own` through the
package's entry points: `fused_ce.head_cross_entropy`, `optim.grad_norm`, `optim.adamw_step` and
`optim.state_values`.  Sizes are those of Qwen2.5-1.5B (hidden 1536, vocabulary 151936,
intermediate 8960, 28 layers, LoRA rank 16 on the seven projections) and generic ones.
"""

import math

import numpy as np
import torch

own = False

IGNORE = -100
BLOCK = 256  # values that share one scale of an 8-bit state
BETAS, EPS, DECAY, LR, MAX_NORM = (0.9, 0.999), 1e-8, 0.01, 2e-4, 1.0
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
LAYERS, HIDDEN, INTER, KV, RANK = 28, 1536, 8960, 256, 16


def listed():
    return [
        # the log-probability of one candidate token (ranking answers, early stopping)
        dict(name="head_score_1", kind="head", tokens=1, ignored=0, vocab=151936, hidden=1536,
             dtype="float16", mode="score"),
        # per-token losses of one evaluation prompt
        dict(name="head_score_301", kind="head", tokens=301, ignored=40, vocab=151936,
             hidden=1536, dtype="float16", mode="score"),
        # a training step's head at 1024 packed tokens, the prompts' positions masked out
        dict(name="head_train_1024", kind="head", tokens=1024, ignored=256, vocab=151936,
             hidden=1536, dtype="float16", mode="frozen"),
        # a long packed batch with every position trained on
        dict(name="head_train_8192", kind="head", tokens=8192, ignored=0, vocab=151936,
             hidden=1536, dtype="bfloat16", mode="frozen"),
        # a trained head with one added token, a ragged batch
        dict(name="head_tied_829", kind="head", tokens=829, ignored=101, vocab=32001,
             hidden=4096, dtype="bfloat16", mode="trained"),
        # the large table trained as well
        dict(name="head_tied_2048", kind="head", tokens=2048, ignored=0, vocab=151936,
             hidden=1536, dtype="float16", mode="trained"),
        # every adapter of the model, clipped, states in 32 bits
        dict(name="adamw_lora", kind="adamw", layers=28, tensors=0, size=0, bits=32,
             dtype="float32", clip=True),
        # a handful of odd little tensors (norms, biases, a soft prompt): latency
        dict(name="adamw_small", kind="adamw", layers=0, tensors=13, size=901, bits=32,
             dtype="float32", clip=False),
        # every adapter of the model, states in 8 bits
        dict(name="adamw8_lora", kind="adamw", layers=28, tensors=0, size=0, bits=8,
             dtype="float32", clip=True),
        # large bf16 weights trained in full, states in 8 bits
        dict(name="adamw8_large", kind="adamw", layers=0, tensors=24, size=1536 * 8960, bits=8,
             dtype="bfloat16", clip=False),
        # the norm of every adapter's gradient
        dict(name="norm_lora", kind="norm", layers=28, tensors=0, size=0, dtype="float32"),
        # the norm over large bf16 gradients
        dict(name="norm_large", kind="norm", layers=0, tensors=24, size=1536 * 8960,
             dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["head", "head", "adamw", "norm"])
    if kind == "head":
        mode = rng.choice(["score", "frozen", "trained"])
        vocab, hidden = _log(rng, 500, 151936), 64 * _log(rng, 2, 64)
        most = {"score": 8192, "frozen": 8192, "trained": 4096}[mode]
        # no more than the largest listed one: 8192 tokens of 151936 x 1536, two products
        room = 8192 * 151936 * 1536 * 2 // (vocab * hidden * 3)
        tokens = _log(rng, 1, max(1, min(most, room)))
        return dict(kind=kind, tokens=tokens, ignored=int(tokens * rng.uniform(0, 0.7)),
                    vocab=vocab, hidden=hidden, dtype=rng.choice(["float16", "bfloat16"]),
                    mode=mode)
    case = dict(kind=kind, layers=0, tensors=_log(rng, 1, 300))
    case["size"] = _log(rng, 30, 2e8 / case["tensors"])
    if kind == "adamw":
        case["bits"] = rng.choice([32, 8])
    case["dtype"] = rng.choice(["float32", "float16", "bfloat16"])
    if kind == "adamw":
        case["clip"] = rng.choice([True, False])
    return case


# ---- inputs -----------------------------------------------------------------------------------


def _sizes(case):
    """The tensors of an optimizer case: LoRA A and B of seven projections a layer, or `tensors`
    sizes around `size`."""
    if case["layers"]:
        widths = [(HIDDEN, HIDDEN), (HIDDEN, KV), (HIDDEN, KV), (HIDDEN, HIDDEN),
                  (HIDDEN, INTER), (HIDDEN, INTER), (INTER, HIDDEN)]
        return [n for k, m in widths * case["layers"] for n in (RANK * k, RANK * m)]
    # from half to one and a half times the size, none alike
    t = case["tensors"]
    return [max(1, case["size"] * (2 * i + t) // (2 * t)) + i % 3 for i in range(t)]


def _arena(sizes, dtype, device):
    """One buffer for tensors of these sizes, each from a multiple of BLOCK on, and its views."""
    starts = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])]).tolist()
    flat = torch.zeros(starts[-1], dtype=dtype, device=device)
    return flat, [flat[s:s + n] for s, n in zip(starts, sizes)]


def _maps(device):
    """The two 8-bit code books, ascending: signed with 2^i and unsigned with 2^(i+1) midpoints
    in the decade below 10^(i-6), i = 0..6, and with 0 and 1."""
    books = []
    for more in (0, 1):
        values = [0.0, 1.0]
        for i in range(7):
            edge = np.array([np.float32(0.1 + 0.9 * j / (1 << (i + more)))
                             for j in range((1 << (i + more)) + 1)], np.float32)
            mids = ((edge[:-1] + edge[1:]) / np.float32(2.0)).astype(np.float64)
            mids = (10.0 ** (i - 6) * mids).astype(np.float32)
            values += mids.tolist() + ([] if more else (-mids).tolist())
        books.append(torch.tensor(sorted(values), dtype=torch.float32, device=device))
    return books


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dt=torch.float32):
        return torch.empty(*shape, dtype=dt, device=dev).normal_(0.0, std, generator=gen)

    if case["kind"] == "head":
        t, v, d = case["tokens"], case["vocab"], case["hidden"]
        weight = normal(v, d, std=0.8 / math.sqrt(d), dt=dtype)
        labels = torch.randint(v, (t,), device=dev, generator=gen)
        # hidden states lean towards their token by different amounts: from hopeless to sure
        lean = torch.rand(t, 1, device=dev, generator=gen) * 18.0
        rows = weight[labels].float()
        hidden = normal(t, d, std=2.5) + lean * rows / rows.square().sum(1, keepdim=True)
        gone = torch.randperm(t, device=dev, generator=gen)[:case["ignored"]]
        labels[gone] = IGNORE
        state = dict(case=case, hidden=hidden.to(dtype), weight=weight, labels=labels,
                     # the loss scale of a half-precision training program
                     scale=torch.tensor(1024.0 if dtype == torch.float16 else 1.0, device=dev))
        if case["mode"] != "score":
            state["hidden"].requires_grad_(True)
            weight.requires_grad_(case["mode"] == "trained")
        return state

    sizes = _sizes(case)
    state = dict(case=case, sizes=sizes)
    state["grad"], state["grads"] = _arena(sizes, dtype, dev)
    for i, g in enumerate(state["grads"]):  # layers' gradients differ in size
        g.normal_(0.0, 1e-3 * (1 + i % 7), generator=gen)
    if case["kind"] == "norm":
        return state
    state["param"], state["params"] = _arena(sizes, dtype, dev)
    for p in state["params"]:
        p.normal_(0.0, 0.02, generator=gen)
    state["step"] = torch.tensor(41.0, device=dev)
    if case["bits"] == 32:
        for name, std in (("m", 1e-3), ("v", 2e-3)):
            state[name], views = _arena(sizes, torch.float32, dev)
            for x in views:
                x.normal_(0.0, std, generator=gen)
            if name == "v":
                state[name].square_()
            state[name + "s"] = views
    else:
        state["maps"] = _maps(dev)
        state["borders"] = [((b[1:].double() + b[:-1].double()) / 2) for b in state["maps"]]
        for name, book in zip(("m", "v"), state["maps"]):
            codes, views = _arena(sizes, torch.uint8, dev)
            scale = 1e-3 * (0.5 + torch.rand(codes.numel() // BLOCK, device=dev, generator=gen))
            scale = scale if name == "m" else scale.square()
            zero = int((book == 0).nonzero())
            codes.fill_(zero)
            middle = (book[1:] + book[:-1]) / 2
            for x in views:
                y = normal(x.numel(), std=0.3).clamp_(-1, 1)
                x.copy_(torch.bucketize(y if name == "m" else y.square_(), middle,
                                        out_int32=True))
            first = np.concatenate([[0], np.cumsum([-(-n // BLOCK) for n in sizes])]).tolist()
            state[name], state[name + "s"] = codes, views
            state[name + "_scale"] = scale
            state[name + "_scales"] = [scale[a:b] for a, b in zip(first[:-1], first[1:])]
    return state


# ---- one pass ---------------------------------------------------------------------------------


def _head_plain(state):
    mode, h, w, labels = (state["case"]["mode"], state["hidden"].detach(),
                          state["weight"].detach(), state["labels"])
    h32, w32 = h.float(), w.float()
    live = labels != IGNORE
    at = torch.where(live, labels, 0)[:, None]
    z = h32 @ w32.t()
    top = z.amax(1, keepdim=True)
    e = (z - top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(live, (top + total.log() - z.gather(1, at))[:, 0], 0.0)
    if mode == "score":
        return [loss]
    n = live.sum()
    mean = (loss.double().sum() / n).float()
    part = live[:, None] * (state["scale"] / n)
    e.mul_(part / total)
    e.scatter_add_(1, at, -part)
    grads = [(e @ w32).to(h.dtype)]
    if mode == "trained":
        grads.append((e.t() @ h32).to(w.dtype))
    return [mean, *grads]


def _head_own(state):
    from mindxsoup_amd import fused_ce

    h, w, labels = state["hidden"], state["weight"], state["labels"]
    if state["case"]["mode"] == "score":
        return [fused_ce.head_cross_entropy(h, w, labels, reduction="none")]
    loss = fused_ce.head_cross_entropy(h, w, labels)
    leaves = [h, w] if w.requires_grad else [h]
    return [loss.detach(), *torch.autograd.grad(loss, leaves, state["scale"])]


def _norm_plain(state):
    # one sum over the buffer that holds the gradients (zeros lie between them)
    return state["grad"].double().square_().sum().sqrt_().float()


def _norm_own(state):
    from mindxsoup_amd import optim

    return optim.grad_norm(state["grads"])


def _adamw_plain(state):
    """The step on the whole buffers; what lies between two tensors is zero and stays zero."""
    clip, (b1, b2) = state["case"]["clip"], BETAS
    step, p, g = state["step"], state["param"], state["grad"]
    step += 1
    t = step.double()
    wide = torch.float64 if state["case"]["bits"] == 8 else torch.float32
    g = g.to(wide)
    norm = None
    if clip:
        norm = _norm_plain(state)
        g = g * (MAX_NORM / (norm.double() + 1e-6)).clamp(max=1.0).to(wide)
    if state["case"]["bits"] == 32:
        m, v = state["m"], state["v"]
        m.mul_(b1).add_(g * (1 - b1))
        v.mul_(b2).add_(g.square().mul_(1 - b2))
    else:  # in 64 bits: a value next to the border of two codes has to take the right one
        both = []
        for name, beta, x in (("m", b1, g), ("v", b2, g.square())):
            book, codes, scale = state["maps"][name == "v"], state[name], state[name + "_scale"]
            old = book[codes.int()].double().view(-1, BLOCK) * scale.double()[:, None]
            new = old.mul_(beta).add_(x.view(-1, BLOCK) * (1 - beta))
            scale.copy_(new.abs().amax(1))
            top = scale.double()[:, None]
            rel = torch.where(top > 0, new / top, 0.0)
            codes.copy_(torch.bucketize(rel, state["borders"][name == "v"],
                                        out_int32=True).view(-1))
            both.append(new.view(-1).float())
        m, v = both
    root = v.sqrt().mul_((1 / (1 - b2 ** t).sqrt()).float()).add_(EPS)
    p32 = p.float() * (1 - LR * DECAY)
    p32 -= (LR / (1 - b1 ** t)).float() * m / root
    p.copy_(p32)
    if state["case"]["bits"] == 8:
        m, v = (state["maps"][k][state[n].int()].view(-1, BLOCK).mul_(state[n + "_scale"][:, None])
                .view(-1) for k, n in ((0, "m"), (1, "v")))
    return [p, m, v, step, *([norm] if clip else [])]


def _adamw_own(state):
    from mindxsoup_amd import optim

    case = state["case"]
    norm = optim.grad_norm(state["grads"]) if case["clip"] else None
    kw = dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, norm=norm,
              max_norm=MAX_NORM if case["clip"] else None)
    if case["bits"] == 8:
        kw["scales"] = (state["m_scales"], state["v_scales"])
    optim.adamw_step(state["params"], state["grads"], state["ms"], state["vs"], state["step"],
                     **kw)
    m, v = state["m"], state["v"]
    if case["bits"] == 8:  # the values that the codes stand for
        m = optim.state_values(m, state["m_scale"], signed=True)
        v = optim.state_values(v, state["v_scale"], signed=False)
    return [state["param"], m, v, state["step"], *([norm] if case["clip"] else [])]


def run(state):
    kind = state["case"]["kind"]
    if kind == "head":
        return _head_own(state) if own else _head_plain(state)
    if kind == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    return _adamw_own(state) if own else _adamw_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    width = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "head":
        t, v, d = case["tokens"], case["vocab"], case["hidden"]
        live = t - case["ignored"]
        products = {"score": 1, "frozen": 2, "trained": 3}[case["mode"]]
        data = width * (live * d + v * d) + 8 * t + 4 * (t if case["mode"] == "score" else 1)
        data += width * t * d * (products > 1) + width * v * d * (products > 2)
        return {"bytes": data, "flops": 2.0 * products * live * v * d}
    n = sum(_sizes(case))
    if case["kind"] == "norm":
        return {"bytes": n * width + 4, "flops": 2.0 * n}
    # gradient read, parameter and both states read and written
    state = 4.0 if case["bits"] == 32 else 1 + 4 / BLOCK
    # 8-bit states also leave as the values that they stand for
    values = 8 if case["bits"] == 8 else 0
    return {"bytes": n * (3 * width + 4 * state + values), "flops": 16.0 * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def _head_exact(state):
    case, labels = state["case"], state["labels"]
    w = state["weight"].detach().double()
    keep = (labels != IGNORE).nonzero()[:, 0]
    h, y = state["hidden"].detach().double(), labels[keep]
    loss = torch.zeros(labels.numel(), dtype=torch.float64, device=w.device)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w) if case["mode"] == "trained" else None
    weight = float(state["scale"]) / max(1, keep.numel())
    for some in torch.arange(keep.numel(), device=w.device).split(1024):
        rows, label = h[keep[some]], y[some]
        logp = torch.log_softmax(torch.mm(rows, w.T), dim=-1)
        pick = torch.arange(some.numel(), device=w.device)
        loss[keep[some]] = -logp[pick, label]
        if case["mode"] != "score":
            slope = torch.exp(logp)
            slope[pick, label] = torch.expm1(logp[pick, label])
            slope *= weight
            dh[keep[some]] = torch.mm(slope, w)
            if dw is not None:
                dw.addmm_(slope.T, rows)
    if case["mode"] == "score":
        return [loss]
    return [loss.sum() / keep.numel(), dh, *([] if dw is None else [dw])]


def _nearest(x, book):
    """The index of the book's value that is nearest, the lower one of two as near."""
    up = torch.searchsorted(book, x).clamp_(1, book.numel() - 1)
    return up - (x - book[up - 1] <= book[up] - x).long()


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "head":
        return _head_exact(state)
    norm = torch.stack([torch.linalg.vector_norm(g.double()) for g in state["grads"]]).norm()
    if case["kind"] == "norm":
        return norm
    t = float(state["step"]) + 1
    # the clipping factor goes by the norm as a 32-bit number: that is what is handed over
    cut = min(1.0, MAX_NORM / (float(norm.float()) + 1e-6)) if case["clip"] else 1.0
    out = {k: torch.zeros(state["param"].numel(), dtype=torch.float64, device="cuda")
           for k in "pmv"}
    at = 0
    for i, (p, g) in enumerate(zip(state["params"], state["grads"])):
        n, g = p.numel(), g.double() * cut
        new = {}
        for k, beta, x in (("m", BETAS[0], g), ("v", BETAS[1], g ** 2)):
            if case["bits"] == 32:
                new[k] = out[k][at:at + n] = beta * state[k + "s"][i].double() + (1 - beta) * x
                continue
            book = state["maps"]["mv".index(k)].double()
            scale = state[k + "_scales"][i].double().repeat_interleave(BLOCK)[:n]
            new[k] = beta * (book[state[k + "s"][i].long()] * scale) + (1 - beta) * x
            # a block's scale is kept in 32 bits
            pad = torch.nn.functional.pad(new[k].abs(), (0, -n % BLOCK)).view(-1, BLOCK)
            top = pad.max(1).values.float().double().repeat_interleave(BLOCK)[:n]
            share = torch.where(top == 0, torch.zeros_like(top), new[k] / top)
            out[k][at:at + n] = book[_nearest(share, book)] * top
        hat = new["m"] / (1 - BETAS[0] ** t), new["v"] / (1 - BETAS[1] ** t)
        out["p"][at:at + n] = p.double() - LR * (DECAY * p.double() + hat[0] / (hat[1].sqrt() + EPS))
        at += -(-n // BLOCK) * BLOCK
    return [out["p"], out["m"], out["v"], torch.tensor(t, dtype=torch.float64),
            *([norm] if case["clip"] else [])]
