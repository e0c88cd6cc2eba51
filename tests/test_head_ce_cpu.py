"""The head's cross entropy without a GPU: refusals and the C entry points' argument checks."""

import pytest
import torch

from mindxsoup_amd import _lib, fused_ce


def test_cpu_tensors_are_refused():
    h, w, y = torch.zeros(2, 64).half(), torch.zeros(5, 64).half(), torch.zeros(2).long()
    with pytest.raises(ValueError, match="GPU"):
        fused_ce.head_cross_entropy(h, w, y)
    with pytest.raises(ValueError, match="reduction"):
        fused_ce.head_cross_entropy(h, w, y, reduction="max")


def test_workspace_is_bounded_whatever_the_rows():
    """The exponentials of at most 1 GiB are held; the rest of the workspace grows with the rows
    (gathered copies, 2 bytes a value) and the vocabulary's statistics."""
    f = _lib.lib().mxs_head_ce_workspace_bytes
    small, large = (f(t, 151936, 1536, 1, 0) for t in (2048, 1 << 17))
    assert 0 < small < (3 << 30) and large - small < (1 << 30) + 2 * 1536 * (1 << 17)
    assert f(1, 151936, 1536, 0, 0) < 16 << 20  # no exponentials for losses alone
    assert f(10, 100, 96, 0, 0) == -4 and f(-1, 100, 64, 0, 0) == -1
    assert f(10, 0, 64, 0, 0) == -1 and f(10, 100, 0, 0, 0) == -1
    assert f(0, 100, 64, 1, 1) > 0


def test_c_entries_check_arguments_before_any_launch():
    L = _lib.lib()
    P = 0x10000

    def run(h=P, ldh=64, w=P, ldw=64, y=P, T=4, V=10, D=64, dt=0, red=2, rg=None, loss=P, dh=P,
            dw=P, keep=0, ws=P):
        return L.mxs_head_ce(h, ldh, w, ldw, y, T, V, D, dt, -100, red, rg, loss, dh, dw, keep, ws,
                             None)

    assert run(h=None) == -1 and run(w=None) == -1 and run(y=None) == -1 and run(ws=None) == -1
    assert run(loss=None, dh=None, dw=None) == -1 and run(red=3) == -1 and run(T=-1) == -1
    assert run(red=0) == -1  # dw of per-row losses needs row_grad
    assert run(ldh=63) == -1 and run(ldw=56) == -1
    assert run(D=96, ldh=96, ldw=96) == -4 and run(T=1 << 25) == -4
    assert run(dt=1) == -2 and run(dt=7) == -2
    assert run(ldw=68) == -3 and run(w=P + 2) == -3 and run(dh=P + 4) == -3
    assert run(ws=P + 16) == -3 and run(dw=P + 8) == -3
    assert run(keep=1) == -1 and run(dw=None, keep=1, red=0) == -1
    assert run(dw=None, keep=1, T=4096, V=1 << 20) == -4  # several pieces
    assert L.mxs_head_ce_one_piece(2048, 151936, 1536) == 1
    assert L.mxs_head_ce_one_piece(2049, 151936, 1536) == 0
    t = L.mxs_head_ce_table_grad
    assert t(None, 4, 10, 64, 0, 2, None, 1, P, P, None) == -1
    assert t(P, 4, 10, 64, 0, 2, None, 1, P, None, None) == -1
    assert t(P, 4, 10, 64, 1, 2, None, 1, P, P, None) == -2
    assert t(P, 4, 10, 64, 0, 2, None, 1, P, P + 8, None) == -3
    assert t(P, 4096, 1 << 20, 64, 0, 2, None, 1, P, P, None) == -4
    g = L.mxs_head_ce_grad
    assert g(None, P, 0, 4, 64, 0, P, None) == -1 and g(P, None, 0, 4, 64, 0, P, None) == -1
    assert g(P, P, 0, 4, 63, 0, P, None) == -4 and g(P, P, 0, 4, 64, 1, P, None) == -2
    assert g(P + 4, P, 0, 4, 64, 0, P, None) == -3 and g(P, P, 0, 0, 64, 0, P, None) == 0


def test_meta_shapes_and_gradients():
    from mindxsoup_amd import ops

    mx = ops.load()
    h = torch.empty(3, 7, 64, device="meta", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(50, 64, device="meta", dtype=torch.bfloat16, requires_grad=True)
    y = torch.empty(3, 7, device="meta", dtype=torch.int64)
    for reduction, shape in ((0, (3, 7)), (1, ()), (2, ())):
        loss = mx.head_cross_entropy(h, w, y, -100, reduction)
        assert loss.shape == shape and loss.dtype == torch.float32
        assert "FusedHeadCE" in loss.grad_fn.name()
        dh, dw = torch.autograd.grad(loss, (h, w), torch.empty_like(loss))
        assert dh.shape == h.shape and dw.shape == w.shape
        assert dh.dtype == dw.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="multiple of 64"):
        mx.head_cross_entropy(h[..., :32], w[:, :32], y, -100, 2)
    with pytest.raises(ValueError, match="GPU"):
        mx.head_cross_entropy(torch.zeros(2, 64).half(), torch.zeros(5, 64).half(),
                              torch.zeros(2).long(), -100, 2)
