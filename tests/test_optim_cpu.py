"""The optimizer's entry points without a GPU: refusals, the operators' Meta kernels, the C entry
points' argument checks and the Trainer patch."""

import ctypes

import pytest
import torch

from mindxsoup_amd import _lib, ops, optim


def test_cpu_tensors_and_empty_lists_are_refused():
    with pytest.raises(ValueError, match="at least one"):
        optim.grad_norm([])
    with pytest.raises(ValueError, match="GPU"):
        optim.grad_norm([torch.zeros(3)])
    x = torch.zeros(3)
    with pytest.raises(ValueError, match="GPU"):
        optim.adamw_step([x], [x], [x], [x], torch.zeros(()), lr=1e-3)
    with pytest.raises(ValueError, match="GPU"):
        optim.state_values(torch.zeros(3, dtype=torch.uint8), torch.zeros(1), True)


@pytest.mark.parametrize("kw", [dict(state_bits=4), dict(lr=-1.0), dict(betas=(1.0, 0.9)),
                                dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                                dict(weight_decay=-1.0), dict(max_grad_norm=0.0),
                                dict(lr=float("nan"))])
def test_optimizer_refuses_bad_arguments(kw):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(2))], **kw)


@pytest.mark.parametrize("kw", [{}, dict(state_bits=8), dict(max_grad_norm=1.0)])
def test_optimizer_refuses_cpu_parameters(kw):
    p = torch.nn.Parameter(torch.ones(5000))
    p.grad = torch.ones(5000)
    with pytest.raises(ValueError, match="GPU"):
        optim.AdamW([p], **kw).step()
    assert bool((p == 1).all())


def test_meta_shapes():
    mx = ops.load()
    g = torch.empty(5, 7, device="meta", dtype=torch.bfloat16)
    out = mx.grad_norm([g, g], None)
    assert out.shape == () and out.dtype == torch.float32 and out.device.type == "meta"
    codes = torch.empty(5, 100, device="meta", dtype=torch.uint8)
    values = mx.state_values(codes, torch.empty(2, device="meta"), True)
    assert values.shape == codes.shape and values.dtype == torch.float32
    with pytest.raises(RuntimeError, match="scale must be"):
        mx.state_values(codes, torch.empty(3, device="meta"), True)


def test_c_entries_check_arguments_before_any_launch():
    """Null pointers, negative sizes, unknown types and bad alignment return an error code; no
    device is touched (there is none here)."""
    L = _lib.lib()
    one = (ctypes.c_void_p * 1)(0x1000)
    none = (ctypes.c_void_p * 1)(None)
    n1, bad = (ctypes.c_int64 * 1)(5), (ctypes.c_int64 * 1)(-1)
    f32, unknown = (ctypes.c_int * 1)(1), (ctypes.c_int * 1)(7)
    assert L.mxs_grad_norm_workspace_bytes(1, n1) >= 8
    assert L.mxs_grad_norm_workspace_bytes(1, bad) < 0
    assert L.mxs_grad_norm_workspace_bytes(-1, n1) < 0
    assert L.mxs_grad_norm(1, none, n1, f32, None, 0x1000, 0x1000, None) == -1
    assert L.mxs_grad_norm(1, one, bad, f32, None, 0x1000, 0x1000, None) == -1
    assert L.mxs_grad_norm(1, one, n1, unknown, None, 0x1000, 0x1000, None) == -2
    assert L.mxs_grad_norm(1, one, n1, f32, None, 0x1000, 0x1004, None) == -3
    assert L.mxs_grad_norm(1, one, n1, f32, None, None, 0x1000, None) == -1

    def step(bits=32, p=one, scales=None, sizes=n1, dtypes=f32, at=0x1000, ws=0x1000):
        return L.mxs_adamw_step(1, p, one, one, one, scales, scales, sizes, dtypes, bits, at, 0.1,
                                None, 0.9, 0.999, 1e-8, 0.0, None, 1.0, None, None, ws, None)

    assert step(bits=16) == -2 and step(dtypes=unknown) == -2
    assert step(p=none) == -1 and step(sizes=bad) == -1 and step(at=None) == -1
    assert step(bits=8) == -1 and step(bits=8, scales=none) == -1 and step(ws=0x1004) == -3
    assert L.mxs_state_values(None, None, 5, 1, None, None) == -1
    assert L.mxs_state_values(None, None, -5, 1, None, None) == -1
    assert L.mxs_state_values(None, None, 0, 1, None, None) == 0


def test_trainer_patch(monkeypatch):
    transformers = pytest.importorskip("transformers")
    trainer = transformers.Trainer
    monkeypatch.setattr(trainer, "get_optimizer_cls_and_kwargs",
                        trainer.get_optimizer_cls_and_kwargs)  # restored after the test
    assert optim.patch_trainer() and optim.patch_trainer()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)

    class Args:
        learning_rate, adam_beta1, adam_beta2, adam_epsilon, optim_args = 1e-4, 0.8, 0.99, 1e-6, None

    for name, bits in (("adamw_torch", 32), ("adamw_torch_fused", 32), ("adamw_8bit", 8),
                       ("adamw_bnb_8bit", 8)):
        args = Args()
        args.optim = name
        cls, kw = trainer.get_optimizer_cls_and_kwargs(args)
        assert cls is optim.AdamW
        assert kw == {"lr": 1e-4, "betas": (0.8, 0.99), "eps": 1e-6, "state_bits": bits}
    args = Args()
    args.optim = transformers.training_args.OptimizerNames.SGD
    assert trainer.get_optimizer_cls_and_kwargs(args)[0] is torch.optim.SGD
