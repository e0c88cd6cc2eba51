"""The language-model head with its cross entropy on the HIP kernels of csrc/head_ce.hip: the loss
and its gradients without the matrix of logits (the reference's solution/fused_ce.py, which
works through it in chunks).

    loss = fused_ce.head_cross_entropy(hidden, lm_head.weight, labels)

The losses take one product with the table; where gradients are wanted the forward also computes
that of the hidden states, from the product's exponentials in 16 bits (a piece of the rows at a
time), and the backward multiplies it by the gradient that comes from above.  A trained table's
gradient is the backward's own product where the rows are one piece, over dz kept from the forward
(16 bits, 1 GiB at most); of several pieces it is summed in fp32 beside them.  Per-token losses
whose table is trained need the factor from above per row, so their backward runs all products
anew.

With FEATURES["torch_ops"] (on) the call is the compiled torch.ops.mxs_nf4.head_cross_entropy,
whose backward runs in C++; FusedHeadCE over ctypes is the other route and gives the same bits.
"""

import torch

from . import _lib, direct, ops

REDUCTIONS = ("none", "sum", "mean")
_DTYPES = {torch.float16: _lib.MXS_DTYPE_F16, torch.bfloat16: _lib.MXS_DTYPE_BF16}


def _rows(t, cols):
    """t [rows, cols] with its columns side by side: (tensor, row stride)."""
    if t.shape[0] <= 1:
        t = t.contiguous()
        return t, cols
    if t.stride(1) != 1 or t.stride(0) < cols:
        t = t.contiguous()
    return t, t.stride(0)


def _run(h, w, labels, ignore_index, reduction, row_grad, want_loss, want_dh, want_dw):
    """One call of mxs_head_ce: (loss, dh, dw), None where not wanted.  dw: fp32 [V, D], or, of one
    piece's rows, the workspace that _table_grad makes it from."""
    rows, cols = h.shape
    vocab, dev = w.shape[0], h.device
    f32 = dict(dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        h, ldh = _rows(h, cols)
        w, ldw = _rows(w, cols)
        if ldw % 8 or w.data_ptr() % 16:
            w, ldw = w.clone(memory_format=torch.contiguous_format), cols
        L = _lib.lib()
        keep = bool(want_dw) and L.mxs_head_ce_one_piece(rows, vocab, cols) == 1
        loss = torch.empty(rows if reduction == "none" else (), **f32) if want_loss else None
        dh = torch.empty(rows, cols, **f32) if want_dh else None
        dw = torch.empty(vocab, cols, **f32) if want_dw and not keep else None
        n = L.mxs_head_ce_workspace_bytes(rows, vocab, cols, want_dh, want_dw)
        if n < 0:
            _lib.check(n, "mxs_head_ce_workspace_bytes")
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.call("mxs_head_ce", _lib.ptr(h), ldh, _lib.ptr(w), ldw, _lib.ptr(labels), rows,
                  vocab, cols, _DTYPES[h.dtype], ignore_index, REDUCTIONS.index(reduction),
                  _lib.ptr(row_grad), _lib.ptr(loss), _lib.ptr(dh), _lib.ptr(dw), int(keep),
                  _lib.ptr(ws), _lib.stream_of(dev))
    return loss, dh, ws if keep else dw


def _table_grad(dw, h, w_shape, reduction, row_grad, want_dh, g):
    """The table's gradient in h's dtype from what _run left for it, times g (one value or None)."""
    if dw.dtype != torch.uint8:
        return dw.to(h.dtype) if g is None else _scaled(dw, g, h.dtype)
    out = torch.empty(w_shape, dtype=h.dtype, device=dw.device)
    if g is not None:
        g = g.to(torch.float32).contiguous()
    with torch.cuda.device(dw.device):
        _lib.call("mxs_head_ce_table_grad", _lib.ptr(dw), h.shape[0], w_shape[0], w_shape[1],
                  _DTYPES[h.dtype], REDUCTIONS.index(reduction), _lib.ptr(row_grad),
                  int(want_dh), _lib.ptr(g), _lib.ptr(out), _lib.stream_of(dw.device))
    return out


def _scaled(unit, g, dtype):
    """unit * g rounded to dtype: g one value, or one per row."""
    out = torch.empty_like(unit, dtype=dtype)
    g = g.to(torch.float32).contiguous()
    with torch.cuda.device(unit.device):
        _lib.call("mxs_head_ce_grad", _lib.ptr(unit), _lib.ptr(g), int(g.dim() > 0),
                  unit.shape[0], unit.shape[1], _DTYPES[dtype], _lib.ptr(out),
                  _lib.stream_of(unit.device))
    return out


class FusedHeadCE(torch.autograd.Function):
    """loss of (hidden [T, D], table [V, D], labels [T]); gradients for the first two."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        want_dh, want_dw = (*ctx.needs_input_grad, False, False)[:2]
        again = want_dw and reduction == "none"
        loss, dh, dw = _run(hidden, weight, labels, ignore_index, reduction, None, True,
                            want_dh and not again, want_dw and not again)
        ctx.again, ctx.args, ctx.w_shape = again, (ignore_index, reduction), weight.shape
        ctx.want_dh = want_dh
        if again:
            ctx.save_for_backward(hidden, weight, labels)
        else:
            ctx.save_for_backward(hidden.new_empty(hidden.shape[0], 0), dh, dw)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        want_dh, want_dw = ctx.needs_input_grad[:2]
        reduction = ctx.args[1]
        if ctx.again:
            hidden, grad = ctx.saved_tensors[0], grad.to(torch.float32).contiguous()
            _, dh, dw = _run(*ctx.saved_tensors, *ctx.args, grad, False, want_dh, want_dw)
            dh = dh.to(hidden.dtype) if want_dh else None
            if want_dw:
                dw = _table_grad(dw, hidden, ctx.w_shape, reduction, grad, want_dh, None)
            return dh, dw, None, None, None
        hidden, dh, dw = ctx.saved_tensors  # hidden: its type and rows
        return (_scaled(dh, grad, hidden.dtype) if want_dh else None,
                _table_grad(dw, hidden, ctx.w_shape, reduction, None, ctx.want_dh, grad)
                if want_dw else None, None, None, None)


def _check(hidden, weight, labels):
    """The operator's own checks, for the other route."""
    for name, t in (("weight", weight), ("labels", labels)):
        if t.device != hidden.device:
            raise ValueError(f"{name} is on {t.device}, hidden on {hidden.device}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden [..., D] and weight [V, D], got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {tuple(labels.shape)} for hidden {tuple(hidden.shape)}")
    if labels.is_floating_point() or labels.is_complex() or labels.dtype == torch.bool:
        raise ValueError(f"labels must be integers, got {labels.dtype}")
    if weight.shape[0] == 0 or weight.shape[1] == 0 or weight.shape[1] % 64:
        raise ValueError(f"the table is [V >= 1, a multiple of 64], got {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or hidden.dtype not in _DTYPES:
        raise ValueError(f"hidden and weight must both be fp16 or both bf16, got {hidden.dtype} "
                         f"and {weight.dtype}")


def head_cross_entropy(hidden, weight, labels, *, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits hidden @ weight.T against `labels`, as
    torch.nn.functional.cross_entropy gives it on fp32 logits, without holding them.

    hidden [..., D] and weight [V, D] are fp16 or bf16 GPU tensors of one type (under autocast both
    are cast to its type first); D is a multiple of 64.  labels: integers of hidden's leading shape;
    positions holding `ignore_index` take no part, whatever their hidden states hold.  A label
    outside [0, V) that is not ignore_index makes the loss and its gradients NaN.
    reduction: "mean" over the positions that take part (NaN if there is none), "sum", or "none":
    fp32 losses in labels' shape, 0 at ignored positions.
    Gradients flow to hidden and, where it requires one, to weight, each summed in fp32 and
    rounded once.

    The call and its backward can be captured into a graph, as long as no autograd graph that was
    made from the same leaves on the default stream is still alive (the compiled operator refuses
    the call then)."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction is one of {REDUCTIONS}, got {reduction!r}")
    for name, t in (("hidden", hidden), ("weight", weight), ("labels", labels)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a GPU tensor")
    if torch.is_autocast_enabled("cuda"):
        kind = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(kind), weight.to(kind)
    if ops.ENABLED:
        return ops.load().head_cross_entropy(hidden, weight, labels, int(ignore_index),
                                             REDUCTIONS.index(reduction))
    _check(hidden, weight, labels)
    loss = direct.run(FusedHeadCE, hidden.reshape(-1, weight.shape[1]), weight,
                      labels.reshape(-1).to(torch.int64).contiguous(), int(ignore_index),
                      reduction)
    return loss.view(labels.shape) if reduction == "none" else loss


def _watched(module):
    """Whether somebody sees the module's calls: hooks, or a forward put on the object itself."""
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or
                module._backward_pre_hooks or "forward" in vars(module))


def _takes(model, labels, logits_to_keep, kwargs):
    """Whether the patched forward serves this call: a training call for the loss of all positions
    from a plain head in a type the kernels take, with nothing asked for beside it."""
    head = model.lm_head
    if not (model.training and isinstance(labels, torch.Tensor) and labels.is_cuda
            and isinstance(logits_to_keep, int) and logits_to_keep == 0):
        return False
    if type(head) is not torch.nn.Linear or head.bias is not None or head.in_features % 64 or \
            not head.weight.is_cuda or _watched(head):
        return False
    asked = kwargs.get("return_dict")  # None: as the configuration says
    if not (getattr(model.config, "return_dict", True) if asked is None else asked):
        return False
    if kwargs.get("output_hidden_states") or kwargs.get("output_attentions") or \
            getattr(model.config, "output_hidden_states", False) or \
            getattr(model.config, "output_attentions", False):
        return False
    if torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda") in _DTYPES
    return head.weight.dtype in _DTYPES


def patch_qwen2_head_ce():
    """Qwen2ForCausalLM's training forward takes its loss from head_cross_entropy and returns no
    logits (the reference's patch of the same method); evaluation, generation and calls that ask
    for more, models with a loss_function of their own and heads with hooks run the original.
    Returns whether transformers' Qwen2 model is importable."""
    try:
        from transformers.loss.loss_utils import ForCausalLMLoss
        from transformers.modeling_outputs import CausalLMOutputWithPast
        from transformers.models.qwen2 import modeling_qwen2
    except Exception:
        return False
    cls = modeling_qwen2.Qwen2ForCausalLM
    if getattr(cls, "_mindx_head_ce", False):
        return True
    original = cls.forward

    def forward(self, input_ids=None, attention_mask=None, position_ids=None,
                past_key_values=None, inputs_embeds=None, labels=None, use_cache=None,
                logits_to_keep=0, **kwargs):
        if not _takes(self, labels, logits_to_keep, kwargs) or \
                self.loss_function is not ForCausalLMLoss:
            return original(self, input_ids, attention_mask, position_ids, past_key_values,
                            inputs_embeds, labels, use_cache, logits_to_keep, **kwargs)
        count = kwargs.pop("num_items_in_batch", None)
        ignore = kwargs.pop("ignore_index", -100)
        shifted = kwargs.pop("shift_labels", None)
        out = self.model(input_ids=input_ids, attention_mask=attention_mask,
                         position_ids=position_ids, past_key_values=past_key_values,
                         inputs_embeds=inputs_embeds, use_cache=use_cache, **kwargs)
        if shifted is None:  # position t predicts token t + 1
            shifted = torch.nn.functional.pad(labels, (0, 1), value=ignore)[..., 1:]
        hidden = out.last_hidden_state
        loss = head_cross_entropy(hidden, self.lm_head.weight, shifted.to(hidden.device),
                                  ignore_index=ignore,
                                  reduction="mean" if count is None else "sum")
        if count is not None:  # the whole accumulated batch's positions
            loss = loss / (count.to(loss.device) if isinstance(count, torch.Tensor) else count)
        return CausalLMOutputWithPast(loss=loss, logits=None,
                                      past_key_values=out.past_key_values)

    forward._mindx_original = original
    cls.forward = forward
    cls._mindx_head_ce = True
    return True
