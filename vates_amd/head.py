"""lm_head over the vocabulary with the argmax fused in (libvmi ``vmi_lm_head``), and
the loss of tokens under a head with its gradients (``head_loss``).

The analogue of the verify forward's tail ``logits = model.lm_head(inner.norm(h))``
followed by ``preds = mx.argmax(logits, -1)`` (mlx_streaming/mtp/generate.py:208-217,
:756) and of the draft step's ``int(mx.argmax(lg))`` (mlx_streaming/mtp/drafter.py:20-40).
Errors raise ``VmiError``; there is no fallback path.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import VMI_BF16, VMI_F32, VmiError, check, load
from .moe import (_matches, _no_tangent, _on_current, _on_stream, _once, _ptr, _require, _stream_handle, _stream_on, scratch,
                  workspace)


class TiledHead:
    """A bf16 [vocab, hidden] head re-laid once in tile-major order
    (``vmi_head_tiles``: each 16-row x 128-value chunk is 4 KB of contiguous
    memory), for callers that run the head every decode step; ``lm_head`` on it
    gives the row-major head's results bit for bit, faster."""

    def __init__(self, weight: torch.Tensor, stream=None):
        if weight.dim() != 2 or weight.dtype != torch.bfloat16 or not weight.is_cuda:
            raise VmiError("weight must be a bf16 [vocab, hidden] device tensor")
        weight = weight.contiguous()
        self.vocab, self.hidden = int(weight.shape[0]), int(weight.shape[1])
        lib = load()
        nbytes = int(lib.vmi_head_tiles_bytes(self.vocab, self.hidden))
        if nbytes == 0:
            raise VmiError(f"unsupported head shape {tuple(weight.shape)}")
        self.tiles = torch.empty(nbytes // 2, dtype=torch.bfloat16, device=weight.device)
        check(lib.vmi_head_tiles(weight.data_ptr(), self.vocab, self.hidden, self.tiles.data_ptr(),
                                 _stream_handle(stream)), "vmi_head_tiles")

    @property
    def device(self):
        return self.tiles.device


def lm_head(x: torch.Tensor, weight, norm_weight: Optional[torch.Tensor] = None, *,
            eps: float = 1e-6, want_logits: bool = True, logits: Optional[torch.Tensor] = None,
            argmax: Optional[torch.Tensor] = None, max_logit: Optional[torch.Tensor] = None,
            top_prob: Optional[torch.Tensor] = None, stream=None):
    """Returns (logits f32 [T, V] or None, argmax int32 [T], max logit f32 [T]).

    x bf16 [T, H] (T <= 16), weight bf16 [V, H] or a TiledHead of one,
    norm_weight bf16 [H] or None.
    top_prob (f32 [T], optional) receives the softmax probability of each
    row's argmax (the draft confidence of drafter.py:42-62).
    """
    dev = x.device
    if x.dim() != 2:
        raise VmiError(f"x must be [T, hidden], got {tuple(x.shape)}")
    T, H = x.shape
    tiled = isinstance(weight, TiledHead)
    if tiled:
        if weight.hidden != H:
            raise VmiError(f"tiled head has hidden {weight.hidden}, x has {H}")
        V, wt = weight.vocab, weight.tiles
    else:
        if weight.dim() != 2 or weight.shape[1] != H:
            raise VmiError(f"weight must be [vocab, {H}], got {tuple(weight.shape)}")
        V, wt = weight.shape[0], weight
    _require(x, "x", 2, dev)
    _require(wt, "weight", 2, dev)
    if norm_weight is not None:
        _require(norm_weight, "norm_weight", 2, dev)
        if norm_weight.numel() != H:
            raise VmiError(f"norm_weight must have {H} elements")
    if want_logits and logits is None:
        logits = torch.empty((T, V), dtype=torch.float32, device=dev)
    if argmax is None:
        argmax = torch.empty(T, dtype=torch.int32, device=dev)
    if max_logit is None:
        max_logit = torch.empty(T, dtype=torch.float32, device=dev)
    for t, name, n in ((logits, "logits", T * V), (argmax, "argmax", T), (max_logit, "max_logit", T),
                       (top_prob, "top_prob", T)):
        if t is not None:
            _require(t, name, 4, dev)
            if t.numel() != n:
                raise VmiError(f"{name} must have {n} elements")
    sh = _stream_handle(stream)
    lib = load()
    nbytes = lib.vmi_lm_head_workspace_bytes(T, V)
    ws = workspace(nbytes, dev, sh, tag="lm_head")
    fn = lib.vmi_lm_head_tiled if tiled else lib.vmi_lm_head
    rc = fn(x.data_ptr(), T, H, None if norm_weight is None else norm_weight.data_ptr(), float(eps),
                         wt.data_ptr(), V, None if logits is None else logits.data_ptr(), argmax.data_ptr(),
                         max_logit.data_ptr(), None if top_prob is None else top_prob.data_ptr(), ws.data_ptr(),
                         ws.numel(), sh)
    check(rc, "vmi_lm_head_tiled" if tiled else "vmi_lm_head")
    return logits, argmax, max_logit


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, status):
        loss, lse = _head_loss(x, weight, targets, ignore_index, status)
        ctx.save_for_backward(x, weight, targets, lse)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    @_once
    def backward(ctx, d_loss, d_lse):
        x, weight, targets, lse = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        if d_loss is None and d_lse is None:
            return None, None, None, None, None
        d_loss = torch.zeros_like(lse) if d_loss is None else d_loss.contiguous()
        dx, dw = _head_loss_grad(x, weight, targets, lse, d_loss, None if d_lse is None else d_lse.contiguous(), need_x,
                                 torch.bfloat16 if need_w else None, ctx.ignore_index)
        return dx, dw, None, None, None


def _check_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor) -> torch.device:
    if isinstance(weight, TiledHead):
        raise VmiError("weight must be the row-major head, not a TiledHead")
    dev = _on_current(x)
    xs, ws = x.shape, weight.shape
    if len(xs) != 2 or len(ws) != 2 or ws[1] != xs[1]:
        raise VmiError(f"x must be [T, hidden] and weight [vocab, hidden], got {tuple(xs)} and {tuple(ws)}")
    _matches(x, "x", xs, torch.bfloat16, dev)
    _matches(weight, "weight", ws, torch.bfloat16, dev)
    if targets.dtype not in (torch.int64, torch.int32):
        raise VmiError(f"targets must be int64 or int32 (got {targets.dtype})")
    _matches(targets, "targets", xs[:1], targets.dtype, dev)
    _no_tangent(x, weight)
    return dev


def _head_loss(x, weight, targets, ignore_index, status):
    T, H = x.shape
    V = weight.shape[0]
    loss, lse = x.new_empty(T, dtype=torch.float32), x.new_empty(T, dtype=torch.float32)
    lib = load()
    ws = scratch(lib.vmi_head_loss_workspace_bytes(T, H, V), x.device)
    check(lib.vmi_head_loss(x.data_ptr(), T, H, weight.data_ptr(), V, targets.data_ptr(), ignore_index, loss.data_ptr(),
                            lse.data_ptr(), _ptr(status), ws.data_ptr(), ws.numel(), _stream_on(x.device, None)),
          "vmi_head_loss")
    return loss, lse


def head_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
              status: Optional[torch.Tensor] = None, stream=None):
    """(loss f32 [T], lse f32 [T]): the softmax cross entropy of every token under a
    head, lse - z[target] with z = x . weight and lse = log sum exp z, without the
    logits in memory (``vmi_head_loss``).  The likelihood of a text is -loss.sum().

    x bf16 [T, hidden] behind the final norm (T <= 65536, hidden a multiple of 64
    up to 8192), weight bf16 [vocab, hidden] (the row-major head), targets int64 or
    int32 [T].  A token with target ignore_index has loss and lse 0 and is not read;
    a target outside the vocabulary gives NaN and ORs VMI_STATUS_BAD_TARGET into
    status (int32 [1] on the device).  Differentiable in x and weight through
    both outputs (``head_loss_grad``; a weight that needs no gradient costs none), once and
    in reverse mode; tokens left out of the loss have zeros and add nothing."""
    dev = _check_loss(x, weight, targets)
    if status is not None:
        _matches(status, "status", (1,), torch.int32, dev)
    return _on_stream(stream, _head_loss_on, x, weight, targets, ignore_index, status)


def _head_loss_on(x, weight, targets, ignore_index, status):
    if targets.dtype is not torch.int64:
        targets = targets.long()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _HeadLoss.apply(x, weight, targets, ignore_index, status)
    return _head_loss(x, weight, targets, ignore_index, status)


def head_loss_grad(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, d_loss: torch.Tensor,
                   d_lse: Optional[torch.Tensor] = None, *, want_dx: bool = True, want_dweight: bool = True,
                   dweight_dtype: torch.dtype = torch.bfloat16, ignore_index: int = -100, stream=None):
    """(dx bf16 [T, hidden] or None, dweight [vocab, hidden] or None): the gradients
    of ``head_loss`` from the lse that it returned and those of its outputs, f32
    [T] (``vmi_head_loss_grad``).  dweight_dtype: bf16, or f32, which spares gradients that a
    caller adds up itself the output's rounding; that of g to bf16 stays above 64 tokens (half a step,
    2^-8, of every token's share).  Not differentiable itself.  The same call gives the same bits."""
    dev = _check_loss(x, weight, targets)
    T = x.shape[0]
    for t, name in ((lse, "lse"), (d_loss, "d_loss"), (d_lse, "d_lse")):
        if t is not None or name != "d_lse":
            _matches(t, name, (T,), torch.float32, dev)
    _no_tangent(lse, d_loss, d_lse)
    if dweight_dtype not in (torch.bfloat16, torch.float32):
        raise VmiError(f"dweight_dtype must be bf16 or f32 (got {dweight_dtype})")
    if not (want_dx or want_dweight):
        raise VmiError("neither dx nor dweight wanted")
    return _on_stream(stream, _head_loss_grad, x, weight, targets, lse, d_loss, d_lse,
                      want_dx, dweight_dtype if want_dweight else None, ignore_index)


def _head_loss_grad(x, weight, targets, lse, d_loss, d_lse, want_dx, dweight_dtype, ignore_index):
    T, H = x.shape
    V = weight.shape[0]
    lib = load()
    if targets.dtype is not torch.int64:
        targets = targets.long()
    dx = torch.empty_like(x) if want_dx else None
    dw = None if dweight_dtype is None else weight.new_empty((V, H), dtype=dweight_dtype)
    ws = scratch(lib.vmi_head_loss_grad_workspace_bytes(T, H, V), x.device)
    check(lib.vmi_head_loss_grad(x.data_ptr(), T, H, weight.data_ptr(), V, targets.data_ptr(), ignore_index, lse.data_ptr(),
                                 d_loss.data_ptr(), _ptr(d_lse), _ptr(dx), _ptr(dw),
                                 VMI_F32 if dweight_dtype is torch.float32 else VMI_BF16, ws.data_ptr(), ws.numel(),
                                 _stream_on(x.device, None)), "vmi_head_loss_grad")
    return dx, dw
