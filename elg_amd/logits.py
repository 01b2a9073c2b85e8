"""Row operators over node logits and probabilities: a teacher's best logits, the loss that distils a policy from them, and the
verification of drafted choices.  They work on rows as `engine.rollout_forward(..., dump="logits" / "probs")` returns them -- closed nodes
-inf / 0 -- and on any other rows of 1 to 2^24 entries in f32, bf16 or f16.

    values, idx, tail = top_logits(teacher_logits, 40, temperature=2.0, with_tail=True)   # once per teacher rollout; 8 bytes per kept logit
    loss = distill_loss(student_logits, values, idx, tail=tail, temperature=2.0)          # differentiable in the student's logits
    loss, grad = distill_loss_grad(student_logits, values, idx, tail=tail, temperature=2.0)   # loss and gradient from one read of the logits
    tokens, accepted = verify_draft(target_probs, drafted, uniforms, draft_probs=draft_probs)

Each is one call into libelg_hip.so (include/elg_hip.h) on the current stream, without a host synchronisation: capturable.  Inputs must
live on the current device; rows may be strided views (the last dimension contiguous), others are copied."""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import _lib as L
from .engine import _need_cuda

_TYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # a tenth of the time of current_stream()'s object


def _stream() -> int:
    """The current stream of the current device (which every input has been checked to live on)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


@functools.lru_cache(maxsize=256)
def _distill_ws_bytes(R: int, V: int, ty: int) -> int:
    return int(L.lib().elg_distill_ws_bytes(R, V, ty))


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _type(t: torch.Tensor, what: str) -> int:
    """The element type of a call's first tensor, which must live on the current device."""
    _need_cuda(t, what)
    ty = _TYPES.get(t.dtype)
    if ty is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return ty


def _beside(t: torch.Tensor, dev: int, what: str):
    """Another tensor of the call: on the same device `dev`, which is the current one."""
    if t.get_device() != dev:
        _need_cuda(t, what)


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """(..., V) as (R, V) with a contiguous last dimension; a view wherever the strides allow one."""
    if t.dim() == 0 or not 1 <= t.shape[-1] <= L.ROW_MAX_V:
        raise ValueError(f"{what} must have rows of 1 .. {L.ROW_MAX_V} entries, got shape {tuple(t.shape)}")
    if t.dim() != 2:
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _temperature(t: float) -> float:
    t = float(t)
    if not 1e-15 <= t <= 1e15:
        raise ValueError(f"the temperature must lie in 1e-15 .. 1e15, got {t}")
    return t


def _per_row(t: Optional[torch.Tensor], lead, dev: int, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    _beside(t, dev, what)
    if t.shape != lead:
        raise ValueError(f"{what} must hold one number per row: {tuple(lead)}, got {tuple(t.shape)}")
    if t.dtype != torch.float32:
        raise ValueError(f"{what} must be float32, got {t.dtype}")
    return t.contiguous()


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0, with_tail: bool = False) -> Tuple[torch.Tensor, ...]:
    """The k best logits of each row: (values (..., k) of the logits' type, idx (..., k) int32), best first; equal logits by the lower
    index, NaN above +inf.  with_tail adds the probability under softmax(logits / temperature) of the nodes not among the k, (...) f32 --
    what `distill_loss` takes as `tail`.  1 <= k <= min(V, 256).  A row with fewer than k open nodes is filled up with its closed ones
    (-inf), lowest index first.  No gradient flows through (the teacher is a constant)."""
    ty = _type(logits, "logits")
    temperature = _temperature(temperature)
    z = _rows(logits, "logits")
    R, V = z.shape
    k = int(k)
    if not 1 <= k <= min(V, L.TOP_MAX_K):
        raise ValueError(f"k must be 1 .. min(V, {L.TOP_MAX_K}), got k = {k} for rows of {V}")
    lead = logits.shape[:-1]
    values = z.new_empty((*lead, k))
    idx = z.new_empty((*lead, k), dtype=torch.int32)
    tail = z.new_empty(lead, dtype=torch.float32) if with_tail else None
    L.check(L.lib().elg_top_logits(_p(z), z.stride(0), ty, R, V, k, temperature, _p(values), _p(idx), _p(tail), _stream()),
            "elg_top_logits")
    return (values, idx, tail) if with_tail else (values, idx)


class _Teacher:
    """The checked arguments of a distillation call."""

    def __init__(self, logits, values, idx, tail, temperature, weight):
        self.type = _type(logits, "logits")
        dev = logits.get_device()
        _beside(values, dev, "top_values")
        _beside(idx, dev, "top_idx")
        if values.dtype not in _TYPES:
            raise ValueError(f"top_values must be float32, bfloat16 or float16, got {values.dtype}")
        if idx.dtype is not torch.int32 and idx.dtype is not torch.int64:
            raise ValueError(f"top_idx must be int32 or int64, got {idx.dtype}")
        lead = logits.shape[:-1]
        if values.shape != idx.shape or values.dim() == 0 or values.shape[:-1] != lead:
            raise ValueError(f"top_values and top_idx must be {tuple(lead)} + (k,), got {tuple(values.shape)} and {tuple(idx.shape)}")
        if not 1 <= values.shape[-1] <= L.TOP_MAX_K:
            raise ValueError(f"1 .. {L.TOP_MAX_K} teacher entries a row, got {values.shape[-1]}")
        if (values.requires_grad or (tail is not None and tail.requires_grad) or (weight is not None and weight.requires_grad)) \
                and torch.is_grad_enabled():
            raise ValueError("no gradient flows to the teacher's logits, the tail or the weights: detach them")
        self.values, self.idx = values.contiguous(), idx.contiguous()
        self.tail = _per_row(tail, lead, dev, "tail")
        self.weight = _per_row(weight, lead, dev, "weight")
        self.temperature = _temperature(temperature)
        self.lead = lead

    def tensors(self):
        return self.values, self.idx, self.tail, self.weight


def _distill_call(z, ty, teacher, temperature, *, cot=None, cot_stride=0, scale=1.0, rows=None, total=None, grad=None):
    values, idx, tail, weight = teacher
    R, V = z.shape
    ws, n = None, 0
    lib = L.lib()
    if total is not None or V > 2048:
        n = _distill_ws_bytes(R, V, ty)
        ws = z.new_empty(n, dtype=torch.uint8) if n else None
    L.check(lib.elg_distill_loss_grad(_p(z), z.stride(0), ty, R, V, _p(values), _TYPES[values.dtype], _p(idx), int(idx.dtype == torch.int64),
                                      values.shape[-1], _p(tail), temperature, _p(weight), _p(cot), cot_stride, scale, _p(rows), _p(total),
                                      _p(grad), _p(ws), n, _stream()), "elg_distill_loss_grad")


def _scale(reduction: str, R: int) -> float:
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    return 1.0 / R if reduction == "mean" and R > 0 else 1.0


class _DistillLoss(torch.autograd.Function):
    """Forward: the loss from one read of the logits.  Backward: the gradient from a second one, scaled by the cotangent on the device."""

    @staticmethod
    def forward(ctx, logits, teacher, reduction, values, idx, tail, weight):
        z = _rows(logits, "logits")
        scale = _scale(reduction, z.shape[0])
        ctx.dtype, ctx.temperature, ctx.scale, ctx.reduction, ctx.shape = logits.dtype, teacher.temperature, scale, reduction, values.shape
        # the teacher's tensors too, and nothing beside: writing to one before the backward is an error, not a wrong gradient, hooks on saved
        # tensors see what the backward reads, and it is all freed with the graph
        ctx.save_for_backward(logits, values, idx, tail, weight)
        if reduction == "none":
            loss = z.new_empty(teacher.lead, dtype=torch.float32)
            if z.shape[0]:
                _distill_call(z, teacher.type, (values, idx, tail, weight), teacher.temperature, rows=loss)
        else:
            loss = z.new_empty((), dtype=torch.float32)
            _distill_call(z, teacher.type, (values, idx, tail, weight), teacher.temperature, total=loss, scale=scale)
        return loss

    @staticmethod
    def gradient(ctx, gout):
        logits, values, idx, tail, weight = ctx.saved_tensors
        # what a hook gives back goes to the kernel by its address: it has to be what was saved
        dev, lead = gout.get_device(), ctx.shape[:-1]
        if logits.shape[:-1] != lead or logits.get_device() != dev or logits.dtype is not ctx.dtype or values.shape != ctx.shape \
                or values.get_device() != dev or values.dtype not in _TYPES or idx.shape != ctx.shape or idx.get_device() != dev \
                or (idx.dtype is not torch.int32 and idx.dtype is not torch.int64):
            raise RuntimeError("elg_amd: a hook on saved tensors gave back other logits or another teacher than were saved")
        for t in (tail, weight):
            if t is not None and (t.shape != lead or t.get_device() != dev or t.dtype is not torch.float32):
                raise RuntimeError("elg_amd: a hook on saved tensors gave back another tail or weight than was saved")
        z = _rows(logits, "logits")
        grad = z.new_empty(logits.shape)
        if z.shape[0]:
            if gout.dtype != torch.float32 or not gout.is_contiguous():
                gout = gout.float().contiguous()
            teacher = (values.contiguous(), idx.contiguous(), None if tail is None else tail.contiguous(),
                       None if weight is None else weight.contiguous())
            _distill_call(z, _TYPES[z.dtype], teacher, ctx.temperature, cot=gout, cot_stride=int(ctx.reduction == "none"), scale=ctx.scale, grad=grad)
        return grad, None, None, None, None, None, None

    @staticmethod
    def backward(ctx, gout):
        # only a backward that builds a graph (create_graph=True) needs its outputs marked as differentiable no further
        return _distill_gradient_once(ctx, gout) if torch.is_grad_enabled() else _DistillLoss.gradient(ctx, gout)


_distill_gradient_once = torch.autograd.function.once_differentiable(_DistillLoss.gradient)


def distill_loss(logits: torch.Tensor, top_values: torch.Tensor, top_idx: torch.Tensor, *, tail: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, weight: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """Distillation of `logits` (..., V) from a teacher's best logits top_values (..., k) at nodes top_idx (..., k):

        q = (1 - tail) softmax(top_values / T),   p = softmax(logits / T)
        L = T^2 weight [ sum_j q_j (log q_j - log p_{i_j})  +  tail (log tail - log p(no entry's node)) ]

    per row; reduction 'none' (...) f32, 'sum', or 'mean' over all rows (0 where there are none). tail (...) f32: the teacher's probability
    outside its entries at the same temperature (`top_logits(with_tail=True)`), None: the entries hold everything. weight (...) f32: 0
    leaves a row out (it is not read) -- finished trajectories. Entries whose node lies outside [0, V) are absent: -1 is padding. An entry
    whose logit is -inf has mass 0, and its node is an entry's all the same, not one of the rest that the tail is spread over. A node listed
    twice carries both masses. Rows without an open node or without an entry above -inf give loss 0 and gradient 0; a teacher probability on
    a closed node gives +inf.

    The gradient reaches `logits` only, in their type, and can be taken once (no double backward); statistics and sums are f32, the sum over
    the rows f64: a loss that cancels is exact to about 1e-7 T^2.  Hooks on saved tensors see the logits and the teacher's tensors."""
    t = _Teacher(logits, top_values, top_idx, tail, temperature, weight)
    return _DistillLoss.apply(logits, t, reduction, *t.tensors())


def distill_loss_grad(logits: torch.Tensor, top_values: torch.Tensor, top_idx: torch.Tensor, *, tail: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, weight: Optional[torch.Tensor] = None,
                      reduction: str = "mean") -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, d loss / d logits) of `distill_loss` in one pass over the logits: for training loops that hand the gradient on themselves
    (`logits.backward(grad)`), with the loss's own cotangent 1.  With reduction 'none' the gradient is that of the rows' sum."""
    t = _Teacher(logits, top_values, top_idx, tail, temperature, weight)
    z = _rows(logits, "logits")
    scale = _scale(reduction, z.shape[0])
    grad = z.new_empty(logits.shape)
    if reduction == "none":
        loss = z.new_empty(t.lead, dtype=torch.float32)
        if z.shape[0]:
            _distill_call(z, t.type, t.tensors(), t.temperature, rows=loss, grad=grad)
    else:
        loss = z.new_empty((), dtype=torch.float32)
        _distill_call(z, t.type, t.tensors(), t.temperature, total=loss, grad=grad, scale=scale)
    return loss, grad


def _steps(t: torch.Tensor) -> torch.Tensor:
    """(..., S, V) as (B, S, V) with a contiguous last dimension; a view wherever the strides allow one."""
    if t.dim() != 3:
        t = t.reshape(t.shape[:-2].numel(), *t.shape[-2:])
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def verify_draft(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor, *,
                 draft_probs: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted choices the target keeps, and what it answers instead of the first one it does not: speculative sampling from given
    uniforms.  target_probs (..., G + 1, V): the target's probabilities at each draft and after the last; draft_tokens (..., G) int32 /
    int64; uniforms (..., G + 1) f32 in [0, 1): one per acceptance test and, last, one for the draw; draft_probs (..., G, V) of the same
    type, or None where the drafts were certain (greedy); lengths (...) int32 / int64: drafts of each sequence (clamped to 0 .. G), None: all G.

    Returns tokens (..., G + 1) int32 -- the accepted drafts, the drawn choice, then -1 -- and accepted (...) int32.  A draft is kept while
    u q(x) < p(x) (exact, in 64 bits); the draw is from max(p - q, 0) at the refused draft, from the target's next row if none was refused,
    from the target's own row where nothing is left of it over the draft, and -1 where that row is empty.  A token outside [0, V) is refused."""
    ty = _type(target_probs, "target_probs")
    dev = target_probs.get_device()
    _beside(draft_tokens, dev, "draft_tokens")
    _beside(uniforms, dev, "uniforms")
    if draft_tokens.dtype is not torch.int32 and draft_tokens.dtype is not torch.int64:
        raise ValueError(f"draft_tokens must be int32 or int64, got {draft_tokens.dtype}")
    if uniforms.dtype != torch.float32:
        raise ValueError(f"uniforms must be float32, got {uniforms.dtype}")
    if draft_tokens.dim() == 0 or target_probs.dim() < 2:
        raise ValueError("draft_tokens is (..., G), target_probs (..., G + 1, V)")
    lead, G = draft_tokens.shape[:-1], draft_tokens.shape[-1]
    V = target_probs.shape[-1]
    if G > L.DRAFT_MAX or not 1 <= V <= L.ROW_MAX_V:
        raise ValueError(f"up to {L.DRAFT_MAX} drafts over rows of 1 .. {L.ROW_MAX_V} probabilities, got {G} over {V}")
    if target_probs.shape != (*lead, G + 1, V) or uniforms.shape != (*lead, G + 1):
        raise ValueError(f"target_probs must be {(*lead, G + 1, V)} and uniforms {(*lead, G + 1)}, got {tuple(target_probs.shape)} "
                         f"and {tuple(uniforms.shape)}")
    p = _steps(target_probs)
    q = None
    if draft_probs is not None and G > 0:
        if draft_probs.shape != (*lead, G, V) or draft_probs.dtype != target_probs.dtype:
            raise ValueError(f"draft_probs must be {(*lead, G, V)} of {target_probs.dtype}, got {tuple(draft_probs.shape)} of {draft_probs.dtype}")
        _beside(draft_probs, dev, "draft_probs")
        q = _steps(draft_probs)
    B = p.shape[0]
    x, u = draft_tokens.contiguous(), uniforms.contiguous()
    if lengths is not None:
        _beside(lengths, dev, "lengths")
        if lengths.shape != lead or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths must be {tuple(lead)} int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")
        if lengths.dtype is torch.int64:
            lengths = lengths.clamp(0, G).to(torch.int32)       # clamped before it is cut to 32 bits
        lengths = lengths.contiguous()
    tokens = p.new_empty((*lead, G + 1), dtype=torch.int32)
    accepted = p.new_empty(lead, dtype=torch.int32)
    lib, ws, n = L.lib(), None, 0
    if V > 1024:
        n = lib.elg_verify_ws_bytes(B, V, ty)
        ws = p.new_empty(n, dtype=torch.uint8) if n else None
    L.check(lib.elg_verify_draft(_p(p), p.stride(0), p.stride(1), _p(q), q.stride(0) if q is not None else 0,
                                     q.stride(1) if q is not None else 0, ty, _p(x), int(x.dtype == torch.int64), G, _p(u), G + 1,
                                     _p(lengths), B, G, V, _p(tokens), _p(accepted), _p(ws), n, _stream()), "elg_verify_draft")
    return tokens, accepted
