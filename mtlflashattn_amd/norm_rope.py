"""RMS norm of query and key heads and the rotation of their positions in one HIP
pass (mfa_norm_rope), with its backward.  The reference has no counterpart: its
callers normalise and rotate with elementwise framework ops before the attention
call."""
from __future__ import annotations

import torch

from . import _hip, _kernel
from ._kernel import MAX_HEAD_DIM

_DTYPES = _kernel._SUPPORTED_DTYPES


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """Norm and rotation of every query and key head, in one launch.

    q: [B, L, Hq, D] (or packed [T, Hq, D]), k: [B, L, Hkv, D] ([T, Hkv, D]),
    fp16 / bf16 / fp32, any strides (views of a packed projection are read in
    place).  Returns (q', k'), contiguous, in the same dtype:

      n = x / sqrt(mean(x^2) + eps),  y = n * weight
      y_a cos - y_b sin, y_b cos + y_a sin    for each pair (a, b) of the rotated part

    q_weight, k_weight: [D] of any of the three dtypes (the same one), or None (1).
    cos, sin: [rows, rotary_dim / 2] tables in q.dtype or fp32; the pairs are
    (i, i + rotary_dim / 2) of the first rotary_dim <= D elements, or (2i, 2i + 1)
    with interleaved=True; the elements behind are normalised only.
    positions: int32 / int64 rows of the tables, [B, L] ([T]) or [L]; None: 0, 1,
    2, ... in each sequence.  They are read on the device: a position outside the
    tables gives NaN in the rotated elements (never a read out of bounds).
    Arithmetic is fp32, rounded once.  Differentiable in q, k and the weights
    (weight gradients are summed in fp32 in an order that sizes, strides and alignment
    decide: the same bits for the same layout); cos and sin are constants.  Forward and backward can be captured into a
    graph; as for every operator, no eager autograd graph of the same leaves may be
    alive while a backward is captured.
    """
    # (numbers, so that the signature holds a value whatever type it came in)
    plan = _plan(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
    _kernel._check_no_tangent(q, k, q_weight, k_weight, cos, sin)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (
            q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad)):
        return _QkNormRopeFn.apply(plan, float(eps), bool(interleaved), q, k, q_weight, k_weight, cos, sin, positions)
    return _forward(plan, q, k, q_weight, k_weight, cos, sin, positions)


class _Plan:
    """Of a call's signature: its parameters (everything but the data pointers),
    whether the tensors are used in place, the backward's parameters for contiguous
    gradients, and its workspace (bytes by which weights have a gradient)."""

    __slots__ = ("params", "direct", "bwd", "ws")

    def __init__(self, params, direct):
        self.params, self.direct, self.ws = params, direct, {}
        self.bwd = b = _hip.MfaNormRopeBwdParams()
        b.fwd = params
        L, D = params.seqlen, params.head_dim
        b.dqo_batch_stride, b.dqo_seq_stride, b.dqo_head_stride = L * params.heads_q * D, params.heads_q * D, D
        b.dko_batch_stride, b.dko_seq_stride, b.dko_head_stride = L * params.heads_kv * D, params.heads_kv * D, D


_plans = {}


def _plan(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    """The plan of a call, its arguments checked at their first use."""
    try:
        if cos.requires_grad or sin.requires_grad:
            raise NotImplementedError("mtlflashattn_amd: cos and sin are constants (no gradient)")
        key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, cos.shape, cos.stride(),
               cos.dtype, cos.device, sin.shape, sin.stride(), sin.dtype, sin.device, eps, interleaved,
               q_weight is not None and (q_weight.shape, q_weight.stride(), q_weight.dtype, q_weight.device),
               k_weight is not None and (k_weight.shape, k_weight.stride(), k_weight.dtype, k_weight.device),
               positions is not None and (positions.shape, positions.stride(), positions.dtype, positions.device))
    except AttributeError:
        raise ValueError("mtlflashattn_amd: q, k, cos and sin (and norm weights and positions, if given) must be "
                         "tensors") from None
    plan = _plans.get(key)
    if plan is None:
        tensors = (q, k, q_weight, k_weight, cos, sin, positions)
        p = _prepare(*tensors, eps, interleaved)
        plan = _Plan(p, all(t is _rows(t) for t in tensors) and cos.stride(0) == sin.stride(0))
        if len(_plans) >= _kernel._PLANS_MAX:
            _plans.clear()
        _plans[key] = plan
    return plan


def _check(q, k, q_weight, k_weight, cos, sin, positions, eps):
    if q.dim() not in (3, 4) or k.dim() != q.dim():
        raise ValueError(f"mtlflashattn_amd: expected q and k [B,L,H,D] or [T,H,D], got {q.dim()}-D and {k.dim()}-D")
    _kernel._check_device(q, k)
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise NotImplementedError(f"mtlflashattn_amd: dtype {q.dtype} (q/k must match, fp16/bf16/fp32)")
    D = q.shape[-1]
    if D > MAX_HEAD_DIM or D == 0:
        raise NotImplementedError(f"mtlflashattn_amd: head_dim {D} outside [1, {MAX_HEAD_DIM}]")
    if k.shape[-1] != D or k.shape[:-2] != q.shape[:-2]:
        raise ValueError(f"mtlflashattn_amd: q {tuple(q.shape)} and k {tuple(k.shape)} differ in tokens or head_dim")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if tuple(w.shape) != (D,) or w.dtype not in _DTYPES or w.dtype != weights[0].dtype:
            raise ValueError(f"mtlflashattn_amd: norm weights must be [{D}] tensors of one fp16/bf16/fp32 dtype")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dtype not in (q.dtype, torch.float32):
        raise ValueError("mtlflashattn_amd: cos and sin must be [rows, rotary_dim / 2] tables in q.dtype or fp32")
    if 2 * cos.shape[1] > D:
        raise ValueError(f"mtlflashattn_amd: rotary_dim {2 * cos.shape[1]} > head_dim {D}")
    if positions is not None:
        if not torch.is_tensor(positions) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("mtlflashattn_amd: positions must be an int32 or int64 tensor")
        if positions.shape not in (q.shape[:-2], q.shape[-3:-2]):
            raise ValueError(f"mtlflashattn_amd: positions {tuple(positions.shape)} must be {tuple(q.shape[:-2])} or "
                             f"{tuple(q.shape[-3:-2])}")
    if not eps >= 0:
        raise ValueError("mtlflashattn_amd: eps must be >= 0")
    _kernel._check_sizes(*q.shape, *k.shape, cos.shape[0])
    _kernel._check_device(q, *weights, cos, sin, *([positions] if positions is not None else []))


def _strides(t):
    """(batch, token, head) element strides of [B, L, H, D] or [T, H, D]; 0 for size-1 dims."""
    st = [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    return (0, st[0], st[1]) if len(st) == 3 else tuple(st[:3])


def _rows(t):
    """t with a contiguous last dim."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _prepare(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    _check(q, k, q_weight, k_weight, cos, sin, positions, eps)
    p = _hip.MfaNormRopeParams()
    q, k, cos, sin, positions = (_rows(t) for t in (q, k, cos, sin, positions))
    p.q_batch_stride, p.q_seq_stride, p.q_head_stride = _strides(q)
    p.k_batch_stride, p.k_seq_stride, p.k_head_stride = _strides(k)
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    p.table_stride = cos.stride(0) if cos.shape[0] > 1 and cos.shape[1] > 0 else 0
    p.batch, p.seqlen = (q.shape[0], q.shape[1]) if q.dim() == 4 else (1, q.shape[0])
    p.heads_q, p.heads_kv, p.head_dim = q.shape[-2], k.shape[-2], q.shape[-1]
    p.rotary_dim, p.table_rows = 2 * cos.shape[1], cos.shape[0]
    if positions is not None:
        p.positions_64 = int(positions.dtype == torch.int64)
        p.positions_batch_stride = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    p.interleaved = int(bool(interleaved))
    p.dtype = _hip.DTYPE_CODES[q.dtype]
    w = q_weight if q_weight is not None else k_weight
    p.dtype_weight = _hip.DTYPE_CODES[w.dtype if w is not None else q.dtype]
    p.dtype_table = _hip.DTYPE_CODES[cos.dtype]
    p.eps = eps
    return p


def _fill(p, plan, q, k, q_weight, k_weight, cos, sin, positions):
    """Sets the data pointers; returns the tensors they point into."""
    if not plan.direct:
        q, k, q_weight, k_weight, cos, sin, positions = (_rows(t) for t in (q, k, q_weight, k_weight, cos, sin, positions))
        if cos.stride(0) != sin.stride(0):
            cos, sin = cos.contiguous(), sin.contiguous()
    p.q, p.k, p.cos, p.sin = q.data_ptr(), k.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if q_weight is not None:
        p.q_weight = q_weight.data_ptr()
    if k_weight is not None:
        p.k_weight = k_weight.data_ptr()
    if positions is not None:
        p.positions = positions.data_ptr()
    return q, k, q_weight, k_weight, cos, sin, positions


def _empty(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(plan, q, k, q_weight, k_weight, cos, sin, positions):
    p = _hip.MfaNormRopeParams.from_buffer_copy(plan.params)
    held = _fill(p, plan, q, k, q_weight, k_weight, cos, sin, positions)  # noqa: F841 (kept until the launch)
    q_out, k_out = _empty(q), _empty(k)
    p.q_out, p.k_out = q_out.data_ptr(), k_out.data_ptr()
    _kernel._launch_on(q.device, _hip.norm_rope, p)
    return q_out, k_out


class _QkNormRopeFn(torch.autograd.Function):
    """qk_norm_rope with the HIP backward, which forms the statistics again from
    q and k (nothing but the inputs is kept).  The backward's plan is that of the
    tensors it gets: saved-tensor hooks (save_on_cpu, activation offload) may give
    back copies with other strides than the forward's views."""

    @staticmethod
    def forward(ctx, plan, eps, interleaved, q, k, q_weight, k_weight, cos, sin, positions):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.options = eps, interleaved
        return _forward(plan, q, k, q_weight, k_weight, cos, sin, positions)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        if q.shape != dq_out.shape or k.shape != dk_out.shape or q.device != dq_out.device:
            raise ValueError(f"mtlflashattn_amd: saved q {tuple(q.shape)} and k {tuple(k.shape)} on {q.device} came back for "
                             f"gradients {tuple(dq_out.shape)} and {tuple(dk_out.shape)} on {dq_out.device}")
        plan, device = _plan(q, k, q_weight, k_weight, cos, sin, positions, *ctx.options), q.device
        b = _hip.MfaNormRopeBwdParams.from_buffer_copy(plan.bwd)
        held = _fill(b.fwd, plan, q, k, q_weight, k_weight, cos, sin, positions)  # noqa: F841 (kept until the launch)
        if dq_out.dtype is not q.dtype or dk_out.dtype is not k.dtype:
            dq_out, dk_out = dq_out.to(q.dtype), dk_out.to(k.dtype)
        dq_out, dk_out = _rows(dq_out), _rows(dk_out)
        if not dq_out.is_contiguous():
            b.dqo_batch_stride, b.dqo_seq_stride, b.dqo_head_stride = _strides(dq_out)
        if not dk_out.is_contiguous():
            b.dko_batch_stride, b.dko_seq_stride, b.dko_head_stride = _strides(dk_out)
        b.dq_out, b.dk_out = dq_out.data_ptr(), dk_out.data_ptr()
        dq, dk = _empty(q), _empty(k)
        b.dq, b.dk = dq.data_ptr(), dk.data_ptr()
        needs = ctx.needs_input_grad
        dqw = _empty(q_weight) if q_weight is not None and needs[5] else None
        dkw = _empty(k_weight) if k_weight is not None and needs[6] else None
        if dqw is not None:
            b.dq_weight = dqw.data_ptr()
        if dkw is not None:
            b.dk_weight = dkw.data_ptr()
        which = (dqw is not None, dkw is not None)
        nbytes = plan.ws.get(which)
        if nbytes is None:
            with _kernel._on(device):
                nbytes = _hip.norm_rope_bwd_workspace_bytes(b)
            plan.ws[which] = nbytes
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _kernel._launch_on(device, _hip.norm_rope_bwd, b, None if ws is None else ws.data_ptr(), nbytes)
        return None, None, None, dq, dk, dqw, dkw, None, None, None
