"""Rows sorted by expert and back, with weights and gradients (csrc/expert_rows.hip): the routing of rows to groups that have
matrices of their own -- what the class-aware head does with its voxels (ops/head_stage.class_rows), for any router.

    plan = expert_plan(ids, n_experts)             # ids [T, k], as torch.topk gives them; -1 drops a pair
    rows = expert_gather(x, plan)                  # [T * k, C]: the rows of expert e are plan.offsets[e] .. plan.offsets[e + 1]
    ...                                            # the experts' layers (me.grouped_conv, int8_linear(plan=plan), ...)
    out = expert_combine(rows, plan, weights)      # [T, C] = sum over the k slots of weights * rows

Nothing is read back to the host: the calls can be captured into a graph.  No sum uses an atomic: results and gradients are the
same from run to run.  Rows behind the last (as many as there are dropped pairs) are zeros in every output of that shape."""
import contextlib
import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import CG3DError, ptr

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int8: 3}       # CG3D_DT_*
FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_EXPERTS = 1024


def on_device(t):
    """The context a call on `t` is made in: the launches go to the current stream of t's device, also where another device is
    the current one."""
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return contextlib.nullcontext()


def need(ok, message, *args):
    if not ok:
        raise CG3DError(message % args)


class ExpertPlan:
    """Where the rows of a routing go.  offsets int32 [n_experts + 1], rows int32 [T * k] (the token of each row, -1 behind the
    last), pairs int32 [T * k] (the pair t * k + s of each row, negative behind the last), pos int32 [T, k] (the row of each pair;
    negative: the pair has none)."""

    __slots__ = ("offsets", "rows", "pairs", "pos", "n_tokens", "k", "n_experts")

    def __init__(self, offsets, rows, pairs, pos, n_experts):
        self.offsets, self.rows, self.pairs, self.pos, self.n_experts = offsets, rows, pairs, pos, n_experts
        self.n_tokens, self.k = pos.shape

    @property
    def n_rows(self):
        return self.n_tokens * self.k


def expert_plan(experts, n_experts):
    """experts int32 / int64 [T, k] (or [T]): the experts of each token; an id outside [0, n_experts) has no row.  A token may
    name an expert twice: it then has two rows.  Rows are in expert order, pairs of one expert in the order of (token, slot)."""
    need(isinstance(experts, torch.Tensor) and experts.dtype in (torch.int32, torch.int64) and experts.dim() in (1, 2),
         "expert_plan: experts must be an int32 or int64 tensor [T, k] or [T]")
    n_experts = int(n_experts)
    need(1 <= n_experts <= MAX_EXPERTS, "expert_plan: n_experts = %d is not in 1 .. %d", n_experts, MAX_EXPERTS)
    ids = (experts if experts.dim() == 2 else experts.unsqueeze(1)).contiguous()
    t, k = ids.shape
    need(k >= 1 and t * k < 2 ** 31, "expert_plan: experts of shape %s (k >= 1, fewer than 2^31 pairs)", tuple(experts.shape))
    lib = _lib.get()
    lib.check(ids)
    with on_device(ids):
        ws_bytes = int(lib.raw("cg3d_expert_plan_ws_bytes")(t, k, n_experts))
        n = t * k
        n_ws = ws_bytes // 4
        out = torch.empty(n_ws + 3 * n + n_experts + 1, dtype=torch.int32, device=ids.device)
        _, rows, pairs, pos, offsets = out.split((n_ws, n, n, n, n_experts + 1))
        pos = pos.view(t, k)
        ws = ptr(out) if n_ws else None
        lib.call("cg3d_expert_plan", ptr(ids), int(ids.dtype == torch.int64), t, k, n_experts, ptr(offsets),
                 ptr(rows), ptr(pairs), ptr(pos), ws, lib.stream())
    return ExpertPlan(offsets, rows, pairs, pos, n_experts)


def _check_rows(who, x, n, plan, what):
    need(isinstance(plan, ExpertPlan), "%s: plan must come from expert_plan", who)
    need(isinstance(x, torch.Tensor) and x.dtype in FLOATS, "%s: %s must be float32, bfloat16 or float16", who, what)
    need(x.dim() == 2 and x.shape[0] == n and x.shape[1] >= 1, "%s: %s must be [%d, C], got %s", who, what, n, tuple(x.shape))
    need(x.device == plan.pos.device, "%s: %s is on %s, the plan on %s", who, what, x.device, plan.pos.device)


def _gather(x, pos, rows):
    lib = _lib.get()
    x = x.contiguous()
    lib.check(x, rows)
    t, k = pos.shape
    with on_device(x):
        out = torch.empty((t * k, x.shape[1]), dtype=x.dtype, device=x.device)
        lib.call("cg3d_expert_gather", ptr(x), DTYPES[x.dtype], ptr(rows), t, k, x.shape[1], ptr(out), lib.stream())
    return out


def _combine(y, pos, w):
    lib = _lib.get()
    lib.check(y, pos, w)
    t, k = pos.shape
    with on_device(y):
        out = torch.empty((t, y.shape[1]), dtype=y.dtype, device=y.device)
        lib.call("cg3d_expert_combine", ptr(y), DTYPES[y.dtype], ptr(pos), ptr(w), 0 if w is None else DTYPES[w.dtype], t, k, y.shape[1],
                 ptr(out), lib.stream())
    return out


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, rows):
        ctx.save_for_backward(pos)
        ctx.set_materialize_grads(False)
        return _gather(x, pos, rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return None if dout is None else _combine(dout.contiguous(), ctx.saved_tensors[0], None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, pos, pairs, w):
        y, w = y.contiguous(), None if w is None else w.contiguous()
        ctx.save_for_backward(y if ctx.needs_input_grad[3] else None, pairs, w)
        ctx.shape = pos.shape
        ctx.set_materialize_grads(False)
        return _combine(y, pos, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        if dout is None:
            return None, None, None, None
        y, pairs, w = ctx.saved_tensors
        (t, k), c = ctx.shape, dout.shape[1]
        need_dy, _, _, need_dw = ctx.needs_input_grad
        lib = _lib.get()
        dout = dout.contiguous()
        with on_device(dout):
            dy = torch.empty((t * k, c), dtype=dout.dtype, device=dout.device) if need_dy else None
            dw = torch.empty_like(w) if need_dw else None
            lib.call("cg3d_expert_combine_bwd", ptr(dout), ptr(y), DTYPES[dout.dtype], ptr(pairs), ptr(w), 0 if w is None else DTYPES[w.dtype], t, k, c,
                     ptr(dy), ptr(dw), lib.stream())
        return dy, None, None, dw


def expert_gather(x, plan):
    """x [T, C] float32 / bfloat16 / float16 -> [T * k, C], the tokens' rows in the plan's order (differentiable in x)."""
    _check_rows("expert_gather", x, getattr(plan, "n_tokens", 0), plan, "x")
    if not (x.requires_grad and torch.is_grad_enabled()):
        return _gather(x, plan.pos, plan.rows)
    return _Gather.apply(x, plan.pos, plan.rows)


def expert_combine(rows, plan, weights=None):
    """rows [T * k, C] in the plan's order -> [T, C]: out[t] = sum_s weights[t, s] * rows[pos[t, s]] over the slots that have a
    row, summed in float32 in slot order (differentiable in rows and weights).  weights [T, k] float32 / bfloat16 / float16;
    None: all ones."""
    _check_rows("expert_combine", rows, getattr(plan, "n_rows", 0), plan, "rows")
    if weights is not None:
        need(isinstance(weights, torch.Tensor) and weights.dtype in FLOATS, "expert_combine: weights must be float32, bfloat16 or float16")
        if weights.dim() == 1 and plan.k == 1:
            weights = weights.unsqueeze(1)
        need(tuple(weights.shape) == (plan.n_tokens, plan.k), "expert_combine: weights must be [%d, %d], got %s", plan.n_tokens, plan.k,
             tuple(weights.shape))
        need(weights.device == rows.device, "expert_combine: weights are on %s, rows on %s", weights.device, rows.device)
    if not (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))):
        return _combine(rows.contiguous(), plan.pos, None if weights is None else weights.contiguous())
    return _Combine.apply(rows, plan.pos, plan.pairs, weights)
