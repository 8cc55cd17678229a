"""Rows sorted by expert and back, with weights and gradients (csrc/expert_rows.hip): the routing of rows to groups that have
matrices of their own -- what the class-aware head does with its voxels (ops/head_stage.class_rows), for any router.

    plan = expert_plan(ids, n_experts)             # ids [T, k], as torch.topk gives them; -1 drops a pair
    rows = expert_gather(x, plan)                  # [T * k, C]: the rows of expert e are plan.offsets[e] .. plan.offsets[e + 1]
    ...                                            # the experts' layers (me.grouped_conv, int8_linear(plan=plan), ...)
    out = expert_combine(rows, plan, weights)      # [T, C] = sum over the k slots of weights * rows

Nothing is read back to the host: the calls can be captured into a graph.  No sum uses an atomic: results and gradients are the
same from run to run.  Rows behind the last (as many as there are dropped pairs) are zeros in every output of that shape."""
import contextlib
import functools
import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import CG3DError, ptr

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int8: 3}       # CG3D_DT_*
FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_EXPERTS = 1024
MAX_COLUMNS = 1 << 30


def on_device(t):
    """The context a call on `t` is made in: the launches go to the current stream of t's device, also where another device is
    the current one."""
    if t.is_cuda and t.device.index != _lib._GET_DEVICE():
        return torch.cuda.device(t.device)
    return _HERE


_HERE = contextlib.nullcontext()


def need(ok, message, *args):
    if not ok:
        raise CG3DError(message % args)


class ExpertPlan:
    """Where the rows of a routing go.  offsets int32 [n_experts + 1], rows int32 [T * k] (the token of each row, -1 behind the
    last), pairs int32 [T * k] (the pair t * k + s of each row, negative behind the last), pos int32 [T, k] (the row of each pair;
    negative: the pair has none).  The tables lie in one allocation; the tensors are made when they are asked for."""

    __slots__ = ("device", "n_tokens", "k", "n_experts", "n_rows", "_tables", "_at")

    def __init__(self, tables, at, n_tokens, k, n_experts):
        self.device, self.n_tokens, self.k, self.n_experts, self.n_rows = tables.device, n_tokens, k, n_experts, n_tokens * k
        self._tables, self._at = tables, at

    def _slice(self, i, n):
        at = self._at + i * self.n_rows
        return self._tables[at:at + n]

    rows = property(lambda self: self._slice(0, self.n_rows))
    pairs = property(lambda self: self._slice(1, self.n_rows))
    pos = property(lambda self: self._slice(2, self.n_rows).view(self.n_tokens, self.k))
    offsets = property(lambda self: self._slice(3, self.n_experts + 1))

    def address(self, i):
        """Of table i: rows, pairs, pos, offsets."""
        return self._tables.data_ptr() + 4 * (self._at + i * self.n_rows)


ROWS, PAIRS, POS, OFFSETS = range(4)


@functools.lru_cache(maxsize=4096)
def _plan_ws_words(lib, t, k, n_experts):
    return int(lib.raw("cg3d_expert_plan_ws_bytes")(t, k, n_experts)) // 4


def expert_plan(experts, n_experts):
    """experts int32 / int64 [T, k] (or [T]): the experts of each token; an id outside [0, n_experts) has no row.  A token may
    name an expert twice: it then has two rows.  Rows are in expert order, pairs of one expert in the order of (token, slot)."""
    if not (isinstance(experts, torch.Tensor) and experts.dtype in (torch.int32, torch.int64) and experts.dim() in (1, 2)):
        raise CG3DError("expert_plan: experts must be an int32 or int64 tensor [T, k] or [T]")
    n_experts = int(n_experts)
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise CG3DError("expert_plan: n_experts = %d is not in 1 .. %d" % (n_experts, MAX_EXPERTS))
    ids = (experts if experts.dim() == 2 else experts.unsqueeze(1)).contiguous()
    t, k = ids.shape
    if k < 1 or t * k >= 2 ** 31:
        raise CG3DError("expert_plan: %d x %d pairs (k >= 1, fewer than 2^31 pairs)" % (t, k))
    lib = _lib.get()
    lib.check(ids)
    with on_device(ids):
        at = _plan_ws_words(lib, t, k, n_experts)
        tables = torch.empty(at + 3 * t * k + n_experts + 1, dtype=torch.int32, device=ids.device)      # workspace | the plan's four tables
        plan = ExpertPlan(tables, at, t, k, n_experts)
        rows = plan.address(ROWS)
        lib.call("cg3d_expert_plan", ids.data_ptr(), int(ids.dtype == torch.int64), t, k, n_experts, plan.address(OFFSETS), rows,
                 plan.address(PAIRS), plan.address(POS), rows - 4 * at if at else None, lib.stream())
    return plan


def _check_rows(who, x, n, plan, what):
    if not isinstance(plan, ExpertPlan):
        raise CG3DError("%s: plan must come from expert_plan" % who)
    if not (isinstance(x, torch.Tensor) and x.dtype in FLOATS and x.dim() == 2 and x.shape[0] == n and 1 <= x.shape[1] <= MAX_COLUMNS):
        raise CG3DError("%s: %s must be [%d, C] float32, bfloat16 or float16 with C in 1 .. 2^30, got %s" % (
            who, what, n, (x.dtype, tuple(x.shape)) if isinstance(x, torch.Tensor) else type(x)))
    if x.device != plan.device:
        raise CG3DError("%s: %s is on %s, the plan on %s" % (who, what, x.device, plan.device))


def _gather(x, plan):
    lib = _lib.get()
    x = x.contiguous()
    lib.check(x)
    with on_device(x):
        out = torch.empty((plan.n_rows, x.shape[1]), dtype=x.dtype, device=x.device)
        lib.call("cg3d_expert_gather", x.data_ptr(), DTYPES[x.dtype], plan.address(ROWS), plan.n_tokens, plan.k, x.shape[1], out.data_ptr(),
                 lib.stream())
    return out


def _combine(y, plan, w, out_dtype):
    lib = _lib.get()
    lib.check(y, w)
    with on_device(y):
        out = torch.empty((plan.n_tokens, y.shape[1]), dtype=out_dtype, device=y.device)
        lib.call("cg3d_expert_combine", y.data_ptr(), DTYPES[y.dtype], plan.address(POS), ptr(w), 0 if w is None else DTYPES[w.dtype],
                 plan.n_tokens, plan.k, y.shape[1], out.data_ptr(), DTYPES[out_dtype], lib.stream())
    return out


def _once(backward):
    """once_differentiable, whose bookkeeping (4 us a call) is for a backward pass that is itself recorded."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        return _gather(x, plan)

    @staticmethod
    @_once
    def backward(ctx, dout):
        return None if dout is None else _combine(dout.contiguous(), ctx.plan, None, dout.dtype), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, plan, w, out_dtype):
        y, w = y.contiguous(), None if w is None else w.contiguous()
        ctx.plan, ctx.dtype = plan, y.dtype
        ctx.save_for_backward(y if ctx.needs_input_grad[2] else None, w)
        ctx.set_materialize_grads(False)
        return _combine(y, plan, w, out_dtype)

    @staticmethod
    @_once
    def backward(ctx, dout):
        if dout is None:
            return None, None, None, None
        y, w = ctx.saved_tensors
        plan, c = ctx.plan, dout.shape[1]
        lib = _lib.get()
        dout = dout.to(ctx.dtype).contiguous()                  # (wider than the output where the rows are)
        with on_device(dout):
            dy = torch.empty((plan.n_rows, c), dtype=dout.dtype, device=dout.device) if ctx.needs_input_grad[0] else None
            dw = torch.empty_like(w) if ctx.needs_input_grad[2] else None
            lib.call("cg3d_expert_combine_bwd", dout.data_ptr(), ptr(y), DTYPES[dout.dtype], plan.address(PAIRS), ptr(w),
                     0 if w is None else DTYPES[w.dtype], plan.n_tokens, plan.k, c, ptr(dy), ptr(dw), lib.stream())
        return dy, None, dw, None


def expert_gather(x, plan):
    """x [T, C] float32 / bfloat16 / float16 -> [T * k, C], the tokens' rows in the plan's order (differentiable in x)."""
    _check_rows("expert_gather", x, getattr(plan, "n_tokens", 0), plan, "x")
    if not (x.requires_grad and torch.is_grad_enabled()):
        return _gather(x, plan)
    return _Gather.apply(x, plan)


def expert_combine(rows, plan, weights=None, out_dtype=None):
    """rows [T * k, C] in the plan's order -> [T, C]: out[t] = sum_s weights[t, s] * rows[pos[t, s]] over the slots that have a
    row, summed in float32 in slot order and rounded once, to out_dtype (default: the rows' own; float32 rows: any of the three)
    -- differentiable in rows and weights.  weights [T, k] float32 / bfloat16 / float16; None: all ones."""
    _check_rows("expert_combine", rows, getattr(plan, "n_rows", 0), plan, "rows")
    out_dtype = out_dtype or rows.dtype
    need(out_dtype == rows.dtype or (rows.dtype == torch.float32 and out_dtype in FLOATS), "expert_combine: out_dtype must be the rows' own, "
         "or float32, bfloat16 or float16 for float32 rows")
    if weights is not None:
        need(isinstance(weights, torch.Tensor) and weights.dtype in FLOATS, "expert_combine: weights must be float32, bfloat16 or float16")
        if weights.dim() == 1 and plan.k == 1:
            weights = weights.unsqueeze(1)
        if weights.shape != (plan.n_tokens, plan.k) or weights.device != rows.device:
            raise CG3DError("expert_combine: weights must be [%d, %d] on %s, got %s on %s" % (plan.n_tokens, plan.k, rows.device,
                                                                                              tuple(weights.shape), weights.device))
    if not (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))):
        return _combine(rows.contiguous(), plan, None if weights is None else weights.contiguous(), out_dtype)
    return _Combine.apply(rows, plan, weights, out_dtype)
