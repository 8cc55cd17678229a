"""Rows sorted by expert and back, with weights and gradients (csrc/expert_rows.hip): the routing of rows to groups that have
matrices of their own -- what the class-aware head does with its voxels (ops/head_stage.class_rows), for any router.

    plan = expert_plan(ids, n_experts)             # ids [T, k], as torch.topk gives them; -1 drops a pair
    rows = expert_gather(x, plan)                  # [T * k, C]: the rows of expert e are plan.offsets[e] .. plan.offsets[e + 1]
    ...                                            # the experts' layers (me.grouped_conv, int8_linear(plan=plan), ...)
    out = expert_combine(rows, plan, weights)      # [T, C] = sum over the k slots of weights * rows

Nothing is read back to the host: the calls can be captured into a graph.  torch.jit.trace records gather and combination (the plan
is made outside of it); there is no forward-mode derivative and no second one.  No sum uses an atomic: results and gradients are the
same from run to run.  Rows behind the last (as many as there are dropped pairs) are zeros in every output of that shape."""
import contextlib
import functools
import torch
from torch.autograd import forward_ad
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


_TRACING = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing
_MODES = getattr(torch._C, "_len_torch_dispatch_stack", None) or (lambda: 0)


def recorded():
    """Whether torch has to see the call also without gradients: torch.jit.trace records it, forward-mode differentiation has its
    tangents refused -- both where it goes through an autograd.Function.  (The kernels take addresses: of a call that goes to them
    directly a trace holds nothing but an uninitialised output.)  A graph of torch's own operators cannot hold it at all."""
    if _MODES():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if get_proxy_mode() is not None:
            raise CG3DError("the operators take the addresses of their inputs: a graph of torch's own operators (make_fx) cannot hold them")
    return forward_ad._current_level >= 0 or _TRACING()


def whole(t):
    """t contiguous, its memory holding its values (that of a lazily negated view holds the opposite ones)."""
    return t.resolve_neg().contiguous() if t.is_neg() else t if t.is_contiguous() else t.contiguous()


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

    def address(self, i, tables=None):
        """Of table i: rows, pairs, pos, offsets -- in `tables`, a saved form of them."""
        return (self._tables if tables is None else tables).data_ptr() + 4 * (self._at + i * self.n_rows)

    def to_save(self):
        """The tables as a saved tensor of a pass, so that one that is written before its backward pass is noticed (None for a plan made
        in inference mode, whose tensors autograd neither saves nor watches)."""
        return None if self._tables.is_inference() else self._tables


ROWS, PAIRS, POS, OFFSETS = range(4)


@functools.lru_cache(maxsize=4096)
def _plan_ws_words(lib, t, k, n_experts):
    return int(lib.raw("cg3d_expert_plan_ws_bytes")(t, k, n_experts)) // 4


def expert_plan(experts, n_experts):
    """experts int32 / int64 [T, k] (or [T]): the experts of each token; an id outside [0, n_experts) has no row.  A token may
    name an expert twice: it then has two rows.  Rows are in expert order, pairs of one expert in the order of (token, slot)."""
    if recorded() and _TRACING():
        raise CG3DError("expert_plan: a trace would keep the plan of the ids it was made with; make the plan outside the trace")
    if not (isinstance(experts, torch.Tensor) and experts.dtype in (torch.int32, torch.int64) and experts.dim() in (1, 2)):
        raise CG3DError("expert_plan: experts must be an int32 or int64 tensor [T, k] or [T]")
    n_experts = int(n_experts)
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise CG3DError("expert_plan: n_experts = %d is not in 1 .. %d" % (n_experts, MAX_EXPERTS))
    ids = whole(experts if experts.dim() == 2 else experts.unsqueeze(1))
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
    # (named behind the launch, here and in the passes: torch.compile stops at an address and resumes with what the rest of the function
    # names, so that it would free copies of inputs before the launch)
    del ids
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
    _check_rows("expert_gather", x, getattr(plan, "n_tokens", 0), plan, "x")
    lib = _lib.get()
    x = whole(x)
    lib.check(x)
    with on_device(x):
        c = x.shape[1]
        c = c if type(c) is int else int(c)                     # (in a trace)
        out = torch.empty((plan.n_rows, c), dtype=x.dtype, device=x.device)
        lib.call("cg3d_expert_gather", x.data_ptr(), DTYPES[x.dtype], plan.address(ROWS), plan.n_tokens, plan.k, c, out.data_ptr(),
                 lib.stream())
    del x, plan
    return out


def _combine_inputs(rows, plan, weights, out_dtype):
    """-> rows and weights [T, k] as the kernels take them, the output's type."""
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
        weights = whole(weights)
    return whole(rows), weights, out_dtype


def _combine(y, plan, w, out_dtype, tables=None):
    lib = _lib.get()
    lib.check(y, w)
    with on_device(y):
        c = y.shape[1]
        c = c if type(c) is int else int(c)
        out = torch.empty((plan.n_tokens, c), dtype=out_dtype, device=y.device)
        lib.call("cg3d_expert_combine", y.data_ptr(), DTYPES[y.dtype], plan.address(POS, tables), ptr(w), 0 if w is None else DTYPES[w.dtype],
                 plan.n_tokens, plan.k, c, out.data_ptr(), DTYPES[out_dtype], lib.stream())
    del y, w, plan, tables
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
        out = _gather(x, plan)
        ctx.plan = plan
        ctx.save_for_backward(plan.to_save())
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        if dout is None:
            return None, None
        tables, = ctx.saved_tensors
        return _combine(whole(dout), ctx.plan, None, dout.dtype, tables), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, plan, weights, out_dtype):
        y, w, out_dtype = _combine_inputs(rows, plan, weights, out_dtype)
        ctx.plan, ctx.dtype, ctx.w_shape = plan, y.dtype, None if w is None else weights.shape
        ctx.save_for_backward(y if ctx.needs_input_grad[2] else None, w, plan.to_save())
        ctx.set_materialize_grads(False)
        return _combine(y, plan, w, out_dtype)

    @staticmethod
    @_once
    def backward(ctx, dout):
        if dout is None:
            return None, None, None, None
        y, w, tables = ctx.saved_tensors
        plan, c = ctx.plan, dout.shape[1]
        lib = _lib.get()
        dout = whole(dout.to(ctx.dtype))                        # (wider than the output where the rows are)
        lib.check(dout, y, w, tables)                           # (what hooks of saved tensors gave back)
        with on_device(dout):
            dy = torch.empty((plan.n_rows, c), dtype=dout.dtype, device=dout.device) if ctx.needs_input_grad[0] else None
            dw = torch.empty_like(w) if ctx.needs_input_grad[2] else None
            lib.call("cg3d_expert_combine_bwd", dout.data_ptr(), ptr(y), DTYPES[dout.dtype], plan.address(PAIRS, tables), ptr(w),
                     0 if w is None else DTYPES[w.dtype], plan.n_tokens, plan.k, c, ptr(dy), ptr(dw), lib.stream())
        return dy, None, None if dw is None else dw.view(ctx.w_shape), None


def expert_gather(x, plan):
    """x [T, C] float32 / bfloat16 / float16 -> [T * k, C], the tokens' rows in the plan's order (differentiable in x)."""
    if recorded() or (torch.is_grad_enabled() and getattr(x, "requires_grad", False)):
        return _Gather.apply(x, plan)
    return _gather(x, plan)


def expert_combine(rows, plan, weights=None, out_dtype=None):
    """rows [T * k, C] in the plan's order -> [T, C]: out[t] = sum_s weights[t, s] * rows[pos[t, s]] over the slots that have a
    row, summed in float32 in slot order and rounded once, to out_dtype (default: the rows' own; float32 rows: any of the three)
    -- differentiable in rows and weights.  weights [T, k] float32 / bfloat16 / float16; None: all ones."""
    if recorded() or (torch.is_grad_enabled() and (getattr(rows, "requires_grad", False) or getattr(weights, "requires_grad", False))):
        return _Combine.apply(rows, plan, weights, out_dtype)
    rows, weights, out_dtype = _combine_inputs(rows, plan, weights, out_dtype)
    return _combine(rows, plan, weights, out_dtype)
