"""Products in 8-bit integers with a scale for each row and each output channel (csrc/int8_linear.hip), dense or with a matrix of
its own for each expert's rows: the served form of the kernel-size-1 convolutions, the RoI contraction and the per-class products.

    weight = int8_weight(conv.kernel)                       # once: [cin, cout] (or [E, cin, cout]), quantised per output channel
    y = int8_linear(x, weight, bias)                        # rows in floats are quantised per row in the call
    q, scale = quantize_rows(x)                             # or once for several products:
    y = int8_linear(q, weight, bias, scale=scale, out_dtype=torch.bfloat16)
    y = int8_linear(x, weight, plan=plan, gather=True)      # each expert's tokens with its matrix (ops/expert_rows.expert_plan)

Results are rounded to the rows' own type unless out_dtype says otherwise.  Rows of 16 bits that are to be combined are therefore rounded
twice, before and after the weighted sum (bf16: results 0.0023 off instead of 0.0016, in the 2-norm), for half the memory traffic between
the two; rounded once:

    y = int8_linear(x, weight, plan=plan, gather=True, out_dtype=torch.float32)
    out = expert_combine(y, plan, gate, out_dtype=x.dtype)

The integer sums are exact, so results do not depend on how the work is split.  There is no gradient: a call on inputs that require
one, with gradients enabled, or that carry a tangent is refused.  torch.jit.trace records the calls; weights are laid out and plans
made outside of it."""
import functools

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import CG3DError, ptr
from .expert_rows import DTYPES, FLOATS, OFFSETS, ROWS, ExpertPlan, need, on_device, recorded, whole

ROWS_IN = tuple(DTYPES)
MAX_CIN = 131071                  # the int32 sum of so many products of 8-bit values cannot overflow


def _no_grad_for(who, wanted):
    if wanted and torch.is_grad_enabled():
        raise CG3DError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % who)


def _no_tangent_for(who, *tensors):
    for t in tensors:
        if forward_ad._current_level >= 0 and isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
            raise CG3DError("%s has no forward-mode derivative" % who)


def _record(who, f, args, tensors):
    tensors = [t for t in tensors if isinstance(t, torch.Tensor)]
    _no_grad_for(who, any(t.requires_grad for t in tensors))
    _no_tangent_for(who, *tensors)
    return _Recorded.apply(f, *args)


class _Recorded(torch.autograd.Function):
    """A call that torch.jit.trace has to see: f(*args), which has no gradient."""

    @staticmethod
    def forward(ctx, f, *args):
        return f(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise CG3DError("products in 8 bits have no gradient")


class Int8Weight:
    """Weights in the product kernels' order.  packed int8 (cg3d_int8_weight_bytes), scale float32 [E, cout]."""

    __slots__ = ("packed", "scale", "n_experts", "cin", "cout", "grouped", "device")

    def __init__(self, packed, scale, n_experts, cin, cout, grouped):
        self.packed, self.scale, self.n_experts, self.cin, self.cout, self.grouped = packed, scale, n_experts, cin, cout, grouped
        self.device = packed.device


def int8_weight(w, scale=None):
    """w [cin, cout] or [E, cin, cout] (the layout of the framework's kernels).  Floats: every output channel is quantised to
    scale * (-127 .. 127), scale = max |w| / 127.  int8: `scale` float32 [cout] ([E, cout]) must be given and w is taken as it is."""
    if recorded():
        need(not torch.jit.is_tracing(), "int8_weight: a trace would keep the weights it was made with; lay them out outside the trace")
        _no_tangent_for("int8_weight", w, scale)
    need(isinstance(w, torch.Tensor) and w.dtype in DTYPES and w.dim() in (2, 3),
         "int8_weight: w must be float32, bfloat16, float16 or int8, [cin, cout] or [experts, cin, cout]")
    grouped = w.dim() == 3
    e, cin, cout = w.shape if grouped else (1,) + tuple(w.shape)
    need(1 <= e <= 1024 and 1 <= cin <= MAX_CIN and 1 <= cout <= 1 << 20,
         "int8_weight: w of shape %s (experts in 1 .. 1024, cin in 1 .. %d, cout in 1 .. 2^20)", tuple(w.shape), MAX_CIN)
    if w.dtype == torch.int8:
        need(isinstance(scale, torch.Tensor) and scale.dtype == torch.float32 and tuple(scale.shape) == ((e, cout) if grouped else (cout,))
             and scale.device == w.device, "int8_weight: weights in 8 bits need their scale, float32 %s, beside them",
             [e, cout] if grouped else [cout])
    else:
        need(scale is None, "int8_weight: the scale of weights in floats is computed here")
    lib = _lib.get()
    w = whole(w.detach())
    lib.check(w)
    with on_device(w):
        packed = torch.empty(int(lib.raw("cg3d_int8_weight_bytes")(e, cin, cout)), dtype=torch.int8, device=w.device)
        if scale is None:
            out, ws = torch.empty((2, e, cout), dtype=torch.float32, device=w.device)
        else:
            out, ws = scale.detach().resolve_neg().clone(memory_format=torch.contiguous_format).view(e, cout), None      # (the handle's own: the caller may reuse the memory)
        lib.call("cg3d_int8_weight", ptr(w), DTYPES[w.dtype], e, cin, cout, ptr(packed),
                 ptr(out) if ws is not None else None, ptr(ws), lib.stream())
    del w, ws                                                     # (held until the launch has been made, under torch.compile too)
    return Int8Weight(packed, out, e, cin, cout, grouped)


def _rows_in(who, x, dtypes):
    if not (isinstance(x, torch.Tensor) and x.dtype in dtypes and x.dim() == 2 and 1 <= x.shape[1] <= MAX_CIN and x.shape[0] < 2 ** 31):
        raise CG3DError("%s: x must be [rows, cin] of %s with cin in 1 .. %d, got %s" % (
            who, " / ".join(str(d).replace("torch.", "") for d in dtypes), MAX_CIN, (x.dtype, tuple(x.shape)) if isinstance(x, torch.Tensor) else type(x)))


@functools.lru_cache(maxsize=4096)
def _ws_bytes(lib, *sizes):
    return int(lib.raw("cg3d_int8_linear_ws_bytes")(*sizes))


def quantize_rows(x):
    """x [rows, cin] float32 / bfloat16 / float16 -> (q int8 [rows, cin], scale float32 [rows]): scale = max |x| / 127 of each row,
    q = the nearest level, ties to the even one.  A row of zeros has the scale 0, one with an infinity or a NaN the scale NaN;
    the scale of a row whose largest magnitude is below 1.5e-36 is subnormal and has fewer bits."""
    return _record("quantize_rows", _quantize, (x,), (x,)) if recorded() else _quantize(x)


def _quantize(x):
    _rows_in("quantize_rows", x, FLOATS)
    _no_grad_for("quantize_rows", x.requires_grad)
    lib = _lib.get()
    x = whole(x.detach())
    lib.check(x)
    n, cin = x.shape
    if type(cin) is not int:                                      # (in a trace)
        n, cin = int(n), int(cin)
    with on_device(x):
        q = torch.empty((n, cin), dtype=torch.int8, device=x.device)
        scale = torch.empty(n, dtype=torch.float32, device=x.device)
        lib.call("cg3d_int8_quantize_rows", ptr(x), DTYPES[x.dtype], n, cin, cin, ptr(q), ptr(scale),
                 lib.stream())
    del x                                                         # (held until the launch has been made, under torch.compile too)
    return q, scale


def int8_linear(x, weight, bias=None, scale=None, out_dtype=None, plan=None, gather=False):
    """x [rows, cin] float32 / bfloat16 / float16 (quantised here) or int8 with `scale` float32 [rows] -> [rows, cout] of out_dtype
    (default: x's own, float32 for int8) = x @ weight (+ bias [cout], or [E, cout] with a plan).

    plan (ops/expert_rows.expert_plan): weight holds plan.n_experts matrices and each row is multiplied by its expert's; x has the
    plan's rows ([T * k, cin], what expert_gather gives), or with gather=True the tokens ([T, cin]), whose rows are picked in the
    product.  Rows behind the last are zeros."""
    if recorded():
        return _record("int8_linear", _linear, (x, weight, bias, scale, out_dtype, plan, gather), (x, bias, scale))
    return _linear(x, weight, bias, scale, out_dtype, plan, gather)


def _linear(x, weight, bias, scale, out_dtype, plan, gather):
    # (plain comparisons before any message is made: the call's host time is that of a small product)
    if not isinstance(weight, Int8Weight):
        raise CG3DError("int8_linear: weight must come from int8_weight")
    _rows_in("int8_linear", x, ROWS_IN)
    n_x, cin = x.shape
    if type(cin) is not int:                                      # (in a trace)
        n_x, cin = int(n_x), int(cin)
    dtype, dev, cout, n_experts = x.dtype, x.device, weight.cout, weight.n_experts
    if cin != weight.cin:
        raise CG3DError("int8_linear: x has %d columns, weight %d rows" % (cin, weight.cin))
    if weight.device != dev:
        raise CG3DError("int8_linear: x is on %s, weight on %s" % (dev, weight.device))
    if dtype is torch.int8:
        need(isinstance(scale, torch.Tensor) and scale.dtype == torch.float32 and scale.shape == (n_x,) and scale.device == dev,
             "int8_linear: rows in 8 bits need their scale beside them, float32 [%d]", n_x)
        out_dtype = out_dtype or torch.float32
        scale = whole(scale)
    else:
        need(scale is None, "int8_linear: the scale of rows in floats is computed here")
        out_dtype = out_dtype or dtype
    if out_dtype not in FLOATS:
        raise CG3DError("int8_linear: out_dtype must be float32, bfloat16 or float16")
    if plan is None:
        if n_experts != 1 or gather:
            raise CG3DError("int8_linear: %d matrices (or gather) need a plan" % n_experts)
        n_rows, offsets, rows = n_x, None, None
    else:
        need(isinstance(plan, ExpertPlan) and plan.device == dev, "int8_linear: plan must come from expert_plan, on %s", dev)
        need(n_experts == plan.n_experts, "int8_linear: %d matrices for a plan of %d experts", n_experts, plan.n_experts)
        n_rows = plan.n_rows
        need(n_x == (plan.n_tokens if gather else n_rows), "int8_linear: x has %d rows, the plan %d tokens and %d rows", n_x, plan.n_tokens, n_rows)
        offsets, rows = plan.address(OFFSETS), plan.address(ROWS) if gather else None
    per_expert = 0
    if bias is not None:
        need(isinstance(bias, torch.Tensor) and bias.dtype in FLOATS and bias.device == dev and (
            bias.shape == (cout,) or (weight.grouped and bias.shape == (n_experts, cout))),
            "int8_linear: bias must be floats [%d] (or [%d, %d] with a matrix for each expert) on %s", cout, n_experts, cout, dev)
        per_expert = int(bias.dim() == 2)
    _no_grad_for("int8_linear", x.requires_grad or (bias is not None and bias.requires_grad) or (scale is not None and scale.requires_grad))
    if bias is not None and not (bias.dtype is torch.float32 and bias.is_contiguous() and not bias.is_neg()):
        bias = whole(bias.detach().to(torch.float32))
    lib = _lib.get()
    x = whole(x)
    lib.check(x)
    code, at = DTYPES[dtype], x.data_ptr()
    with on_device(x):
        ws_bytes = _ws_bytes(lib, code, n_x, cin, n_rows, cout, n_experts, int(plan is not None) | (0 if at & 15 else 2))
        y = torch.empty((n_rows, cout), dtype=out_dtype, device=dev)
        ws = torch.empty(ws_bytes, dtype=torch.int8, device=dev) if ws_bytes > 0 else None
        lib.call("cg3d_int8_linear", at, code, ptr(scale), n_x, cin, weight.packed.data_ptr(), weight.scale.data_ptr(), ptr(bias), per_expert,
                 offsets, rows, y.data_ptr(), DTYPES[out_dtype], n_rows, cout, n_experts, ptr(ws), lib.stream())
    # (named behind the launch: torch.compile stops at an address and resumes with what the rest of the function names, so that it would
    # free workspaces and copies of inputs before the launch)
    del x, scale, weight, bias, plan, ws
    return y
