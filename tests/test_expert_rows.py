"""Rows sorted by expert and back (ops/expert_rows.py, csrc/expert_rows.hip).

CPU (-m "not gpu"): the oracle's restatement against a plain implementation in 64 bits, the refusals.  -m gpu: the HIP kernels
against the same -- every type, widths that no vector load divides, routings that leave experts and tokens empty, more pairs than
one workgroup sorts -- the gradients against the formulas and against differences, a captured graph, another stream, a run together
with the grouped product of the framework."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from cagroup3d_amd import _lib, me
from cagroup3d_amd.ops.expert_rows import MAX_EXPERTS, expert_combine, expert_gather, expert_plan

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative to the value
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}                     # half a step below the normal range


def plain_plan(ids, n_experts):
    t, k = ids.shape
    flat = ids.reshape(-1).tolist()
    pairs = [p for e in range(n_experts) for p in range(t * k) if flat[p] == e] if t * k <= 4096 else None
    if pairs is None:
        key = torch.where((ids >= 0) & (ids < n_experts), ids, n_experts).reshape(-1).cpu()
        order = torch.sort(key, stable=True)[1]
        pairs = order[key[order] < n_experts].tolist()
    counts = torch.bincount(ids[(ids >= 0) & (ids < n_experts)].reshape(-1).cpu(), minlength=n_experts)
    rows = torch.full((t * k,), -1, dtype=torch.int32)
    pos = torch.full((t * k,), -1, dtype=torch.int32)
    pairs = torch.tensor(pairs, dtype=torch.int64)
    rows[:pairs.numel()] = (pairs // k).int()
    pos[pairs] = torch.arange(pairs.numel(), dtype=torch.int32)
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int(), rows, pos.view(t, k)


def routing(t, k, n_experts, kind, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        ids = torch.randint(0, n_experts, (t, k), generator=g)
    elif kind == "one expert":
        ids = torch.full((t, k), n_experts - 1)
    elif kind == "none":
        ids = torch.full((t, k), -1)
    elif kind == "dropped":                  # ids on both sides of the range, whole tokens dropped
        ids = torch.randint(-2, n_experts + 3, (t, k), generator=g)
        ids[torch.rand(t, generator=g) < 0.3] = -1
    elif kind == "wild":                     # ids no int32 holds, and the ends of the type
        ids = torch.randint(0, n_experts, (t, k), generator=g)
        far = torch.iinfo(dtype)
        pick = torch.randint(0, 4, (t, k), generator=g)
        ids = torch.where(pick == 0, torch.tensor(far.min), torch.where(pick == 1, torch.tensor(far.max), ids))
    return ids.to(dtype)


def check_plan(ids, n_experts):
    plan = expert_plan(ids, n_experts)
    offsets, rows, pos = plain_plan(ids.cpu(), n_experts)
    assert torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(plan.rows.cpu(), rows)
    got = plan.pos.cpu()
    assert torch.equal(torch.where(got >= 0, got, -1), pos)
    behind = torch.sort(~got[got < 0])[0]                    # the pairs without a row own the rows behind the last, once each
    flat, pairs = got.view(-1).long(), plan.pairs.cpu()
    assert torch.equal(pairs[torch.where(flat >= 0, flat, ~flat)], torch.where(flat >= 0, 1, -1).int() * torch.arange(ids.numel(), dtype=torch.int32) - (flat < 0).int())
    assert torch.equal(behind, torch.arange(int(offsets[-1]), ids.numel(), dtype=torch.int32))
    return plan, offsets, rows, pos


def reference(x, y, w, pos, dr, do):
    """Both passes and their gradients in 64 bits, pair by pair -> (gathered, combined, dx, dy, dw) and, for the sums, the sums of
    the absolute values of their terms."""
    t, k = pos.shape
    x, y, w, dr, do = (v.double().cpu() for v in (x, y, w, dr, do))
    there = (pos >= 0).unsqueeze(2)
    at = pos.clamp(min=0).long()
    gathered, dy = torch.zeros_like(y), torch.zeros_like(y)
    tok = torch.arange(t).unsqueeze(1).expand(t, k)
    m = pos >= 0
    gathered[at[m]] = x[tok[m]]
    dy[at[m]] = w[m].unsqueeze(1) * do[tok[m]]
    py, pdr = y[at] * there, dr[at] * there
    return dict(gathered=gathered, combined=(py * w.unsqueeze(2)).sum(1), dx=pdr.sum(1), dy=dy, dw=(py * do.unsqueeze(1)).sum(2),
                abs_combined=(py * w.unsqueeze(2)).abs().sum(1), abs_dx=pdr.abs().sum(1), abs_dw=(py * do.unsqueeze(1)).abs().sum(2))


def run_all(ids, n_experts, c, dtype, wdtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    t, k = ids.shape
    x, y = (torch.randn(n, c, generator=g).to(dtype).to(dev).requires_grad_() for n in (t, t * k))
    w = torch.rand(t, k, generator=g).to(wdtype).to(dev).requires_grad_()
    dr, do = (torch.randn(n, c, generator=g).to(dtype).to(dev) for n in (t * k, t))
    plan, _, _, pos = check_plan(ids.to(dev), n_experts)
    gathered, combined = expert_gather(x, plan), expert_combine(y, plan, w)
    dx, dy, dw = torch.autograd.grad([gathered, combined], [x, y, w], [dr, do])
    ref = reference(x.detach(), y.detach(), w.detach(), pos, dr, do)
    got = dict(gathered=gathered, combined=combined, dx=dx, dy=dy, dw=dw)

    # a sum of n terms in fp32 is off by at most n half-steps of the sum of the absolute values (each product one more), and each
    # result is rounded once to its type
    u = 2.0 ** -24
    slack = dict(gathered=0.0, dy=0.0, combined=(k + 1) * u * ref["abs_combined"], dx=k * u * ref["abs_dx"],
                 dw=(c + 1) * u * ref["abs_dw"])
    for name, v in got.items():
        dt = wdtype if name == "dw" else dtype
        assert v.dtype == dt and v.device.type == torch.device(dev).type
        want = ref[name]
        extra = slack[name] if isinstance(slack[name], torch.Tensor) else torch.zeros_like(want)
        # (dy: one product rounded to fp32, then to the type)
        tol = (HALF[dt] + (u if name == "dy" else 0.0)) * (want.abs() + extra) * (1 + 2.0 ** -7) + extra + TINY[dt]
        if name == "gathered":
            assert torch.equal(v.detach().cpu().double(), want)
        else:
            off = (v.detach().cpu().double() - want).abs()
            assert bool((off <= tol).all()), (name, float((off - tol).max()))
    return got


SMALL = [  # tokens, k, experts, c, kind
    (1, 1, 1, 1, "uniform"), (1, 2, 18, 64, "uniform"), (3, 4, 5, 7, "dropped"), (64, 1, 2, 8, "uniform"), (65, 3, 18, 9, "dropped"),
    (130, 2, 10, 33, "one expert"), (40, 2, 6, 16, "none"), (257, 8, 61, 5, "dropped"), (200, 2, 1024, 12, "uniform"),
    (31, 3, 4, 130, "wild"),
]


@pytest.mark.parametrize("t,k,n_experts,c,kind", SMALL)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_oracle_is_the_definition(oracle, t, k, n_experts, c, kind, dtype):
    with _lib.use_library(oracle):
        run_all(routing(t, k, n_experts, kind, 1), n_experts, c, dtype, torch.float32, 2, "cpu")
        check_plan(routing(t, k, n_experts, kind, 3, torch.int32), n_experts)


def test_oracle_empty_and_one_slot(oracle):
    with _lib.use_library(oracle):
        plan = expert_plan(torch.zeros(0, 2, dtype=torch.int64), 3)
        assert plan.offsets.tolist() == [0, 0, 0, 0]
        assert expert_gather(torch.zeros(0, 4), plan).shape == (0, 4)
        assert expert_combine(torch.zeros(0, 4), plan).shape == (0, 4)
        plan = expert_plan(torch.tensor([1, 0, 1]), 2)                       # [T]: one slot
        x = torch.tensor([[1.0], [2.0], [3.0]])
        assert expert_gather(x, plan).view(-1).tolist() == [2.0, 1.0, 3.0]
        assert expert_combine(expert_gather(x, plan), plan, torch.tensor([1.0, 10.0, 100.0])).view(-1).tolist() == [1.0, 20.0, 300.0]


def refusals(dev):
    ids = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    x, y, w = torch.zeros(4, 8, device=dev), torch.zeros(8, 8, device=dev), torch.zeros(4, 2, device=dev)
    plan = expert_plan(ids, 3)
    for bad in (lambda: expert_plan(ids.float(), 3), lambda: expert_plan(ids, 0), lambda: expert_plan(ids, MAX_EXPERTS + 1),
                lambda: expert_plan(ids.view(2, 2, 2), 3), lambda: expert_plan(ids[:, :0], 3), lambda: expert_plan([[0]], 3),
                lambda: expert_plan(ids.short(), 3),
                lambda: expert_gather(x, ids), lambda: expert_gather(x[:3], plan), lambda: expert_gather(x[:, :0], plan),
                lambda: expert_gather(x.double(), plan), lambda: expert_gather(x[0], plan), lambda: expert_gather(None, plan),
                lambda: expert_combine(x, plan), lambda: expert_combine(y.long(), plan), lambda: expert_combine(y, plan, w[:3]),
                lambda: expert_combine(y, plan, w.t()), lambda: expert_combine(y, plan, w.double()), lambda: expert_combine(y, None, w),
                lambda: expert_combine(y, plan, w, torch.float64), lambda: expert_combine(y.half(), plan, w, torch.float32),
                lambda: expert_combine(y.half(), plan, w, torch.bfloat16)):
        with pytest.raises(_lib.CG3DError):
            bad()


def test_refusals(oracle):
    with _lib.use_library(oracle):
        refusals("cpu")


def test_entry_points_refuse(oracle):
    """The C-ABI's own checks (the same conditions in the library and in its restatement)."""
    i, f = torch.zeros(64, dtype=torch.int32), torch.zeros(64)
    h = _lib.bind(_lib.HIP_LIB_PATH)
    for lib in (oracle, h):                       # every call below is refused before anything is launched
        ok = dict(p=i.data_ptr(), x=f.data_ptr())
        for bad in ((ok["p"], 2, 4, 2, 3), (ok["p"], 0, -1, 2, 3), (ok["p"], 0, 4, 0, 3), (ok["p"], 0, 4, 2, 0), (ok["p"], 0, 4, 2, 1025),
                    (ok["p"], 0, 2 ** 31, 1, 3), (None, 0, 4, 2, 3), (ok["p"] + 2, 0, 4, 2, 3), (ok["p"] + 4, 1, 4, 2, 3)):
            assert lib.raw("cg3d_expert_plan")(*bad, ok["p"], ok["p"], ok["p"], ok["p"], None, None) == -1, bad
        assert lib.raw("cg3d_expert_plan")(ok["p"], 0, 4, 2, 3, None, ok["p"], ok["p"], ok["p"], None, None) == -1
        assert lib.raw("cg3d_expert_plan_ws_bytes")(2 ** 31, 1, 3) == -1
        for dt, t, k, c in ((3, 4, 2, 8), (-1, 4, 2, 8), (0, -1, 2, 8), (0, 4, 0, 8), (0, 4, 2, 0), (0, 2 ** 31, 1, 8)):
            assert lib.raw("cg3d_expert_gather")(ok["x"], dt, ok["p"], t, k, c, ok["x"], None) == -1
            assert lib.raw("cg3d_expert_combine")(ok["x"], dt, ok["p"], None, 0, t, k, c, ok["x"], max(dt, 0), None) == -1
            assert lib.raw("cg3d_expert_combine_bwd")(ok["x"], None, dt, ok["p"], None, 0, t, k, c, ok["x"], None, None) == -1
        assert lib.raw("cg3d_expert_gather")(ok["x"] + 2, 0, ok["p"], 4, 2, 8, ok["x"], None) == -1
        assert lib.raw("cg3d_expert_combine")(ok["x"], 0, ok["p"], ok["x"], 3, 4, 2, 8, ok["x"], 0, None) == -1
        for dt, out in ((0, 3), (0, -1), (1, 0), (1, 2), (2, 0)):
            assert lib.raw("cg3d_expert_combine")(ok["x"], dt, ok["p"], None, 0, 4, 2, 8, ok["x"], out, None) == -1
        assert lib.raw("cg3d_expert_combine_bwd")(ok["x"], ok["x"], 0, ok["p"], ok["x"], 0, 4, 2, 8, None, None, None) == -1
        assert lib.raw("cg3d_expert_combine_bwd")(ok["x"], None, 0, ok["p"], ok["x"], 0, 4, 2, 8, ok["x"], ok["x"], None) == -1
        assert lib.raw("cg3d_expert_gather")(None, 0, ok["p"], 4, 2, 8, ok["x"], None) == -1
    if h.raw("cg3d_expert_plan_ws_bytes")(100000, 2, 18) > 0:
        assert h.raw("cg3d_expert_plan")(i.data_ptr(), 0, 100000, 2, 18, i.data_ptr(), i.data_ptr(), i.data_ptr(), i.data_ptr(), None, None) == -1


def test_too_many_columns_are_refused(oracle):
    """A number of columns that the C-ABI's 32 bits do not hold (no memory behind the tensors' one element)."""
    p = torch.zeros(64).data_ptr()
    for lib in (oracle, _lib.bind(_lib.HIP_LIB_PATH)):
        assert lib.raw("cg3d_expert_gather")(p, 0, p, 4, 2, (1 << 30) + 1, p, None) == -1
        assert lib.raw("cg3d_expert_combine")(p, 0, p, None, 0, 4, 2, (1 << 30) + 1, p, 0, None) == -1
        assert lib.raw("cg3d_expert_combine_bwd")(p, None, 0, p, None, 0, 4, 2, (1 << 30) + 1, p, None, None) == -1
    with _lib.use_library(oracle):
        plan = expert_plan(torch.zeros(2, 1, dtype=torch.int32), 1)
        for wide in ((1 << 30) + 1, (1 << 32) + 8):
            x = torch.zeros(1).expand(2, wide)
            with pytest.raises(_lib.CG3DError):
                expert_gather(x, plan)
            with pytest.raises(_lib.CG3DError):
                expert_combine(x, plan)


def test_no_cpu_fallback():
    with _lib.use_library(_lib.bind(_lib.HIP_LIB_PATH)):
        with pytest.raises(_lib.CG3DError):
            expert_plan(torch.zeros(4, 2, dtype=torch.int64), 3)


# ------------------------------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("t,k,n_experts,kind", [
    (0, 2, 3, "uniform"), (1, 1, 1, "uniform"), (1, 2, 18, "uniform"), (33, 3, 18, "dropped"), (512, 2, 18, "uniform"),
    (1000, 1, 1024, "uniform"), (8192, 2, 1024, "dropped"), (8193, 2, 18, "dropped"), (5000, 8, 61, "wild"), (20000, 2, 1, "none"),
    (200000, 2, 18, "uniform"), (150001, 8, 256, "dropped"), (40000, 3, 7, "one expert")])
def test_hip_plan(hip, t, k, n_experts, kind):
    for dtype in (torch.int64, torch.int32):
        check_plan(routing(t, k, n_experts, kind, 5, dtype).cuda(), n_experts)


@pytest.mark.gpu
@pytest.mark.parametrize("n_experts", [1, 64, 65, 300, 1024])
@pytest.mark.parametrize("t", [2, 63, 64, 65, 257, 1023, 1025, 2048, 2049, 4095, 4096, 4097, 21505, 600001])
def test_hip_plan_at_the_borders_of_its_launches(hip, t, n_experts):
    check_plan(routing(t, 1, n_experts, "dropped", 8, torch.int32).cuda(), n_experts)


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,n_experts,c,kind", SMALL + [(5000, 2, 18, 64, "uniform"), (3001, 8, 61, 251, "dropped"), (900, 3, 4, 1030, "dropped"),
                                                          (20011, 2, 18, 128, "uniform")])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.bfloat16)])
def test_hip_passes_and_gradients(hip, t, k, n_experts, c, kind, dtype, wdtype):
    run_all(routing(t, k, n_experts, kind, 6), n_experts, c, dtype, wdtype, 7, "cuda")


@pytest.mark.gpu
def test_hip_gradients_against_differences(hip):
    ids = routing(23, 3, 5, "dropped", 8).cuda()
    plan = expert_plan(ids, 5)
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn(23, 6, generator=g).cuda(), torch.rand(23, 3, generator=g).cuda()
    do = torch.randn(23, 6, generator=g).cuda()

    def f(x, w):                                              # multilinear in x and in w: central differences are exact but for rounding
        return (expert_combine(expert_gather(x, plan), plan, w).double() * do.double()).sum()
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(f(xl, wl), [xl, wl])
    h = 0.5
    for grad, v, which in ((dx, x, 0), (dw, w, 1)):
        for i in range(0, v.numel(), 7):
            d = torch.zeros_like(v).view(-1)
            d[i] = h
            d = d.view_as(v)
            up, dn = (f(x + d, w), f(x - d, w)) if which == 0 else (f(x, w + d), f(x, w - d))
            # each forward's entries are off by at most a few half-steps of numbers below 16: 23 * 6 entries, sums in 64 bits
            assert abs(float(grad.reshape(-1)[i]) - float((up - dn) / (2 * h))) < 1e-3


@pytest.mark.gpu
def test_hip_shared_and_broadcast_inputs(hip):
    """One tensor as x twice, a broadcast weight, a broadcast output gradient, views that are not contiguous."""
    ids = routing(100, 2, 6, "dropped", 10).cuda()
    plan = expert_plan(ids, 6)
    base = torch.randn(16, 100, device="cuda", requires_grad=True)
    gate = torch.full((1, 1), 0.75, device="cuda", requires_grad=True)
    out = expert_combine(expert_gather(base.t(), plan) + expert_gather(base.t(), plan), plan, gate.expand(100, 2))
    out.sum().backward()
    n = (plan.pos >= 0).sum(1).double()
    want = (2 * 0.75 * n).unsqueeze(0).expand(16, 100)
    assert torch.equal(base.grad.double(), want)              # multiples of 0.75: exact
    ref = (2 * base.detach().double() * n).sum()
    assert abs(float(gate.grad) - float(ref)) < 1e-4 * float((2 * base.detach().double().abs() * n).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c", [3, 64, 129])
def test_hip_fp32_rows_to_a_narrower_output(hip, out, c):
    """One rounding only: fp32 rows, a 16-bit output, and its gradients, which are formed in fp32."""
    ids = routing(300, 3, 7, "dropped", 50).cuda()
    plan = expert_plan(ids, 7)
    g = torch.Generator().manual_seed(51)
    y, w = torch.randn(900, c, generator=g).cuda().requires_grad_(), torch.rand(300, 3, generator=g).cuda().requires_grad_()
    do = torch.randn(300, c, generator=g).to(out).cuda()
    got = expert_combine(y, plan, w, out)
    wide = expert_combine(y, plan, w)
    assert got.dtype == out and torch.equal(got, wide.to(out))
    for a, b in zip(torch.autograd.grad(got, [y, w], do), torch.autograd.grad(wide, [y, w], do.float())):
        assert a.dtype == torch.float32 and torch.equal(a, b)


@pytest.mark.gpu
def test_hip_nonfinite_rows_stay_where_they_are(hip):
    """Infinities and NaN in rows that no pair names, and in rows behind the last, reach nothing."""
    ids = torch.tensor([[0, -1], [1, 0], [-1, -1]]).cuda()
    plan = expert_plan(ids, 2)
    y = torch.full((6, 8), float("nan"), device="cuda")
    y[:3] = torch.arange(24, device="cuda").view(3, 8).float()
    y.requires_grad_()
    w = torch.tensor([[2.0, float("inf")], [3.0, 4.0], [float("nan"), float("nan")]], device="cuda", requires_grad=True)
    out = expert_combine(y, plan, w)
    rows = y.detach()[:3]
    # rows: expert 0 holds (0, 0) and (1, 1), expert 1 holds (1, 0)
    assert torch.equal(out.detach(), torch.stack([2 * rows[0], 3 * rows[2] + 4 * rows[1], torch.zeros(8, device="cuda")]))
    dy, dw = torch.autograd.grad(out, [y, w], torch.ones_like(out))
    assert torch.equal(dy[3:], torch.zeros(3, 8, device="cuda")) and bool(torch.isfinite(dy).all())
    assert torch.equal(dw, torch.stack([torch.stack([rows[0].sum(), rows.new_zeros(())]), torch.stack([rows[2].sum(), rows[1].sum()]),
                                        torch.zeros(2, device="cuda")]))


@pytest.mark.gpu
def test_hip_graph_replays_with_new_inputs(hip):
    """Captured once, replayed on new ids and rows with eager calls between; two graphs at once share no workspace."""
    t, k, e, c = 12000, 2, 18, 32
    ids = [routing(t, k, e, "dropped", s).cuda() for s in (20, 21, 22)]
    xs = [torch.randn(t, c, generator=torch.Generator().manual_seed(s)).cuda() for s in (20, 21, 22)]

    def step(i, x):
        plan = expert_plan(i, e)
        return plan.rows, expert_combine(expert_gather(x, plan), plan)
    static = [(ids[0].clone(), xs[0].clone()) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i, x in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i, x))
        graphs.append(g)
    for turn in range(3):
        for j in range(2):
            static[j][0].copy_(ids[(turn + j) % 3])
            static[j][1].copy_(xs[(turn + j) % 3])
        for g in graphs:
            g.replay()
        for j in range(2):
            want = step(ids[(turn + j) % 3], xs[(turn + j) % 3])           # eager, between the replays
            assert all(torch.equal(a, b) for a, b in zip(outs[j], want))


@pytest.mark.gpu
def test_hip_offsets_past_32_bits(hip):
    """More than 2^31 elements of rows: gather, combination and gradient at the far end."""
    t, k, e, c = 1100000, 2, 5, 1024
    ids = routing(t, k, e, "uniform", 60).cuda()
    plan = expert_plan(ids, e)
    x = torch.randn(t, 8, device="cuda").to(torch.bfloat16).repeat(1, c // 8)
    rows = expert_gather(x, plan)
    tail = slice(t * k - 50, t * k)
    assert torch.equal(rows[tail], x[plan.rows[tail].long()]) and torch.equal(rows[:50], x[plan.rows[:50].long()])
    rows.requires_grad_()
    w = torch.ones(t, k, device="cuda", requires_grad=True)
    out = expert_combine(rows, plan, w)
    assert torch.equal(out[-50:], (2 * x[-50:].float()).to(torch.bfloat16))
    dy, dw = torch.autograd.grad(out, [rows, w], x)
    assert torch.equal(dy[tail], x[plan.rows[tail].long()])
    want = x[-50:].double().square().sum(1, keepdim=True).expand(50, k)
    assert bool(((dw[-50:].double() - want).abs() <= (c + 1) * 2.0 ** -24 * want).all())


@pytest.mark.gpu
def test_hip_second_gradients_are_refused(hip):
    ids = routing(20, 2, 3, "uniform", 61).cuda()
    plan = expert_plan(ids, 3)
    x, w = torch.randn(20, 8, device="cuda", requires_grad=True), torch.rand(20, 2, device="cuda", requires_grad=True)
    out = expert_combine(expert_gather(x, plan), plan, w)
    (g,) = torch.autograd.grad(out.square().sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("t,n_experts", [(3, 1024), (2000, 1024), (30000, 1024), (30000, 18)])
def test_hip_plans_in_a_graph(hip, t, n_experts):
    """Every shape of the plan's launches captured once and replayed with other ids, eager plans in between."""
    fixed = routing(t, 2, n_experts, "uniform", 62, torch.int32).cuda()
    expert_plan(fixed, n_experts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = expert_plan(fixed, n_experts)
    for seed in range(3):
        ids = routing(t, 2, n_experts, "dropped", 63 + seed, torch.int32).cuda()
        fixed.copy_(ids)
        graph.replay()
        want = expert_plan(ids, n_experts)
        torch.cuda.synchronize()
        for a, b in ((held.offsets, want.offsets), (held.rows, want.rows), (held.pairs, want.pairs), (held.pos, want.pos)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_hip_on_another_stream(hip):
    ids, x = routing(30000, 2, 18, "uniform", 30).cuda(), torch.randn(30000, 64, device="cuda")
    want = expert_gather(x, expert_plan(ids, 18))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = expert_gather(x, expert_plan(ids, 18))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_hip_same_bits_every_run(hip):
    ids, w = routing(9000, 4, 18, "dropped", 31).cuda(), torch.rand(9000, 4, device="cuda")
    y = torch.randn(36000, 48, device="cuda")
    first = expert_combine(y, expert_plan(ids, 18), w)
    for _ in range(3):
        assert torch.equal(expert_combine(y, expert_plan(ids, 18), w), first)


@pytest.mark.gpu
def test_hip_layer_of_experts_trains(hip):
    """Plan, gather, the grouped product of the framework (per-expert matrices) and the combination as one layer: outputs and
    gradients against the same layer in 64 bits."""
    t, k, e, c, n = 700, 2, 6, 32, 48
    ids = routing(t, k, e, "uniform", 40).cuda()
    plan = expert_plan(ids, e)
    g = torch.Generator().manual_seed(41)
    x, w = torch.randn(t, c, generator=g).cuda().requires_grad_(), torch.rand(t, k, generator=g).cuda().requires_grad_()
    mats = [(torch.randn(1, c, n, generator=g) / c ** 0.5).cuda().requires_grad_() for _ in range(e)]
    bounds = tuple(plan.offsets.tolist())
    rows = expert_gather(x, plan)
    y = me.grouped_conv(rows, mats, me.KernelMap.identity(t * k, rows.device), bounds)
    out = expert_combine(y, plan, w)
    do = torch.randn(t, n, generator=g).cuda()
    got = torch.autograd.grad(out, [x, w] + mats, do)
    xd, wd = x.detach().double().cpu().requires_grad_(), w.detach().double().cpu().requires_grad_()
    md = [m.detach().double().cpu().requires_grad_() for m in mats]
    per = torch.stack([xd @ m[0] for m in md], 1)                                       # [t, e, n]
    ref = (per[torch.arange(t).unsqueeze(1), ids.cpu()] * wd.unsqueeze(2)).sum(1)
    want = torch.autograd.grad(ref, [xd, wd] + md, do.double().cpu())
    # fp32 throughout; the longest sums run over ~t * k / e rows of numbers of order 1 (matrices) and over c + n terms (the rest)
    for a, b in zip([out.detach()] + list(got), [ref.detach()] + list(want)):
        torch.testing.assert_close(a.cpu().double(), b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


@pytest.mark.gpu
def test_hip_refusals(hip):
    refusals("cuda")
    plan = expert_plan(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 3)
    for bad in (lambda: expert_gather(torch.zeros(4, 8), plan), lambda: expert_combine(torch.zeros(8, 8, device="cuda"), plan, torch.zeros(4, 2))):
        with pytest.raises(_lib.CG3DError):
            bad()


def empty_batch(dev):
    """No tokens: every gradient exists and is empty, whichever inputs ask for one, with and without weights."""
    for k in (1, 3):
        plan = expert_plan(torch.zeros(0, k, dtype=torch.int64, device=dev), 3)
        for dtype, out in ((torch.float32, None), (torch.bfloat16, None), (torch.float32, torch.float16)):
            for need_y, need_w in ((True, True), (True, False), (False, True)):
                x = torch.zeros(0, 4, dtype=dtype, device=dev, requires_grad=True)
                y = torch.zeros(0, 4, dtype=dtype, device=dev, requires_grad=need_y)
                w = torch.zeros(0, k, device=dev, requires_grad=need_w)
                (expert_gather(x, plan).sum() + expert_combine(y, plan, w, out).sum()).backward()
                assert x.grad.shape == (0, 4) and (y.grad is not None) == need_y and (w.grad is not None) == need_w
                assert not need_y or y.grad.shape == (0, 4) and y.grad.dtype == dtype
                assert not need_w or w.grad.shape == (0, k)
            y = torch.zeros(0, 4, dtype=dtype, device=dev, requires_grad=True)
            expert_combine(y, plan, None, out).sum().backward()
            assert y.grad.shape == (0, 4)


def test_empty_batch_has_gradients(oracle):
    with _lib.use_library(oracle):
        empty_batch("cpu")
    for lib in (oracle, _lib.bind(_lib.HIP_LIB_PATH)):           # no addresses behind empty tensors: nothing is launched
        assert lib.raw("cg3d_expert_combine_bwd")(None, None, 0, None, None, 0, 0, 2, 8, None, None, None) == 0


@pytest.mark.gpu
def test_hip_empty_batch_has_gradients(hip):
    empty_batch("cuda")


def traced_and_dual(dev):
    """What torch has to see of a call -- a trace, forward-mode differentiation -- is seen by it without gradients too: a trace
    computes, and has its checks, on new inputs; a tangent is refused and not dropped; a plan, which is no tensor, is not made in a
    trace."""
    ids = routing(9, 2, 3, "dropped", 70).to(dev)
    plan = expert_plan(ids, 3)
    g = torch.Generator().manual_seed(71)
    x, y, w = torch.randn(9, 8, generator=g).to(dev), torch.randn(18, 8, generator=g).to(dev), torch.rand(9, 2, generator=g).to(dev)
    calls = ((lambda a: expert_gather(a, plan), x), (lambda a: expert_combine(a, plan, w), y), (lambda a: expert_combine(a, plan), y),
             (lambda a: expert_combine(y, plan, a, torch.bfloat16), w))
    for f, a in calls:
        for grad in (False, True):
            traced = torch.jit.trace(f, (a.clone().requires_grad_(grad),))
            junk = [torch.full_like(f(a), 7.0) for _ in range(4)]            # (memory that an output without a kernel would show)
            del junk
            assert torch.equal(traced(3 * a), f(3 * a))
            with pytest.raises(RuntimeError, match="must be"):               # (TorchScript's own error around the refusal)
                traced(a[:-1].contiguous())
        with forward_ad.dual_level():
            assert torch.equal(f(a), f(a))                                   # (no tangent)
            with pytest.raises(NotImplementedError):
                f(forward_ad.make_dual(a, torch.ones_like(a)))
        with pytest.raises(_lib.CG3DError):
            make_fx(f)(a)
    with pytest.raises(_lib.CG3DError):
        torch.jit.trace(lambda i: expert_plan(i, 3).rows, (ids,))
    with pytest.raises(_lib.CG3DError):
        make_fx(lambda i: expert_plan(i, 3).rows)(ids)


def test_traces_and_tangents(oracle):
    with _lib.use_library(oracle):
        traced_and_dual("cpu")


@pytest.mark.gpu
def test_hip_traces_and_tangents(hip):
    traced_and_dual("cuda")


def tables_are_saved(dev):
    """A plan's tables are saved tensors of both passes: one that is written between forward and backward is noticed, hooks of
    saved tensors see it, and the backward pass reads what they give back."""
    ids = routing(9, 2, 3, "dropped", 80).to(dev)
    g = torch.Generator().manual_seed(81)
    x, y, w = torch.randn(9, 8, generator=g).to(dev), torch.randn(18, 8, generator=g).to(dev), torch.rand(9, 2, generator=g).to(dev)

    def passes(plan):
        a, b, c = (t.clone().requires_grad_() for t in (x, y, w))
        return (lambda: (expert_gather(a, plan), (a,)), lambda: (expert_combine(b, plan, c), (b, c)), lambda: (expert_combine(b, plan), (b,)))
    for i in range(3):
        plan = expert_plan(ids, 3)
        want = [t.clone() for o, v in [passes(plan)[i]()] for t in torch.autograd.grad(o.sum(), v)]
        out, leaves = passes(plan)[i]()
        plan.pos[0, 0] = 5
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaves)
        plan, packed = expert_plan(ids, 3), []

        def pack(t):
            packed.append(t)
            return t.clone()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.clone()):
            out, leaves = passes(plan)[i]()
        assert any(t.dtype == torch.int32 for t in packed)
        with torch.no_grad():
            for t in (plan.rows, plan.pairs, plan.pos):
                t.fill_(0)                                                   # (the hooks gave copies)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(out.sum(), leaves), want))
        with torch.inference_mode():                                         # a router's plan, made without any bookkeeping
            plan = expert_plan(ids, 3)
        out, leaves = passes(plan)[i]()
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(out.sum(), leaves), want))


def test_tables_are_saved_tensors(oracle):
    with _lib.use_library(oracle):
        tables_are_saved("cpu")


@pytest.mark.gpu
def test_hip_tables_are_saved_tensors(hip):
    tables_are_saved("cuda")


def negated_views(dev):
    """Views whose memory holds the opposite of their values (as torch's conjugates make them) count with their values."""
    g = torch.Generator().manual_seed(90)
    ids = routing(9, 2, 3, "dropped", 91).to(dev)
    x, y, w = torch.randn(9, 8, generator=g).to(dev), torch.randn(18, 8, generator=g).to(dev), torch.rand(9, 2, generator=g).to(dev)
    plan, neg = expert_plan(ids, 3), torch._neg_view
    other = expert_plan(neg((-ids).contiguous()), 3)
    assert torch.equal(other.rows, plan.rows) and torch.equal(other.pos, plan.pos)
    for grad in (False, True):
        a, b, c = (t.clone().requires_grad_(grad) for t in (x, y, w))
        out = expert_gather(neg(a), plan)
        assert torch.equal(out, expert_gather(-x, plan))
        both = expert_combine(neg(b), plan, neg(c))
        assert torch.equal(both, expert_combine(-y, plan, -w)) and torch.equal(expert_combine(neg(b), plan), expert_combine(-y, plan))
        if grad:
            got = torch.autograd.grad([out, both], [a, b, c], [neg(y), neg(x)])
            l, m, n = (t.clone().requires_grad_() for t in (x, y, w))
            want = torch.autograd.grad([expert_gather(-l, plan), expert_combine(-m, plan, -n)], [l, m, n], [-y, -x])
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_negated_views(oracle):
    with _lib.use_library(oracle):
        negated_views("cpu")


@pytest.mark.gpu
def test_hip_negated_views(hip):
    negated_views("cuda")


def weights_of_one_slot(dev):
    """Weights [T] of a plan of one slot: their gradient has their shape."""
    plan = expert_plan(torch.tensor([1, 0, 1, -1]).to(dev), 2)
    y = torch.arange(8.0).view(4, 2).to(dev).requires_grad_()
    for w in (torch.tensor([1.0, 10.0, 100.0, 1000.0]).to(dev), torch.tensor([[1.0], [10.0], [100.0], [1000.0]]).to(dev)):
        w.requires_grad_()
        out = expert_combine(y, plan, w)
        dy, dw = torch.autograd.grad(out.sum(), [y, w])
        assert out.tolist() == [[2.0, 3.0], [0.0, 10.0], [400.0, 500.0], [0.0, 0.0]]
        assert dw.shape == w.shape and dw.view(-1).tolist() == [5.0, 1.0, 9.0, 0.0]
        assert dy.tolist() == [[10.0, 10.0], [1.0, 1.0], [100.0, 100.0], [0.0, 0.0]]


def test_weights_of_one_slot(oracle):
    with _lib.use_library(oracle):
        weights_of_one_slot("cpu")


@pytest.mark.gpu
def test_hip_weights_of_one_slot(hip):
    weights_of_one_slot("cuda")


@pytest.mark.gpu
def test_hip_training_pass_in_a_graph(hip):
    """Plan, both passes and all gradients captured once and replayed with other ids and rows, eager passes in between."""
    t, k, e, c = 3000, 2, 18, 40
    g = torch.Generator().manual_seed(95)

    def inputs(seed):
        ids = routing(t, k, e, "dropped", seed).cuda()
        return [ids] + [torch.randn(*s, generator=g).cuda() for s in ((t, c), (t * k, c), (t, k), (t * k, c), (t, c))]

    def step(ids, x, y, w, dr, do):
        plan = expert_plan(ids, e)
        x, y, w = (v.detach().requires_grad_() for v in (x, y, w))
        outs = expert_gather(x, plan), expert_combine(y, plan, w)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [x, y, w], [dr, do]))
    static = inputs(96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*static)
    for seed in (97, 98, 99):
        new = inputs(seed)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
