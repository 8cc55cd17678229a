"""Products in 8-bit integers (ops/int8_linear.py, csrc/int8_linear.hip).

CPU (-m "not gpu"): the oracle's restatement against a plain implementation in 64 bits, the refusals.  -m gpu: the HIP kernels
against the same -- every type in and out, sizes around the tiles, long contractions, single rows, experts without rows, dropped
pairs, gathered rows -- the levels at exact ties and at the ends of the types' ranges, a captured graph, another stream, a layer of
experts as it is served."""
import copy
import pickle

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from cagroup3d_amd import _lib
from cagroup3d_amd.ops.expert_rows import expert_combine, expert_gather, expert_plan
from cagroup3d_amd.ops.int8_linear import MAX_CIN, int8_linear, int8_weight, quantize_rows

F32, BF16, F16, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}       # half a step, relative to the value
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -25}    # below the normal range a step is this and not relative


def plain_levels(x):
    """(q, scale in 64 bits) of each row: products and quotient in 64 bits place every value on its own side of a border."""
    v = x.double()
    top = v.abs().amax(1, keepdim=True)
    q = torch.round(v * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return q, (top / 127).squeeze(1)


def check_levels(x, q, scale):
    want_q, want_s = plain_levels(x.cpu())
    assert q.dtype == I8 and scale.dtype == F32
    assert torch.equal(q.cpu().double(), want_q)
    assert bool(((scale.cpu().double() - want_s).abs() <= 2.0 ** -24 * want_s + 2.0 ** -150).all())


def make(n, cin, cout, dtype, seed, experts=None):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((experts, cin, cout) if experts else (cin, cout), generator=g) / cin ** 0.5
    if dtype == I8:
        x, sx = torch.randint(-128, 128, (n, cin), generator=g).to(I8), torch.rand(n, generator=g) + 0.1
    else:
        x, sx = (torch.randn(n, cin, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype), None
        x[torch.rand(n, generator=g) < 0.1] = 0
    return x, sx, w, torch.randn((experts, cout) if experts else (cout,), generator=g)


def reference(x, sx, wq, sw, bias, expert, token):
    """64 bits: rows token[r] of x times the matrix of expert[r] -> (result, sum of the absolute values of its two terms)."""
    q, s = (x.cpu().double(), sx.cpu().double()) if x.dtype == I8 else plain_levels(x.cpu())
    wq, sw = wq.cpu().double(), sw.cpu().double()
    y = torch.zeros(len(expert), wq.shape[2], dtype=torch.float64)
    for e in expert.unique().tolist():
        if e >= 0:
            m = expert == e
            y[m] = q[token[m]] @ wq[e] * s[token[m]].unsqueeze(1) * sw[e]
    size = y.abs()
    if bias is not None:
        b = bias.cpu().double()
        b = torch.where((expert >= 0).unsqueeze(1), b[expert.clamp(min=0)] if b.dim() == 2 else b, 0.0)
        y, size = y + b, size + b.abs()
    return y, size


def close(got, want, size, out):
    """fp32: the sum converted, two products with scales that are themselves rounded once, one addition -- 6 half-steps of the
    terms' sizes -- and one rounding to the output's type."""
    assert got.dtype == out and bool(torch.isfinite(got).all())
    tol = (6 * 2.0 ** -24 * size) * (1 + HALF[out]) + HALF[out] * want.abs() * (1 + 2.0 ** -7) + TINY[out]
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def dense(n, cin, cout, dtype, out, bias, seed, dev, offset=0):
    x, sx, w, b = make(n, cin, cout, dtype, seed)
    wq, sw = plain_levels(w.t().contiguous())                     # a channel of w is a row here
    weight = int8_weight(w.to(dev))
    assert bool(((weight.scale.cpu().double().view(-1) - sw).abs() <= 2.0 ** -24 * sw).all())
    if offset:                                                    # x behind an odd number of elements of its storage
        x = torch.cat([torch.zeros(offset, dtype=x.dtype), x.reshape(-1)]).to(dev)[offset:].view(n, cin)
    y = int8_linear(x.to(dev), weight, b.to(dev) if bias else None, scale=None if sx is None else sx.to(dev), out_dtype=out)
    want, size = reference(x, sx, wq.t().unsqueeze(0), sw.unsqueeze(0), b if bias else None, torch.zeros(n, dtype=torch.long), torch.arange(n))
    assert y.shape == (n, cout)
    close(y, want, size, out)
    return y


def grouped(ids, experts, cin, cout, dtype, out, bias, gather, seed, dev):
    t, k = ids.shape
    x, sx, w, b = make(t if gather else t * k, cin, cout, dtype, seed, experts)
    if bias == 1:
        b = b[0]
    wq, sw = plain_levels(w.transpose(1, 2).reshape(-1, cin))
    wq, sw = wq.view(experts, cout, cin).transpose(1, 2), sw.view(experts, cout)
    plan = expert_plan(ids.to(dev), experts)
    rows, off = plan.rows.cpu().long(), plan.offsets.cpu().long()
    expert = torch.bucketize(torch.arange(t * k), off[1:], right=True)
    expert[expert == experts] = -1
    y = int8_linear(x.to(dev), int8_weight(w.to(dev)), b.to(dev) if bias else None, scale=None if sx is None else sx.to(dev), out_dtype=out,
                    plan=plan, gather=gather)
    want, size = reference(x, sx, wq, sw, b if bias else None, expert, rows.clamp(min=0) if gather else torch.arange(t * k))
    close(y, want, size, out)
    assert bool((y[int(off[-1]):] == 0).all())
    return y


def ids_of(t, k, experts, kind, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (t, k), generator=g)
    if kind == "dropped":
        ids[torch.rand(t, k, generator=g) < 0.4] = -1
    elif kind == "one":
        ids[:] = experts // 2
    elif kind == "none":
        ids[:] = -1
    return ids


ODD = [(1, 1, 1), (1, 64, 64), (2, 16, 8), (15, 63, 65), (17, 65, 63), (33, 100, 7), (16, 128, 128), (70, 200, 77), (129, 257, 130)]


@pytest.mark.parametrize("n,cin,cout", ODD)
@pytest.mark.parametrize("dtype,out,bias", [(F32, F32, True), (BF16, BF16, False), (F16, F16, True), (I8, F32, False), (I8, BF16, True)])
def test_oracle_is_the_definition(oracle, n, cin, cout, dtype, out, bias):
    with _lib.use_library(oracle):
        dense(n, cin, cout, dtype, out, bias, 1, "cpu")


@pytest.mark.parametrize("kind", ["uniform", "dropped", "one", "none"])
@pytest.mark.parametrize("gather", [False, True])
def test_oracle_grouped(oracle, kind, gather):
    with _lib.use_library(oracle):
        grouped(ids_of(20, 2, 5, kind, 2), 5, 33, 18, F32, F32, 2, gather, 3, "cpu")
        grouped(ids_of(20, 2, 5, kind, 2), 5, 33, 18, I8, F16, 1, gather, 3, "cpu")


def levels_cases():
    """Rows whose elements sit on and beside the borders between levels, at the ends of the type's range too."""
    m = torch.arange(-127, 127).double()
    ties = (2 * m + 1) / 254                                     # times the largest magnitude: half-way between two levels
    rows = []
    for top in (1.0, 254.0, 127.0, 3.0, 2.0 ** -20, 254 * 2.0 ** -149, 127 * 2.0 ** -140, 2.0 ** -126, 3.3e38, 1.7e-37):
        r = torch.cat([torch.tensor([top]).double(), ties * top]).float()
        rows += [r, torch.nextafter(r, torch.zeros(())), torch.cat([r[:1], torch.nextafter(r[1:], 2 * r[1:])])]
    rows.append(torch.zeros(255))
    rows.append(torch.cat([torch.tensor([2.0 ** -149]), torch.zeros(254)]))
    return torch.stack(rows)


def levels(dev):
    x = levels_cases().to(dev)
    check_levels(x, *quantize_rows(x))
    g = torch.Generator().manual_seed(4)
    for dtype in (BF16, F16):                                    # short significands: exact ties everywhere
        v = torch.randint(-254, 255, (300, 61), generator=g).to(dtype).to(dev)
        check_levels(v, *quantize_rows(v))
        v = (torch.randn(300, 130, generator=g) * 1e-6).to(dtype).to(dev)
        check_levels(v, *quantize_rows(v))


def short_levels(dev, dtype):
    """Every pair of significands of the type, over the octaves where a level is not 0: a row for each largest magnitude."""
    bits = 8 if dtype == BF16 else 11
    step = 1 if dev == "cuda" or dtype == BF16 else 37            # (fp16 has 1024 x 1024 pairs an octave)
    sig = torch.arange(2 ** (bits - 1), 2 ** bits, step).double()
    if step > 1:                                                  # multiples of 127 are where halves can be met away from 63.5
        sig = torch.cat([sig, torch.arange(9, 17).double() * 127])
    x = torch.cat([sig.unsqueeze(1)] + [torch.arange(2 ** (bits - 1), 2 ** bits).double().unsqueeze(0).expand(sig.numel(), -1) * 2.0 ** -s for s in range(1, 9)], 1)
    x[:, 1::2] *= -1
    x = (x * 2.0 ** -6).to(dtype).to(dev)                         # (exact: no subnormals of fp16)
    check_levels(x, *quantize_rows(x))


def nonfinite(dev):
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(5)).to(dev)
    x[1, 7], x[2, 39], x[3, 0], x[4] = float("inf"), float("nan"), float("-inf"), 0.0
    q, s = quantize_rows(x)
    bad = torch.tensor([False, True, True, True, False, False]).to(dev)
    assert torch.equal(torch.isnan(s), bad) and bool((q[bad] == 0).all()) and float(s[4]) == 0.0
    w = int8_weight(torch.randn(40, 9, generator=torch.Generator().manual_seed(6)).to(dev))
    b = torch.ones(9, device=dev)
    for dt in (F32, BF16):
        y = int8_linear(x.to(dt), w, b)
        assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all()) and bool((y[4] == 1).all())


def test_oracle_levels_and_nonfinite(oracle):
    with _lib.use_library(oracle):
        levels("cpu")
        short_levels("cpu", BF16)
        short_levels("cpu", F16)
        nonfinite("cpu")


def test_oracle_weights_in_8_bits(oracle):
    with _lib.use_library(oracle):
        eight_bit_weights("cpu")


def eight_bit_weights(dev):
    g = torch.Generator().manual_seed(7)
    wq, sw = torch.randint(-128, 128, (3, 70, 20), generator=g).to(I8), torch.rand(3, 20, generator=g)
    x = torch.randint(-128, 128, (12, 70), generator=g).to(I8)
    sx = torch.rand(12, generator=g)
    plan = expert_plan(torch.arange(12).view(6, 2).remainder(3).to(dev), 3)
    handle_scale = sw.clone().to(dev)
    handle = int8_weight(wq.to(dev), handle_scale)
    handle_scale.zero_()                                          # the handle keeps its own
    y = int8_linear(x.to(dev), handle, scale=sx.to(dev), plan=plan)
    expert = torch.bucketize(torch.arange(12), plan.offsets.cpu().long()[1:], right=True)
    want, size = reference(x, sx, wq, sw, None, expert, torch.arange(12))
    close(y, want, size, F32)
    assert torch.equal(int8_linear(x.to(dev), int8_weight(wq[0].to(dev), sw[0].to(dev)), scale=sx.to(dev))[:1],
                       int8_linear(x[:1].to(dev), int8_weight(wq[0].to(dev), sw[0].to(dev)), scale=sx[:1].to(dev)))


def refusals(dev):
    x, w = torch.zeros(4, 8, device=dev), int8_weight(torch.ones(8, 6, device=dev))
    w3 = int8_weight(torch.ones(3, 8, 6, device=dev))
    q, s = torch.zeros(4, 8, dtype=I8, device=dev), torch.zeros(4, device=dev)
    plan = expert_plan(torch.zeros(2, 2, dtype=torch.int64, device=dev), 3)
    one = torch.ones(6, device=dev)
    for bad in (lambda: int8_weight(torch.ones(8, device=dev)), lambda: int8_weight(torch.ones(8, 6, device=dev).double()),
                lambda: int8_weight(torch.ones(0, 6, device=dev)), lambda: int8_weight(torch.ones(8, 0, device=dev)),
                lambda: int8_weight(torch.ones(MAX_CIN + 1, 1, device=dev)), lambda: int8_weight(torch.ones(1025, 1, 1, device=dev)),
                lambda: int8_weight(q), lambda: int8_weight(q, s), lambda: int8_weight(x, one), lambda: int8_weight(q, torch.zeros(8, device=dev).double()),
                lambda: quantize_rows(x[0]), lambda: quantize_rows(x.double()), lambda: quantize_rows(q), lambda: quantize_rows(x[:, :0]),
                lambda: quantize_rows(x.clone().requires_grad_()),
                lambda: int8_linear(x, x), lambda: int8_linear(x[:, :7], w), lambda: int8_linear(x[0], w), lambda: int8_linear(x.double(), w),
                lambda: int8_linear(q, w), lambda: int8_linear(q, w, scale=s[:3]), lambda: int8_linear(q, w, scale=s.double()), lambda: int8_linear(x, w, scale=s),
                lambda: int8_linear(x, w, one[:5]), lambda: int8_linear(x, w, one.long()), lambda: int8_linear(x, w, one.view(1, 6)),
                lambda: int8_linear(x, w, out_dtype=torch.float64), lambda: int8_linear(x, w, out_dtype=I8),
                lambda: int8_linear(x, w3), lambda: int8_linear(x, w, gather=True), lambda: int8_linear(x, w, plan=plan),
                lambda: int8_linear(x[:3], w3, plan=plan), lambda: int8_linear(x, w3, plan=plan, gather=True), lambda: int8_linear(x, w3, plan=(1, 2)),
                lambda: int8_linear(x, w3, one.view(1, 6).expand(2, 6), plan=plan), lambda: int8_linear(x.clone().requires_grad_(), w)):
        with pytest.raises(_lib.CG3DError):
            bad()
    with torch.no_grad():
        assert int8_linear(x.clone().requires_grad_(), w).shape == (4, 6)


def test_refusals(oracle):
    with _lib.use_library(oracle):
        refusals("cpu")
        assert int8_linear(torch.zeros(0, 8), int8_weight(torch.ones(8, 6))).shape == (0, 6)
        assert quantize_rows(torch.zeros(0, 8))[0].shape == (0, 8)


def test_entry_points_refuse(oracle):
    """The C-ABI's own checks (the same conditions in the library and in its restatement; nothing is launched)."""
    f = torch.zeros(4096)
    a = f.data_ptr()
    for lib in (oracle, _lib.bind(_lib.HIP_LIB_PATH)):
        for e, cin, cout in ((0, 8, 8), (1025, 8, 8), (1, 0, 8), (1, MAX_CIN + 1, 8), (1, 8, 0), (1, 8, (1 << 20) + 1)):
            assert lib.raw("cg3d_int8_weight_bytes")(e, cin, cout) == -1
            assert lib.raw("cg3d_int8_weight")(a, 0, e, cin, cout, a, a, a, None) == -1
        for args in ((None, 0, 1, 8, 8, a, a, a), (a, 4, 1, 8, 8, a, a, a), (a, 0, 1, 8, 8, None, a, a), (a, 0, 1, 8, 8, a + 4, a, a),
                     (a, 0, 1, 8, 8, a, None, a), (a, 0, 1, 8, 8, a, a, None), (a + 2, 0, 1, 8, 8, a, a, a), (a + 1, 1, 1, 8, 8, a, a, a)):
            assert lib.raw("cg3d_int8_weight")(*args, None) == -1, args
        for args in ((a, 3, 4, 8, 8, a, a), (a, 0, -1, 8, 8, a, a), (a, 0, 4, 0, 8, a, a), (a, 0, 4, 8, 7, a, a), (None, 0, 4, 8, 8, a, a),
                     (a, 0, 4, 8, 8, None, a), (a, 0, 4, 8, 8, a, None), (a + 2, 0, 4, 8, 8, a, a), (a, 0, 4, 8, 8, a, a + 2)):
            assert lib.raw("cg3d_int8_quantize_rows")(*args, None) == -1, args
        good = dict(x=a, dtype=0, sx=None, n_x=4, cin=8000, w=a, sw=a, bias=None, bpe=0, offsets=None, rows=None, y=a, out=0, n_rows=4, cout=6, e=1, ws=a)
        for change in (dict(dtype=4), dict(dtype=-1), dict(out=3), dict(out=-1), dict(bpe=2), dict(n_x=3), dict(e=2), dict(rows=a), dict(x=None),
                       dict(w=None), dict(sw=None), dict(y=None), dict(ws=None), dict(ws=a + 4), dict(x=a + 2), dict(w=a + 8), dict(y=a + 2),
                       dict(sw=a + 2), dict(bias=a + 1), dict(dtype=3, ws=None), dict(dtype=3, sx=a + 2), dict(n_x=-4, n_rows=-4), dict(cin=0), dict(cout=0),
                       dict(offsets=a, n_x=3), dict(offsets=a, rows=a, n_x=0), dict(offsets=a + 2), dict(offsets=a, rows=a + 1), dict(n_rows=1 << 31, n_x=1 << 31)):
            assert lib.raw("cg3d_int8_linear")(*{**good, **change}.values(), None) == -1, change


@pytest.mark.parametrize("cin,cout", [(1, 1), (512, 512), (4096, 4096), (4096, 16384), (131071, 1 << 20)])
@pytest.mark.parametrize("grouped_call", [0, 1])
def test_no_rows_need_no_workspace(oracle, cin, cout, grouped_call):
    """Any weights, no rows: nothing is launched, and the choice of a kernel has no sizes to divide by."""
    for lib in (oracle, _lib.bind(_lib.HIP_LIB_PATH)):
        for dtype in range(4):
            assert lib.raw("cg3d_int8_linear_ws_bytes")(dtype, 0, cin, 0, cout, 3 if grouped_call else 1, grouped_call) == 0


def test_no_cpu_fallback():
    with _lib.use_library(_lib.bind(_lib.HIP_LIB_PATH)):
        with pytest.raises(_lib.CG3DError):
            int8_weight(torch.zeros(4, 2))
        with pytest.raises(_lib.CG3DError):
            quantize_rows(torch.zeros(4, 2))


# ------------------------------------------------------------------------------------------------------------------- GPU
def weights_that_are_views_or_copies(dev):
    g = torch.Generator().manual_seed(60)
    w, scale = torch.randint(-127, 128, (3, 40, 20), generator=g).to(I8).to(dev), (torch.rand(20, 3, generator=g) + 0.1).to(dev)
    x, plan = torch.randn(12, 40, generator=g).to(dev), expert_plan(torch.arange(12).remainder(3).to(dev), 3)
    weight = int8_weight(w, scale.t())                            # (its columns are the neighbours in memory)
    y = int8_linear(x, weight, plan=plan, gather=True)
    assert torch.equal(y, int8_linear(x, int8_weight(w, scale.t().contiguous()), plan=plan, gather=True))
    for other in (copy.deepcopy(weight), pickle.loads(pickle.dumps(weight))):      # own memory, also when the first is gone
        weight.packed.zero_()
        assert torch.equal(int8_linear(x, other, plan=plan, gather=True), y)
        weight.packed.copy_(other.packed)


def test_weights_that_are_views_or_copies(oracle):
    with _lib.use_library(oracle):
        weights_that_are_views_or_copies("cpu")


@pytest.mark.gpu
def test_hip_levels_and_nonfinite(hip):
    levels("cuda")
    short_levels("cuda", BF16)
    short_levels("cuda", F16)
    nonfinite("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin", [(1, 1), (3, 15), (1000, 64), (77, 250), (513, 512), (130, 1025), (65, 4096), (9, 5000), (3, 43904), (2, MAX_CIN)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_hip_quantize_rows(hip, n, cin, dtype):
    x = make(n, cin, 1, dtype, 11)[0].cuda()
    check_levels(x, *quantize_rows(x))


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout", [
    (20, 500, 70), (50, 1000, 70), (50, 1900, 40), (20, 4000, 70), (20, 6000, 70),                          # few rows, by the chunks a wave holds
    (25000, 60, 60), (25000, 60, 130), (25000, 120, 130), (25000, 120, 250), (25000, 300, 250), (25000, 300, 60), (25000, 300, 130),
    (1700, 300, 250), (70000, 40, 520), (66500, 130, 1100), (21000, 700, 130), (20001, 832, 300),   # one pass: panels of a wave, chunks held
    (3000, 4100, 130), (3000, 700, 700), (53000, 600, 70)])                                                                   # tiles, in parts and whole
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (I8, F32)])
def test_hip_each_kernel_of_the_choice(hip, n, cin, cout, dtype, out):
    dense(n, cin, cout, dtype, out, True, 50, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts,cin,cout", [(1500, 2, 5, 4200, 130), (300, 2, 18, 1000, 200), (60, 2, 64, 1000, 520), (12000, 2, 7, 600, 100)])
@pytest.mark.parametrize("dtype,out,gather", [(F32, F32, True), (BF16, BF16, True), (I8, F32, False)])
def test_hip_grouped_long_rows(hip, t, k, experts, cin, cout, dtype, out, gather):
    grouped(ids_of(t, k, experts, "dropped", 51), experts, cin, cout, dtype, out, 2, gather, 52, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin", [(70, 257), (70, 1000), (30, 2047), (30, 4095), (20, 8193), (20, 16384), (20, 16385), (600, 17001), (20, 32768), (20, 32769), (600, 49152), (520, 49153)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_hip_quantize_long_rows(hip, n, cin, dtype):
    x = make(n, cin, 1, dtype, 14)[0].cuda()
    check_levels(x, *quantize_rows(x))


@pytest.mark.gpu
def test_hip_weights_that_are_views_or_copies(hip):
    weights_that_are_views_or_copies("cuda")


@pytest.mark.gpu
def test_hip_large_tiles_are_reached(hip):
    """Sizes whose products go to the largest tiles, dense and grouped, with a ragged last tile each way."""
    dense(6500, 530, 1900, BF16, F32, True, 40, "cuda")
    dense(6401, 576, 2052, I8, BF16, False, 41, "cuda")
    grouped(ids_of(9000, 2, 4, "dropped", 42), 4, 600, 700, F32, F32, 2, True, 43, "cuda")
    grouped(ids_of(20000, 1, 3, "uniform", 44), 3, 528, 640, I8, F16, 1, False, 45, "cuda")


WIDE = [(1, 64, 64), (1, 4096, 256), (5, 512, 320), (16, 1000, 72), (31, 2048, 100), (64, 512, 512), (65, 576, 64), (127, 64, 128), (128, 128, 64),
        (300, 512, 192), (1003, 200, 77), (513, 1024, 300), (2050, 384, 136), (4099, 64, 64), (700, 1100, 520), (40, 43904, 128), (300, 9000, 64),
        (3, MAX_CIN, 5), (5000, 130, 40), (256, 2048, 512), (1000, 640, 640), (25001, 70, 260), (25000, 200, 130), (13000, 500, 264), (26000, 33, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout", ODD + WIDE)
@pytest.mark.parametrize("dtype,out,bias", [(F32, F32, True), (BF16, BF16, True), (F16, F16, False), (I8, F32, True), (I8, BF16, False)])
def test_hip_dense(hip, n, cin, cout, dtype, out, bias):
    dense(n, cin, cout, dtype, out, bias, 12, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout", [(70, 200, 77), (130, 64, 64), (5, 512, 64), (260, 1024, 128), (3000, 1024, 192),
                                        (2000, 320, 320)])
def test_hip_dense_at_odd_addresses(hip, n, cin, cout):
    for dtype, out in ((F32, F32), (BF16, BF16), (F16, F16), (I8, F32)):
        dense(n, cin, cout, dtype, out, True, 13, "cuda", offset=1)


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,experts,cin,cout,kind", [
    (1, 1, 1, 64, 64, "uniform"), (1, 2, 18, 128, 64, "uniform"), (4, 2, 64, 512, 512, "uniform"), (20, 2, 5, 33, 18, "dropped"),
    (300, 2, 18, 128, 64, "dropped"), (300, 2, 18, 128, 64, "one"), (50, 2, 7, 70, 90, "none"), (900, 4, 61, 96, 200, "uniform"),
    (64, 1, 200, 100, 70, "uniform"), (1500, 2, 3, 640, 256, "dropped"), (700, 2, 4, 1024, 130, "uniform"), (3000, 2, 10, 64, 64, "uniform"),
    (16, 4, 1024, 64, 32, "uniform"), (13000, 2, 5, 130, 300, "dropped"), (9000, 3, 7, 500, 130, "uniform")])
@pytest.mark.parametrize("dtype,out,bias,gather", [(F32, F32, 2, True), (BF16, BF16, 0, True), (F16, F16, 1, False), (I8, F32, 2, True), (I8, BF16, 2, False)])
def test_hip_grouped(hip, t, k, experts, cin, cout, kind, dtype, out, bias, gather):
    grouped(ids_of(t, k, experts, kind, 14), experts, cin, cout, dtype, out, bias, gather, 15, "cuda")


@pytest.mark.gpu
def test_hip_largest_sum_does_not_wrap(hip):
    """Every product at its largest: -128 * -128 over the longest contraction."""
    x = torch.full((3, MAX_CIN), -128, dtype=I8, device="cuda")
    w = int8_weight(torch.full((MAX_CIN, 2), -128, dtype=I8, device="cuda"), torch.ones(2, device="cuda"))
    y = int8_linear(x, w, scale=torch.ones(3, device="cuda"))
    want = 16384.0 * MAX_CIN
    assert bool(((y.double() - want).abs() <= 2.0 ** -24 * want).all())


@pytest.mark.gpu
def test_hip_weights_in_8_bits(hip):
    eight_bit_weights("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_hip_quantised_first_is_the_same(hip, dtype):
    """A row quantised in the call and one quantised before it give the same bits, whichever kernel takes them."""
    for n, cin, cout in ((1, 512, 512), (40, 100, 70), (3000, 256, 128), (600, 1500, 64), (9, 6000, 130)):
        x, _, w, b = make(n, cin, cout, dtype, 16)
        x, weight, b = x.cuda(), int8_weight(w.cuda()), b.cuda()
        q, s = quantize_rows(x)
        assert torch.equal(int8_linear(x, weight, b, out_dtype=F32), int8_linear(q, weight, b, scale=s))


@pytest.mark.gpu
def test_hip_gather_is_the_gathered_product(hip):
    for t, cin in ((5, 128), (2000, 128), (300, 700)):
        ids = ids_of(t, 2, 18, "dropped", 17).cuda()
        plan = expert_plan(ids, 18)
        x, _, w, b = make(t, cin, 64, BF16, 18, 18)
        x, weight, b = x.cuda(), int8_weight(w.cuda()), b.cuda()
        assert torch.equal(int8_linear(x, weight, b, plan=plan, gather=True), int8_linear(expert_gather(x, plan), weight, b, plan=plan))


@pytest.mark.gpu
def test_hip_views_and_bias_types(hip):
    x, _, w, b = make(64, 96, 40, BF16, 19)
    x, w, b = x.cuda(), w.cuda(), b.cuda()
    want = int8_linear(x, int8_weight(w), b.to(BF16).float())
    assert torch.equal(int8_linear(x.t().contiguous().t(), int8_weight(w.t().contiguous().t()), b.to(BF16)), want)
    wide = torch.randn(64, 200, device="cuda").to(BF16)
    wide[:, 50:146] = x
    assert torch.equal(int8_linear(wide[:, 50:146], int8_weight(w), b.to(BF16)), want)


@pytest.mark.gpu
def test_hip_graph_replays_with_new_inputs(hip):
    """A served layer of experts captured once, replayed on new tokens with eager calls between; two graphs share nothing."""
    t, k, e = 700, 2, 18
    weight = int8_weight(make(1, 640, 128, F32, 20, e)[2].cuda())
    small = int8_weight(make(1, 128, 64, F32, 21, e)[2].cuda())
    ids = [ids_of(t, k, e, "dropped", s).cuda() for s in (22, 23, 24)]
    xs = [make(t, 640, 1, BF16, s)[0].cuda() for s in (22, 23, 24)]
    gate = torch.rand(t, k, device="cuda")

    def step(i, x):
        plan = expert_plan(i, e)
        return expert_combine(int8_linear(int8_linear(x, weight, plan=plan, gather=True), small, plan=plan), plan, gate)
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
            assert torch.equal(outs[j], step(ids[(turn + j) % 3], xs[(turn + j) % 3]))


@pytest.mark.gpu
def test_hip_large_tiles_in_a_graph(hip):
    x, _, w, b = make(6500, 600, 1900, BF16, 46)
    x, weight, b = x.cuda(), int8_weight(w.cuda()), b.cuda()
    other = make(6500, 600, 1, BF16, 47)[0].cuda()
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    int8_linear(static, weight, b)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = int8_linear(static, weight, b)
    for v in (x, other, x):
        static.copy_(v)
        graph.replay()
        assert torch.equal(out, int8_linear(v, weight, b))


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout", [(2200000, 64, 1024), (600000, 4096, 64), (36, 512, 1 << 20)])
def test_hip_offsets_past_32_bits(hip, n, cin, cout):
    """Results (or rows, or a matrix) of more than 2^31 bytes: the last rows and channels are those of a small call."""
    g = torch.Generator(device="cuda").manual_seed(48)
    x = torch.randint(-128, 128, (n, cin), generator=g, device="cuda", dtype=torch.int32).to(I8) if n * cin < 2 ** 28 else \
        torch.randint(-128, 128, (n // 8, cin), generator=g, device="cuda", dtype=torch.int32).to(I8).repeat(8, 1)
    sx = torch.rand(n, generator=g, device="cuda") + 0.1
    wq = torch.randint(-128, 128, (cin, cout), generator=g, device="cuda", dtype=torch.int32).to(I8)
    sw = torch.rand(cout, generator=g, device="cuda") + 0.1
    y = int8_linear(x, int8_weight(wq, sw), scale=sx, out_dtype=BF16)
    for rows in (slice(0, 20), slice(n - 20, n)):
        for cols in (slice(0, 70), slice(max(0, cout - 70), cout)):
            want = int8_linear(x[rows], int8_weight(wq[:, cols].contiguous(), sw[cols].contiguous()), scale=sx[rows], out_dtype=BF16)
            assert torch.equal(y[rows, cols], want)


@pytest.mark.gpu
def test_hip_on_another_stream(hip):
    x, _, w, b = make(3000, 700, 192, BF16, 25)
    x, weight, b = x.cuda(), int8_weight(w.cuda()), b.cuda()
    want = int8_linear(x, weight, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8_linear(x, weight, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_hip_served_layer_of_experts(hip):
    """Two products of each token's experts and the weighted combination, against the same in 64 bits on the same levels."""
    t, k, e, c, n = 500, 2, 10, 128, 256
    ids = ids_of(t, k, e, "uniform", 26)
    x, _, w1, b1 = make(t, c, n, BF16, 27, e)
    w2 = make(1, n, c, F32, 28, e)[2]
    gate = torch.rand(t, k)
    plan = expert_plan(ids.cuda(), e)
    h = torch.relu(int8_linear(x.cuda(), int8_weight(w1.cuda()), b1.cuda(), plan=plan, gather=True, out_dtype=F32))
    y = int8_linear(h, int8_weight(w2.cuda()), plan=plan)
    out = expert_combine(y, plan, gate.cuda())
    rows, off = plan.rows.cpu().long(), plan.offsets.cpu().long()
    expert = torch.bucketize(torch.arange(t * k), off[1:], right=True)

    def levels_of(w):
        q, s = plain_levels(w.transpose(1, 2).reshape(-1, w.shape[1]))
        return q.view(e, w.shape[2], w.shape[1]).transpose(1, 2), s.view(e, w.shape[2])
    want, size = reference(x, None, *levels_of(w1), b1, expert, rows)
    close(h, torch.relu(want), size, F32)
    want, size = reference(h, None, *levels_of(w2), None, expert, torch.arange(t * k))
    close(y, want, size, F32)
    pos = plan.pos.cpu().long()
    terms = y.cpu().double()[pos] * gate.double().unsqueeze(2)
    assert bool(((out.cpu().double() - terms.sum(1)).abs() <= (k + 2) * 2.0 ** -24 * terms.abs().sum(1)).all())


@pytest.mark.gpu
def test_hip_refusals(hip):
    refusals("cuda")
    w = int8_weight(torch.ones(8, 6, device="cuda"))
    for bad in (lambda: int8_linear(torch.zeros(4, 8), w), lambda: int8_linear(torch.zeros(4, 8, device="cuda"), w, torch.zeros(6))):
        with pytest.raises(_lib.CG3DError):
            bad()
    assert int8_linear(torch.zeros(0, 8, device="cuda"), w).shape == (0, 6)


def traced_and_dual(dev):
    """torch.jit.trace records the calls (and their checks run on new inputs); a tangent, a graph of torch's own operators and weights
    laid out inside a trace are refused."""
    x, _, w, b = make(12, 40, 20, F32, 70, 3)
    x, w, b = x.to(dev), w.to(dev), b.to(dev)
    weight, one, plan = int8_weight(w), int8_weight(w[0]), expert_plan(torch.arange(12).remainder(3).to(dev), 3)
    q, s = quantize_rows(x)
    calls = ((lambda a: int8_linear(a, one, b[0]), x), (lambda a: int8_linear(a, weight, b, plan=plan, gather=True, out_dtype=BF16), x),
             (lambda a: int8_linear(a, weight, plan=plan), x.to(BF16)), (lambda a: int8_linear(q, one, scale=a), s), (lambda a: int8_linear(x, one, a), b[0]),
             (lambda a: quantize_rows(a)[0], x), (lambda a: quantize_rows(a)[1], x))
    for f, a in calls:
        traced = torch.jit.trace(f, (a,))
        junk = [torch.full_like(f(a), 7.0) for _ in range(4)]
        del junk
        other = (a.flip(0) * 3).contiguous()
        assert torch.equal(traced(other), f(other))
        with torch.no_grad():
            traced = torch.jit.trace(f, (a.clone().requires_grad_(),))
        assert torch.equal(traced(other), f(other))
        with forward_ad.dual_level():
            assert torch.equal(f(a), f(a))
            with pytest.raises(_lib.CG3DError):
                f(forward_ad.make_dual(a, torch.ones_like(a)))
        with pytest.raises(_lib.CG3DError):
            make_fx(f)(a)
        with pytest.raises(_lib.CG3DError):
            torch.jit.trace(f, (a.clone().requires_grad_(),))
    with pytest.raises(RuntimeError, match="columns"):
        torch.jit.trace(calls[0][0], (x,))(x[:, 1:].contiguous())
    with pytest.raises(_lib.CG3DError):
        torch.jit.trace(lambda a: int8_linear(x, int8_weight(a)), (w[0],))
    with forward_ad.dual_level(), pytest.raises(_lib.CG3DError):
        int8_weight(forward_ad.make_dual(w, torch.ones_like(w)))


def test_traces_and_tangents(oracle):
    with _lib.use_library(oracle):
        traced_and_dual("cpu")


@pytest.mark.gpu
def test_hip_traces_and_tangents(hip):
    traced_and_dual("cuda")


def negated_views(dev):
    """Views whose memory holds the opposite of their values count with their values."""
    x, _, w, b = make(12, 40, 20, F32, 80, 3)
    x, w, b, neg = x.to(dev), w.to(dev), b.to(dev), torch._neg_view
    weight, one, plan = int8_weight(w), int8_weight(w[0]), expert_plan(torch.arange(12).remainder(3).to(dev), 3)
    q, s = quantize_rows(x)
    assert torch.equal(quantize_rows(neg(x))[0], -q) and torch.equal(quantize_rows(neg(x))[1], s)
    assert torch.equal(int8_linear(neg(x), one, neg(b[0])), int8_linear(-x, one, -b[0]))
    assert torch.equal(int8_linear(neg(x), weight, neg(b.to(BF16)), plan=plan, gather=True), int8_linear(-x, weight, -b.to(BF16), plan=plan, gather=True))
    assert torch.equal(int8_linear(neg(q), one, scale=neg(s)), int8_linear(q, one, scale=s))       # (both signs)
    assert torch.equal(int8_linear(x, int8_weight(neg(w)), plan=plan), int8_linear(x, int8_weight(-w), plan=plan))
    wq = quantize_rows(w[0].t().contiguous())[0].t()
    assert torch.equal(int8_linear(x, int8_weight(neg(wq), neg(b[0]))), int8_linear(x, int8_weight(-wq, -b[0])))


def test_negated_views(oracle):
    with _lib.use_library(oracle):
        negated_views("cpu")


@pytest.mark.gpu
def test_hip_negated_views(hip):
    negated_views("cuda")


def compiled(dev):
    """torch.compile stops at the addresses that a call takes and resumes behind them: workspaces, copies of inputs, weights and plans made
    for one call are there until it has been made."""
    x, _, w, b = make(60, 40, 20, F32, 90, 3)
    x, w, b, gate, ids = x.to(dev), w.to(dev), b.to(dev), torch.rand(60, 2).to(dev), ids_of(60, 2, 3, "dropped", 91).to(dev)
    weight, plan = int8_weight(w), expert_plan(ids, 3)
    turned = lambda t: t.t().contiguous().t()                     # (copied by the call)
    for f in (lambda t: expert_gather(turned(t), expert_plan(turned(ids), 3)), lambda t: expert_combine(turned(expert_gather(t, plan)), plan, turned(gate)),
              lambda t: quantize_rows(turned(t))[0], lambda t: int8_linear(turned(t), int8_weight(turned(w[0])), b[0].to(BF16)),
              lambda t: expert_combine(int8_linear(t, weight, b, plan=plan, gather=True), plan, gate),
              lambda t: torch.autograd.grad(expert_combine(expert_gather(t.requires_grad_(), plan), plan, gate).sum(), [t])[0]):
        torch._dynamo.reset()
        g = torch.compile(f, backend="eager")
        for i in range(20):
            assert torch.equal(g(x * i), f(x * i))


def test_compiled(oracle):
    with _lib.use_library(oracle):
        compiled("cpu")


@pytest.mark.gpu
def test_hip_compiled(hip):
    compiled("cuda")


def far_scales(dev, sizes):
    """Row and channel scales at both ends of fp32's range whose product with the sum is back in it: no step on the way leaves the range
    or its full precision.  In floats (rows of 1e35 against weights of 1e-5 and the like) and in 8 bits, where the scales are given; a
    result beyond the type is an infinity, one below it rounds once more."""
    g = torch.Generator().manual_seed(100)
    for n, cin, cout in sizes:
        for top, low in ((3e37, 1e-3), (1e35, 1e-5), (3e38, 1e-30), (1e-30, 1e20), (1e-5, 1e35), (1e-30, 3e38)):
            x = torch.randn(n, cin, generator=g).clamp(-3, 3) * (top / 3.1)
            w = torch.randn(cin, cout, generator=g).clamp(-3, 3) * (low / 3.1)
            wq, sw = plain_levels(w.t().contiguous())
            for dtype in (F32, BF16):
                v = x.to(dtype)
                y = int8_linear(v.to(dev), int8_weight(w.to(dev)), out_dtype=F32)
                want, size = reference(v, None, wq.t().unsqueeze(0), sw.unsqueeze(0), None, torch.zeros(n, dtype=torch.long), torch.arange(n))
                assert bool((want.abs().amax() < 2.0 ** 127))
                close(y, want, size, F32)
        q = torch.randint(-128, 128, (n, cin), generator=g).to(I8)
        wq = torch.randint(-128, 128, (cin, cout), generator=g).to(I8)
        for a, b in ((2.0 ** 120, 2.0 ** -149), (2.0 ** 126, 2.0 ** -140), (2.0 ** -149, 2.0 ** 100), (1.5 * 2.0 ** -126, 1.25 * 2.0 ** 127), (2.0 ** -140, 2.0 ** 127),
                     (1.7 * 2.0 ** -70, 1.3 * 2.0 ** -70), (2.0 ** -100, 1.1), (1.9 * 2.0 ** 64, 1.1 * 2.0 ** -64)):
            sx = torch.full((n,), a) * (1 + torch.arange(n) % 2)     # (exact: whole and twice as much)
            sw = torch.full((cout,), b) if b < 2.0 ** -126 else b * (1 + torch.rand(cout, generator=g) / 8)
            y = int8_linear(q.to(dev), int8_weight(wq.to(dev), sw.to(dev)), scale=sx.to(dev))
            want, size = reference(q, sx, wq.unsqueeze(0), sw.unsqueeze(0), None, torch.zeros(n, dtype=torch.long), torch.arange(n))
            assert bool((want.abs().amax() < 2.0 ** 127))
            close(y, want, size, F32)                             # (2^-126 covers what is below the normal range)
        zero = torch.zeros(1, cin, dtype=I8)
        big = int8_weight(wq.to(dev), torch.full((cout,), 3e38, device=dev))
        assert bool((int8_linear(zero.to(dev), big, scale=torch.full((1,), 3e38, device=dev)) == 0).all())
        ones = int8_weight(torch.ones(cin, cout, dtype=I8, device=dev), torch.full((cout,), 3e38, device=dev))
        for sign in (1, -1):
            y = int8_linear(torch.full((1, cin), sign, dtype=I8, device=dev), ones, scale=torch.full((1,), 3e38, device=dev))
            assert bool((y == sign * float("inf")).all())


def test_far_scales(oracle):
    with _lib.use_library(oracle):
        far_scales("cpu", [(3, 64, 5), (20, 33, 18)])


@pytest.mark.gpu
def test_hip_far_scales(hip):
    far_scales("cuda", [(3, 64, 5), (20, 500, 70), (1700, 300, 130), (3000, 700, 70), (600, 4200, 130), (6500, 600, 300)])


@pytest.mark.parametrize("n,cin,cout", [(4000000, 1024, 64), (3000, 1024, 192), (4096, 4096, 4096), (512, 43904, 128), (5, 512, 64), (300000, 64, 64)])
@pytest.mark.parametrize("grouped_call", [0, 1])
def test_aligned_rows_in_8_bits_need_no_copy(n, cin, cout, grouped_call):
    """Rows in 8 bits that the kernels read where they are ask for no memory to be copied to; other rows, and a query that does not say
    how they are aligned, for theirs."""
    ws = _lib.bind(_lib.HIP_LIB_PATH).raw("cg3d_int8_linear_ws_bytes")
    copy = n * cin
    for c, flags, copied in ((cin, grouped_call | 2, False), (cin, grouped_call, None), (cin + 1, grouped_call | 2, None)):
        got = ws(3, n, c, n, cout, 1, flags)
        parts = ws(3, n, cin, n, cout, 1, grouped_call | 2)       # (partial sums of a long contraction: less than the rows)
        assert 0 <= got and (copied is None or got < copy) and got in (parts, parts + n * ((c + 63) // 64 * 64) + (4 * n + 255) // 256 * 256)
    assert ws(3, n, cin, n, cout, 1, 4) == -1
    for dtype in range(3):                                        # rows in floats: the same either way
        assert ws(dtype, n, cin, n, cout, 1, grouped_call | 2) == ws(dtype, n, cin, n, cout, 1, grouped_call)


@pytest.mark.gpu
def test_hip_aligned_rows_in_8_bits_need_no_copy(hip):
    """A product of rows that are aligned allocates its result and nothing of the rows' size; at an odd address it copies them, with
    the same bits; the workspace of one does not serve the other."""
    g = torch.Generator(device="cuda").manual_seed(110)
    n, cin = 60000, 1024
    store = torch.randint(-128, 127, (n * cin + 16,), generator=g, device="cuda", dtype=I8)
    sx, w = torch.rand(n, generator=g, device="cuda") + 0.1, int8_weight(torch.randn(cin, 64, generator=g, device="cuda"))
    x = store[:n * cin].view(n, cin)

    def extra(rows):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = int8_linear(rows, w, scale=sx, out_dtype=BF16)
        torch.cuda.synchronize()
        return y, torch.cuda.max_memory_allocated() - before
    int8_linear(x[:300], w, scale=sx[:300])
    for _ in range(2):
        y, more = extra(x)
        assert more < 2 * 2 * n * 64
        for off in (1, 4, 8, 15):
            odd = store[off:off + n * cin].view(n, cin)
            z, more = extra(odd)
            assert more >= n * cin and torch.equal(z, int8_linear(odd.clone(), w, scale=sx, out_dtype=BF16))
    assert torch.equal(y, int8_linear(x, w, scale=sx, out_dtype=BF16))


def test_large_tiles_take_whole_contractions():
    """Only the smaller tiles are used in parts (the larger ones have no code for it): partial sums ask for memory, whole contractions do not."""
    ws = _lib.bind(_lib.HIP_LIB_PATH).raw("cg3d_int8_linear_ws_bytes")
    for cin in (4096, 43904, 131056):
        for n, cout in ((8192, 4096), (65536, 256), (16384, 1024)):
            assert ws(3, n, cin, n, cout, 1, 2) == 0
    assert ws(3, 512, 43904, 512, 128, 1, 2) > 0                  # (shorter ones of so few rows go to the kernel for few rows)


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout", [(36, 4160, 1 << 20), (36, 131056, 33000)])
def test_hip_matrix_past_32_bits(hip, n, cin, cout):
    """A matrix, and its packed form, of more than 2^32 bytes, for the larger and the smaller tiles: its first and last channels are those
    of a small call."""
    assert cin * cout > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(120)
    x = torch.randint(-128, 127, (n, cin), generator=g, device="cuda", dtype=I8)
    sx, sw = torch.rand(n, generator=g, device="cuda") + 0.1, torch.rand(cout, generator=g, device="cuda") + 0.1
    wq = torch.randint(-128, 127, (cin, cout), generator=g, device="cuda", dtype=I8)
    y = int8_linear(x, int8_weight(wq, sw), scale=sx, out_dtype=F32)
    for cols in (slice(0, 70), slice(cout // 2, cout // 2 + 70), slice(cout - 70, cout)):
        assert torch.equal(y[:, cols], int8_linear(x, int8_weight(wq[:, cols].contiguous(), sw[cols].contiguous()), scale=sx))


@pytest.mark.gpu
@pytest.mark.parametrize("t,cin,cout,dtype", [(20, 2048, 2112, I8), (20, 2048, 2112, BF16), (300, 512, 8320, I8), (700, 2048, 2080, I8)])
def test_hip_experts_past_32_bits(hip, t, cin, cout, dtype):
    """The matrices of 1024 experts, of more than 2^32 bytes, for few rows, one pass and tiles: rows of the first, a middle and the last
    expert are those of a product with its matrix alone."""
    e = 1024
    assert e * cin * cout > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(121)
    x = torch.randn(t, cin, generator=g, device="cuda").to(BF16)
    ids = torch.randint(0, e, (t, 1), generator=g, device="cuda")
    ids[::3], ids[1::7] = e - 1, 0
    ids[2], ids[4] = 513, -1
    wq = torch.randint(-128, 127, (e, cin, cout), generator=g, device="cuda", dtype=I8) if dtype == I8 else \
        torch.randn(e, cin, cout, generator=g, device="cuda", dtype=BF16)
    sw = torch.rand(e, cout, generator=g, device="cuda") + 0.1 if dtype == I8 else None
    plan = expert_plan(ids, e)
    y = int8_linear(x, int8_weight(wq, sw), plan=plan, gather=True, out_dtype=F32)
    for i in (0, 513, e - 1):
        at = plan.pos[:, 0][ids[:, 0] == i].long()
        assert at.numel() > 0
        assert torch.equal(y[at], int8_linear(x[ids[:, 0] == i], int8_weight(wq[i], None if sw is None else sw[i]), out_dtype=F32))
    assert bool((y[int(plan.offsets[-1]):] == 0).all())


def layer_rounds_once(dev):
    """A layer of experts on 16-bit rows whose results stay in fp32 until they are combined is off by one rounding to the type; with the
    default types by two."""
    t, k, e, cin, cout = 200, 2, 5, 64, 40
    ids, gate = ids_of(t, k, e, "dropped", 130), torch.rand(t, k, generator=torch.Generator().manual_seed(131))
    for dtype in (BF16, F16):
        x, _, w, b = make(t, cin, cout, dtype, 132, e)
        wq, sw = plain_levels(w.transpose(1, 2).reshape(-1, cin))
        plan = expert_plan(ids.to(dev), e)
        rows, off, pos = plan.rows.cpu().long(), plan.offsets.cpu().long(), plan.pos.cpu().long()
        expert = torch.bucketize(torch.arange(t * k), off[1:], right=True)
        expert[expert == e] = -1
        y, size = reference(x, None, wq.view(e, cout, cin).transpose(1, 2), sw.view(e, cout), b, expert, rows.clamp(min=0))
        terms = torch.where((pos >= 0).unsqueeze(2), y[pos.clamp(min=0)] * gate.double().unsqueeze(2), 0.0)
        sizes = torch.where((pos >= 0).unsqueeze(2), size[pos.clamp(min=0)] * gate.double().unsqueeze(2), 0.0).sum(1)
        want, fp32 = terms.sum(1), (6 + k + 2) * 2.0 ** -24 * sizes     # the product's 6 half-steps and the sum's
        weight = int8_weight(w.to(dev))
        once = expert_combine(int8_linear(x.to(dev), weight, b.to(dev), plan=plan, gather=True, out_dtype=F32), plan, gate.to(dev), dtype)
        twice = expert_combine(int8_linear(x.to(dev), weight, b.to(dev), plan=plan, gather=True), plan, gate.to(dev))
        assert once.dtype == twice.dtype == dtype
        for got, before in ((once, 0.0), (twice, HALF[dtype] * terms.abs().sum(1))):
            off_by = (got.cpu().double() - want).abs()
            assert bool((off_by <= HALF[dtype] * want.abs() * (1 + 2.0 ** -7) + (before + fp32) * (1 + 2.0 ** -7) + 2 * TINY[dtype] * k).all())


def test_layer_of_experts_rounds_once(oracle):
    with _lib.use_library(oracle):
        layer_rounds_once("cpu")


@pytest.mark.gpu
def test_hip_layer_of_experts_rounds_once(hip):
    layer_rounds_once("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,cin,cout,dtype", [(64 * (768 + 40) + 5, 600, 520, BF16), (64 * (768 + 239) + 1, 832, 530, F16), (64 * (768 + 300), 700, 520, BF16),
                                              (64 * (1024 + 30) + 63, 500, 520, I8)])
def test_hip_last_tiles_behind_whole_rounds(hip, n, cin, cout, dtype):
    """Tiles whose panels are shared out, behind whole rounds of three and of four workgroups a CU."""
    dense(n, cin, cout, dtype, F32 if dtype == I8 else dtype, True, 140, "cuda")
