"""The residual add + norm and the microscaled quantisation on the GPU, against 64-bit references
(mx_ref.py).  Codes, scales and the rounded sums must be the references' exactly: the kernels
decide in 64 bits (norm) or on exact values (quantisation)."""
import numpy as np
import pytest
import torch

import mx_ref
from gpu_helpers import bf, dev, host

pytestmark = pytest.mark.gpu


def _rows(g, rows, cols, scale=1.0):
    v = g.standard_normal((rows, cols)) * scale
    v[:, g.integers(0, cols, max(1, cols // 200))] *= 15
    return v.astype(np.float32)


def _norm_ref(x, res, w, eps):
    s = x.astype(np.float64) + (0 if res is None else res.astype(np.float64))
    with np.errstate(all="ignore"):
        inv = 1 / np.sqrt((s * s).sum(1, keepdims=True) / s.shape[1] + eps)
        return s, s * inv * w.astype(np.float64)


def _check_bf16(got, want, what):
    """Half a bf16 step: 2^-8 of the value (2^-134 among the smallest numbers)."""
    g = bf(got).astype(np.float64)
    with np.errstate(all="ignore"):
        near = np.abs(g - want) <= np.abs(want) * 2.0 ** -8 + 2.0 ** -134
    over = np.abs(want) >= 2.0 ** 128 * (1 - 2.0 ** -9)
    ok = near | (np.isnan(g) & np.isnan(want)) | (over & (g == np.copysign(np.inf, want)))
    assert ok.all(), (what, np.argwhere(~ok)[:4])


def _run_norm(x, res, w, eps, quant=True, normed=True, sums=True):
    from pegainfer_amd import ops
    rows, cols = x.shape
    new = lambda: torch.full((rows, cols), 7.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    s, y = new() if sums else None, new() if normed else None
    q = ops.MxTensor.empty(rows, cols, ops.MxFormat.Fp8E4M3) if quant else None
    xd = dev(x) if x.dtype == np.float32 else dev(x, bf16=True)
    ops.add_rmsnorm(xd, None if res is None else dev(res, bf16=True), dev(w, bf16=True), eps,
                    residual_out=s, normed=y, quantized=q)
    return (host(s) if sums else None, host(y) if normed else None,
            (host(q.codes), host(q.scales)) if quant else None)


@pytest.mark.parametrize("x32", [False, True])
@pytest.mark.parametrize("rows,cols", [
    (1, 7168), (3, 2048), (5, 32), (1, 8), (2, 40), (9, 96), (333, 2048), (257, 1408), (4, 520),
    (6, 1024), (5, 1032), (2, 4096), (3, 4104), (2, 8192), (2, 16384), (2, 32768), (3, 20000)])
def test_norm_matches_the_formula(rows, cols, x32):
    g = np.random.default_rng(rows * 7 + cols)
    quant = cols % 32 == 0
    xb = mx_ref.bf16_round(_rows(g, rows, cols, 0.5))
    x = _rows(g, rows, cols, 0.5) if x32 else xb
    xf = x if x32 else bf(x)
    res = mx_ref.bf16_round(_rows(g, rows, cols, 2.0))
    w = mx_ref.bf16_round(1 + 0.2 * g.standard_normal(cols))
    for r in (res, None):
        s, y = _norm_ref(xf, None if r is None else bf(r), bf(w), 1e-6)
        gs, gy, gq = _run_norm(x, r, w, 1e-6, quant=quant)
        assert np.array_equal(gs, mx_ref.bf16_round(s))
        _check_bf16(gy, y, "normed")
        if quant:
            codes, scales = mx_ref.quantize(y, "fp8")
            assert np.array_equal(gq[1], scales)
            assert np.array_equal(gq[0], codes)


def test_norm_outputs_alone_are_the_joint_calls():
    g = np.random.default_rng(3)
    x, res = (mx_ref.bf16_round(_rows(g, 6, 1408)) for _ in range(2))
    w = mx_ref.bf16_round(g.standard_normal(1408))
    s, y, q = _run_norm(x, res, w, 1e-5)
    assert np.array_equal(_run_norm(x, res, w, 1e-5, quant=False, normed=False)[0], s)
    assert np.array_equal(_run_norm(x, res, w, 1e-5, quant=False, sums=False)[1], y)
    alone = _run_norm(x, res, w, 1e-5, normed=False, sums=False)[2]
    assert np.array_equal(alone[0], q[0]) and np.array_equal(alone[1], q[1])


def test_norm_extremes():
    """Zero rows, rows whose squares pass fp32's range on either side, infinities and NaN."""
    cols = 2048
    g = np.random.default_rng(4)
    x = _rows(g, 8, cols)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 77] = np.inf
    x[4, 2047] = np.nan
    x[5] = 0
    x[5, 5] = -3.0
    x[6] *= 1e-38
    w = mx_ref.bf16_round(1 + 0.1 * g.standard_normal(cols))
    for eps in (1e-6, 0.0):
        s, y = _norm_ref(x, None, bf(w), eps)
        gs, gy, (gc, gsc) = _run_norm(x, None, w, eps)
        nan = np.isnan(s)
        assert np.array_equal(gs[~nan], mx_ref.bf16_round(s)[~nan]) and np.isnan(bf(gs)[nan]).all()
        _check_bf16(gy, y, "normed")
        codes, scales = mx_ref.quantize(y, "fp8")
        assert np.array_equal(gsc, scales) and np.array_equal(gc, codes)


def test_norm_in_place_and_rows_are_independent():
    from pegainfer_amd import ops
    g = np.random.default_rng(5)
    x, res = (mx_ref.bf16_round(_rows(g, 300, 7168)) for _ in range(2))
    w = mx_ref.bf16_round(1 + 0.1 * g.standard_normal(7168))
    s, y, q = _run_norm(x, res, w, 1e-6)
    xd, rd = dev(x, bf16=True), dev(res, bf16=True)
    ops.add_rmsnorm(xd, rd, dev(w, bf16=True), 1e-6, residual_out=rd, normed=xd)
    assert np.array_equal(host(rd), s) and np.array_equal(host(xd), y)
    one = _run_norm(x[123:124], res[123:124], w, 1e-6)
    assert np.array_equal(one[0], s[123:124]) and np.array_equal(one[1], y[123:124])
    assert np.array_equal(one[2][0], q[0][123:124])


def test_norm_leaves_rows_past_its_own_alone():
    from pegainfer_amd import ops
    big = torch.full((9, 512), 3.0, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(5, 512, device="cuda").to(torch.bfloat16)
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    q = ops.MxTensor.empty(9, 512, ops.MxFormat.Fp8E4M3)
    q.codes.fill_(0x55), q.scales.fill_(0x66)
    ops.add_rmsnorm(x, None, w, 1e-6, normed=big[:5], quantized=q.head(5))
    torch.cuda.synchronize()
    assert (big[5:] == 3).all() and (q.codes[5:] == 0x55).all() and (q.scales[5:] == 0x66).all()


FORMATS = [("fp8", 0), ("fp4", 1)]


def _mx(name, n):
    from pegainfer_amd import ops
    return ops.MxFormat(n)


@pytest.mark.parametrize("name,n", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (5, 96), (2, 128), (7, 544), (37, 2048),
                                       (130, 1408), (3, 9728)])
def test_quantize_matches_the_definition(rows, cols, name, n):
    from pegainfer_amd import ops
    g = np.random.default_rng(rows + cols)
    v = g.standard_normal((rows, cols)) * 10.0 ** g.integers(-8, 8, (rows, 1))
    v.reshape(rows, -1, 32)[:, 0] = 0  # a zero block (signed zeros among it)
    v[:, 0] = -0.0
    x = mx_ref.bf16_round(v)
    q = ops.MxTensor.empty(rows, cols, _mx(name, n))
    ops.mx_quantize(dev(x, bf16=True), q)
    codes, scales = mx_ref.quantize(bf(x), name)
    assert np.array_equal(host(q.scales), scales) and np.array_equal(host(q.codes), codes)
    back = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    ops.mx_dequantize(q, back)
    want = mx_ref.values(codes, scales, name)
    assert np.array_equal(bf(host(back)).astype(np.float64), want)


@pytest.mark.parametrize("name,n", FORMATS)
def test_quantize_every_bf16(name, n):
    """Every bf16 as the largest of its block (alone, and beside smaller ones), and every bf16
    beside a block maximum of 1."""
    from pegainfer_amd import ops
    every = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    g = np.random.default_rng(1)
    with np.errstate(all="ignore"):
        lone = np.zeros((65536, 32), np.uint16)
        lone[:, 13] = every
        fill = mx_ref.bf16_round(np.nan_to_num(bf(every).astype(np.float64), posinf=0, neginf=0)[:, None]
                                 * g.uniform(-1, 1, (65536, 32)))
        fill[:, 31] = every
    small = every.reshape(-1, 32)[np.abs(bf(every)).reshape(-1, 32).max(1) <= 1].copy()
    small[:, 0] = 0x3F80
    for x in (lone, fill, small):
        q = ops.MxTensor.empty(len(x), 32, _mx(name, n))
        ops.mx_quantize(dev(x, bf16=True), q)
        codes, scales = mx_ref.quantize(bf(x), name)
        assert np.array_equal(host(q.scales), scales)
        bad = np.argwhere(host(q.codes) != codes)
        assert not len(bad), (bad[:3], x[bad[0][0]])


@pytest.mark.parametrize("name,n", FORMATS)
def test_dequantize_every_code(name, n):
    from pegainfer_amd import ops
    scales = np.array([0, 1, 5, 100, 127, 130, 200, 246, 255], np.uint8)
    codes = np.tile(np.arange(256, dtype=np.uint8), 1).reshape(1, -1)
    if name == "fp8":
        codes = np.where((codes & 127) == 127, 0, codes).astype(np.uint8)
    cols = codes.shape[1] * (1 if name == "fp8" else 2)
    c = np.repeat(codes, len(scales), 0)
    s = np.repeat(scales[:, None], cols // 32, 1)
    q = ops.MxTensor(len(scales), cols, _mx(name, n), dev(c), dev(s))
    out = torch.zeros(len(scales), cols, dtype=torch.bfloat16, device="cuda")
    ops.mx_dequantize(q, out)
    want = mx_ref.values(c, s, name)
    got = bf(host(out)).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    # bf16's smallest step is 2^-133: values below its normal range are within half of it
    assert (np.abs(got - want)[fine] <= 2.0 ** -134).all()
    normal = fine & (np.abs(want) >= 2.0 ** -126)
    assert np.array_equal(got[normal], want[normal])


@pytest.mark.parametrize("name,n", FORMATS)
@pytest.mark.parametrize("rows,inter", [(1, 32), (37, 2048), (5, 1408), (3, 96)])
def test_swiglu_quantize_is_the_two_calls(rows, inter, name, n):
    from pegainfer_amd import ops
    g = np.random.default_rng(inter)
    w13 = dev(mx_ref.bf16_round(g.standard_normal((rows, 2 * inter)) * 3), bf16=True)
    act = torch.zeros(rows, inter, dtype=torch.bfloat16, device="cuda")
    ops.kimi_marlin_w13_swiglu(w13, act, rows, inter)
    a, b = (ops.MxTensor.empty(rows, inter, _mx(name, n)) for _ in range(2))
    ops.mx_quantize(act, a)
    ops.mx_swiglu_quantize(w13, b)
    assert np.array_equal(host(a.codes), host(b.codes))
    assert np.array_equal(host(a.scales), host(b.scales))
    codes, scales = mx_ref.quantize(bf(host(act)), name)
    assert np.array_equal(host(b.codes), codes) and np.array_equal(host(b.scales), scales)


@pytest.mark.parametrize("u", [1.0, -0.3, 2.0 ** 100, 2.0 ** -100, np.inf, np.nan, 0.0])
def test_swiglu_quantize_every_gate(u):
    """All 65536 bf16 gates, a block each (the others of its block zero), against the two calls."""
    from pegainfer_amd import ops
    bits = np.zeros((1 << 11, 32, 32), np.uint16)
    bits[..., 5] = np.arange(1 << 16, dtype=np.uint16).reshape(1 << 11, 32)
    gate = bits.reshape(1 << 11, 1024)
    up = np.broadcast_to(mx_ref.bf16_round(np.float64(u)), gate.shape).astype(np.uint16)
    w13 = dev(np.concatenate([gate, up], 1), bf16=True)
    act = torch.zeros(1 << 11, 1024, dtype=torch.bfloat16, device="cuda")
    ops.kimi_marlin_w13_swiglu(w13, act, 1 << 11, 1024)
    for name, n in FORMATS:
        a, b = (ops.MxTensor.empty(1 << 11, 1024, _mx(name, n)) for _ in range(2))
        ops.mx_quantize(act, a)
        ops.mx_swiglu_quantize(w13, b)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_swiglu_quantize_random_pairs():
    """Four million pairs of gates and values: fp8 codes of the two calls."""
    from pegainfer_amd import ops
    torch.manual_seed(1)
    w13 = (torch.randn(2048, 4096, device="cuda") * 4).bfloat16()
    act = torch.zeros(2048, 2048, dtype=torch.bfloat16, device="cuda")
    ops.kimi_marlin_w13_swiglu(w13, act, 2048, 2048)
    a, b = (ops.MxTensor.empty(2048, 2048, ops.MxFormat.Fp8E4M3) for _ in range(2))
    ops.mx_quantize(act, a)
    ops.mx_swiglu_quantize(w13, b)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def test_norm_then_quantized_swiglu_in_a_graph_and_on_a_side_stream():
    """The operators in the order a block uses them, captured once and replayed on new inputs."""
    from pegainfer_amd import layer, ops
    rows, cols = 5, 1024
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    res, y = torch.zeros_like(x), torch.zeros_like(x)
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    q, a = (ops.MxTensor.empty(rows, c, ops.MxFormat.Fp8E4M3) for c in (cols, cols // 2))

    def step():
        ops.add_rmsnorm(x, res, w, 1e-6, normed=y, quantized=q)
        ops.mx_swiglu_quantize(y, a)
    graph = layer.capture_graph(step)
    side = torch.cuda.Stream()
    for seed in range(3):
        torch.manual_seed(seed)
        x.copy_(torch.randn(rows, cols))
        res.copy_(torch.randn(rows, cols))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, q.codes, q.scales, a.codes, a.scales)]
        for t in (y, q.codes, a.codes):
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for g0, t in zip(got, (y, q.codes, q.scales, a.codes, a.scales)):
            assert torch.equal(g0, t)


@pytest.mark.parametrize("rows,cols,x32", [(1025, 4128, False), (1100, 7168, True), (1024, 7168, False),
                                           (4097, 256, False)])
def test_norm_of_many_rows(rows, cols, x32):
    """Either side of the rule that gives long batches more vectors a lane: the same results."""
    g = np.random.default_rng(cols)
    x = _rows(g, rows, cols, 0.5)
    x = x if x32 else mx_ref.bf16_round(x)
    res = mx_ref.bf16_round(_rows(g, rows, cols, 2.0))
    w = mx_ref.bf16_round(1 + 0.1 * g.standard_normal(cols).astype(np.float32))
    s, y, q = _run_norm(x, res, w, 1e-6)
    at = np.unique(np.r_[0:8, rows // 2, rows - 9:rows])
    want_s, want_y = _norm_ref((x if x32 else bf(x))[at], bf(res)[at], bf(w), 1e-6)
    _check_bf16(s[at], want_s, "sums")
    _check_bf16(y[at], want_y, "normed")
    codes, scales = mx_ref.quantize(want_y, "fp8")
    assert np.array_equal(q[0][at], codes) and np.array_equal(q[1][at], scales)
    for lo in range(0, rows, 300):  # each row as in a short batch
        part = _run_norm(x[lo:lo + 300], res[lo:lo + 300], w, 1e-6)
        for a, b in ((part[0], s), (part[1], y), (part[2][0], q[0]), (part[2][1], q[1])):
            assert np.array_equal(a, b[lo:lo + 300])


@pytest.mark.parametrize("name,n", FORMATS)
def test_offsets_past_32_bits(name, n):
    """17 GB of rows, more vectors than a launch indexes: the last rows are those of a short call."""
    from pegainfer_amd import ops
    cols, block = 1 << 13, 1 << 10
    rows = (1 << 20) + 5
    torch.manual_seed(n)
    some = torch.randn(block, cols, device="cuda").bfloat16()
    few = ops.MxTensor.empty(block, cols, _mx(name, n))
    ops.mx_quantize(some, few)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:rows - 5].view(-1, block, cols).copy_(some)
    x[rows - 5:].copy_(some[7:12])
    q = ops.MxTensor.empty(rows, cols, _mx(name, n))
    ops.mx_quantize(x, q)
    for got, want in ((q.codes, few.codes), (q.scales, few.scales)):
        assert (got[:rows - 5].view(-1, block, got.shape[1]) == want).all()
        assert torch.equal(got[rows - 5:], want[7:12])
    back = torch.empty(block, cols, dtype=torch.bfloat16, device="cuda")
    ops.mx_dequantize(few, back)
    ops.mx_dequantize(q, x)
    assert (x[:rows - 5].view(-1, block, cols).view(torch.int16) == back.view(torch.int16)).all()
    assert torch.equal(x[rows - 5:], back[7:12])
    del q
    a = ops.MxTensor.empty(rows, cols // 2, _mx(name, n))
    ops.mx_swiglu_quantize(x, a)
    b = ops.MxTensor.empty(block, cols // 2, _mx(name, n))
    ops.mx_swiglu_quantize(back, b)
    assert (a.codes[:rows - 5].view(-1, block, b.codes.shape[1]) == b.codes).all()
    assert torch.equal(a.codes[rows - 5:], b.codes[7:12])
    assert torch.equal(a.scales[rows - 5:], b.scales[7:12])


def test_norm_of_more_rows_than_a_launch_takes():
    from pegainfer_amd import ops
    rows, cols, block = (1 << 26) + 5, 8, 1 << 12
    torch.manual_seed(0)
    some, w = torch.randn(block, cols, device="cuda").bfloat16(), torch.randn(cols, device="cuda").bfloat16()
    want, y = torch.empty_like(some), torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    ops.add_rmsnorm(some, some, w, 1e-6, normed=want)
    x = torch.empty_like(y)
    x[:rows - 5].view(-1, block, cols).copy_(some)
    x[rows - 5:].copy_(some[7:12])
    ops.add_rmsnorm(x, x, w, 1e-6, normed=y)
    assert (y[:rows - 5].view(-1, block, cols).view(torch.int16) == want.view(torch.int16)).all()
    assert torch.equal(y[rows - 5:], want[7:12])


def test_norm_rounds_once_below_fp32s_normal_range():
    """Results a little off the middle between two of bf16's smallest numbers (2^-133 apart) and
    between two MXFP8 values of the lowest scale (2^-136 apart), nearer to it than fp32's smallest
    step: rounded to fp32 first, they would lie on it."""
    cols = 1024
    x, w = np.zeros((3, cols)), np.full(cols, 2.0 ** -132)
    # half of a row at the middle and a bit: above 0.5, below 1.5 steps of bf16, above 0.5 of MXFP8
    # (ties go to the even one, the other side); the rest brings the mean of the squares to 1
    for row, (base, off) in enumerate(((0.25, 2.0 ** -18), (0.75, -2.0 ** -19), (2.0 ** -5, 2.0 ** -15))):
        a = base * (1 + off)
        x[row, ::2] = a
        x[row, 1::2] = np.sqrt(2 - a * a)
        x[row, ::4] *= -1
    x, w = x.astype(np.float32), mx_ref.bf16_round(w)
    s, y = _norm_ref(x, None, bf(w), 0.0)
    small = np.abs(y[:, ::2])
    middle = np.array([[2.0 ** -134], [1.5 * 2.0 ** -133], [2.0 ** -137]])
    assert (small != middle).all() and (np.abs(small - middle) < 2.0 ** -151).all()
    _, gy, (gc, gsc) = _run_norm(x, None, w, 0.0)
    assert np.array_equal(gy, mx_ref.bf16_round(y))
    codes, scales = mx_ref.quantize(y, "fp8")
    assert np.array_equal(gsc, scales) and np.array_equal(gc, codes)


@pytest.mark.parametrize("x32", [False, True])
def test_norm_of_tiny_weights(x32):
    """Weights and so results throughout bf16's and MXFP8's smallest numbers."""
    rows, cols = 61, 4096
    g = np.random.default_rng(8)
    xb = mx_ref.bf16_round(_rows(g, rows, cols))
    x = _rows(g, rows, cols) if x32 else xb
    res = mx_ref.bf16_round(_rows(g, rows, cols))
    w = mx_ref.bf16_round(2.0 ** g.uniform(-140, -120, cols) * g.choice([-1, 1], cols))
    _, y = _norm_ref(x if x32 else bf(x), bf(res), bf(w), 1e-6)
    _, gy, (gc, gsc) = _run_norm(x, res, w, 1e-6)
    assert np.array_equal(gy, mx_ref.bf16_round(y))
    codes, scales = mx_ref.quantize(y, "fp8")
    assert np.array_equal(gsc, scales) and np.array_equal(gc, codes)
