"""Norms on both sides of a block on the GPU against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import decode_ref as ref
import mx_ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _bits(t):
    return t.view(torch.int16).cpu().numpy().view(np.uint16)


def _bf(v):
    return torch.from_numpy(ref.to_bf16_bits(v).view(np.int16)).cuda().view(torch.bfloat16)


def _val(t):
    return t.float().cpu().numpy()


def _inputs(seed, rows, cols, x32, gate, post=True, residual=True, big=1.0):
    g = np.random.default_rng(seed)
    n = lambda *s: g.standard_normal(s).astype(np.float32)  # noqa: E731
    x = torch.from_numpy(n(rows, cols) * big).cuda() if x32 else _bf(n(rows, cols) * big)
    shape = {"none": None, "col": (cols,), "row": (rows, 1), "full": (rows, cols)}[gate]
    return dict(x=x, residual=_bf(n(rows, cols) * 2) if residual else None, pre=_bf(1 + 0.2 * n(cols)),
                post=_bf(1 + 0.2 * n(cols)) if post else None, gate=None if shape is None else _bf(n(*shape)))


def _run(v, *, scale=1.0, offset=False, sums=True, normed=True, quant=False, eps=EPS):
    from pegainfer_amd import ops
    rows, cols = v["x"].shape
    bf = dict(dtype=torch.bfloat16, device="cuda")
    s = torch.empty(rows, cols, **bf) if sums else None
    y = torch.empty(rows, cols, **bf) if normed else None
    q = ops.MxTensor.empty(rows, cols, ops.MxFormat.Fp8E4M3) if quant else None
    ops.sandwich_rmsnorm(v["x"], v["residual"], v["pre"], eps, post_weight=v["post"], gate=v["gate"],
                         residual_scale=scale, unit_offset=offset, residual_out=s, normed=y, quantized=q)
    torch.cuda.synchronize()
    return s, y, q


def _want(v, scale=1.0, offset=False, eps=EPS):
    opt = lambda t: None if t is None else _val(t)  # noqa: E731
    return ref.sandwich(_val(v["x"]), opt(v["residual"]), opt(v["pre"]), eps, opt(v["post"]), opt(v["gate"]),
                        scale, offset)


def _check_codes(q, z):
    """Where z is not within 2^-40 of a border, codes and scales are the reference's."""
    lo, hi = (mx_ref.quantize(z * f, "fp8") for f in (1 - 2.0 ** -40, 1 + 2.0 ** -40))
    codes, scales = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    same = np.repeat(lo[1] == hi[1], 32, 1)
    assert ((scales == lo[1]) | (scales == hi[1])).all()
    assert (((codes == lo[0]) | (codes == hi[0])) | ~same).all() and same.mean() > 0.9


@pytest.mark.parametrize("gate", ["none", "col", "row", "full"])
@pytest.mark.parametrize("rows,cols,x32,post,residual,offset,scale", [
    (1, 8, False, True, True, False, 1.0), (1, 7168, False, True, True, True, 0.5),
    (3, 2048, True, True, True, False, 0.83), (5, 520, False, False, True, False, 1.0),
    (4, 1032, True, True, False, True, 1.0), (7, 4096, False, True, True, False, -2.0),
    (9, 32768, False, True, True, True, 1.0), (6, 16392, True, True, True, False, 1.0),
    (13, 504, True, False, False, False, 1.0), (1100, 4104, False, True, True, False, 0.25)])
def test_formula(gate, rows, cols, x32, post, residual, offset, scale):
    v = _inputs(rows + cols, rows, cols, x32, gate, post, residual)
    s, y, _ = _run(v, scale=scale, offset=offset)
    ws, wz = _want(v, scale, offset)
    ref.assert_rounded(_bits(s), ws, "sum")
    ref.assert_rounded(_bits(y), wz, "normed")


@pytest.mark.parametrize("rows,cols,x32", [
    (2, 5120, True), (2, 5128, True), (256, 4104, False), (257, 4104, False), (3, 5120, False), (2, 5128, False),
    (1024, 8192, False), (1025, 8192, False), (3, 8200, True), (3, 8200, False), (2, 16384, True), (2, 16384, False),
    (2, 16392, False), (1030, 5120, True)])
def test_borders_of_forms(rows, cols, x32):
    """Either side of each border in rows, columns and type between the kernel's forms."""
    v = _inputs(rows * 7 + cols, rows, cols, x32, "row")
    s, y, _ = _run(v, scale=0.5)
    ws, wz = _want(v, 0.5)
    ref.assert_rounded(_bits(s), ws, "sum")
    ref.assert_rounded(_bits(y), wz, "normed")


@pytest.mark.parametrize("gate", ["none", "col", "row", "full"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (5, 2048), (2, 7168), (4, 8224)])
def test_quantized(gate, rows, cols):
    v = _inputs(cols, rows, cols, rows % 2 == 0, gate)
    s, y, q = _run(v, quant=True)
    ws, wz = _want(v)
    ref.assert_rounded(_bits(s), ws)
    ref.assert_rounded(_bits(y), wz)
    _check_codes(q, wz)
    only = _run(v, quant=True, sums=False, normed=False)[2]
    assert torch.equal(only.codes, q.codes) and torch.equal(only.scales, q.scales)
    assert torch.equal(_run(v, sums=False)[1], y) and torch.equal(_run(v, normed=False)[0], s)


def test_is_add_rmsnorm_without_its_extras():
    """No norm after the block, no gate, scale 1: add_rmsnorm's values, rounded once from 64 bits."""
    from pegainfer_amd import ops
    v = _inputs(0, 33, 2056, True, "none", post=False)
    s, y, _ = _run(v)
    s2, y2 = torch.empty_like(s), torch.empty_like(y)
    ops.add_rmsnorm(v["x"], v["residual"], v["pre"], EPS, residual_out=s2, normed=y2)
    assert torch.equal(s, s2) and torch.equal(y, y2)


def test_sum_alone_needs_no_pre_weight():
    v = _inputs(1, 5, 640, False, "row")
    v["pre"] = None
    ref.assert_rounded(_bits(_run(v, normed=False)[0]), _want(v)[0])


@pytest.mark.parametrize("big", [0.0, 1e-30, 1e-20, 1e18])
def test_magnitudes(big):
    """All zeros, rows whose squares lie far outside fp32 and results below its normal numbers."""
    v = _inputs(2, 6, 512, False, "col", big=big)
    v["residual"] = None
    v["gate"] *= 2.0 ** -60
    for post in (True, False):
        w = dict(v) if post else dict(v, post=None)
        s, y, _ = _run(w, eps=1e-38)
        ws, wz = _want(w, eps=1e-38)
        ref.assert_rounded(_bits(s), ws)
        ref.assert_rounded(_bits(y), wz)


def test_a_row_that_is_not_finite_stays_apart():
    v = _inputs(3, 8, 1024, False, "full")
    s0, y0, _ = _run(v)
    v["x"][2, 5], v["x"][5, 0] = float("inf"), float("nan")
    s, y, _ = _run(v)
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(s[keep], s0[keep]) and torch.equal(y[keep], y0[keep])
    assert torch.isnan(y[5]).all() and torch.isnan(y[2]).any()


@pytest.mark.parametrize("rows,cols", [(5, 2048), (3, 7168), (1030, 4104)])
def test_in_place(rows, cols):
    from pegainfer_amd import ops
    v = _inputs(4, rows, cols, False, "full")
    s, y, _ = _run(v)
    x, r = v["x"].clone(), v["residual"].clone()
    ops.sandwich_rmsnorm(x, r, v["pre"], EPS, post_weight=v["post"], gate=v["gate"], residual_out=r, normed=x)
    assert torch.equal(r, s) and torch.equal(x, y)


def test_no_rows_and_untouched_rows():
    from pegainfer_amd import ops
    v = _inputs(5, 4, 256, False, "row")
    whole = torch.full((6, 256), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.sandwich_rmsnorm(v["x"], v["residual"], v["pre"], EPS, post_weight=v["post"], gate=v["gate"],
                         normed=whole[1:5])
    assert (whole[0] == 9).all() and (whole[5] == 9).all() and torch.equal(whole[1:5], _run(v)[1])
    e = v["x"][:0]
    ops.sandwich_rmsnorm(e, e, v["pre"], EPS, gate=v["gate"][:0], normed=whole[:0])


def test_offsets_past_32_bits():
    rows, cols = 150_000, 16384  # 4.9 GB a tensor
    from pegainfer_amd import ops
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    v = _inputs(6, 40, cols, False, "row")
    x[-40:] = v["x"]
    gate = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    gate[-40:] = v["gate"]
    ops.sandwich_rmsnorm(x, None, v["pre"], EPS, post_weight=v["post"], gate=gate, normed=x)
    v["residual"] = None
    assert torch.equal(x[-40:], _run(v)[1]) and (x[:1000] == 0).all()


def test_captured():
    from pegainfer_amd import ops
    v = _inputs(7, 17, 2048, True, "col")
    s = torch.empty(17, 2048, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sandwich_rmsnorm(v["x"], v["residual"], v["pre"], EPS, post_weight=v["post"], gate=v["gate"],
                             residual_out=s, normed=y)
    for _ in range(3):
        v["x"].copy_(v["x"].roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        es, ey, _ = _run(v)
        assert torch.equal(s, es) and torch.equal(y, ey)
