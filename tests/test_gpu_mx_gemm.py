"""Products of microscaled operands on the GPU against 64-bit products of the values that the codes
stand for.

Tolerance, element by element: half a bf16 step of the result (2^-8 of it), plus what the sums may
lose.  An instruction adds 128 products in one go; E4M3 products are aligned to the largest of them
and keep about 12 bits below it, so 2^-11 of the largest product of each 128 k is allowed (E2M1
with E2M1: 2^-20); from instruction to instruction the sums are fp32: 2^-23 of the sum of
magnitudes for each."""
import numpy as np
import pytest
import torch

import mx_ref
from gpu_helpers import bf, dev, host

pytestmark = pytest.mark.gpu
FORMATS = {"fp8": 0, "fp4": 1}


def _operand(g, rows, cols, name, spread=3):
    """Random codes with uneven blocks' scales, on the GPU, and their values."""
    from pegainfer_amd import ops
    if name == "fp8":
        v = torch.from_numpy(g.standard_normal((rows, cols)).astype(np.float32) * 60)
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    else:
        codes = g.integers(0, 256, (rows, cols // 2)).astype(np.uint8)
    scales = g.integers(120 - spread, 121 + spread, (rows, cols // 32)).astype(np.uint8)
    return (ops.MxTensor(rows, cols, ops.MxFormat(FORMATS[name]), dev(codes), dev(scales)),
            mx_ref.values(codes, scales, name))


def _bounds(x, w, name):
    """want [N, M] and the tolerance."""
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    want = (t(x) @ t(w).T).cpu().numpy()
    ax, aw = np.abs(x), np.abs(w)
    peak = lambda a: a.reshape(len(a), -1, 128).max(-1)  # noqa: E731
    steps = x.shape[1] // 128
    lost = (2.0 ** -11 if name == "fp8" else 2.0 ** -20) * (t(peak(ax)) @ t(peak(aw)).T).cpu().numpy()
    sums = steps * 2.0 ** -23 * (t(ax) @ t(aw).T).cpu().numpy()
    return want, np.abs(want) * 2.0 ** -8 + lost + sums


def _check(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("n,m,k", [
    (1, 16, 128), (2, 48, 256), (3, 256, 384), (1, 9728, 2560), (15, 272, 512), (16, 64, 640),
    (17, 80, 1152), (31, 512, 2048), (33, 1408, 128), (64, 4096, 1024), (48, 16, 7168),
    (65, 16, 128), (100, 272, 256), (129, 640, 384), (300, 400, 2560), (128, 256, 640),
    (257, 2816, 2048), (500, 32, 512), (1000, 1040, 128),
    # the tile shapes, ragged: 64 x 64, 128 x 64, 128 x 128, 256 x 128, 256 x 256
    (200, 4080, 1152), (300, 4112, 640), (999, 4048, 512), (1001, 7088, 2048), (3990, 4080, 1408)])
def test_dense(n, m, k, name):
    from pegainfer_amd import ops
    g = np.random.default_rng(n * 31 + m + k)
    x, xv = _operand(g, n, k, name)
    w, wv = _operand(g, m, k, "fp4")
    y = torch.full((n + 1, m), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.mx_gemm(w, x, y[:n])
    got = bf(host(y)).astype(np.float64)
    assert (got[n] == 5).all()  # the row behind the last one
    _check(got[:n], *_bounds(xv, wv, name))


@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("n", [3, 40, 200])
def test_dense_extremes(n, name):
    """Scales at the ends of their range, all-zero rows, and NaN scales, which stay in their own
    row of X or W."""
    from pegainfer_amd import ops
    g = np.random.default_rng(n)
    k, m = 512, 96
    x, xv = _operand(g, n, k, name)
    w, wv = _operand(g, m, k, "fp4")
    xs, ws = host(x.scales), host(w.scales)
    xs[0], ws[5] = 0, 10     # 2^-127 and 2^-117: below fp32's range together
    xs[1], ws[7] = 254, 130  # 2^127: past bf16's range
    xc = host(x.codes)
    xc[2] = 0
    x.codes.copy_(dev(xc)), x.scales.copy_(dev(xs)), w.scales.copy_(dev(ws))
    xv, wv = mx_ref.values(xc, xs, name), mx_ref.values(host(w.codes), ws, "fp4")
    y = torch.zeros(n, m, dtype=torch.bfloat16, device="cuda")
    ops.mx_gemm(w, x, y)
    got = bf(host(y)).astype(np.float64)
    want, tol = _bounds(xv, wv, name)
    tiny = np.abs(want) < 2.0 ** -100
    assert (np.abs(got[tiny]) <= 2.0 ** -99).all()
    rest = ~tiny & (np.abs(want) < 2.0 ** 120)
    rest[1] = False
    _check(got[rest], want[rest], tol[rest])
    assert (got[2] == 0).all()
    assert not np.isnan(got[[0] + list(range(2, n))]).any()
    xs[n - 1, 3], ws[11, 15] = 255, 255
    x.scales.copy_(dev(xs)), w.scales.copy_(dev(ws))
    ops.mx_gemm(w, x, y)
    again = bf(host(y)).astype(np.float64)
    assert np.isnan(again[n - 1]).all() and np.isnan(again[:, 11]).all()
    keep = np.ones((n, m), bool)
    keep[n - 1], keep[:, 11], keep[1] = False, False, False
    assert np.array_equal(again[keep], got[keep])


def _route(tokens, topk, experts, local, start, bs, seed, lean=False):
    from pegainfer_amd import ops
    g = np.random.default_rng(seed)
    if lean:  # every route to one or two experts
        idx = np.stack([g.choice([start, start + local - 1, (start + local) % experts], topk, replace=False)
                        for _ in range(tokens)])
    else:
        idx = np.stack([g.permutation(experts)[:topk] for _ in range(tokens)])
    idx = idx.astype(np.int32)
    ws = ops.KimiMarlinRouteWorkspace(tokens, bs, topk=topk, local_experts=local)
    return idx, ops.moe_align_block_size(ws, dev(idx), tokens, tokens, start)


@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("tokens,topk,experts,local,start,bs,m,k", [
    (1, 1, 4, 4, 0, 8, 16, 128), (1, 8, 384, 48, 48, 8, 256, 1024), (5, 2, 8, 4, 4, 8, 48, 384),
    (64, 8, 96, 48, 48, 16, 512, 640), (64, 6, 64, 64, 0, 16, 80, 256), (33, 3, 16, 8, 8, 32, 272, 512),
    (90, 4, 12, 6, 0, 48, 128, 384), (200, 6, 16, 16, 0, 64, 400, 2048), (300, 2, 6, 3, 3, 64, 16, 128),
    (40, 2, 40, 3, 7, 64, 256, 256),
    # blocks of 8 and 32 rows in tiles, K split and not
    (100, 4, 32, 32, 0, 8, 1040, 640), (400, 8, 32, 32, 0, 32, 1360, 512), (150, 8, 48, 48, 0, 16, 4096, 4096)])
def test_grouped(tokens, topk, experts, local, start, bs, m, k, name):
    """W13's use (top_k rows a token) and W2's (one row a route, the routing weight applied)."""
    from pegainfer_amd import ops
    g = np.random.default_rng(tokens + m + k)
    idx, routing = _route(tokens, topk, experts, local, start, bs, tokens)
    w, wv = _operand(g, local * m, k, "fp4")
    wv = wv.reshape(local, m, k)
    weights = g.random(tokens * topk).astype(np.float32)
    flat = idx.reshape(-1) - start
    for top_k, mul in ((topk, False), (1, True)):
        rows = tokens if top_k == topk and not mul else tokens * topk
        x, xv = _operand(g, rows, k, name)
        y = torch.full((tokens * topk, m), 3.0, dtype=torch.bfloat16, device="cuda")
        ops.mx_grouped_gemm(routing, x, w, dev(weights) if mul else None, y, top_k=top_k,
                            mul_topk_weights=mul, size_m=rows)
        got = bf(host(y)).astype(np.float64)
        for e in range(local):
            r = np.flatnonzero(flat == e)
            if len(r):
                want, tol = _bounds(xv[r // top_k], wv[e], name)
                f = weights[r].astype(np.float64)[:, None] if mul else 1.0
                # the factor's product rounds once more in fp32
                _check(got[r], want * f, tol * f + np.abs(want * f) * 2.0 ** -23, f"expert {e}")
        away = (flat < 0) | (flat >= local)
        assert (got[away] == 3).all()


def test_grouped_skewed_and_without_local_routes():
    from pegainfer_amd import ops
    g = np.random.default_rng(9)
    w, wv = _operand(g, 4 * 64, 256, "fp4")
    for bs in (8, 32, 64):
        idx, routing = _route(150, 2, 16, 4, 8, bs, 1, lean=True)
        x, xv = _operand(g, 150, 256, "fp8")
        y = torch.zeros(300, 64, dtype=torch.bfloat16, device="cuda")
        ops.mx_grouped_gemm(routing, x, w, None, y, top_k=2, mul_topk_weights=False, size_m=150)
        got, flat = bf(host(y)).astype(np.float64), idx.reshape(-1) - 8
        for e in (0, 3):
            r = np.flatnonzero(flat == e)
            _check(got[r], *_bounds(xv[r // 2], wv.reshape(4, 64, 256)[e], "fp8"))
        assert (got[(flat < 0) | (flat > 3)] == 0).all()
        # no route of this GPU at all: nothing is written
        ws = ops.KimiMarlinRouteWorkspace(7, bs, topk=2, local_experts=4)
        none = ops.moe_align_block_size(ws, dev(np.full((7, 2), 100, np.int32)), 7, 7, 0)
        y.fill_(9.0)
        ops.mx_grouped_gemm(none, x, w, None, y, top_k=2, mul_topk_weights=False, size_m=7)
        assert (bf(host(y)) == 9).all()


@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("tokens,bs,m,k,lean", [
    (1500, 8, 272, 512, True), (1500, 16, 272, 1152, False), (700, 48, 528, 640, True), (300, 32, 144, 768, False),
    (500, 64, 256, 512, False), (160, 8, 272, 640, False), (2300, 64, 16, 640, True)])
def test_grouped_blocks_of_one_expert_together(tokens, bs, m, k, lean, name):
    """Many blocks an expert, which workgroups take several of: all on two experts (of a run of over
    64 blocks), or spread unevenly."""
    from pegainfer_amd import ops
    g = np.random.default_rng(tokens + bs)
    idx, routing = _route(tokens, 2, 16, 4, 8, bs, tokens, lean=lean)
    w, wv = _operand(g, 4 * m, k, "fp4")
    x, xv = _operand(g, tokens, k, name)
    y = torch.full((tokens * 2, m), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.mx_grouped_gemm(routing, x, w, None, y, top_k=2, mul_topk_weights=False, size_m=tokens)
    got, flat = bf(host(y)).astype(np.float64), idx.reshape(-1) - 8
    for e in range(4):
        r = np.flatnonzero(flat == e)
        if len(r):
            _check(got[r], *_bounds(xv[r // 2], wv.reshape(4, m, k)[e], name), f"expert {e}")
    assert (got[(flat < 0) | (flat > 3)] == 3).all()


def test_repeat_and_graph_give_the_same_bits():
    from pegainfer_amd import layer, ops
    g = np.random.default_rng(2)
    for n in (5, 200):
        x, _ = _operand(g, n, 1024, "fp8")
        w, _ = _operand(g, 512, 1024, "fp4")
        y = torch.zeros(n, 512, dtype=torch.bfloat16, device="cuda")
        ops.mx_gemm(w, x, y)
        first = y.clone()
        graph = layer.capture_graph(lambda: ops.mx_gemm(w, x, y))
        for _ in range(3):
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, first)


def _exact(rows, cols, seed):
    """Random MXFP4 rows of one scale: every sum of their products is exact in fp32."""
    from pegainfer_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    codes.random_(0, 256, generator=gen)
    return ops.MxTensor(rows, cols, ops.MxFormat.Fp4E2M1, codes,
                        torch.full((rows, cols // 32), 127, dtype=torch.uint8, device="cuda"))


def _part(q, lo, hi):
    from pegainfer_amd import ops
    return ops.MxTensor(hi - lo, q.cols, q.format, q.codes[lo:hi].clone(), q.scales[lo:hi].clone())


def _product(w, x):
    from pegainfer_amd import ops
    y = torch.empty(x.rows, w.rows, dtype=torch.bfloat16, device="cuda")
    ops.mx_gemm(w, x, y)
    return y


@pytest.mark.parametrize("rows", [5, 40, 200])
def test_weights_past_32_bits(rows):
    m, k = (1 << 20) + 16, 8192
    w, x = _exact(m, k, 1), _exact(rows, k, 2)
    y = _product(w, x)
    for lo, hi in ((0, 64), (m // 2, m // 2 + 64), (m - 64, m)):
        assert torch.equal(y[:, lo:hi], _product(_part(w, lo, hi), x))


def test_results_past_32_bits():
    n, m, k = 70001, 65536, 512
    w, x = _exact(m, k, 3), _exact(n, k, 4)
    y = _product(w, x)
    for lo, hi in ((0, 9), (n // 2, n // 2 + 40), (n - 130, n)):
        assert torch.equal(y[lo:hi], _product(w, _part(x, lo, hi)))


@pytest.mark.parametrize("tokens,bs", [(4, 8), (300, 16), (300, 64)])
def test_grouped_weights_past_32_bits(tokens, bs):
    from pegainfer_amd import ops
    e, m, k = 66, 16384, 8192
    w, x = _exact(e * m, k, 5), _exact(tokens, k, 6)
    idx = torch.randint(0, 2, (tokens, 1), dtype=torch.int32, device="cuda") * (e - 1)
    ws = ops.KimiMarlinRouteWorkspace(tokens, bs, topk=1, local_experts=e)
    routing = ops.moe_align_block_size(ws, idx, tokens, tokens, 0)
    y = torch.empty(tokens, m, dtype=torch.bfloat16, device="cuda")
    ops.mx_grouped_gemm(routing, x, w, None, y, top_k=1, mul_topk_weights=False, size_m=tokens)
    for expert in (0, e - 1):
        want = _product(_part(w, expert * m, (expert + 1) * m), x)
        at = (idx[:, 0] == expert).nonzero()[:, 0]
        assert torch.equal(y[at], want[at])


def _small(rows, cols, name, seed):
    """Rows of few bits with two scales: with MXFP4 weights of the same kind no sum of their products
    loses any (a product is a multiple of 1/2 up to 48), so the results are bf16 of the exact ones.
    Also the values, in float64 on the GPU."""
    from pegainfer_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pick = lambda hi, shape: torch.randint(0, hi, shape, device="cuda", generator=gen)  # noqa: E731
    if name == "fp8":
        table = torch.tensor([0.0, 1.0, -1.0, 2.0, -2.0], device="cuda")
        v = table[pick(5, (rows, cols))]
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        table = torch.tensor(np.concatenate([mx_ref.E2M1, -mx_ref.E2M1]), device="cuda", dtype=torch.float32)
        nibbles = pick(16, (rows, cols))
        v, codes = table[nibbles], (nibbles[:, 0::2] | nibbles[:, 1::2] << 4).to(torch.uint8)
    scales = 127 + pick(2, (rows, cols // 32))
    v = v.double() * torch.exp2((scales - 127).double()).repeat_interleave(32, 1)
    return ops.MxTensor(rows, cols, ops.MxFormat(FORMATS[name]), codes, scales.to(torch.uint8)), v


# The streaming kernel's forms by their rules (256 CUs): 32 features a workgroup where that is one for
# most CUs; eight steps in flight for up to 8 MXFP8 rows of k over 4096; 64 features where that is still
# three quarters of the CUs.  Steps that do and do not divide by the waves and by the steps in flight.
@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("n,m,k", [
    (1, 8192, 640), (5, 6144, 1408), (16, 8160, 1152), (16, 6176, 4096),
    (5, 272, 4224), (8, 256, 9728), (1, 9728, 4480), (2, 528, 7168), (7, 80, 4352),
    (32, 12288, 256), (17, 12352, 384), (64, 6144, 4224), (100, 3200, 4352), (33, 8192, 4992)])
def test_streaming_forms(n, m, k, name):
    from pegainfer_amd import ops
    (x, xv), (w, wv) = _small(n, k, name, n + m), _small(m, k, "fp4", k)
    y = torch.full((n + 1, m), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.mx_gemm(w, x, y[:n])
    assert torch.equal(y[:n], (xv @ wv.T).float().bfloat16()) and (y[n] == 5).all()


# Grouped: four steps in flight to one workgroup a CU, eight with more, by 16 or 32 features (short k,
# and k over 6144 below five tiles a CU); two sets of rows for blocks of 32.
@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("tokens,topk,experts,bs,m,k", [
    (40, 4, 40, 8, 928, 6272), (40, 4, 40, 16, 912, 6528), (60, 3, 60, 8, 1056, 384), (60, 3, 60, 16, 1040, 384),
    (30, 2, 24, 8, 1536, 7040), (6, 2, 12, 8, 544, 7168), (6, 2, 12, 8, 528, 4480), (90, 4, 40, 32, 912, 6272),
    (90, 4, 40, 32, 912, 384), (90, 4, 40, 48, 912, 384)])
def test_grouped_streaming_forms(tokens, topk, experts, bs, m, k, name):
    from pegainfer_amd import ops
    idx, routing = _route(tokens, topk, experts, experts, 0, bs, tokens)
    (x, xv), (w, wv) = _small(tokens, k, name, tokens), _small(experts * m, k, "fp4", k)
    y = torch.full((tokens * topk, m), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.mx_grouped_gemm(routing, x, w, None, y, top_k=topk, mul_topk_weights=False, size_m=tokens)
    flat = torch.from_numpy(idx.reshape(-1)).cuda()
    for e in range(experts):
        r = (flat == e).nonzero()[:, 0]
        want = (xv[r // topk] @ wv[e * m:(e + 1) * m].T).float().bfloat16()
        assert torch.equal(y[r], want), e


@pytest.mark.parametrize("name", ["fp8", "fp4"])
@pytest.mark.parametrize("tokens,bs", [(280, 64), (300, 64), (270, 32), (320, 48)])
def test_grouped_either_side_of_the_widest_tile(tokens, bs, name):
    """About 70, 75, 68 and 80 rows an expert: 128 x 64 tiles below 72, 256 x 128 above, several blocks an
    expert."""
    from pegainfer_amd import ops
    topk, experts, m, k = 2, 8, 528, 1152
    idx, routing = _route(tokens, topk, experts, experts, 0, bs, tokens)
    (x, xv), (w, wv) = _small(tokens, k, name, tokens), _small(experts * m, k, "fp4", k)
    y = torch.full((tokens * topk, m), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.mx_grouped_gemm(routing, x, w, None, y, top_k=topk, mul_topk_weights=False, size_m=tokens)
    flat = torch.from_numpy(idx.reshape(-1)).cuda()
    for e in range(experts):
        r = (flat == e).nonzero()[:, 0]
        assert torch.equal(y[r], (xv[r // topk] @ wv[e * m:(e + 1) * m].T).float().bfloat16()), e
