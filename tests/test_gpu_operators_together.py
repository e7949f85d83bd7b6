"""The norm, the microscaled operators and the few-token layer in the order a model calls them.
Every step is checked against the 64-bit formula on what the step before it wrote, so each
tolerance is the step's own, and a captured chain gives the eager chain's bits on new inputs."""
import numpy as np
import pytest
import torch

import mx_ref
from gpu_helpers import bf, dev, host
from test_gpu_few_tokens import Case
from test_gpu_few_tokens import _check as check_layer
from test_gpu_mx_gemm import _bounds
from test_gpu_mx_gemm import _check as check_product
from test_gpu_norm_mx import _check_bf16, _norm_ref

pytestmark = pytest.mark.gpu


def _f64(t):
    return bf(host(t)).astype(np.float64)


def _values(q):
    name = "fp8" if q.format.value == 0 else "fp4"
    return mx_ref.values(host(q.codes), host(q.scales), name)


def _same(q, want, name="fp8"):
    codes, scales = mx_ref.quantize(want, name)
    assert np.array_equal(host(q.codes), codes) and np.array_equal(host(q.scales), scales)


def _bf16_rows(g, rows, cols, scale=1.0):
    return dev(mx_ref.bf16_round(g.standard_normal((rows, cols)) * scale), bf16=True)


def _mx_weight(g, rows, cols):
    """bf16 weights quantised on the GPU as at load time, checked against the reference."""
    from pegainfer_amd import ops
    w = _bf16_rows(g, rows, cols, 0.03)
    q = ops.MxTensor.empty(rows, cols, ops.MxFormat.Fp4E2M1)
    ops.mx_quantize(w, q)
    _same(q, _f64(w), "fp4")
    return q, _values(q)


def _replays(step, inputs, outputs, g):
    """The captured chain against the eager one, on three sets of inputs."""
    from pegainfer_amd import layer
    graph = layer.capture_graph(step)
    for _ in range(3):
        for t in inputs:
            t.copy_(dev(mx_ref.bf16_round(g.standard_normal(t.shape)), bf16=True))
        graph.replay()
        got = [host(t) for t in outputs]
        for t in outputs:
            t.zero_()
        step()
        for a, t in zip(got, outputs):
            assert np.array_equal(a, host(t))


@pytest.mark.parametrize("rows,h,inter", [(1, 512, 384), (37, 1024, 640), (200, 768, 1408)])
def test_mlp_block(rows, h, inter):
    """norm -> gate and up product -> SwiGLU -> down product -> the next block's norm."""
    from pegainfer_amd import ops
    g = np.random.default_rng(rows)
    (w13, v13), (w2, v2) = _mx_weight(g, 2 * inter, h), _mx_weight(g, h, inter)
    gamma = dev(mx_ref.bf16_round(1 + 0.1 * g.standard_normal(h)), bf16=True)
    x, res = _bf16_rows(g, rows, h), _bf16_rows(g, rows, h)
    new = lambda c: torch.zeros(rows, c, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    s, up, down, s2, y2 = new(h), new(2 * inter), new(h), new(h), new(h)
    q, a = (ops.MxTensor.empty(rows, c, ops.MxFormat.Fp8E4M3) for c in (h, inter))

    def step():
        ops.add_rmsnorm(x, res, gamma, 1e-6, residual_out=s, quantized=q)
        ops.mx_gemm(w13, q, up)
        ops.mx_swiglu_quantize(up, a)
        ops.mx_gemm(w2, a, down)
        ops.add_rmsnorm(down, s, gamma, 1e-6, residual_out=s2, normed=y2)
    step()
    want_s, want_y = _norm_ref(_f64(x), _f64(res), _f64(gamma), 1e-6)
    _check_bf16(host(s), want_s, "sums")
    _same(q, want_y)
    check_product(_f64(up), *_bounds(_values(q), v13, "fp8"), "gate and up")
    act = torch.zeros(rows, inter, dtype=torch.bfloat16, device="cuda")
    ops.kimi_marlin_w13_swiglu(up, act, rows, inter)
    _same(a, _f64(act))
    check_product(_f64(down), *_bounds(_values(a), v2, "fp8"), "down")
    want_s, want_y = _norm_ref(_f64(down), _f64(s), _f64(gamma), 1e-6)
    _check_bf16(host(s2), want_s, "sums after")
    _check_bf16(host(y2), want_y, "normed after")
    _replays(step, (x, res), (s, q.codes, q.scales, up, a.codes, a.scales, down, s2, y2), g)


@pytest.mark.parametrize("tokens,bs", [(3, 8), (70, 16), (160, 64)])
def test_routed_block(tokens, bs):
    """norm -> routing -> experts' gate and up -> SwiGLU -> experts' down, weighted -> the routes'
    sum in fp32 -> the next block's norm, which adds it."""
    from pegainfer_amd import ops
    h, inter, experts, local, start, topk = 512, 384, 16, 8, 4, 4
    g = np.random.default_rng(tokens)
    (w13, v13), (w2, v2) = _mx_weight(g, local * 2 * inter, h), _mx_weight(g, local * h, inter)
    v13, v2 = v13.reshape(local, 2 * inter, h), v2.reshape(local, h, inter)
    gamma = dev(mx_ref.bf16_round(1 + 0.1 * g.standard_normal(h)), bf16=True)
    x, res = _bf16_rows(g, tokens, h), _bf16_rows(g, tokens, h)
    logits, bias = dev(g.standard_normal((tokens, experts)).astype(np.float32)), dev(np.zeros(experts, np.float32))
    ws = ops.KimiMarlinRouteWorkspace(tokens, bs, topk=topk, local_experts=local)
    topk_w = torch.zeros(tokens, topk, device="cuda")
    topk_idx = torch.zeros(tokens, topk, dtype=torch.int32, device="cuda")
    n = tokens * topk
    new = lambda r, c: torch.zeros(r, c, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    s, up, route_out, s2, y2 = new(tokens, h), new(n, 2 * inter), new(n, h), new(tokens, h), new(tokens, h)
    total = torch.zeros(tokens, h, device="cuda")
    q, a = ops.MxTensor.empty(tokens, h, ops.MxFormat.Fp8E4M3), ops.MxTensor.empty(n, inter, ops.MxFormat.Fp8E4M3)

    def step():
        ops.add_rmsnorm(x, res, gamma, 1e-6, residual_out=s, quantized=q)
        ops.kimi_router_select(logits, bias, topk_w, topk_idx, tokens, topk=topk)
        routing = ops.moe_align_block_size(ws, topk_idx, tokens, tokens, start)
        ops.mx_grouped_gemm(routing, q, w13, None, up, top_k=topk, mul_topk_weights=False, size_m=tokens)
        ops.mx_swiglu_quantize(up, a)
        ops.mx_grouped_gemm(routing, a, w2, topk_w, route_out, top_k=1, mul_topk_weights=True, size_m=n)
        ops.moe_combine_local_f32(route_out, topk_idx, None, tokens, total, topk, h, start, local)
        ops.add_rmsnorm(total, s, gamma, 1e-6, residual_out=s2, normed=y2)
    step()
    want_s, want_y = _norm_ref(_f64(x), _f64(res), _f64(gamma), 1e-6)
    _check_bf16(host(s), want_s, "sums")
    _same(q, want_y)
    flat, weights = host(topk_idx).reshape(-1) - start, host(topk_w).reshape(-1).astype(np.float64)
    qv, av, upv, outv = _values(q), _values(a), _f64(up), _f64(route_out)
    act = new(n, inter)
    ops.kimi_marlin_w13_swiglu(up, act, n, inter)
    _same(a, _f64(act))
    for e in range(local):
        r = np.flatnonzero(flat == e)
        if not len(r):
            continue
        check_product(upv[r], *_bounds(qv[r // topk], v13[e], "fp8"), f"gate and up {e}")
        want, tol = _bounds(av[r], v2[e], "fp8")
        f = weights[r][:, None]
        check_product(outv[r], want * f, tol * f + np.abs(want * f) * 2.0 ** -23, f"down {e}")
    here = ((flat >= 0) & (flat < local)).reshape(tokens, topk)
    rows = np.where(here[..., None], outv.reshape(tokens, topk, h), 0.0)
    # fp32 sums of up to four rows
    assert (np.abs(host(total) - rows.sum(1)) <= 4 * 2.0 ** -24 * np.abs(rows).sum(1)).all()
    want_s, want_y = _norm_ref(host(total).astype(np.float64), _f64(s), _f64(gamma), 1e-6)
    _check_bf16(host(s2), want_s, "sums after")
    _check_bf16(host(y2), want_y, "normed after")
    _replays(step, (x, res), (s, q.codes, up, a.codes, route_out, total, s2, y2), g)


@pytest.mark.parametrize("tokens", [1, 5])
def test_few_token_block(tokens):
    """norm -> the whole MoE layer, which joins the residual -> the next block's norm."""
    from pegainfer_amd import layer, ops
    c = Case(1024, 256, 8, 16, 4, 4, "bf16", tokens, 128)
    routed = layer.RoutedExperts(c.w13, c.w2, max_tokens=8, topk=4, block_size=8, global_start=4)
    shared = layer.KimiSharedExpert(*c.shared, max_tokens=8)
    moe = layer.KimiMoeDecodeLayer(routed, shared, n_experts=16, few_tokens=8)
    g = c.g
    gamma = dev(mx_ref.bf16_round(1 + 0.1 * g.standard_normal(c.h)), bf16=True)
    x, res = _bf16_rows(g, tokens, c.h), _bf16_rows(g, tokens, c.h)
    _, lg, bi, _ = c.inputs(tokens)
    logits, bias = dev(lg), dev(bi)
    s, y, out, y2 = (torch.zeros(tokens, c.h, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    q = ops.MxTensor.empty(tokens, c.h, ops.MxFormat.Fp8E4M3)

    def step():
        ops.add_rmsnorm(x, res, gamma, 1e-6, residual_out=s, normed=y)
        moe.forward(s, y, logits, bias, out)
        ops.add_rmsnorm(out, None, gamma, 1e-6, normed=y2, quantized=q)
    step()
    want_s, want_y = _norm_ref(_f64(x), _f64(res), _f64(gamma), 1e-6)
    _check_bf16(host(s), want_s, "sums")
    _check_bf16(host(y), want_y, "normed")
    check_layer(host(out), *c.want(host(y), host(moe.topk_idx)[:tokens], host(moe.topk_w)[:tokens], host(s),
                                   ops.KIMI_K2_ROUTER_SCALE))
    _, want_y = _norm_ref(_f64(out), None, _f64(gamma), 1e-6)
    _check_bf16(host(y2), want_y, "normed after")
    _same(q, want_y)
    _replays(step, (x, res), (s, y, out, y2, q.codes, q.scales), g)


def test_no_rows():
    from pegainfer_amd import ops
    e = lambda c: torch.zeros(0, c, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    w, _ = _mx_weight(np.random.default_rng(0), 128, 128)
    for f in ops.MxFormat:
        q = ops.MxTensor.empty(0, 128, f)
        ops.mx_quantize(e(128), q)
        ops.mx_swiglu_quantize(e(256), q)
        ops.mx_dequantize(q, e(128))
        ops.mx_gemm(w, q, e(128))
    ops.add_rmsnorm(e(128), e(128), torch.ones(128, dtype=torch.bfloat16, device="cuda"), 1e-6, normed=e(128))
    torch.cuda.synchronize()


def test_strided_parts_are_refused_and_offset_parts_are_not():
    """Column slices are not rows one after another; row slices are, wherever they begin."""
    from pegainfer_amd import ops
    g = np.random.default_rng(7)
    w, _ = _mx_weight(g, 64, 128)
    big = _bf16_rows(g, 12, 256)
    q, y = ops.MxTensor.empty(4, 128, ops.MxFormat.Fp8E4M3), torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    ones = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: ops.mx_quantize(big[:4, :128], q), lambda: ops.mx_gemm(w, q, big[:4, :64]),
                lambda: ops.add_rmsnorm(big[:4, 128:], None, ones, 1e-6, quantized=q),
                lambda: ops.add_rmsnorm(big[:8].reshape(16, 128)[:4], big[4:8, :128], ones, 1e-6, quantized=q)):
        with pytest.raises(ValueError):
            bad()
    rows = big.reshape(24, 128)
    for lo in (0, 1, 5, 20):
        ops.add_rmsnorm(rows[lo:lo + 4], rows[20 - lo:24 - lo], ones, 1e-6, quantized=q)
        _same(q, _norm_ref(_f64(rows[lo:lo + 4]), _f64(rows[20 - lo:24 - lo]), np.ones(128), 1e-6)[1])
        ops.mx_quantize(rows[lo:lo + 4], q)
        _same(q, _f64(rows[lo:lo + 4]))
        part = ops.MxTensor.empty(9, 128, ops.MxFormat.Fp8E4M3)
        ops.mx_quantize(rows[:9], part)
        at = lo % 5
        some = ops.MxTensor(4, 128, part.format, part.codes[at:at + 4], part.scales[at:at + 4])
        ops.mx_gemm(w, some, y)
        first = host(y)
        ops.mx_gemm(w, ops.MxTensor(4, 128, part.format, some.codes.clone(), some.scales.clone()), y)
        assert np.array_equal(host(y), first)
