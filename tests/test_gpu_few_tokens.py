"""The two-launch MoE layer for a few tokens against the layer's formula in 64 bits, and its router
outputs against the select stages bit for bit.

Tolerance: the SwiGLU rows are rounded to 16 bits (2^-8 of each at most, in the sum 2^-8 of the sum of
magnitudes of their products), out once (2^-8 of it); fp32 sums and silu's exponential add 2^-19 of the
magnitudes of a product chain with room to spare."""
import numpy as np
import pytest
import torch

from gpu_helpers import bf, dev, host, pack_ckpt

pytestmark = pytest.mark.gpu


def _bits(v):
    import mx_ref
    return mx_ref.bf16_round(v)


def _int4(g, e, out_dim, in_dim, scale=0.02):
    """A checkpoint pair and its weights in float64: (nibble - 8) * scale."""
    q = g.integers(-8, 8, (e, out_dim, in_dim)).astype(np.int8)
    s = _bits(np.abs(g.standard_normal((e, out_dim, in_dim // 32))) * scale / 4 + 1e-4)
    return (pack_ckpt(q), s), q * np.repeat(bf(s).astype(np.float64), 32, 2)


def _silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


class Case:
    """A layer's weights on both sides."""

    def __init__(self, h, i, e, n, topk, start, kind, seed, shared_i=None):
        from pegainfer_amd import layer
        g = self.g = np.random.default_rng(seed)
        self.h, self.i, self.e, self.n, self.topk, self.start, self.kind = h, i, e, n, topk, start, kind
        (gate, self.G), (up, self.U), (down, self.D) = (_int4(g, e, i, h), _int4(g, e, i, h), _int4(g, e, h, i))
        self.w13, self.w2 = layer.package_w13(gate, up), layer.package_projection(*down)
        si = self.si = shared_i or i
        self.shared = None
        if kind == "bf16":
            gu, dn = _bits(g.standard_normal((2 * si, h)) * 0.02), _bits(g.standard_normal((h, si)) * 0.02)
            self.shared = (dev(gu, bf16=True), dev(dn, bf16=True))
            self.sG, self.sU, self.sD = (bf(v).astype(np.float64) for v in (gu[:si], gu[si:], dn))
        elif kind == "int4":
            (a, G), (b, U), (c, D) = (_int4(g, 1, si, h), _int4(g, 1, si, h), _int4(g, 1, h, si))
            self.shared = (layer.package_w13(a, b), layer.package_projection(*c))
            self.sG, self.sU, self.sD = G[0], U[0], D[0]

    def workspace(self, tokens):
        from pegainfer_amd import ops
        return ops.FewTokensWorkspace(tokens, self.h, self.i, topk=self.topk, local_experts=self.e,
                                      shared_inter=self.si if self.shared else 0)

    def inputs(self, t, residual=True):
        g = self.g
        x = _bits(g.standard_normal((t, self.h)))
        logits = g.standard_normal((t, self.n)).astype(np.float32)
        bias = (g.standard_normal(self.n) * 0.05).astype(np.float32)
        res = _bits(g.standard_normal((t, self.h))) if residual else None
        return x, logits, bias, res

    def run(self, ws, x, logits, bias, res, softmax, scale, out=None):
        from pegainfer_amd import ops
        t = len(x)
        o = torch.full((t, self.h), 9.0, dtype=torch.bfloat16, device="cuda") if out is None else out
        w = torch.zeros(t, self.topk, device="cuda")
        idx = torch.zeros(t, self.topk, dtype=torch.int32, device="cuda")
        ops.moe_few_tokens(ws, dev(x, bf16=True), dev(logits), self.w13, self.w2, w, idx, o,
                           bias=None if softmax else dev(bias), routed_scale=scale,
                           global_start=self.start, residual=None if res is None else dev(res, bf16=True),
                           shared=self.shared)
        return host(o), host(w), host(idx)

    def want(self, x, idx, w, res, scale):
        """The formula on the given routes, and the tolerance."""
        xv = bf(x).astype(np.float64)
        out, mag = np.zeros((len(x), self.h)), np.zeros((len(x), self.h))

        def add(rows, G, U, D, f):
            act = _silu(rows @ G.T) * (rows @ U.T) * f
            room = np.abs(rows) @ np.abs(G).T * np.abs(rows @ U.T) + np.abs(rows @ G.T) * (np.abs(rows) @ np.abs(U).T)
            return act @ D.T, (np.abs(act) * 2.0 ** -8 + room * np.abs(f) * 2.0 ** -19) @ np.abs(D).T
        for t in range(len(x)):
            for k in range(self.topk):
                e = idx[t, k] - self.start
                if 0 <= e < self.e:
                    a, m = add(xv[t:t + 1], self.G[e], self.U[e], self.D[e], float(w[t, k]) * scale)
                    out[t] += a[0]
                    mag[t] += m[0]
        if self.shared:
            a, m = add(xv, self.sG, self.sU, self.sD, 1.0)
            out, mag = out + a, mag + m
        if res is not None:
            out = out + bf(res)
        return out, np.abs(out) * 2.0 ** -8 + mag * (1 + 2.0 ** -4)


def _check(got, want, tol):
    g = bf(got).astype(np.float64)
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4], tol[bad][:4])


def _select(logits, bias, topk, softmax):
    from pegainfer_amd import ops
    t = len(logits)
    w = torch.zeros(t, topk, device="cuda")
    idx = torch.zeros(t, topk, dtype=torch.int32, device="cuda")
    if softmax:
        ops.dsv2_router_select(dev(logits), w, idx, t, topk)
    else:
        ops.kimi_router_select(dev(logits), dev(bias), w, idx, t, topk=topk)
    return host(w), host(idx)


SHAPES = [  # h, i, e, n, topk, start, shared kind, shared inter
    (64, 64, 1, 1, 1, 0, "none", None), (128, 64, 4, 16, 2, 8, "bf16", 64),
    (256, 192, 8, 8, 3, 0, "int4", 384), (512, 256, 48, 384, 8, 48, "bf16", 256),
    (1024, 448, 16, 64, 6, 16, "int4", 64), (448, 128, 5, 100, 4, 95, "none", None),
    (2048, 320, 12, 12, 6, 0, "int4", 640), (192, 64, 100, 700, 8, 300, "bf16", 128)]


@pytest.mark.parametrize("h,i,e,n,topk,start,kind,si", SHAPES)
@pytest.mark.parametrize("softmax", [False, True])
def test_matches_the_formula(h, i, e, n, topk, start, kind, si, softmax):
    c = Case(h, i, e, n, topk, start, kind, h + n, si)
    ws = c.workspace(16)
    for t in (1, 2, 3, 4, 5, 9, 16):
        x, logits, bias, res = c.inputs(t, residual=t % 2 == 1)
        out, w, idx = c.run(ws, x, logits, bias, res, softmax, 2.5)
        sw, sidx = _select(logits, bias, topk, softmax)
        assert np.array_equal(idx, sidx) and np.array_equal(w, sw)
        _check(out, *c.want(x, idx, w, res, 2.5))
    assert (host(ws.counters) == 0).all()


def test_tokens_without_a_local_route_and_all_on_one_expert():
    c = Case(256, 128, 4, 64, 4, 20, "bf16", 1)
    ws = c.workspace(8)
    x, logits, bias, res = c.inputs(8)
    logits[:, 20:24] = -30.0  # nobody picks the local experts
    bias[:] = 0
    out, w, idx = c.run(ws, x, logits, bias, res, False, 1.0)
    assert not ((idx >= 20) & (idx < 24)).any()
    _check(out, *c.want(x, idx, w, res, 1.0))
    logits[::2, 23] = 30.0  # every other token picks one
    out, w, idx = c.run(ws, x, logits, bias, res, False, 1.0)
    assert (idx[::2, 0] == 23).all()
    _check(out, *c.want(x, idx, w, res, 1.0))


def test_not_finite_rows_stay_their_own():
    """A token with a NaN or an infinity gives NaN and leaves the other tokens' bits alone."""
    for t, softmax in ((6, True), (3, False), (13, True)):
        c = Case(256, 64, 6, 6, 2, 0, "bf16", 3)
        ws = c.workspace(t)
        x, logits, bias, res = c.inputs(t)
        clean, w, idx = c.run(ws, x, logits, bias, res, softmax, 1.0)
        for at, v in ((1, 0x7FC0), (2, 0x7F80), (t - 1, 0xFF80)):
            bad = x.copy()
            bad[at, 17] = v
            out, _, _ = c.run(ws, bad, logits, bias, res, softmax, 1.0)
            assert np.isnan(bf(out)[at]).all()
            keep = np.arange(t) != at
            assert np.array_equal(out[keep], clean[keep])


@pytest.mark.parametrize("kind", ["none", "int4"])
def test_rows_of_any_magnitude(kind):
    """Rows far from 1, all zero, and with values far below their largest (the products are exact down
    to 2^-25 of it, and each value to 2^-40 of it below)."""
    c = Case(512, 128, 5, 5, 2, 0, kind, 11)
    ws = c.workspace(16)
    for t in (4, 7, 16):
        x, logits, bias, _ = c.inputs(t, residual=False)
        v = bf(x).astype(np.float64)
        v[0] *= 2.0 ** 40
        v[1] *= 2.0 ** -60
        v[2] = 0
        v[3, ::2] *= 2.0 ** -20
        if t > 4:
            v[4, 1:] *= 2.0 ** -24
            v[5] *= 2.0 ** -130  # bf16's smallest numbers
        x = _bits(v)
        out, w, idx = c.run(ws, x, logits, bias, None, True, 1.0)
        want, tol = c.want(x, idx, w, None, 1.0)
        assert (out[2] == 0).all()
        tiny = np.abs(want) < 2.0 ** -120
        assert (np.abs(bf(out))[tiny] <= 2.0 ** -118).all()
        got = np.where(tiny, 0, bf(out))
        _check(_bits(got), np.where(tiny, 0, want), tol + 2.0 ** -118)


def test_in_place_batches_of_any_size_and_stale_workspaces():
    c = Case(512, 128, 8, 16, 4, 8, "int4", 5, 256)
    ws = c.workspace(16)
    for t in (ws.act, ws.act_factors, ws.act_shared, ws.act_shared_factors, ws.partials):
        t.fill_(float("nan"))
    ws.slots.fill_(7)
    for t in (16, 2, 11, 1):
        x, logits, bias, res = c.inputs(t)
        out, w, idx = c.run(ws, x, logits, bias, res, False, 1.5)
        _check(out, *c.want(x, idx, w, res, 1.5))
        again, _, _ = c.run(c.workspace(t), x, logits, bias, res, False, 1.5)
        assert np.array_equal(again, out)
        rd = dev(res, bf16=True)
        from pegainfer_amd import ops
        xd = dev(x, bf16=True)
        wd, idxd = torch.zeros(t, 4, device="cuda"), torch.zeros(t, 4, dtype=torch.int32, device="cuda")
        ops.moe_few_tokens(ws, xd, dev(logits), c.w13, c.w2, wd, idxd, rd, bias=dev(bias),
                           routed_scale=1.5, global_start=8, residual=rd, shared=c.shared)
        assert np.array_equal(host(rd), out)


def test_kimi_sizes():
    """The decode layer's real sizes, and the layer's own general path beside it."""
    from pegainfer_amd import layer, ops
    c = Case(7168, 2048, 4, 32, 8, 12, "bf16", 7)
    routed = layer.RoutedExperts(c.w13, c.w2, max_tokens=8, topk=8, block_size=8, global_start=12, ep_size=8)
    shared = layer.KimiSharedExpert(*c.shared, max_tokens=8)
    few = layer.KimiMoeDecodeLayer(routed, shared, n_experts=32, few_tokens=6)
    general = layer.KimiMoeDecodeLayer(routed, shared, n_experts=32)
    for t in (1, 6, 8):  # 8: past few_tokens, the general path
        x, logits, bias, res = c.inputs(t)
        outs = []
        for lay in (few, general):
            out = torch.zeros(t, 7168, dtype=torch.bfloat16, device="cuda")
            lay.forward(dev(res, bf16=True), dev(x, bf16=True), dev(logits), dev(bias), out)
            outs.append(host(out))
        idx, w = host(few.topk_idx[:t]), host(few.topk_w[:t])
        assert np.array_equal(idx, host(general.topk_idx[:t]))
        want, tol = c.want(x, idx, w, res, ops.KIMI_K2_ROUTER_SCALE)
        if t <= 6:
            _check(outs[0], want, tol)
        else:
            assert np.array_equal(outs[0], outs[1])
        assert np.abs(bf(outs[0]) - bf(outs[1])).max() < 0.05 * np.abs(want).max()


def test_dsv2_layer_graph_replays():
    from pegainfer_amd import layer
    c = Case(2048, 192, 16, 16, 6, 0, "int4", 9, 384)
    routed = layer.RoutedExperts(c.w13, c.w2, max_tokens=4, topk=6, block_size=8)
    shared = layer.ExpertFFN(*c.shared, max_rows=4)
    moe = layer.Dsv2MoeLayer(routed, shared, few_tokens=4)
    x, logits, _, _ = c.inputs(4)
    xd, ld = dev(x, bf16=True), dev(logits)
    out = torch.zeros(4, 2048, dtype=torch.bfloat16, device="cuda")
    graph = layer.capture_graph(lambda: moe.forward(xd, ld, out))
    for seed in range(3):
        x, logits, _, _ = c.inputs(4)
        xd.copy_(dev(x, bf16=True)), ld.copy_(dev(logits))
        graph.replay()
        got = host(out)
        moe.forward(xd, ld, out)
        assert np.array_equal(host(out), got)
        _check(got, *c.want(x, host(moe.topk_idx), host(moe.topk_w), None, 1.0))


@pytest.mark.parametrize("tokens", [2, 7])
def test_packages_past_32_bits(tokens):
    """Experts whose weights lie past 4 GB: the bits of a package of the last few alone, as many as the
    tokens have routes (the launch, and so the order of the sums, is by the smaller of the two)."""
    from pegainfer_amd import ops
    e, h, i = 300, 7168, 2048
    gen = torch.Generator(device="cuda").manual_seed(tokens)

    def package(out_dim, in_dim):
        q = torch.empty(e, out_dim * in_dim // 2, dtype=torch.uint8, device="cuda").random_(0, 256, generator=gen)
        s = torch.empty(e, out_dim * in_dim // 32, device="cuda").uniform_(0.001, 0.02, generator=gen).bfloat16()
        return q, s
    w13, w2 = package(2 * i, h), package(h, i)
    pick = lambda p, lo, o, k: ops.MarlinInt4Weight(e - lo, k, o, p[0][lo:].contiguous(), p[1][lo:].contiguous())  # noqa: E731
    x = torch.randn(tokens, h, device="cuda", generator=gen).bfloat16()
    logits = torch.randn(tokens, e, device="cuda", generator=gen)
    logits[:, e - 2:] += 100.0  # every token to the last two
    outs = []
    for lo in (0, e - 2 * tokens):
        ws = ops.FewTokensWorkspace(tokens, h, i, topk=2, local_experts=e - lo)
        out = torch.zeros(tokens, h, dtype=torch.bfloat16, device="cuda")
        w, idx = torch.zeros(tokens, 2, device="cuda"), torch.zeros(tokens, 2, dtype=torch.int32, device="cuda")
        ops.moe_few_tokens(ws, x, logits, pick(w13, lo, 2 * i, h), pick(w2, lo, h, i), w, idx, out, global_start=lo)
        assert (idx >= e - 2).all()
        outs.append(out)
    assert outs[0].abs().max() > 0 and torch.equal(*outs)


def test_two_streams_with_a_workspace_each():
    """Calls at the same time do not meet: the bits of each call alone."""
    from pegainfer_amd import ops
    c = Case(1024, 448, 16, 64, 6, 16, "int4", 3, 64)
    jobs = []
    for t in (3, 11):
        x, logits, bias, res = c.inputs(t)
        jobs.append(dict(t=t, x=dev(x, bf16=True), l=dev(logits), b=dev(bias), r=dev(res, bf16=True), ws=c.workspace(t),
                         w=torch.zeros(t, 6, device="cuda"), i=torch.zeros(t, 6, dtype=torch.int32, device="cuda"),
                         out=[torch.zeros(t, c.h, dtype=torch.bfloat16, device="cuda") for _ in range(31)],
                         stream=torch.cuda.Stream()))

    def call(j, n):
        ops.moe_few_tokens(j["ws"], j["x"], j["l"], c.w13, c.w2, j["w"], j["i"], j["out"][n], bias=j["b"],
                           global_start=c.start, residual=j["r"], shared=c.shared)
    for j in jobs:
        call(j, 30)
    torch.cuda.synchronize()
    for n in range(30):
        for j in jobs:
            with torch.cuda.stream(j["stream"]):
                call(j, n)
    torch.cuda.synchronize()
    for j in jobs:
        assert all(torch.equal(o, j["out"][30]) for o in j["out"])


@pytest.mark.parametrize("kind", ["none", "int4", "bf16"])
@pytest.mark.parametrize("t", [3, 7, 16])
def test_rows_whose_swiglu_is_near_the_largest_floats(t, kind):
    """SwiGLU rows of 2^118 to 2^126, whose factor from fp16 to the nibbles' products is no float, and
    down projections of them that bf16 holds, beside ordinary rows."""
    c = Case(512, 128, 5, 5, 2, 0, kind, 11)
    ws = c.workspace(16)
    x, logits, bias, _ = c.inputs(t, residual=False)
    v = bf(x).astype(np.float64)
    v[0] *= 2.0 ** 59
    v[t // 2] *= 2.0 ** 61
    v[t - 1] *= 2.0 ** 63
    x = _bits(v)
    out, w, idx = c.run(ws, x, logits, bias, None, True, 1.0)
    want, tol = c.want(x, idx, w, None, 1.0)
    act = _silu(bf(x)[0].astype(np.float64) @ c.G.transpose(0, 2, 1)) * (bf(x)[0] @ c.U.transpose(0, 2, 1))
    assert np.abs(act).max() > 2.0 ** 117 and np.abs(want).max() < 2.0 ** 127
    _check(out, want, tol)


@pytest.mark.parametrize("kind", ["kimi", "dsv2"])
def test_layers_take_the_inputs_of_their_general_form(kind):
    """Logits of a larger batch's buffer: the layer with and without few_tokens, and the bits of
    logits of the batch's own rows."""
    from pegainfer_amd import layer
    c = Case(512, 128, 8, 16, 4, 4, "bf16" if kind == "kimi" else "int4", 21, 128)
    routed = layer.RoutedExperts(c.w13, c.w2, max_tokens=8, topk=4, block_size=8, global_start=4)
    if kind == "kimi":
        shared = layer.KimiSharedExpert(*c.shared, max_tokens=8)
        make = lambda n: layer.KimiMoeDecodeLayer(routed, shared, n_experts=16, few_tokens=n)  # noqa: E731
    else:
        shared = layer.ExpertFFN(*c.shared, max_rows=8)
        make = lambda n: layer.Dsv2MoeLayer(routed, shared, few_tokens=n)  # noqa: E731
    x, lg, bi, res = c.inputs(8)
    xd, ld, bd, rd = dev(x, bf16=True), dev(lg), dev(bi), dev(res, bf16=True)
    for n in (0, 8):
        lay, outs = make(n), []
        for logits in (ld, ld[:5]):
            out = torch.zeros(5, 512, dtype=torch.bfloat16, device="cuda")
            if kind == "kimi":
                lay.forward(rd[:5], xd[:5], logits, bd, out)
            else:
                lay.forward(xd[:5], logits, out)
            outs.append(out)
        assert torch.equal(*outs)
        idx, w = host(lay.topk_idx[:5]), host(lay.topk_w[:5])
        if n:
            _check(host(outs[0]), *c.want(x[:5], idx, w, res[:5] if kind == "kimi" else None,
                                          2.827 if kind == "kimi" else 1.0))


@pytest.mark.parametrize("t", [3, 9])
def test_not_finite_rows_that_no_local_expert_takes(t):
    """Only the other tokens have local routes: without a shared expert the residual stays as it is,
    with one the row is NaN; the other rows keep their bits."""
    for kind in ("none", "int4", "bf16"):
        c = Case(256, 64, 4, 16, 2, 8, kind, 8)
        ws = c.workspace(t)
        x, logits, bias, res = c.inputs(t)
        logits[:, 8:12] = 20.0
        logits[1, 8:12] = -20.0
        clean, _, _ = c.run(ws, x, logits, bias, res, False, 1.0)
        keep = np.arange(t) != 1
        for v in (0x7FC0, 0x7F80, 0xFF80):
            bad = x.copy()
            bad[1, 100] = v
            out, _, idx = c.run(ws, bad, logits, bias, res, False, 1.0)
            local = (idx >= 8) & (idx < 12)
            assert not local[1].any() and local[keep].any(1).all()
            assert np.array_equal(out[keep], clean[keep])
            if kind == "none":
                assert np.array_equal(out[1], res[1])
            else:
                assert np.isnan(bf(out)[1]).all()


@pytest.mark.parametrize("t,topk,live", [(8, 2, 2), (3, 3, 3), (16, 6, 6)])
def test_every_expert_here_and_the_tokens_on_the_same(t, topk, live):
    """No route to another GPU, and fewer experts than there could be: the first launch's K is cut."""
    c = Case(1024, 128, 16, 16, topk, 0, "int4", t, 64)
    ws = c.workspace(t)
    x, logits, bias, res = c.inputs(t)
    logits[:] = logits[0]
    for softmax in (True, False):
        out, w, idx = c.run(ws, x, logits, bias, res, softmax, 1.25)
        assert len(np.unique(idx)) == live
        _check(out, *c.want(x, idx, w, res, 1.25))
    assert (host(ws.counters) == 0).all()
