"""The end of a decode step as a model runs it (norms on both sides, 4-bit head, draw) and a shared
expert with 4-bit projections in its layer: every step against the 64-bit formula on what the step
before it wrote, and captured chains against eager ones."""
import numpy as np
import pytest
import torch

import decode_ref as ref
from test_gpu_sample import _params
from test_gpu_w4 import _bf, _case, _pack

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _f(t):
    return t.float().cpu().numpy()


def _head(rows, hidden, vocab, group, zeros, post, seed=0):
    from pegainfer_amd import layer
    _, q, s, z = _case(seed, 1, vocab, hidden, group, zeros)
    s = ref.to_bf16_bits(ref.bf16_values(s) * 4)  # logits with a spread of a few
    g = np.random.default_rng(seed + 1)
    n = lambda *sh: _bf(ref.to_bf16_bits(g.standard_normal(sh).astype(np.float32)))  # noqa: E731
    head = layer.TokenHead(_pack(q, s, z, group), n(hidden), max_rows=rows, eps=EPS,
                           post_norm=n(hidden) if post else None, unit_offset=True)
    return head, (q, s, z), n


@pytest.mark.parametrize("rows,hidden,vocab,group,zeros,post", [
    (1, 2048, 32003, 128, True, True), (7, 512, 5001, 32, False, False), (40, 1408, 16384, 64, True, True),
    (130, 256, 3000, 128, False, True)])
def test_head(rows, hidden, vocab, group, zeros, post):
    head, (q, s, z), n = _head(rows + 3, hidden, vocab, group, zeros, post)
    x, res, gate = n(rows, hidden), n(rows, hidden), n(hidden)
    p = _params(rows, rows)
    dev = {k: torch.from_numpy(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda() for k, v in p.items()}
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    logprobs = torch.empty(rows, device="cuda")
    run = lambda: head.forward(x, res, dev["u"], tokens, gate=gate, residual_scale=0.5, logprobs=logprobs,  # noqa: E731
                               **{k: dev[k] for k in ("temperature", "top_k", "top_p", "min_p")})
    run()
    torch.cuda.synchronize()
    opt = lambda t: None if t is None else _f(t)  # noqa: E731
    _, want = ref.sandwich(_f(x), _f(res), _f(head.final_norm), EPS, opt(head.post_norm), _f(gate), 0.5, True)
    normed = head.normed[:rows]
    ref.assert_rounded(normed.view(torch.int16).cpu().numpy().view(np.uint16), want)
    y, mag = ref.w4_product(_f(normed), q, ref.bf16_values(s), z, group)
    logits = head.logits[:rows].cpu().numpy()
    assert (np.abs(logits - y) <= ref.w4_bound(mag, hidden, group, y, True)).all()
    for r in range(rows):
        token, logprob = ref.sample_row(logits[r], p["u"][r], np.float32(p["temperature"][r]), int(p["top_k"][r]),
                                        np.float32(p["top_p"][r]), np.float32(p["min_p"][r]))
        assert tokens[r].item() == token
        assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * (1 + abs(logprob))
    from pegainfer_amd import layer
    graph = layer.capture_graph(run)
    for _ in range(3):
        x.copy_(x.roll(1, 0))
        dev["u"].copy_(dev["u"].roll(1))
        graph.replay()
        torch.cuda.synchronize()
        got = tokens.clone(), logprobs.clone()
        tokens.zero_(), logprobs.zero_()
        run()
        torch.cuda.synchronize()
        assert torch.equal(got[0], tokens) and torch.equal(got[1], logprobs)


def test_two_heads_on_two_streams():
    """Each with a workspace of its own, at the same time."""
    heads = [_head(24, 512, 20011, 128, True, True, seed=i) for i in (3, 4)]
    work = []
    for head, _, n in heads:
        p = _params(5, 24)
        dev = {k: torch.from_numpy(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda() for k, v in p.items()}
        work.append((head, n(24, 512), n(24, 512), dev, torch.empty(24, dtype=torch.int32, device="cuda")))

    def run(head, x, res, dev, tokens):
        d = dict(dev)
        head.forward(x, res, d.pop("u"), tokens, **d)
    alone = []
    for w in work:
        run(*w)
        torch.cuda.synchronize()
        alone.append(w[4].clone())
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    for _ in range(20):
        for w, st in zip(work, streams):
            with torch.cuda.stream(st):
                run(*w)
    torch.cuda.synchronize()
    for w, a in zip(work, alone):
        assert torch.equal(w[4], a)


def test_head_refuses():
    from pegainfer_amd import layer
    head, _, n = _head(4, 512, 300, 128, False, False)
    t = torch.empty(5, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="exceed"):
        head.forward(n(5, 512), None, torch.rand(5, device="cuda"), t)
    with pytest.raises(ValueError, match="norm has"):
        layer.TokenHead(head.head, n(256), max_rows=4, eps=EPS)


@pytest.mark.parametrize("rows", [1, 16, 70, 300])
def test_shared_expert(rows):
    from pegainfer_amd import layer
    hidden, inter = 512, 384
    x, q1, s1, z1 = _case(rows, rows, 2 * inter, hidden, 64, True)
    _, q2, s2, z2 = _case(rows + 1, rows, hidden, inter, 128, False)
    shared = layer.KimiSharedExpert(_pack(q1, s1, z1, 64), _pack(q2, s2, z2, 128), max_tokens=rows)
    y = torch.empty(rows, hidden, dtype=torch.bfloat16, device="cuda")
    shared.forward(_bf(x), y)
    torch.cuda.synchronize()
    h13, act = _f(shared.h13[:rows]).astype(np.float64), _f(shared.act[:rows])
    want, mag = ref.w4_product(ref.bf16_values(x), q1, ref.bf16_values(s1), z1, 64)
    assert (np.abs(h13 - want) <= ref.w4_bound(mag, hidden, 64, want, False)).all()
    g, u = h13[:, :inter], h13[:, inter:]
    # bf16(silu), then its product rounded to bf16: half a step (2^-8) each
    silu = g / (1 + np.exp(-g)) * u
    assert (np.abs(act - silu) <= (2.0 ** -7 + 2.0 ** -15) * np.abs(silu) + 2.0 ** -130).all()
    want, mag = ref.w4_product(act, q2, ref.bf16_values(s2), z2, 128)
    assert (np.abs(_f(y) - want) <= ref.w4_bound(mag, inter, 128, want, False)).all()


def test_layer_takes_a_4_bit_shared_expert():
    """KimiMoeDecodeLayer's general form: what its shared expert adds is the 4-bit expert's output."""
    from pegainfer_amd import layer, ops, synth
    from gpu_helpers import dev
    g = synth.rng(5, 1)
    E, H, I, T = 4, 512, 256, 6
    gate, up, down = (synth.int4_checkpoint(g, E, a, b) for a, b in ((I, H), (I, H), (H, I)))
    _, q1, s1, _ = _case(1, 1, 2 * I, H, 32, False)
    _, q2, s2, _ = _case(2, 1, H, I, 32, False)
    shared = layer.KimiSharedExpert(_pack(q1, s1, None, 32), _pack(q2, s2, None, 32), max_tokens=T)
    routed = layer.RoutedExperts(layer.package_w13(gate, up), layer.package_projection(*down), max_tokens=T, topk=2,
                                 block_size=8, ep_size=1)
    with pytest.raises(ValueError, match="two-launch"):
        layer.KimiMoeDecodeLayer(routed, shared, n_experts=E, few_tokens=4)
    moe = layer.KimiMoeDecodeLayer(routed, shared, n_experts=E)
    hidden, normed = (dev(synth.normal_bf16(g, (T, H)).view(np.int16)).view(torch.bfloat16) for _ in range(2))
    logits, bias = torch.randn(T, E, device="cuda"), torch.zeros(E, device="cuda")
    out = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    moe.forward(hidden, normed, logits, bias, out)
    projected = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    shared.forward(normed, projected)
    want = torch.empty_like(out)
    ops.kimi_residual_add_scaled_f32(hidden, projected, moe.routed_f32[:T], ops.KIMI_K2_ROUTER_SCALE, want)
    assert torch.equal(out, want) and moe.routed_f32[:T].abs().max() > 0
