"""Token draws on the GPU against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import decode_ref as ref

pytestmark = pytest.mark.gpu
INF = float("inf")


def _draw(logits, u, ws=None, **kw):
    from pegainfer_amd import ops
    rows, vocab = logits.shape
    ws = ws or ops.SampleWorkspace(rows, vocab)
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logprobs = torch.full((rows,), 7.0, device="cuda")
    dev = {k: None if v is None else torch.from_numpy(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda()
           for k, v in kw.items()}
    ops.sample_tokens(ws, logits, torch.from_numpy(np.asarray(u, np.float32)).cuda(), tokens, logprobs=logprobs, **dev)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), logprobs.cpu().numpy()


def _check(logits, u, **kw):
    """Tokens are the definition's; log probabilities are off by half an fp32 step and by what the
    weights' rounding to 2^-44 moves the sum: below vocab * 2^-45 of at least 1."""
    tokens, logprobs = _draw(logits, u, **kw)
    host = logits.float().cpu().numpy()
    for r in range(len(host)):
        one = {k: np.asarray(v)[r] for k, v in kw.items() if v is not None}
        one = {k: int(v) if k == "top_k" else np.float32(v) for k, v in one.items()}
        token, logprob = ref.sample_row(host[r], np.float32(u[r]), **one)
        assert tokens[r] == token, (r, tokens[r], token, one)
        if token >= 0:
            assert abs(logprobs[r] - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -24, (r, logprobs[r], logprob)
        else:
            assert logprobs[r] == -INF


def _logits(seed, rows, vocab, sigma=2.2, bf16=False, masked=0.0):
    g = np.random.default_rng(seed)
    v = (g.standard_normal((rows, vocab)) * sigma).astype(np.float32)
    v[g.random((rows, vocab)) < masked] = -INF
    t = torch.from_numpy(v).cuda()
    return t.to(torch.bfloat16) if bf16 else t


def _params(seed, rows):
    g = np.random.default_rng(seed + 1000)
    pick = lambda *v: np.array([v[i % len(v)] for i in g.permutation(rows)])  # noqa: E731
    return dict(u=g.random(rows, dtype=np.float32), temperature=pick(1.0, 0.7, 0.0, 1.5, 0.2),
                top_k=pick(0, 50, 1, 1000, 3), top_p=pick(1.0, 0.9, 0.95, 0.3), min_p=pick(0.0, 0.05, 0.3))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,vocab", [
    (1, 1), (2, 2), (3, 3), (4, 5), (5, 63), (6, 255), (5, 1023), (5, 1024), (5, 1025), (3, 4097),
    (20, 32003), (7, 50021), (1, 163840), (3, 163840), (40, 163840), (300, 2048), (2, 524288)])
def test_every_step(rows, vocab, bf16):
    p = _params(rows + vocab, rows)
    _check(_logits(vocab, rows, vocab, bf16=bf16, masked=0.2 if vocab > 5 else 0.0), **p)


@pytest.mark.parametrize("steps", [(), ("temperature",), ("top_k",), ("top_p",), ("min_p",), ("top_k", "top_p"),
                                   ("temperature", "min_p"), ("top_p", "min_p")])
@pytest.mark.parametrize("rows,vocab", [(1, 40000), (24, 9001), (200, 3001)])
def test_steps_left_out(steps, rows, vocab):
    p = _params(rows, rows)
    _check(_logits(3, rows, vocab), u=p["u"], **{k: p[k] for k in steps})


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("vocab", [7000, 163840])
@pytest.mark.parametrize("sigma,bf16", [(0.0, False), (0.0, True), (0.02, True), (0.3, True), (0.3, False), (1e-4, False)])
def test_many_equal_or_close(rows, vocab, sigma, bf16):
    """Cuts that fall among thousands of equal logits, or into a bin with more elements than the list."""
    n = rows
    g = np.random.default_rng(vocab)
    _check(_logits(8, n, vocab, sigma, bf16), u=g.random(n, dtype=np.float32), top_k=np.tile([0, 5001], n // 2),
           top_p=np.tile([0.37, 0.5], n // 2), temperature=np.tile([1.0, 2.5], n // 2))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows", [1, 5, 300])
@pytest.mark.parametrize("k", [2, 50, 1024, 1025])
def test_small_k_among_more_equal_logits_than_are_listed(rows, k, bf16):
    """A few tokens ahead, then thousands that share the k-th place: cut by index."""
    v = 20000
    l = torch.full((rows, v), 1.25, device="cuda")
    l[:, 9::5000] = 1.5
    l[:, 3] = float("nan")
    l = l.to(torch.bfloat16) if bf16 else l
    g = np.random.default_rng(k)
    _check(l, u=g.random(rows, dtype=np.float32), top_k=[k] * rows, top_p=[0.9] * rows)


def test_equal_logits_in_closed_form():
    """V equal logits, top-k k: k equal weights; a draw with u is token floor(u k)."""
    v, k = 100000, 6250
    u = np.array([0.0, 0.25, 0.5, 0.7503, 1 - 2.0 ** -24], np.float32)
    tokens, logprobs = _draw(torch.full((5, v), -3.5, device="cuda"), u, top_k=[k] * 5)
    assert tokens.tolist() == [int(np.floor(float(x) * k)) for x in u]
    assert np.allclose(logprobs, -np.log(k), rtol=2.0 ** -23)
    tokens, _ = _draw(torch.full((5, v), -3.5, device="cuda"), u, top_p=[0.5] * 5)
    assert tokens.tolist() == [int(np.floor(float(x) * (v // 2))) for x in u]


@pytest.mark.parametrize("rows", [1, 90])  # few rows, many
def test_extreme_parameters(rows):
    for name, values in (("temperature", [0.0, -1.0, 1e-30, 1e-42, 1e30, INF, float("nan")]),
                         ("top_k", [-5, 0, 1, 2, 4999, 5000, 5001, 2 ** 31 - 1]),
                         ("top_p", [-1.0, 0.0, 1e-30, 1e-7, 1 - 2.0 ** -24, 1.0, 2.0, float("nan")]),
                         ("min_p", [-1.0, 0.0, 1e-30, 0.999999, 1.0, 5.0, float("nan")])):
        for v in values:
            _check(_logits(1, rows, 5000), u=np.full(rows, 0.61, np.float32), **{name: [v] * rows})
    for u in (0.0, 2.0 ** -149, 1 - 2.0 ** -24, 1.0, 3.0, -1.0, float("nan")):
        for kw in ({}, {"top_k": [7] * rows}, {"top_p": [0.8] * rows}):
            _check(_logits(2, rows, 3001), u=np.full(rows, u, np.float32), **kw)


@pytest.mark.parametrize("pad", [0, 70])  # few rows, many
@pytest.mark.parametrize("kw", [{}, {"top_k": 3}, {"top_p": 0.9}, {"temperature": 0.0}, {"min_p": 0.1, "top_p": 0.5}])
def test_masked_and_odd_rows(kw, pad):
    v = 3000
    low = float(np.finfo(np.float32).min)
    base = np.random.default_rng(0).standard_normal((10 + pad, v)).astype(np.float32)
    base[0] = -INF                      # nothing left
    base[1] = np.nan                    # nothing either
    base[2] = -INF
    base[2, 1234] = -5.0                # one left
    base[3, ::2] = np.nan
    base[4, [7, 900]] = INF             # two that take all
    base[5] = low                       # a mask of the type's lowest value everywhere: all equal
    base[6] = low
    base[6, [5, 6]] = 1.0, 1.5
    base[7] = np.where(np.arange(v) % 2, 0.0, -0.0)  # one value
    base[8] = np.float32(3e38)
    base[8, :1500] = -3e38
    base[9] = -INF
    base[9, v - 1] = low
    n = 10 + pad
    _check(torch.from_numpy(base).cuda(), u=np.random.default_rng(1).random(n, dtype=np.float32),
           **{k: [x] * n for k, x in kw.items()})


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows", [5, 80])
@pytest.mark.parametrize("off,stride", [(0, 4099), (1, 4100), (3, 4103), (2, 4098)])
def test_strided_and_offset_rows(rows, bf16, off, stride):
    whole = _logits(5, rows, stride, bf16=bf16)
    view = whole[:, off:off + 4096]
    p = _params(off, rows)
    _check(view, **p)
    assert view.data_ptr() % 16 != 0 or off == 0


def test_same_result_however_often_and_for_any_batch():
    logits, p = _logits(6, 64, 60001, bf16=True), _params(2, 64)
    first = _draw(logits, **p)
    for _ in range(3):
        again = _draw(logits, **p)
        assert (again[0] == first[0]).all() and (again[1] == first[1]).all()
    for r in (0, 13, 63):  # alone, as in the batch
        one = _draw(logits[r:r + 1], **{k: v[r:r + 1] for k, v in p.items()})
        assert one[0][0] == first[0][r] and one[1][0] == first[1][r]


def test_offsets_past_32_bits():
    rows, vocab = 9000, 131072  # 4.7 GB of fp32 logits
    from pegainfer_amd import ops
    logits = torch.zeros(rows, vocab, device="cuda")
    tail = _logits(7, 6, vocab)
    logits[-6:] = tail
    p = _params(3, 6)
    ws = ops.SampleWorkspace(rows, vocab)
    u = torch.zeros(rows, device="cuda")
    u[-6:] = torch.from_numpy(p["u"]).cuda()
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    ops.sample_tokens(ws, logits, u, tokens)
    assert tokens[-6:].tolist() == _draw(tail, p["u"])[0].tolist() and (tokens[:-6] == 0).all()


def test_workspace_is_left_fit_for_the_next_call():
    from pegainfer_amd import ops
    ws = ops.SampleWorkspace(80, 40000)
    ws.buffer.fill_(0xA5)
    for rows, vocab in ((80, 40000), (1, 40000), (3, 17), (80, 900), (2, 39999)):
        logits, p = _logits(rows, rows, vocab), _params(rows, rows)
        got = _draw(logits, ws=ws, **p)
        new = _draw(logits, **p)
        assert (got[0] == new[0]).all() and (got[1] == new[1]).all()


@pytest.mark.parametrize("rows", [2, 100])
def test_captured(rows):
    from pegainfer_amd import ops
    logits, p = _logits(9, rows, 20011), _params(4, rows)
    dev = {k: torch.from_numpy(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda() for k, v in p.items()}
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    logprobs = torch.zeros(rows, device="cuda")
    ws = ops.SampleWorkspace(rows, 20011)
    u = dev.pop("u")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_tokens(ws, logits, u, tokens, logprobs=logprobs, **dev)
    for _ in range(4):
        u.copy_(u.roll(1))
        logits.copy_(logits.roll(7, 1))
        graph.replay()
        torch.cuda.synchronize()
        want = _draw(logits, u.cpu().numpy(), **{k: v.cpu().numpy() for k, v in dev.items()})
        assert (tokens.cpu().numpy() == want[0]).all() and (logprobs.cpu().numpy() == want[1]).all()


@pytest.mark.parametrize("rows", [1, 80])  # of each kind: few rows, many
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kw", [{}, {"top_k": 3}, {"top_k": 2000}, {"top_p": 0.9}, {"temperature": 0.0},
                                {"top_k": 40, "top_p": 0.8}, {"top_p": 0.9, "min_p": 0.01}])
def test_signaling_nans_hide_nothing_beside_them(kw, bf16, rows):
    """In every place of every vector of 16 bytes, the largest logit's among them."""
    vec, v = (8, 3001) if bf16 else (4, 3001)
    patterns = [0x7F81, 0xFF81, 0x7FBF] if bf16 else [0x7F800001, 0xFF800001, 0x7FBFFFFF]
    kind = np.uint16 if bf16 else np.uint32
    for e in range(vec):
        plain = _logits(e, rows, v, 1.0, bf16)
        bits = plain.view(torch.int16 if bf16 else torch.int32).cpu().numpy().view(kind).copy()
        top = np.array([1496 + (e + 1 + r % (vec - 1)) % vec for r in range(rows)])  # 1496: a vector's first
        for r in range(rows):
            bits[r, e::vec] = patterns[(r + e) % 3]
            bits[r, top[r]] = 0x40E0 if bf16 else 0x40E00000  # 7
        logits = torch.from_numpy(bits.view(np.int16 if bf16 else np.int32)).cuda().view(plain.dtype)
        g = np.random.default_rng(e)
        _check(logits, u=g.random(rows, dtype=np.float32), **{k: [x] * rows for k, x in kw.items()})
        greedy = _draw(logits, [0.5] * rows, temperature=[0.0] * rows)[0]
        assert (greedy == top).all()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.5])
@pytest.mark.parametrize("kw", [{}, {"top_k": 2}, {"top_k": 4000}, {"top_p": 1 - 2.0 ** -24}])
@pytest.mark.parametrize("vocab", [2, 5, 5000])
def test_weights_on_the_border_of_the_range(vocab, kw, temperature, bf16, rows):
    """The largest logit is 28 T, all others are all but zero: in 64 bits they lie 28 T below it, the
    smallest weight that there is, and the sum of the two in fp32 is lost."""
    g = np.random.default_rng(vocab)
    l = torch.zeros(rows, vocab)
    l[:, 1::3], l[:, 2::3] = -1e-20, -1e-38
    l[:, vocab // 2] = 28 * temperature
    l = (l.to(torch.bfloat16) if bf16 else l).cuda()
    for u in (0.0, 0.5, 1 - 2.0 ** -24, 1.0, 3.0):
        _check(l, u=[u] * rows, temperature=[temperature] * rows, **{k: [x] * rows for k, x in kw.items()})
    _check(l, u=g.random(rows, dtype=np.float32), temperature=[temperature] * rows)


@pytest.mark.parametrize("rows", [5, 300])
def test_the_largest_sum_of_weights(rows):
    """2^19 equal logits, whose weights add up to 2^63: cut by count, by mass, by both, or not at all."""
    v = 1 << 19
    logits = torch.full((rows, v), 2.5, dtype=torch.bfloat16, device="cuda")
    u = np.resize(np.array([0.0, 0.25, 0.5, 0.7503, 1 - 2.0 ** -24], np.float32), rows)
    p = np.float32(0.3)
    for kept, kw in ((v, {}), (v, {"top_k": v}), (v - 1, {"top_k": v - 1}), (6250, {"top_k": 6250}), (3, {"top_k": 3}),
                     (int(np.ceil(float(p) * v)), {"top_p": p}), (v, {"top_p": 1 - 2.0 ** -24}),
                     (int(np.ceil(float(p) * (v - 1))), {"top_k": v - 1, "top_p": p})):
        tokens, logprobs = _draw(logits, u, **{k: [x] * rows for k, x in kw.items()})
        # a uniform number of 24 bits times a count of 20: exact in 64 bits
        assert tokens.tolist() == [int(float(x) * kept) for x in u], kw
        assert np.abs(logprobs + np.log(kept)).max() <= 2.0 ** -24 * (1 + np.log(kept)), kw
