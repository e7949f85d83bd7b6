"""The 4-bit product, the norms on both sides and the token draw without a GPU: every refusal of the C
entry points and of the Python wrappers, the device layout's sizes, and the references themselves."""
import numpy as np
import pytest
import torch

import decode_ref as ref

A = 0x10000  # addresses that no accepted call of these tests dereferences


def _call(name, *args):
    from pegainfer_amd import _lib
    return getattr(_lib.lib(), name)(*args)


NORM = [A, False, A << 1, 1.0, A << 2, A << 3, 3, A << 4, False, 1e-6, A << 5, A << 6, A << 7, A << 8, 2, 64, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (5, None, 1), (7, None, 1), (6, -1, 1), (6, 4, 1), (9, -1.0, 1), (9, float("nan"), 1),
    (14, -1, 1), (15, 0, 1), (15, -8, 1), (12, None, 1), (13, None, 1),
    (15, 60, 801), (15, 40, 801), (15, 32776, 801),
    (0, A + 2, 801), (2, (A << 1) + 8, 801), (4, (A << 2) + 2, 801), (5, (A << 3) + 2, 801),
    (7, (A << 4) + 4, 801), (10, (A << 5) + 2, 801), (11, (A << 6) + 8, 801), (12, (A << 7) + 8, 801),
    (13, (A << 8) + 2, 801),
    (10, A << 6, 1), (10, (A << 6) + 16, 1),  # two outputs in one place
    (10, A + 16, 1), (11, (A << 1) + 128, 1),  # across other rows of an input
    (10, A << 3, 1), (11, (A << 3) + 128, 1),  # on the gate
    (11, A << 4, 1), (11, A << 2, 1), (12, A, 1), (12, A << 1, 1), (13, A << 3, 1)])
def test_norm_refuses(at, value, code):
    args = list(NORM)
    args[at] = value
    assert _call("pega_sandwich_rmsnorm", *args) == code


def test_norm_refuses_gates_rows_and_missing_outputs():
    args = list(NORM)
    args[6], args[5] = 2, (A << 3) + 1  # one a row: 2-byte aligned
    assert _call("pega_sandwich_rmsnorm", *args) == 801
    args = list(NORM)
    args[1], args[10] = True, A  # bf16 rows over fp32 rows: other rows' bytes
    assert _call("pega_sandwich_rmsnorm", *args) == 1
    args = list(NORM)
    args[10:14] = [None] * 4
    assert _call("pega_sandwich_rmsnorm", *args) == 1
    args = list(NORM)
    args[14], args[0] = 0, None  # no rows: nothing to do
    assert _call("pega_sandwich_rmsnorm", *args) == 0


PACK = [A, A << 1, A << 2, A << 3, A << 4, 20, 256, 64, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (1, None, 1), (3, None, 1), (4, None, 1), (5, 0, 1), (5, -3, 1), (6, 0, 1), (6, 96, 1),
    (6, -64, 1), (7, 16, 801), (7, 0, 801), (7, 256, 801), (6, 1 << 21, 801), (5, (1 << 26) + 1, 801),
    (0, A + 2, 801), (1, (A << 1) + 1, 801), (3, (A << 3) + 8, 801), (4, (A << 4) + 4, 801),
    (3, A, 1), (4, A << 1, 1), (3, A << 2, 1), (4, (A << 3) + 1024, 1)])
def test_pack_refuses(at, value, code):
    args = list(PACK)
    args[at] = value
    assert _call("pega_w4_pack", *args) == code


GEMM = [A, A << 2, True, 64, A << 4, A << 6, True, 20, 3, 256, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (1, None, 1), (4, None, 1), (5, None, 1), (7, 0, 1), (8, -1, 1), (9, 0, 1), (9, 100, 1),
    (3, 48, 801), (9, 1 << 21, 801), (8, 16 * 65535 + 1, 801),
    (0, A + 8, 801), (1, (A << 2) + 4, 801), (4, (A << 4) + 2, 801), (5, (A << 6) + 2, 801), (7, (1 << 26) + 1, 801),
    (5, A, 1), (5, A << 2, 1), (5, (A << 4) + 16, 1)])
def test_gemm_refuses(at, value, code):
    args = list(GEMM)
    args[at] = value
    assert _call("pega_w4_gemm", *args) == code


def test_gemm_of_no_rows_is_nothing():
    args = list(GEMM)
    args[8], args[4], args[5] = 0, None, None
    assert _call("pega_w4_gemm", *args) == 0


SAMPLE = [A, False, 100, 3, 100, A << 4, A << 5, A << 6, A << 7, A << 8, A << 9, A << 10, A << 12, 1 << 30, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (5, None, 1), (10, None, 1), (12, None, 1), (3, -1, 1), (4, 0, 1), (2, 99, 1), (13, 8, 1),
    (0, A + 2, 801), (12, (A << 12) + 8, 801),
    (10, A + 16, 1), (11, A << 9, 1), (11, (A << 9) + 8, 1), (10, A << 4, 1), (10, A << 5, 1), (11, A << 8, 1),
    (12, A, 1), (12, A << 9, 1)])
def test_sample_refuses(at, value, code):
    args = list(SAMPLE)
    args[at] = value
    assert _call("pega_sample_tokens", *args) == code


def test_sample_sizes():
    args = list(SAMPLE)
    args[2] = args[4] = (1 << 19) + 1
    assert _call("pega_sample_tokens", *args) == 801
    args = list(SAMPLE)
    args[3], args[0] = 0, None
    assert _call("pega_sample_tokens", *args) == 0
    size = lambda *a: _call("pega_sample_workspace_bytes", *a)  # noqa: E731
    assert size(0, 5) == 0 and size(5, 0) == 0 and 0 < size(1, 10) <= size(2, 10) <= size(2, 1 << 19)
    args = list(SAMPLE)
    args[13] = size(3, 100) - 1
    assert _call("pega_sample_tokens", *args) == 1


# ---------------------------------------------------------------- the wrappers
def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_wrappers_refuse_shapes_and_types():
    from pegainfer_amd import ops
    x, w = _bf(3, 64), _bf(64)
    norm = lambda x=x, r=x, pre=w, **kw: ops.sandwich_rmsnorm(x, r, pre, 1e-6, **{"normed": _bf(3, 64), **kw})  # noqa: E731
    for bad in (dict(x=_bf(64)), dict(x=x.half()), dict(r=_bf(2, 64)), dict(pre=_bf(32)), dict(pre=None),
                dict(post_weight=_bf(65)), dict(gate=torch.zeros(64)), dict(gate=_bf(3)), dict(gate=_bf(2, 1)),
                dict(gate=_bf(1, 64)), dict(normed=_bf(2, 64)), dict(normed=None), dict(residual_out=_bf(3, 63)),
                dict(quantized=ops.MxTensor.empty(3, 64, ops.MxFormat.Fp4E2M1, "cpu")),
                dict(quantized=ops.MxTensor.empty(2, 64, ops.MxFormat.Fp8E4M3, "cpu"))):
        with pytest.raises(ValueError):
            norm(**bad)
    same = _bf(3, 64)
    with pytest.raises(ValueError, match="different buffers"):
        norm(residual_out=same, normed=same)
    with pytest.raises(ValueError, match="current GPU"):
        norm()  # host tensors
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for args, group in (((u8(4, 64), _bf(4, 2)), 32), ((u8(4, 64), _bf(4, 4)), 48), ((u8(4, 24), _bf(4, 1)), 32),
                        ((u8(4, 64).int(), _bf(4, 4)), 32), ((u8(4, 64), torch.zeros(4, 4)), 32),
                        ((u8(4, 64), _bf(4, 4), u8(4, 3)), 32), ((u8(4, 64), _bf(4, 4), _bf(4, 4)), 32),
                        ((u8(0, 64), _bf(0, 4)), 32), ((u8(256), _bf(4, 4)), 32)):
        with pytest.raises(ValueError):
            ops.w4_pack(*args, group=group)
    wt = ops.W4Weight(20, 128, 32, True, u8(2 * 1024), u8(2 * 16 * 16))
    for bad_x, bad_y in ((_bf(3, 64), _bf(3, 20)), (_bf(3, 128), _bf(3, 21)), (_bf(3, 128), _bf(2, 20)),
                         (torch.zeros(3, 128), _bf(3, 20)), (_bf(3, 128), _bf(3, 20).half())):
        with pytest.raises(ValueError):
            ops.w4_gemm(wt, bad_x, bad_y)
    for kw in (dict(out_dim=33), dict(in_dim=130), dict(group=16), dict(with_zeros=False)):
        with pytest.raises(ValueError):
            ops.W4Weight(**{**dict(out_dim=20, in_dim=128, group=32, with_zeros=True, codes=wt.codes, meta=wt.meta), **kw})


def test_sample_wrapper_refuses():
    from pegainfer_amd import ops
    for bad in ((0, 10), (3, 0), (3, ops.SAMPLE_MAX_VOCAB + 1)):
        with pytest.raises(ValueError):
            ops.SampleWorkspace(*bad, device="cpu")
    ws = ops.SampleWorkspace(3, 100, device="cpu")
    l, f, i = torch.zeros(3, 100), torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    good = dict(logits=l, uniform=f, tokens=i)
    for bad in (dict(logits=torch.zeros(300)), dict(logits=l.double()), dict(logits=torch.zeros(4, 100)),
                dict(logits=torch.zeros(3, 101)), dict(logits=torch.zeros(3, 200)[:, ::2]),
                dict(logits=torch.zeros(1, 100).expand(3, 100)), dict(uniform=f.double()), dict(uniform=f[:2]),
                dict(uniform=None), dict(tokens=None), dict(tokens=i.long()), dict(tokens=i[:1]),
                dict(temperature=f[:2]), dict(top_k=f), dict(top_p=i), dict(min_p=torch.zeros(3, 1)), dict(logprobs=i)):
        with pytest.raises((ValueError, AttributeError)):
            ops.sample_tokens(ws, **{**good, **bad})
    with pytest.raises(ValueError, match="current GPU"):
        ops.sample_tokens(ws, **good)


# ---------------------------------------------------------------- the references
def test_reference_draw_by_hand():
    l = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    draw = lambda u, **kw: ref.sample_row(l, u, **kw)[0]  # noqa: E731
    assert [draw(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [draw(u, top_k=2) for u in (0.0, 0.56, 0.58)] == [1, 1, 3]
    assert [draw(u, top_p=0.75) for u in (0.0, 0.45, 0.66, 0.68)] == [1, 2, 2, 3]  # .4, .3, then .2 from .7 on
    assert [draw(u, min_p=0.6) for u in (0.5, 0.6)] == [1, 3]
    assert draw(0.99, temperature=0.0) == 1
    assert ref.sample_row([1.0, 1.0, 1.0], 0.5, top_k=2) == (1, np.log(0.5))
    assert ref.sample_row([-np.inf, np.nan], 0.5)[0] == -1


def test_reference_product_by_hand():
    q = np.array([[0, 15] * 16])
    x = np.ones((1, 32))
    s, z = np.array([[0.5]]), np.array([[3]])
    assert ref.w4_product(x, q, s, None, 32)[0][0, 0] == (0 * 16 + 15 * 16 - 8 * 32) * 0.5
    assert ref.w4_product(x, q, s, z, 32)[0][0, 0] == (15 * 16 - 3 * 32) * 0.5
    assert ref.pack(q)[0, 0] == 0xF0
