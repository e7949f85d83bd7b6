"""The norm and microscaled operators without a GPU: their 64-bit references against torch's own
conversions, and every refusal of the C entry points and of the Python wrappers."""
import numpy as np
import pytest
import torch

import mx_ref

A = 0x10000  # addresses that no accepted call of these tests dereferences


def _call(name, *args):
    from pegainfer_amd import _lib
    return getattr(_lib.lib(), name)(*args)


def test_reference_codes_are_torch_casts():
    g = np.random.default_rng(0)
    v = np.concatenate([g.standard_normal((40, 64)) * 10.0 ** g.integers(-6, 6, (40, 1)),
                        np.arange(-464, 464, 0.25)[:3712].reshape(58, 64)])
    for fmt in ("fp8", "fp4"):
        codes, sc = mx_ref.quantize(v, fmt)
        u = (v.reshape(len(v), -1, 32) / 2.0 ** (sc[..., None].astype(float) - 127)).reshape(v.shape)
        if fmt == "fp8":
            want = torch.from_numpy(u).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
            assert np.array_equal(codes, want.numpy())
        back = mx_ref.values(codes, sc, fmt)
        # half a step of the value's binade, or of the smallest normal's
        step = 2.0 ** -3 if fmt == "fp8" else 2.0 ** -1
        low = 2.0 ** -6 if fmt == "fp8" else 1.0
        unit = np.repeat(2.0 ** (sc.astype(float) - 127), 32, 1)
        binade = 2.0 ** np.floor(np.log2(np.maximum(np.abs(v) / unit, low)))
        assert (np.abs(back - v) <= binade * unit * step / 2).all()


def test_reference_scale_is_the_smallest_that_holds():
    for fmt, top in (("fp8", 464.0), ("fp4", 7.0)):
        for s in (-126, -3, 0, 50, 110):
            lim = top * 2.0 ** s
            over = np.nextafter(lim, np.inf)
            under = np.nextafter(lim, 0)
            want = [s, s + 1, s] if fmt == "fp8" else [s + 1, s + 1, s]
            got = mx_ref.scale_bytes([lim, over, under], fmt).astype(int) - 127
            assert got.tolist() == want
    assert mx_ref.scale_bytes([0.0, np.inf, 1e-45], "fp8").tolist() == [0, 255, 0]


def test_reference_bf16_rounds_once():
    one = 1.0
    half = 2.0 ** -8  # half a bf16 step above 1
    v = [one + half, one + half + 2.0 ** -40, one + 3 * half, -(one + half), 0.0, -0.0]
    assert mx_ref.bf16_round(v).tolist() == [0x3F80, 0x3F81, 0x3F82, 0xBF80, 0, 0x8000]


NORM = [A, False, A << 1, A << 2, 1e-6, A << 3, A << 4, A << 5, A << 6, 2, 64, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (3, None, 1), (9, -1, 1), (10, 0, 1), (10, -8, 1), (4, -1.0, 1),
    (4, float("nan"), 1),
    (7, None, 1), (8, None, 1),              # codes without scales, scales without codes
    (10, 60, 801), (10, 40, 801),            # not a multiple of 8, of 32
    (10, 32776, 801), (10, 65536, 801),      # past the registers
    (0, A + 2, 801), (2, (A << 1) + 8, 801), (3, (A << 2) + 4, 801), (5, (A << 3) + 2, 801),
    (6, (A << 4) + 8, 801), (7, (A << 5) + 8, 801), (8, (A << 6) + 2, 801),
    (5, A << 4, 1), (5, (A << 4) + 16, 1),   # two outputs in one place
    (5, A + 16, 1), (6, (A << 1) + 128, 1),  # an output across other rows of an input
    (7, A, 1), (7, A << 1, 1), (8, A << 2, 1), (6, A << 2, 1),
])
def test_norm_refuses(at, value, code):
    args = list(NORM)
    args[at] = value
    assert _call("pega_add_rmsnorm", *args) == code


def test_norm_refuses_an_output_over_fp32_rows():
    args = list(NORM)
    args[1] = True
    args[5] = A  # bf16 rows over fp32 rows: other rows' bytes
    assert _call("pega_add_rmsnorm", *args) == 1


def test_norm_needs_an_output_and_takes_no_rows():
    args = list(NORM)
    args[5] = args[6] = args[7] = args[8] = None
    assert _call("pega_add_rmsnorm", *args) == 1
    args = list(NORM)
    args[9] = 0
    assert _call("pega_add_rmsnorm", *args) == 0


@pytest.mark.parametrize("name", ["pega_mx_quantize", "pega_mx_swiglu_quantize", "pega_mx_dequantize"])
@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (1, None, 1), (2, None, 1), (3, 2, 1), (3, -1, 1), (4, -1, 1), (5, 0, 1),
    (5, -32, 1), (5, 48, 801), (0, A + 4, 801), (1, (A << 1) + 2, 801), (1, A, 1), (2, A + 16, 1),
    (2, A << 1, 1),
])
def test_mx_refuses(name, at, value, code):
    args = [A, A << 1, A << 2, 0, 2, 64, None]
    args[at] = value
    assert _call(name, *args) == code
    args = [A, A << 1, A << 2, 1, 0, 64, None]
    assert _call(name, *args) == 0  # no rows


def test_mx_tensor_checks_its_shape():
    from pegainfer_amd import ops
    t = ops.MxTensor.empty(3, 64, ops.MxFormat.Fp4E2M1, device="cpu")
    assert tuple(t.codes.shape) == (3, 32) and tuple(t.scales.shape) == (3, 2)
    assert tuple(ops.MxTensor.empty(0, 32, ops.MxFormat.Fp8E4M3, device="cpu").codes.shape) == (0, 32)
    assert t.head(2).rows == 2 and t.head(2).codes.data_ptr() == t.codes.data_ptr()
    with pytest.raises(ValueError):
        t.head(4)
    with pytest.raises(ValueError):
        ops.MxTensor.empty(3, 48, ops.MxFormat.Fp8E4M3, device="cpu")
    with pytest.raises(ValueError):
        ops.MxTensor(3, 64, ops.MxFormat.Fp8E4M3, t.codes, t.scales)
    with pytest.raises(ValueError):
        ops.MxTensor(3, 64, ops.MxFormat.Fp4E2M1, t.codes.int(), t.scales)
    with pytest.raises(ValueError):
        ops.MxTensor(3, 64, 1, t.codes, t.scales)


def test_wrappers_refuse_shapes_and_types_before_the_device():
    from pegainfer_amd import ops
    bf = dict(dtype=torch.bfloat16)
    x, w = torch.zeros(2, 64, **bf), torch.zeros(64, **bf)
    q8 = ops.MxTensor.empty(2, 64, ops.MxFormat.Fp8E4M3, device="cpu")
    q4 = ops.MxTensor.empty(2, 64, ops.MxFormat.Fp4E2M1, device="cpu")
    out = torch.zeros(2, 64, **bf)
    for bad in (lambda: ops.add_rmsnorm(x, None, w, 1e-6),
                lambda: ops.add_rmsnorm(x.half(), None, w, 1e-6, normed=out),
                lambda: ops.add_rmsnorm(x[0], None, w, 1e-6, normed=out),
                lambda: ops.add_rmsnorm(x, x[:1], w, 1e-6, normed=out),
                lambda: ops.add_rmsnorm(x, None, w[:32], 1e-6, normed=out),
                lambda: ops.add_rmsnorm(x, None, w.float(), 1e-6, normed=out),
                lambda: ops.add_rmsnorm(x, None, w, 1e-6, normed=out, residual_out=out),
                lambda: ops.add_rmsnorm(x, None, w, 1e-6, normed=out.float()),
                lambda: ops.add_rmsnorm(x, None, w, 1e-6, quantized=q4),
                lambda: ops.add_rmsnorm(x, None, w, 1e-6, quantized=q8.head(1)),
                lambda: ops.mx_quantize(x[:1], q8), lambda: ops.mx_quantize(x.float(), q8),
                lambda: ops.mx_swiglu_quantize(x, q8),
                lambda: ops.mx_dequantize(q8, out[:, :32])):
        with pytest.raises(ValueError):
            bad()


GEMM = [A, A << 1, A << 2, A << 3, 0, A << 4, 32, 4, 256, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (1, None, 1), (2, None, 1), (3, None, 1), (5, None, 1), (4, 2, 1), (4, -1, 1),
    (6, 0, 1), (7, -1, 1), (8, 0, 1), (6, 24, 801), (8, 96, 801), (8, 64, 801), (8, 1 << 23, 801),
    (0, A + 8, 801), (2, (A << 2) + 4, 801), (5, (A << 4) + 8, 801), (1, (A << 1) + 2, 801),
    (3, (A << 3) + 1, 801)])
def test_mx_gemm_refuses(at, value, code):
    args = list(GEMM)
    args[at] = value
    assert _call("pega_mx_gemm", *args) == code


def test_mx_gemm_takes_no_rows():
    args = list(GEMM)
    args[7] = 0
    assert _call("pega_mx_gemm", *args) == 0


GROUPED = [A, A << 1, 0, A << 2, A << 3, A << 4, A << 5, A << 6, A << 7, A << 8, 64, 16, 2, True,
           4, 32, 256, 3, 1, None]


@pytest.mark.parametrize("at,value,code", [
    (0, None, 1), (1, None, 1), (3, None, 1), (4, None, 1), (5, None, 1), (6, None, 1),
    (7, None, 1), (8, None, 1), (9, None, 1), (2, 2, 1), (10, -1, 1), (11, 24, 1), (11, 0, 1),
    (11, 128, 1), (12, 0, 1), (12, 1 << 30, 1), (14, -1, 1), (15, 40, 801), (16, 192, 801),
    (16, 0, 1), (17, 0, 1), (18, 0, 1), (3, (A << 2) + 2, 801), (14, 1 << 24, 801)])
def test_mx_grouped_gemm_refuses(at, value, code):
    args = list(GROUPED)
    args[at] = value
    assert _call("pega_mx_grouped_gemm", *args) == code


def test_mx_grouped_gemm_with_nothing_to_do():
    for at in (10, 14):
        args = list(GROUPED)
        args[at] = 0
        assert _call("pega_mx_grouped_gemm", *args) == 0


@pytest.mark.parametrize("operand,size", [(0, 32 * 128), (1, 32 * 8), (2, 4 * 256), (3, 4 * 8)])
def test_mx_products_refuse_an_output_on_an_operand(operand, size):
    for y in (0, 16, size - 16):
        args = list(GEMM)
        args[operand] = A << 20
        args[5] = (A << 20) + y
        assert _call("pega_mx_gemm", *args) == 1
    place = {0: 4, 1: 5, 2: 0, 3: 1}[operand]
    args = list(GROUPED)
    args[place] = A << 20
    args[3] = (A << 20) + (size if operand < 2 else 0)  # the weights are three experts'
    assert _call("pega_mx_grouped_gemm", *args) == 1


def test_mx_gemm_wrappers_refuse_before_the_device():
    from pegainfer_amd import ops
    q = lambda r, c, f=ops.MxFormat.Fp4E2M1: ops.MxTensor.empty(r, c, f, device="cpu")  # noqa: E731
    w, x = q(32, 256), q(4, 256, ops.MxFormat.Fp8E4M3)
    y = torch.zeros(4, 32, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    routing = ops.KimiMarlinRouting(4, 4, 8, 0, 8, 64, 8, 2, 2, i, i, i)
    g = lambda **kw: ops.mx_grouped_gemm(**{**dict(  # noqa: E731
        routing=routing, x=x, w=w, topk_weight=None, output=torch.zeros(8, 16, dtype=torch.bfloat16),
        top_k=2, mul_topk_weights=False, size_m=4), **kw})
    for bad in (lambda: ops.mx_gemm(q(32, 256, ops.MxFormat.Fp8E4M3), x, y),
                lambda: ops.mx_gemm(w, q(4, 128), y), lambda: ops.mx_gemm(w, x, y.float()),
                lambda: ops.mx_gemm(w, x, y[:3]),
                lambda: g(w=q(33, 256)), lambda: g(x=q(4, 128)), lambda: g(size_m=5),
                lambda: g(output=torch.zeros(7, 16, dtype=torch.bfloat16)), lambda: g(top_k=0),
                lambda: g(mul_topk_weights=True), lambda: g(mul_topk_weights=True, topk_weight=torch.zeros(7)),
                lambda: g(output=torch.zeros(8, 16))):
        with pytest.raises(ValueError):
            bad()


def _few(**kw):
    from pegainfer_amd import _lib
    a = _lib.MoeFew()
    for i, (name, _) in enumerate(_lib.MoeFew._fields_[:22]):
        setattr(a, name, A << i)
    a.route_scale = a.routed_scale = 1.0
    a.softmax, a.shared_kind, a.tokens, a.hidden_dim, a.inter, a.shared_inter = 0, 1, 4, 128, 64, 64
    a.n_experts, a.local_experts, a.global_start, a.topk = 16, 4, 4, 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _few_call(**kw):
    import ctypes
    return _call("pega_moe_few_tokens", ctypes.byref(_few(**kw)), None)


@pytest.mark.parametrize("name", [
    "x", "logits", "bias", "w13", "w13_scales", "w2", "w2_scales", "shared_w13", "shared_w2", "out",
    "topk_weight", "topk_idx", "act", "act_factors", "act_shared", "slots", "partials", "counters"])
def test_few_tokens_refuses_null(name):
    assert _few_call(**{name: None}) == 1


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=0), 1), (dict(tokens=-1), 1), (dict(tokens=17), 801), (dict(hidden_dim=96), 801),
    (dict(hidden_dim=0), 1), (dict(inter=32), 801), (dict(inter=0), 1), (dict(shared_inter=100), 801),
    (dict(shared_inter=0), 1), (dict(n_experts=3), 1), (dict(global_start=13), 1),
    (dict(global_start=-1), 1), (dict(topk=0), 1), (dict(topk=17), 1), (dict(topk=33, n_experts=64), 801),
    (dict(local_experts=513, n_experts=1000), 801), (dict(n_experts=1025), 801),
    (dict(local_experts=0), 1), (dict(shared_kind=3), 1), (dict(shared_kind=-1), 1),
    (dict(shared_kind=2, shared_w13_scales=None), 1), (dict(shared_kind=2, shared_w2_scales=None), 1),
    (dict(shared_kind=2, act_shared_factors=None), 1),
    (dict(route_scale=0.0), 1), (dict(route_scale=float("nan")), 1), (dict(x=A + 8), 801),
    (dict(w13=A + 4), 801), (dict(act=A + 2), 801), (dict(shared_w2=A + 2), 801),
    (dict(hidden_dim=1 << 20, inter=1024), 801)])
def test_few_tokens_refuses(kw, code):
    assert _few_call(**kw) == code


@pytest.mark.parametrize("kw", [
    dict(out=A << 40, residual=(A << 40) + 256), dict(out=(A << 40) + 256, residual=A << 40),
    dict(logits=A << 40, topk_weight=(A << 40) + 64), dict(logits=A << 40, topk_idx=(A << 40) + 64),
    dict(topk_weight=A << 40, topk_idx=(A << 40) + 16)])
def test_few_tokens_refuses_overlaps(kw):
    assert _few_call(**kw) == 1


def test_few_tokens_struct_matches_the_header(tmp_path):
    import ctypes
    import os
    import subprocess
    from conftest import ROOT
    from pegainfer_amd import _lib
    src = tmp_path / "s.c"
    fields = [n for n, _ in _lib.MoeFew._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "pega_moe.h"\nint main(void) {\n'
                   'printf("%zu", sizeof(pega_moe_few));\n'
                   + "".join(f'printf(" %zu", offsetof(pega_moe_few, {n}));\n' for n in fields)
                   + "return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got[0] == ctypes.sizeof(_lib.MoeFew) == 224
    assert got[1:] == [getattr(_lib.MoeFew, n).offset for n in fields]


def test_few_tokens_wrappers_refuse_before_the_device():
    from pegainfer_amd import ops
    ws = ops.FewTokensWorkspace(4, 128, 64, topk=2, local_experts=4, shared_inter=64, device="cpu")
    assert ws.act.numel() == 4 * 4 * 64 and ws.counters.numel() == 2 + 512 and ws.slots.numel() == 5
    for bad in (dict(max_tokens=17), dict(max_tokens=0), dict(hidden=96), dict(inter=100),
                dict(topk=0), dict(topk=33), dict(shared_inter=32), dict(local_experts=0)):
        kw = {**dict(max_tokens=4, hidden=128, inter=64, topk=2, local_experts=4, shared_inter=64), **bad}
        with pytest.raises(ValueError):
            ops.FewTokensWorkspace(kw.pop("max_tokens"), kw.pop("hidden"), kw.pop("inter"), device="cpu", **kw)

    def pack(e, k, n):
        return ops.MarlinInt4Weight(e, k, n, torch.zeros(e * k * n // 2, dtype=torch.uint8),
                                    torch.zeros(e * n * (k // 32), dtype=torch.bfloat16))
    bf = dict(dtype=torch.bfloat16)
    good = dict(x=torch.zeros(3, 128, **bf), logits=torch.zeros(3, 16), w13=pack(4, 128, 128),
                w2=pack(4, 64, 128), topk_weight=torch.zeros(3, 2),
                topk_idx=torch.zeros(3, 2, dtype=torch.int32), out=torch.zeros(3, 128, **bf))
    for bad in (dict(x=torch.zeros(3, 128)), dict(x=torch.zeros(5, 128, **bf)),
                dict(x=torch.zeros(0, 128, **bf)), dict(x=torch.zeros(3, 64, **bf)),
                dict(logits=torch.zeros(2, 16)), dict(logits=torch.zeros(3, 16, **bf)),
                dict(w13=pack(3, 128, 128)), dict(w2=pack(4, 128, 128)), dict(w13=pack(4, 128, 256)),
                dict(topk_weight=torch.zeros(3, 1)), dict(topk_idx=torch.zeros(3, 2)),
                dict(out=torch.zeros(2, 128, **bf)), dict(residual=torch.zeros(3, 64, **bf)),
                dict(bias=torch.zeros(15)), dict(global_start=13), dict(global_start=-1),
                dict(shared=(torch.zeros(64, 128, **bf), torch.zeros(128, 64, **bf))),
                dict(shared=(torch.zeros(128, 128, **bf), torch.zeros(128, 32, **bf))),
                dict(shared=(pack(1, 128, 64), pack(1, 64, 128)))):
        with pytest.raises(ValueError):
            ops.moe_few_tokens(ws, **{**good, **bad})


def test_no_rows_is_nothing_to_do():
    """Empty tensors have no address: nothing is asked of it, sizes are still checked."""
    for fmt in (0, 1):
        assert _call("pega_mx_quantize", None, None, None, fmt, 0, 64, None) == 0
        assert _call("pega_mx_swiglu_quantize", None, None, None, fmt, 0, 64, None) == 0
        assert _call("pega_mx_dequantize", None, None, None, fmt, 0, 64, None) == 0
        assert _call("pega_mx_gemm", A, A << 1, None, None, fmt, None, 32, 0, 256, None) == 0
        assert _call("pega_mx_quantize", None, None, None, fmt, 0, 40, None) == 801
        assert _call("pega_mx_gemm", A, A << 1, None, None, fmt, None, 32, 0, 200, None) == 801
    assert _call("pega_add_rmsnorm", None, False, None, A, 1e-6, None, None, None, None, 0, 64, None) == 0
    assert _call("pega_add_rmsnorm", None, False, None, A, -1.0, None, None, None, None, 0, 64, None) == 1


@pytest.mark.parametrize("bad", [dict(local_experts=513), dict(hidden=1 << 20, inter=1024),
                                 dict(hidden=1 << 20, inter=64, shared_inter=1024)])
def test_few_tokens_workspace_refuses_what_its_calls_would(bad):
    """The entry's limits, and the same sizes refused there."""
    from pegainfer_amd import ops
    kw = {**dict(hidden=128, inter=64, topk=2, local_experts=4, shared_inter=64), **bad}
    with pytest.raises(ValueError):
        ops.FewTokensWorkspace(1, kw.pop("hidden"), kw.pop("inter"), device="meta", **kw)
    entry = {**{"hidden" if k == "hidden_dim" else k: v for k, v in bad.items()}, "n_experts": 1000}
    entry["hidden_dim"] = entry.pop("hidden", 128)
    assert _few_call(**entry) == 801


def test_few_tokens_workspace_takes_the_limits():
    from pegainfer_amd import ops
    ops.FewTokensWorkspace(1, 128, 64, topk=2, local_experts=512, device="meta")
    ops.FewTokensWorkspace(1, 1 << 20, 448, topk=2, local_experts=4, device="meta")


def test_decode_layers_refuse_few_tokens_of_other_sizes_when_built():
    from pegainfer_amd import layer, ops

    def pack(e, k, n):
        u8, bf = dict(dtype=torch.uint8, device="meta"), dict(dtype=torch.bfloat16, device="meta")
        return ops.MarlinInt4Weight(e, k, n, torch.empty(e * k * n // 2, **u8), torch.empty(e * n * (k // 32), **bf))
    routed = layer.RoutedExperts(pack(513, 128, 128), pack(513, 64, 128), max_tokens=8, topk=2, block_size=8,
                                 device="meta")
    bf = dict(dtype=torch.bfloat16, device="meta")
    kimi = layer.KimiSharedExpert(torch.empty(128, 128, **bf), torch.empty(128, 64, **bf), max_tokens=8, device="meta")
    dsv2 = layer.ExpertFFN(pack(1, 128, 128), pack(1, 64, 128), max_rows=8, device="meta")
    for make in (lambda n: layer.KimiMoeDecodeLayer(routed, kimi, device="meta", few_tokens=n),
                 lambda n: layer.Dsv2MoeLayer(routed, dsv2, device="meta", few_tokens=n)):
        make(0)
        with pytest.raises(ValueError, match="local experts"):
            make(4)


@pytest.mark.parametrize("shape", [(3, 16), (8, 16), (1, 4, 16)])
def test_few_tokens_takes_logits_as_the_selects_do(shape):
    """Whatever covers the tokens' rows (a buffer of a larger batch): refused for its place alone."""
    from pegainfer_amd import ops
    u8, bf = dict(dtype=torch.uint8), dict(dtype=torch.bfloat16)
    pack = lambda e, k, n: ops.MarlinInt4Weight(  # noqa: E731
        e, k, n, torch.zeros(e * k * n // 2, **u8), torch.zeros(e * n * (k // 32), **bf))
    ws = ops.FewTokensWorkspace(4, 128, 64, topk=2, local_experts=4, device="cpu")
    with pytest.raises(ValueError, match="current GPU"):
        ops.moe_few_tokens(ws, torch.zeros(3, 128, **bf), torch.zeros(*shape), pack(4, 128, 128), pack(4, 64, 128),
                           torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 128, **bf))
    with pytest.raises(ValueError, match="logits"):
        ops.moe_few_tokens(ws, torch.zeros(3, 128, **bf), torch.zeros(2, 16), pack(4, 128, 128), pack(4, 64, 128),
                           torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 128, **bf))


@pytest.mark.parametrize("at,value", [(6, 1 << 28), (6, (1 << 31) - 16), (7, (1 << 21) - 31), (7, (1 << 31) - 1)])
def test_mx_gemm_refuses_more_than_a_launch_holds(at, value):
    args = list(GEMM)
    args[at], args[8] = value, 128
    for operand in range(4):
        args[operand] = (A << 40) + (operand << 60)
    assert _call("pega_mx_gemm", *args) == 801


@pytest.mark.parametrize("ids,bs", [((1 << 31) - 1, 8), (65535 * 8 + 1, 8), (65535 * 64 + 1, 64)])
def test_mx_grouped_gemm_refuses_more_blocks_than_a_launch_holds(ids, bs):
    args = list(GROUPED)
    args[10], args[11] = ids, bs
    assert _call("pega_mx_grouped_gemm", *args) == 801
    args = list(GROUPED)
    args[15] = 1 << 28
    assert _call("pega_mx_grouped_gemm", *args) == 801


@pytest.mark.parametrize("output", ["topk_weight", "topk_idx", "out"])
@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("operand,size", [
    ("x", 1024), ("bias", 64), ("w13", 32768), ("w13_scales", 4096), ("w2", 16384), ("w2_scales", 2048),
    ("shared_w13", (32768, 8192)), ("shared_w13_scales", (0, 1024)), ("shared_w2", (16384, 4096)),
    ("shared_w2_scales", (0, 512)), ("residual", 1024)])
def test_few_tokens_refuses_outputs_on_operands(output, kind, operand, size):
    """128 columns, 64 between, 4 tokens of top 2, 4 local experts: the operand's first and last bytes."""
    size = size if isinstance(size, int) else size[kind - 1]
    if not size or output == "out" and operand not in ("w2", "w2_scales", "shared_w2", "shared_w2_scales"):
        return  # not an operand of this kind; out may be on what only the first launch reads
    for place in (A << 40, (A << 40) + size - 16):
        assert _few_call(**{"shared_kind": kind, operand: A << 40, output: place}) == 1
        assert "overlap" in _last_error()


def _last_error():
    from pegainfer_amd import _lib
    return _lib.last_error()
