"""The 4-bit dense product on the GPU against the formula in 64 bits."""
import numpy as np
import pytest
import torch

import decode_ref as ref

pytestmark = pytest.mark.gpu


def _case(seed, rows, n, k, group, zeros):
    g = np.random.default_rng(seed)
    x = ref.to_bf16_bits(g.standard_normal((rows, k)).astype(np.float32))
    q = g.integers(0, 16, (n, k))
    s = ref.to_bf16_bits((np.abs(g.standard_normal((n, k // group))) * 0.01).astype(np.float32))
    z = g.integers(0, 17, (n, k // group)).astype(np.uint8) if zeros else None
    return x, q, s, z


def _bf(bits):
    return torch.from_numpy(bits.view(np.int16).copy()).cuda().view(torch.bfloat16)


def _pack(q, s, z, group):
    from pegainfer_amd import ops
    return ops.w4_pack(torch.from_numpy(ref.pack(q)).cuda(), _bf(s),
                       None if z is None else torch.from_numpy(z).cuda(), group=group)


def _run(x, w, f32=False):
    from pegainfer_amd import ops
    y = torch.full((x.shape[0], w.out_dim), 7.0, device="cuda", dtype=torch.float32 if f32 else torch.bfloat16)
    ops.w4_gemm(w, x, y)
    torch.cuda.synchronize()
    return y


def _check(x, q, s, z, group, f32=False):
    y = _run(_bf(x), _pack(q, s, z, group), f32).double().cpu().numpy()
    want, mag = ref.w4_product(ref.bf16_values(x), q, ref.bf16_values(s), z, group)
    bound = ref.w4_bound(mag, x.shape[1], group, want, f32)
    bad = ~(np.abs(y - want) <= bound)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], y[bad][:4], want[bad][:4], bound[bad][:4])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,n,ksteps", [
    (1, 1, 1), (1, 16, 1), (1, 17, 3), (1, 250, 11), (2, 15, 2), (4, 64, 5), (5, 2051, 11), (8, 33, 9),
    (9, 129, 4), (15, 31, 7), (16, 48, 16), (17, 16, 8), (31, 100, 3), (33, 65, 5), (48, 200, 6),
    (64, 128, 9), (65, 70, 2), (100, 257, 5), (128, 256, 3), (129, 300, 7), (300, 513, 4)])
def test_product(rows, n, ksteps, group, zeros):
    _check(*_case(rows * 7 + n, rows, n, ksteps * group, group, zeros), group, f32=(rows + n) % 2 == 1)


@pytest.mark.parametrize("rows", [1, 3, 16, 40, 96, 200])
@pytest.mark.parametrize("k,group", [(7168, 32), (1408, 64), (1376, 32), (8192, 128)])
def test_long_rows(rows, k, group):
    _check(*_case(rows, rows, 96, k, group, rows % 2 == 0), group, f32=True)


@pytest.mark.parametrize("rows,n,k", [(1, 40, 256), (7, 40, 160), (50, 64, 96), (70, 130, 320), (150, 260, 128)])
def test_exact_integers(rows, n, k):
    """Small whole activations and scales that are powers of two: every sum is a whole number below
    2^24 steps, so the result is the formula's, bit for bit, whatever the order."""
    g = np.random.default_rng(k)
    xv = g.integers(-4, 5, (rows, k)).astype(np.float32)
    q = g.integers(0, 16, (n, k))
    s = ref.to_bf16_bits(np.float32(2.0) ** g.integers(-2, 3, (n, k // 32)))
    z = g.integers(0, 128, (n, k // 32)).astype(np.uint8)
    y = _run(_bf(ref.to_bf16_bits(xv)), _pack(q, s, z, 32), True).double().cpu().numpy()
    want, _ = ref.w4_product(xv, q, ref.bf16_values(s), z, 32)
    assert np.array_equal(y, want)


@pytest.mark.parametrize("rows", [3, 20, 70, 140])
def test_rows_that_are_not_finite_stay_apart(rows):
    x, q, s, z = _case(5, rows, 50, 256, 64, True)
    clean = _run(_bf(x), _pack(q, s, z, 64), True)
    bad = x.copy()
    bad[1, 7], bad[2, 200] = 0x7F80, 0x7FC0  # an infinity, a NaN
    y = _run(_bf(bad), _pack(q, s, z, 64), True)
    assert torch.isnan(y[1:3]).all()
    keep = [r for r in range(rows) if r not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("rows", [1, 16, 48, 130])
def test_repeats_and_writes_nothing_else(rows):
    from pegainfer_amd import ops
    x, q, s, z = _case(9, rows, 77, 384, 128, False)
    w, xd = _pack(q, s, z, 128), _bf(x)
    big = torch.full((rows * 77 + 64,), 3.0, device="cuda")
    out = big[32:32 + rows * 77].view(rows, 77)
    ops.w4_gemm(w, xd, out)
    first = out.clone()
    for _ in range(3):
        ops.w4_gemm(w, xd, out)
        assert torch.equal(out, first)
    assert (big[:32] == 3).all() and (big[32 + rows * 77:] == 3).all()
    odd = torch.full((rows * 77 + 3,), 3.0, device="cuda")  # a result that starts and ends anywhere
    part = odd[1:1 + rows * 77].view(rows, 77)
    ops.w4_gemm(w, xd, part)
    assert torch.equal(part, first) and odd[0] == 3 and (odd[-2:] == 3).all()
    ops.w4_gemm(w, xd[:0], out[:0])  # no rows: nothing to do


def test_row_does_not_depend_on_the_others():
    x, q, s, z = _case(4, 16, 90, 640, 32, True)
    w = _pack(q, s, z, 32)
    whole = _run(_bf(x), w, True)
    for r in (0, 5, 15):
        other = x.copy()
        other[[i for i in range(16) if i != r]] = x[::-1][:15]
        assert torch.equal(_run(_bf(other), w, True)[r], whole[r])


def test_codes_past_32_bit_offsets():
    """4.4 GB of codes: the last features, at offsets past 2^32, against their own small weight."""
    from pegainfer_amd import ops
    n, k, last = 1_200_016, 7168, 33
    packed = torch.full((n, k // 2), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.ones(n, k // 128, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    packed[-last:] = torch.randint(0, 256, (last, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    w = ops.w4_pack(packed, scales, group=128)
    small = ops.w4_pack(packed[-last:].contiguous(), scales[-last:].contiguous(), group=128)
    del packed
    for rows in (2, 20):
        x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
        y, z = _run(x, w, True), _run(x, small, True)
        # w4_bound with q = z = 8 and s = 1, where the formula gives 0 (other features' codes give about
        # 4.6 sqrt(k) = 390); both sides are within it
        off = (2 * 128 + k // 128 + 18) * 2.0 ** -23 * 48 * x.float().abs().sum(1, keepdim=True)
        assert off.max() < 20
        assert (y[:, :-last].abs() <= off).all() and ((y[:, -last:] - z).abs() <= 2 * off).all()
        assert z.abs().max() > 200
        del y


@pytest.mark.parametrize("n", [65536])
def test_results_past_32_bit_offsets(n):
    rows, k = 36000, 32
    x, q, s, z = _case(2, 300, n, k, 32, False)
    w = _pack(q, s, z, 32)
    xd = _bf(x).repeat(rows // 300, 1).contiguous()
    y = _run(xd, w, True)
    part = _run(_bf(x), w, True)
    for at in (0, 300 * 50, rows - 300):
        assert torch.allclose(y[at:at + 300], part, rtol=0, atol=1e-4)


def test_captured_on_another_stream():
    from pegainfer_amd import ops
    x, q, s, z = _case(3, 24, 160, 512, 64, True)
    w, xd = _pack(q, s, z, 64), _bf(x)
    y = torch.zeros(24, 160, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.w4_gemm(w, xd, y)
    for i in range(4):
        xd.copy_(xd.roll(1, 0))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(xd, w, True)
        assert torch.equal(y, eager)


# sizes that take each form of the kernels (five streaming ones, then tiles from narrow to wide), with an odd
# number of features and, where the group allows it, a last step that is not whole
FORMS = {
    32: [(1, 2051, 7136), (1, 1000, 448), (3, 33001, 448), (17, 12003, 448), (40, 20011, 1376), (130, 33001, 1376),
         (1500, 4083, 448), (420, 8200, 448), (600, 12003, 1376)],
    64: [(1, 2051, 7104), (1, 1000, 448), (3, 33001, 448), (17, 12003, 448), (40, 20011, 1344), (40, 33001, 448),
         (900, 2051, 1344), (3000, 1000, 448), (600, 12003, 448), (300, 20011, 1344)],
    128: [(1, 2051, 7168), (1, 1000, 384), (1, 33001, 1408), (17, 12003, 384), (40, 20011, 1408), (40, 33001, 384),
          (1500, 4083, 384), (3000, 1000, 384), (768, 5001, 7168), (600, 33001, 384)],
}


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,rows,n,k", [(g, *c) for g, cs in FORMS.items() for c in cs])
def test_every_form(group, rows, n, k, zeros):
    """The reference in float64 on the GPU, features in blocks."""
    from pegainfer_amd import ops
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    s = (torch.randn(n, k // group, device="cuda", generator=g) * 0.01).to(torch.bfloat16)
    z = torch.randint(0, 17, (n, k // group), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    y = _run(x, ops.w4_pack(packed, s, z, group=group), True)
    q = torch.stack((packed & 15, packed >> 4), -1).reshape(n, k).double()
    zr = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    sr = s.double().repeat_interleave(group, 1)
    for at in range(0, n, 4096):
        part = slice(at, at + 4096)
        qp, zp = q[part], zr if z is None else zr[part]
        want = x.double() @ ((qp - zp) * sr[part]).T
        mag = x.double().abs() @ ((32 + qp + zp) * sr[part].abs()).T
        bound = (2 * group + k // group + 18) * 2.0 ** -23 * mag + want.abs() * 2.0 ** -24  # w4_bound
        bad = (y[:, part].double() - want).abs() > bound
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())
        # and far inside it for most: a wrong scale, code or row would not be
        assert ((y[:, part].double() - want).abs() <= 1e-5 * mag).float().mean() > 0.999


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,rows,n,k", [(g, *c) for g, cs in FORMS.items() for c in cs])
def test_every_form_bit_for_bit(group, rows, n, k, zeros):
    """Whole activations up to 3, scales of 2^-20 to 2^-18: in units of the smallest scale every sum of a row is a
    whole number below 3 * 127 * 4 * 7168 < 2^24, so the result is exact in any order.  Then the same with the
    activations just below the largest that rows of finite values may have: 3 * 2^115 < 2^117 with zero points up
    to 127, 3 * 2^117 < 2^119 without.  The first row has the largest value everywhere."""
    from pegainfer_amd import ops
    assert 3 * 127 * 4 * k < 2 ** 24
    g = torch.Generator(device="cuda").manual_seed(rows * 3 + n)
    x = torch.randint(-3, 4, (rows, k), device="cuda", generator=g).to(torch.bfloat16)
    x[0] = 3
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.exp2(torch.randint(-20, -17, (n, k // group), device="cuda", generator=g).float()).to(torch.bfloat16)
    z = torch.randint(0, 128, (n, k // group), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    if zeros:
        z[0], z[-1] = 127, 127
    w = ops.w4_pack(packed, s, z, group=group)
    up = 2.0 ** (115 if zeros else 117)
    y, high = _run(x, w, True), _run(x * up, w, True)
    q = torch.stack((packed & 15, packed >> 4), -1).reshape(n, k).double()
    zr = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    sr = s.double().repeat_interleave(group, 1)
    for at in range(0, n, 4096):
        part = slice(at, at + 4096)
        want = x.double() @ ((q[part] - (zr if z is None else zr[part])) * sr[part]).T
        assert torch.equal(y[:, part].double(), want)
        assert torch.equal(high[:, part].double(), want * up)
