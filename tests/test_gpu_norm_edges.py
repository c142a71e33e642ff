"""Codes of the residual's addition with RMS norm where the arithmetic is at its edges, exactly as the definition says.

With every x + r equal to a power of two and eps = 0, the mean of the squares, its root and the normalised row are exact:
y is the norm's weight, whatever it is.  Scale, zero point and codes then follow from 32-bit divisions alone."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import ipex_b200

    ipex_b200.load_ops()
    return torch.ops.torch_ipex


def quotient(a, b):
    """a / b of fp32 numbers in fp32: 53 digits are more than twice 24 and two, so that rounding twice is rounding once."""
    return (a.double() / b.double()).float()


def definition(y, asym):
    """y bf16 [k] (CPU) -> scale, zero point, codes, in 32-bit arithmetic."""
    y = y.float()
    if not asym:
        s = quotient(y.abs().max(), torch.tensor(127.0))
        return s, 0, quotient(y, s).round().clamp(-128, 127).int()
    s = quotient(y.max() - y.min(), torch.tensor(255.0))
    z = -quotient(y.min(), s).round()
    return s, int(z), (quotient(y, s) + z).round().clamp(0, 255).int()


def run(ops, y, asym, base=1.0, rows=1):
    """The operator on rows whose normalised values are y."""
    k = y.numel()
    x = torch.full((rows, k), base / 2, device="cuda").bfloat16()
    h, qa, sa, zpa = ops.woq_add_rmsnorm_quant(x, x, y.cuda(), 0.0, 2 if asym else 6)
    assert (h == base).all()
    codes = qa.view(torch.uint8) if asym else qa
    return sa.cpu(), zpa.cpu(), codes.cpu().int()


def check(ops, y, asym, base=1.0, rows=1):
    sa, zpa, codes = run(ops, y, asym, base, rows)
    s, z, c = definition(y, asym)
    assert (sa == s).all() and (not asym or (zpa == z).all())
    assert torch.equal(codes, c.expand(rows, -1))


@pytest.mark.parametrize("rows, k", [(1, 64), (1, 8192), (150, 14336), (1, 16400), (3, 4112)])
@pytest.mark.parametrize("low, sign", [(0.0, 1), (1.0, 1), (4.0, 1), (4.0, -1), (16.0, -1), (64.0, 1), (64.0, -1), (100.0, 1)])
def test_rows_on_one_side(ops, rows, k, low, sign):
    """Quotients of up to 2^15 before the zero point is added: neighbours in bf16 lie up to 255 codes apart, and many halfway
    between two codes."""
    gen = torch.Generator().manual_seed(int(low) + k)
    for _ in range(4 if k > 64 else 60):
        check(ops, (sign * (low + torch.rand(k, generator=gen))).bfloat16(), True, rows=rows)


@pytest.mark.parametrize("asym", [False, True])
def test_ties(ops, asym):
    """Values at and next to every half code."""
    for top in (127.0, 127.5, 254.0, 255.0, 63.5):
        y = torch.arange(0, 256, 1).float() * 0.5 * (top / 127.5)
        y = torch.cat((y, -y if not asym else y + 1.0, torch.tensor([top] + [0.0] * 15))).bfloat16()
        check(ops, y, asym)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("power", [-133, -132, -130, -128, -126, -124, -120, -110])
def test_scales_with_no_reciprocal(ops, asym, power):
    """Rows whose largest value is so small that the scale's reciprocal passes the largest fp32 number."""
    gen = torch.Generator().manual_seed(-power)
    for spread in (1, 3, 100, 255):
        y = (torch.randint(-spread, spread + 1, (64,), generator=gen).double() * 2.0 ** power).bfloat16()
        check(ops, y, asym)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows, k", [(1, 64), (1, 8192), (150, 14336), (2, 16400)])
def test_weights_that_are_not_finite(ops, asym, bad, rows, k):
    """A y that is not finite makes the row's scale NaN, wherever it stands."""
    for at in (0, k // 2, k - 1):
        y = torch.linspace(-1, 1, k).bfloat16()
        y[at] = bad
        assert run(ops, y, asym, rows=rows)[0].isnan().all()


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("base, weight", [(2.0 ** 60, 2.0 ** 70), (2.0 ** -40, 2.0 ** -100)])
def test_products_out_of_range_on_the_way(ops, asym, base, weight):
    """y is in range though the sum times the weight, without the norm's factor, is not."""
    gen = torch.Generator().manual_seed(3)
    check(ops, (torch.randn(64, generator=gen) * weight).bfloat16(), asym, base)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("low", [-1.0, 0.0, 3.0])
def test_the_same_as_without_a_residual(ops, asym, low):
    """Where the sums of squares are exact in any order, the operator and woq_rmsnorm_quant on the sum agree in every bit."""
    gen = torch.Generator().manual_seed(4)
    for k in (64, 2048, 4096):
        x = torch.randint(-8, 9, (20, k), generator=gen).bfloat16().cuda()  # sums of squares below 2^24
        r = torch.randint(-8, 9, (20, k), generator=gen).bfloat16().cuda()
        g = (low + 2 * torch.rand(k, generator=gen)).bfloat16().cuda()
        mode = 2 if asym else 6
        h, qa, sa, zpa = ops.woq_add_rmsnorm_quant(x, r, g, 1e-5, mode)
        qb, sb, zpb = ops.woq_rmsnorm_quant(h, g, 1e-5, mode)
        # (the roots may differ in their last place: rows where they do have scales that do)
        same = sa == sb
        assert torch.equal(qa[same], qb[same])
        assert not asym or torch.equal(zpa[same], zpb[same])
        assert same.float().mean() > 0.9


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("rows, k", [(1, 64), (1, 8192), (40, 8192), (150, 14336), (2, 16400), (300, 4096)])
def test_the_sum_in_the_place_of_an_operand(ops, rows, k, asym):
    """The C entry writes the sum over x or over r, rows of any distance apart."""
    from ipex_b200 import _capi

    gen = torch.Generator().manual_seed(5)
    x, r = (torch.randn(rows, k + 24, generator=gen).bfloat16().cuda() for _ in range(2))
    g = torch.rand(k, generator=gen).bfloat16().cuda()
    h, qa, sa, zpa = ops.woq_add_rmsnorm_quant(x[:, :k].contiguous(), r[:, :k].contiguous(), g, 1e-5, 2 if asym else 6)
    for over in (0, 1):
        a = [x.clone(), r.clone()]
        behind = a[over][:, k:].clone()
        codes, scales, zeros = torch.zeros_like(qa), torch.zeros_like(sa), torch.zeros(rows, dtype=torch.int32, device="cuda")
        assert _capi.lib().woq_b200_add_rmsnorm_quant(a[0].data_ptr(), k + 24, a[1].data_ptr(), k + 24, g.data_ptr(), 1e-5, rows, k,
                                                      2 if asym else 6, a[over].data_ptr(), k + 24, codes.data_ptr(), scales.data_ptr(),
                                                      zeros.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(a[over][:, :k], h) and torch.equal(codes, qa) and torch.equal(scales, sa)
        assert not asym or torch.equal(zeros, zpa)
        assert torch.equal(a[over][:, k:], behind) and torch.equal(a[1 - over], (x, r)[1 - over])
