"""The 4-bit key/value cache where its arithmetic and its arguments are at their edges."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ipex():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import ipex_b200

    ipex_b200.load_ops()
    yield ipex_b200
    torch.ops.torch_ipex.woq_check_status()


def cache_of(num_pages, heads, d, page, group, t):
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    return _IPEXPagedKv4Cache(num_pages, heads, d, page, group, t)


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def stored(c, x):
    """What the cache holds after x [tokens, 1, D] was appended as keys and as values."""
    slots = torch.arange(x.shape[0], device="cuda")
    c.append(x.cuda(), x.cuda(), slots)
    k, v = c.read(slots)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    return k.cpu().double()


@pytest.mark.parametrize("t, power", [(BF, -133), (BF, -131), (BF, -129), (BF, -127), (BF, -125), (BF, -120), (FP, -24), (FP, -20)])
def test_steps_with_no_reciprocal(ipex, t, power):
    """Groups whose step is so small that its reciprocal passes the largest fp32 number (bf16 below 2^-127)."""
    c = cache_of(2, 1, 64, 16, 32, t)
    x = (torch.randint(0, 256, (20, 1, 64), generator=torch.Generator().manual_seed(1)).double() * 2.0 ** power).to(t)
    x[:, :, 0] = 0  # (the lowest element of a group has code 0)
    assert torch.equal(stored(c, x), R.quantise(x, 32)[0])


def digits(x, bits, how):
    """A Fraction of normal size to a number of `bits` digits: toward zero (math.floor) or to the nearest, even (round)."""
    if x == 0:
        return x
    e = math.frexp(float(abs(x)))[1]  # (of the number rounded to 64 bits: one too large just below a power of two)
    e -= abs(x) < Fraction(2) ** (e - 1)
    unit = Fraction(2) ** (e - bits)
    return how(abs(x) / unit) * unit * (1 if x > 0 else -1)


def quantised_exactly(row, t):
    """One group in rational numbers: 64 bits do not hold the difference of a large and a tiny number."""
    bits = 8 if t == BF else 11
    x = [Fraction(float(v)) for v in row]
    lo, hi = min(x), max(x)
    s = digits((hi - lo) / 15, bits, math.floor)
    return [digits(min(round((v - lo) / s), 15) * s + lo, bits, round) for v in x], s


@pytest.mark.parametrize("t, low", [(BF, 2.0 ** -30), (BF, 2.0 ** -100), (FP, 2.0 ** -24), (BF, -2.0 ** -30), (FP, -2.0 ** -23)])
def test_the_step_is_rounded_toward_zero_once(ipex, t, low):
    """max - min just below (or above) 15 numbers of the type: 32 bits round it to all 15, the step is the number below."""
    c = cache_of(1, 1, 64, 16, 64, t)
    x = torch.zeros(6, 1, 64)
    for i, top in enumerate((15.0, 7.5, 60.0, 30.0, 3.75, 120.0)):
        x[i] = top * torch.linspace(0, 1, 64)
        x[i, 0, 63], x[i, 0, 0] = top, low
        x[i, 0, 1] = low
    x = x.to(t)
    got = stored(c, x)[:, 0].tolist()
    for row, have in zip(x[:, 0], got):
        want, s = quantised_exactly(row, t)
        assert have[0] == want[0] == low and have[63] == want[63]
        # codes of the others may lie on a border of two: a step apart at most there
        assert all(abs(Fraction(h) - w) <= s for h, w in zip(have, want))


@pytest.mark.parametrize("batch, heads, new, length", [(1, 4, 1, 60000), (300, 4, 1, 1000), (160, 2, 6, 1000), (1, 4, 70, 30000),
                                                       (80, 4, 70, 1000)])
@pytest.mark.parametrize("t", [BF, FP])
def test_many_small_weights_beside_a_large_one(ipex, t, batch, heads, new, length):
    """One key far above up to tens of thousands of others, each of 2^-25 of its weight: together they are the result, since the
    large one's value is zero.  All sequences read the same pages; more of them leave more of the keys to one CTA."""
    c = cache_of(-(-length // 64), 1, 64, 64, 64, t)
    k, v = torch.zeros(length, 1, 64), 0.5 + torch.rand(length, 1, 64, generator=torch.Generator().manual_seed(2))
    k[0, 0, 0], v[0] = 17.5, 0.0
    k, v = k.to(t), v.to(t)
    c.append(k.cuda(), v.cuda(), torch.arange(length, device="cuda"))
    q = torch.zeros(batch * new, heads, 64)
    q[..., 0] = 1.0
    q = q.to(t)
    table = torch.arange(c.num_pages, device="cuda").int().repeat(batch, 1)
    starts = None if new == 1 else (torch.arange(batch + 1) * new).int().cuda()
    lens = torch.full((batch,), length).int().cuda()
    got = c.attention(q.cuda(), table, lens, starts, scale=1.0).cpu().double().unflatten(0, (batch, new))
    want, tol = R.attend(q[:new].double(), R.quantise(k, 64)[0], R.quantise(v, 64)[0], 1.0, True)
    assert want.abs().min() > 2.0 ** -17
    assert ((got - want).abs() <= tol(R.EPS[t])).all()


def test_a_wait_that_gave_up_is_reported_before_a_missing_page(ipex):
    """Kernels record a wait that they gave up with a compare-and-swap on the first word of the workspace: a page that the
    cache does not have, met before, must not stand in its way."""
    from ipex_b200 import _capi

    L = _capi.lib()
    c = cache_of(4, 1, 64, 16, 64, BF)
    x = randn(1, 16, 1, 64).to(BF).cuda()
    c.append(x, x, torch.arange(16, device="cuda"))
    d = _capi.Kv4Desc(4, 1, 64, 16, 64, _capi.T_BF16)
    for new in (1, 80):  # both kernels
        ws = torch.zeros(L.woq_b200_kv4_attention_workspace_bytes(ctypes.byref(d), 1, new, 4), dtype=torch.uint8, device="cuda")
        q, out = randn(2, new, 4, 64).to(BF).cuda(), torch.zeros(new, 4, 64, dtype=BF, device="cuda")
        table, lens, starts = torch.tensor([[0, 9]]).int().cuda(), torch.tensor([32]).int().cuda(), torch.tensor([0, new]).int().cuda()
        stream = torch.cuda.current_stream().cuda_stream

        def call():
            assert L.woq_b200_kv4_attention(ctypes.byref(d), c.tensor.data_ptr(), q.data_ptr(), 256, 64, 4, table.data_ptr(), 2, 2,
                                            lens.data_ptr(), starts.data_ptr(), 1, new, 0.125, 0, out.data_ptr(), 256, 64,
                                            ws.data_ptr(), ws.numel(), stream) == 0

        call()
        assert L.woq_b200_workspace_status(ws.data_ptr(), stream) == 1 and b"page" in L.woq_b200_last_error()
        assert L.woq_b200_workspace_status(ws.data_ptr(), stream) == 0 and not ws[:L.woq_b200_workspace_header_bytes()].any()
        call()
        first = ws[:4].view(torch.int32)
        first.copy_(torch.where(first == 0, 910, first))  # what a kernel that gives up does
        assert L.woq_b200_workspace_status(ws.data_ptr(), stream) == 6 and b"910" in L.woq_b200_last_error()
        assert b"page" in L.woq_b200_last_error()
        assert L.woq_b200_workspace_status(ws.data_ptr(), stream) == 0 and not ws[:L.woq_b200_workspace_header_bytes()].any()


def test_numbers_of_64_bits_do_not_wrap(ipex):
    """int64 tables, lengths and starts: a page of 2^32 + 1 is none that the cache has, a length of 2^32 + 5 is cut to the
    table, negative ones stay negative."""
    c = cache_of(4, 1, 64, 16, 64, BF)
    x = randn(1, 64, 1, 64).to(BF)
    c.append(x.cuda(), x.cuda(), torch.arange(64, device="cuda"))
    kv = R.quantise(x, 64)[0]
    q = randn(2, 3, 4, 64).to(BF)
    table = torch.tensor([[0, (1 << 32) + 1, 2], [3, 2, -(1 << 32)], [1, 0, 1 << 62]]).cuda()
    lens = torch.tensor([48, (1 << 32) + 5, 5 - (1 << 40)]).cuda()
    torch.ops.torch_ipex.woq_check_status()
    for starts, rows in ((None, [1, 1, 1]), (torch.tensor([-(1 << 33), 2, 3, (1 << 32) + 2]).cuda(), [2, 1, 0])):
        got = c.attention(q.cuda(), table, lens, starts, causal=False).cpu().double()
        with pytest.raises(RuntimeError, match="page"):
            torch.ops.torch_ipex.woq_check_status()
        row = 0
        for n, keys in zip(rows, (list(range(16)) + list(range(32, 48)), list(range(48, 64)) + list(range(32, 48)), [])):
            want, tol = R.attend(q[row:row + n].double(), kv[keys], kv[keys], 0.125, False)
            assert ((got[row:row + n] - want).abs() <= tol(R.EPS[BF])).all()
            row += n
    torch.ops.torch_ipex.woq_check_status()


@pytest.mark.parametrize("d, heads, kv_heads", [(64, 4, 8), (128, 4, 8), (256, 2, 4), (128, 1, 160), (64, 64, 1)])
def test_a_workspace_serves_every_smaller_call(ipex, d, heads, kv_heads):
    """Its size does not shrink with the sequences or the rows: a program makes one for its largest call."""
    from ipex_b200 import _capi

    L = _capi.lib()
    desc = _capi.Kv4Desc(64, kv_heads, d, 16, 32, _capi.T_BF16)

    def size(batch, tokens):
        return L.woq_b200_kv4_attention_workspace_bytes(ctypes.byref(desc), batch, tokens, heads * kv_heads)

    counts = [1, 2, 3, 5, 8, 9, 16, 17, 31, 33, 40, 64, 65, 100, 127, 128, 129, 255, 300, 1000, 4097, 20000]
    for batch in (1, 2, 4, 7, 32, 100, 600):
        sizes = [size(batch, n) for n in counts]
        assert sizes == sorted(sizes), (batch, sizes)
    for n in counts:
        sizes = [size(batch, n) for batch in (1, 2, 4, 7, 32, 100, 600)]
        assert sizes == sorted(sizes), (n, sizes)
    # and the smaller calls are taken
    ws = torch.zeros(size(4, 4000), dtype=torch.uint8, device="cuda")
    cache = torch.zeros(L.woq_b200_kv4_bytes(ctypes.byref(desc)), dtype=torch.uint8, device="cuda")
    for batch, n in ((1, 1), (4, 4), (3, 30), (1, 100), (4, 100), (1, 400), (4, 4000)):
        q = torch.zeros(n, heads * kv_heads, d, dtype=BF, device="cuda")
        out = torch.ones_like(q)
        starts = (torch.arange(batch + 1, device="cuda") * (n // batch)).int()
        table, lens = torch.arange(4, device="cuda").int().repeat(batch, 1), torch.full((batch,), 64, device="cuda").int()
        rc = L.woq_b200_kv4_attention(ctypes.byref(desc), cache.data_ptr(), q.data_ptr(), q.stride(0), d, heads * kv_heads,
                                      table.data_ptr(), 4, 4, lens.data_ptr(), starts.data_ptr(), batch, n, 0.1, 0, out.data_ptr(),
                                      q.stride(0), d, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0, (batch, n, L.woq_b200_last_error())
        torch.cuda.synchronize()
        assert (out[:batch * (n // batch)] == 0).all()
        assert L.woq_b200_workspace_status(ws.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
