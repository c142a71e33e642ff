"""Appending to the paged 4-bit cache, reading it back and attention over it, against plain 64-bit implementations."""
import math

import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.fixture(scope="module")
def ipex():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import ipex_b200

    ipex_b200.load_ops()
    yield ipex_b200
    torch.ops.torch_ipex.woq_check_status()


def cache_of(num_pages, heads, d, page, group, t, fill=0):
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    c = _IPEXPagedKv4Cache(num_pages, heads, d, page, group, t)
    c.tensor.fill_(fill)
    return c


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ---- append and read ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, group", SHAPES)
def test_values_without_a_rotation_are_exact(ipex, t, d, group):
    """Keys and values as slices of one projection, slots in any order, some for padding or outside the cache: what is
    read back is what the definition gives, bit for bit, and no other slot changes."""
    n, hq, hk, page, pages = 37, 3, 3, 32, 5
    qkv = randn(1, n, (hq + 2 * hk) * d).to(t)
    qkv[3] = 0.5           # a constant row: scale 0
    qkv[4, : hq * d + 7] *= 100
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(2))[:n]
    slots[5], slots[11], slots[12] = -1, pages * page, 1 << 40
    q, k, v = qkv.cuda().view(n, -1, d).split([hq, hk, hk], 1)
    c = cache_of(pages, hk, d, page, group, t, fill=0x35)
    before = c.read(torch.arange(pages * page, device="cuda"))
    assert c.append(k, v, slots.cuda()) is None
    kk, vv = c.read(slots.cuda())
    live = [i for i in range(n) if i not in (5, 11, 12)]
    for got, x in ((kk, k), (vv, v)):
        assert torch.equal(got.cpu().double()[live], R.quantise(x.cpu(), group)[0][live])
        assert (got[[5, 11, 12]] == 0).all()
    others = torch.ones(pages * page, dtype=torch.bool)
    others[slots[live]] = False
    after = c.read(torch.arange(pages * page, device="cuda"))
    for a, b in zip(after, before):
        assert torch.equal(a.cpu().view(torch.int16)[others], b.cpu().view(torch.int16)[others])
    # int32 slots, and appending again: the same
    c.append(k, v, slots.clamp(-1, 10 ** 6).int().cuda())
    assert torch.equal(c.read(slots.cuda())[0], kk)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, rot, interleaved, tokens, hq, hk", [
    (64, 64, False, 1, 4, 1), (64, 16, True, 50, 5, 5), (128, 128, False, 300, 32, 8), (128, 32, False, 7, 3, 1),
    (128, 128, True, 9, 8, 2), (256, 256, False, 5, 4, 2), (256, 64, True, 33, 2, 1), (256, 160, False, 3, 1, 1)])
def test_rotation_on_the_way(ipex, t, d, rot, interleaved, tokens, hq, hk):
    """Queries: one rounding of the rotated ones (half a step), on top of 32-bit arithmetic that is off by at most two
    units of 2^-24 of the result.  Keys: within half a quantisation step of the rotated ones, where the step comes from
    keys that are rounded to T first."""
    q, k, v = randn(3, tokens, hq, d).to(t), (3 * randn(4, tokens, hk, d)).to(t), randn(5, tokens, hk, d).to(t)
    pos = torch.randint(0, 9000, (tokens,), generator=torch.Generator().manual_seed(6))
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    table = _IPEXPagedKv4Cache.rotary_table(9000, rot, 5e5)
    c = cache_of(3 + tokens // 16, hk, d, 16, 32, t)
    slots = torch.arange(tokens, device="cuda")
    got = c.append(k.cuda(), v.cuda(), slots, q.cuda(), pos.cuda(), table, interleaved)
    want = R.rotate(q, pos, table.cpu(), interleaved)
    eps = R.EPS[t]
    tiny = 2.0 ** -25  # half the smallest fp16 number
    assert ((got.cpu().double() - want).abs() <= want.abs() * (eps / 2 + 2.0 ** -22) + tiny).all()
    kk, vv = (x.cpu().double() for x in c.read(slots))
    assert torch.equal(vv, R.quantise(v, 32)[0])
    exact = R.rotate(k, pos, table.cpu(), interleaved)
    step = R.quantise(exact.to(t), 32)[1].repeat_interleave(32, -1)
    # half a step; a key on a rounding border may be rounded either way: one step of T on it and on both ends of the
    # range; 15 scales too small by eps each; the value's own rounding
    slack = step * (0.5 + 15 * eps) * (1 + eps) + 3 * eps * exact.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
    assert ((kk - exact).abs() <= slack + kk.abs() * eps / 2).all()


def test_positions_outside_the_table(ipex):
    """They store nothing and make the query NaN; padding (slot -1) with a good position still rotates its query."""
    c = cache_of(2, 2, 64, 16, 32, BF, fill=0x11)
    before = c.tensor.clone()
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    table = _IPEXPagedKv4Cache.rotary_table(10, 64)
    x = randn(1, 4, 2, 64).to(BF).cuda()
    q = c.append(x, x, torch.tensor([0, 1, 2, -1]).cuda(), x, torch.tensor([-1, 10, 1 << 40, 3]).cuda(), table)
    assert q[:3].isnan().all() and torch.equal(c.tensor, before)
    want = R.rotate(x[3:].cpu(), torch.tensor([3]), table.cpu(), False)
    assert ((q[3:].cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all()


@pytest.mark.parametrize("t", [BF, FP])
def test_values_that_are_not_finite(ipex, t):
    """The key says it, so that rows that do not see the token are not touched; extreme finite values stay finite, and
    come through attention: bf16 ones below 2^61, beyond which they count as not finite."""
    d, top = 128, 2.0 ** 60.5 if t == BF else torch.finfo(t).max
    k, v = randn(1, 5, 1, d).to(t), randn(2, 5, 1, d).to(t)
    k[0, 0, 3], v[1, 0, 100], k[2, 0, 0] = math.nan, math.inf, -math.inf
    k[3, 0, 0], k[3, 0, 1], v[3, 0, 64], v[3, 0, 65] = top, -top, -top, top
    v[4, 0, :] = top
    c = cache_of(1, 1, d, 16, 64, t)
    c.append(k.cuda(), v.cuda(), torch.arange(5).cuda())
    kk, vv = (x.cpu() for x in c.read(torch.arange(5).cuda()))
    assert kk[[0, 1, 2]].isnan().all() and (vv[1] == 0).all()
    assert torch.equal(vv[[0, 2]].double(), R.quantise(v[[0, 2]], 64)[0])
    assert torch.equal(kk[[3, 4]].double(), R.quantise(k[[3, 4]], 64)[0]) and kk[3].isfinite().all()
    assert torch.equal(vv[[3, 4]].double(), R.quantise(v[[3, 4]], 64)[0]) and vv[3:].isfinite().all()
    if t == BF:
        k3 = randn(5, 2, 1, d).to(t)
        k3[1, 0, 9] = 2.0 ** 61
        c.append(k3.cuda(), k3.flip(0).cuda(), torch.arange(5, 7).cuda())
        kk, vv = (x.cpu() for x in c.read(torch.arange(5, 7).cuda()))
        assert kk.isnan().all() and (vv[0] == 0).all() and torch.equal(vv[1].double(), R.quantise(k3[:1], 64)[0][0])
    # the extreme values: one key each, so that the output is the value
    for i in (3, 4):
        table = torch.zeros(1, 1).int().cuda()
        c.append(torch.zeros(1, 1, d, dtype=t, device="cuda"), v[i:i + 1].cuda(), torch.zeros(1).long().cuda())
        o = c.attention(torch.ones(1, 2, d, dtype=t, device="cuda"), table, torch.tensor([1]).int().cuda())
        want = R.quantise(v[i:i + 1], 64)[0]
        assert ((o.cpu().double() - want).abs() <= want.abs() * 2.0 ** -20).all()
    # queries of 2 tokens: the first does not see token 4 (made NaN), the second does
    k2 = randn(3, 5, 1, d).to(t)
    v2 = k2.clone()
    v2[4, 0, 0] = math.nan
    c.append(k2.cuda(), v2.cuda(), torch.arange(5).cuda())
    q = randn(4, 2, 1, d).to(t).cuda()
    o = c.attention(q, torch.zeros(1, 1).int().cuda(), torch.tensor([5]).int().cuda(), torch.tensor([0, 2]).int().cuda())
    assert o[0].isfinite().all() and o[1].isnan().all()


# ---- attention ---------------------------------------------------------------------------------------------------
def fill(c, lens, seed, wide=1.0):
    """Appends sum(lens) tokens over shuffled pages.  Returns per sequence (k, v) in 64 bits, and the block table, whose
    unused entries name no page."""
    page = c.page_size
    need = [-(-n // page) for n in lens]
    order = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
    slots, at = [], 0
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
        slots += [pages[i // page] * page + i % page for i in range(n)]
    total = sum(lens)
    k = (wide * randn(seed + 1, total, c.kv_heads, c.head_dim)).to(c.dtype)
    v = randn(seed + 2, total, c.kv_heads, c.head_dim).to(c.dtype)
    if total:
        c.append(k.cuda(), v.cuda(), torch.tensor(slots).cuda())
    kq, vq = R.quantise(k, c.group_size)[0], R.quantise(v, c.group_size)[0]
    return list(zip(kq.split(lens), vq.split(lens))), table.cuda()


def check(c, lens, new, heads, seed, causal=True, scale=None, wide=1.0, starts=True, q=None):
    """Attention of new[b] query rows a sequence against the plain one."""
    kv, table = fill(c, lens, seed, wide)
    hq = heads * c.kv_heads
    q = randn(seed + 3, sum(new), hq, c.head_dim).to(c.dtype) if q is None else q
    at = torch.tensor([0] + new).cumsum(0).int().cuda() if starts else None
    got = c.attention(q.cuda(), table, torch.tensor(lens).int().cuda(), at, scale, causal)
    compare(got, q, kv, new, c, causal, scale)
    return got, table, q


def compare(got, q, kv, new, c, causal, scale=None):
    got = got.cpu().double()
    row = 0
    for (k, v), n in zip(kv, new):
        want, tol = R.attend(q[row:row + n].double(), k, v, scale if scale is not None else c.head_dim ** -0.5, causal)
        off = (got[row:row + n] - want).abs() - tol(R.EPS[c.dtype])
        assert n == 0 or off.max() <= 0, (k.shape[0], n, float(off.max()))
        row += n


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, group", SHAPES)
def test_one_token_a_sequence(ipex, t, d, group):
    """Lengths around the blocks and pages, among them none; unused slots and pages hold NaN parameters."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 200, 481]
    c = cache_of(80, 2, d, 32, group, t, fill=0xff)
    got, _, _ = check(c, lens, [1] * len(lens), 4, 10, starts=False)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("heads", [1, 2, 3, 5, 7, 8, 9, 12, 16, 20, 32, 40])
def test_query_heads_of_a_kv_head(ipex, heads):
    c = cache_of(30, 3, 128, 16, 64, BF, fill=0xff)
    check(c, [100, 7, 33], [1, 1, 1], heads, 20, starts=False)


@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_page_sizes(ipex, page):
    c = cache_of(40, 2, 64, page, 32, FP, fill=0xff)
    check(c, [300, 1, 255, 64], [1] * 4, 4, 30, starts=False)


@pytest.mark.parametrize("lens", [[20000], [5000, 3, 9000, 1], [1] * 333, [17, 40] * 50, [0] * 5 + [4097]])
@pytest.mark.parametrize("d, kv_heads", [(64, 1), (128, 2)])
def test_shares_of_long_and_many_sequences(ipex, lens, d, kv_heads):
    """One sequence over every CTA, many sequences a CTA, and both."""
    pages = sum(-(-n // 32) for n in lens) + 1
    c = cache_of(pages, kv_heads, d, 32, 32, BF, fill=0xff)
    check(c, lens, [1] * len(lens), 4, 40, starts=False)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, heads, causal", [(64, 1, True), (64, 4, False), (128, 4, True), (128, 3, True), (128, 8, False),
                                              (256, 2, True), (256, 8, True)])
def test_several_tokens_a_sequence(ipex, t, d, heads, causal):
    """Rows of a sequence over several tiles; sequences without queries; more queries than tokens (rows that see nothing)."""
    lens, new = [40, 7, 100, 5, 0, 333, 16], [3, 7, 1, 0, 2, 17, 20]
    c = cache_of(60, 2, d, 16, 32, t, fill=0xff)
    got, _, _ = check(c, lens, new, heads, 50, causal=causal)
    assert (got[11:13] == 0).all()
    if causal:
        assert (got[30:34] == 0).all() and (got[34:].abs().sum((1, 2)) > 0).all()


@pytest.mark.parametrize("d, heads, group, t, lens, new", [
    (128, 4, 64, BF, [512], [512]), (128, 8, 32, FP, [300, 129, 64], [300, 65, 64]), (64, 3, 64, BF, [777], [500]),
    (256, 2, 128, BF, [200, 90], [200, 90]), (128, 1, 128, BF, [1000], [257]), (64, 16, 32, FP, [65], [33])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(ipex, d, heads, group, t, lens, new, causal):
    c = cache_of(80, 2, d, 64, group, t, fill=0xff)
    check(c, lens, new, heads, 60, causal=causal)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, heads, lens, new", [
    (128, 4, [5000, 700], [70, 33]), (64, 8, [3001], [64]), (256, 2, [2000, 40], [100, 1]), (128, 16, [900, 0, 1500], [5, 6, 20]),
    (128, 4, [2500], [2500])])
def test_short_prompts_behind_long_prefixes(ipex, t, d, heads, lens, new):
    """Several CTAs share a tile of rows: parts that see nothing of a tile, a tile without rows, and the same bits again."""
    c = cache_of(200, 1, d, 64, 32, t, fill=0xff)
    got, table, q = check(c, lens, new, heads, 65)
    starts = torch.tensor([0] + new).cumsum(0).int().cuda()
    for _ in range(5):
        assert torch.equal(c.attention(q.cuda(), table, torch.tensor(lens).int().cuda(), starts), got)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, heads, new, length", [(128, 8, 1, 30000), (64, 1, 1, 26000), (256, 3, 2, 30001), (64, 16, 2, 20000)])
def test_one_sequence_for_all(ipex, t, d, heads, new, length):
    """One kv head of one sequence, so that as many CTAs share an item as may; the same bits again."""
    c = cache_of(480, 1, d, 64, 32, t)
    got, table, q = check(c, [length], [new], heads, 67)
    starts = torch.tensor([0, new]).int().cuda()
    for _ in range(5):
        assert torch.equal(c.attention(q.cuda(), table, torch.tensor([length]).int().cuda(), starts), got)


@pytest.mark.parametrize("new", [1, 5, 70])
def test_values_that_are_not_finite_in_a_shared_item(ipex, new):
    """A token of the new ones that holds a NaN: rows before it keep their results, rows from it on are NaN, whichever CTA
    had its keys.  One of the old ones: all rows are."""
    c = cache_of(200, 1, 128, 64, 64, BF, fill=0xff)
    got, table, q = check(c, [5000], [new], 4, 69)
    starts, lens = torch.tensor([0, new]).int().cuda(), torch.tensor([5000]).int().cuda()
    bad = torch.full((1, 1, 128), math.nan, dtype=BF, device="cuda")
    for token in (5000 - 1 - new // 2, 2500):
        slot = table[0, token // 64].long().reshape(1) * 64 + token % 64
        c.append(torch.zeros_like(bad), bad, slot)
        o = c.attention(q.cuda(), table, lens, starts)
        first = max(0, token - (5000 - new))  # the first row that sees the token
        assert torch.equal(o[:first], got[:first]) and o[first:].isnan().all()


@pytest.mark.parametrize("batch, heads, new", [(3, 4, 16), (3, 4, 17), (200, 4, 8), (200, 4, 9), (200, 1, 33)])
def test_where_the_tiles_of_rows_change(ipex, batch, heads, new):
    """Numbers of rows around those from which tiles of 128 rows take a call, with few and with many sequences."""
    c = cache_of(batch * 3, 1, 128, 32, 64, BF, fill=0xff)
    lens = [(7 * b) % 60 + new - 5 for b in range(batch)]
    check(c, lens, [new] * batch, heads, 68)


@pytest.mark.parametrize("batch", [31, 257, 700])
def test_shares_of_many_sequences(ipex, batch):
    """More sequences than a warp, a CTA and a round of its warps look at; lengths all over, one long."""
    lens = [(i * 37) % 90 for i in range(batch)]
    lens[batch // 2] = 3000
    c = cache_of(sum(-(-n // 16) for n in lens) + 1, 1, 64, 16, 64, BF, fill=0xff)
    check(c, lens, [1] * batch, 4, 45, starts=False)


def test_a_table_without_pages(ipex):
    c = cache_of(3, 2, 64, 16, 32, BF)
    o = c.attention(torch.ones(2, 4, 64).to(BF).cuda(), torch.zeros(2, 0).int().cuda(), torch.tensor([5, 0]).int().cuda())
    assert (o == 0).all()


def test_scores_of_any_size(ipex):
    """A scale of 0 is an average, a negative one turns the order round, wide keys make one token win."""
    c = cache_of(40, 2, 128, 16, 64, BF)
    for scale, wide in ((0.0, 1.0), (-0.3, 1.0), (1.0, 8.0), (1e-30, 1.0)):
        check(c, [70, 300], [1, 1], 4, 70, scale=scale, wide=wide, starts=False)


def test_growing_scores_raise_the_reference(ipex):
    """Every block's scores pass the ones before by far."""
    c = cache_of(40, 1, 64, 16, 64, BF)
    kv, table = fill(c, [600], 80)
    k = (torch.arange(600)[:, None, None] * 0.05 + 0 * randn(1, 600, 1, 64)).to(BF)
    v = randn(82, 600, 1, 64).to(BF)
    slots = (table[0].cpu().long()[torch.arange(600) // 16] * 16 + torch.arange(600) % 16).cuda()
    c.append(k.cuda(), v.cuda(), slots)
    q = torch.ones(1, 4, 64).to(BF)
    got = c.attention(q.cuda(), table, torch.tensor([600]).int().cuda(), scale=1.0)
    compare(got, q, [(R.quantise(k, 64)[0], R.quantise(v, 64)[0])], [1], c, True, 1.0)


def test_strided_queries_and_other_index_types(ipex):
    c = cache_of(40, 2, 128, 16, 64, BF)
    lens = [50, 20, 300]
    kv, table = fill(c, lens, 90)
    wide = randn(93, 3, 24, 128).to(BF).cuda()
    q = wide[:, 5:13]                       # a slice of a projection
    odd = randn(93, 3, 8, 129).to(BF).cuda()[..., 1:]  # not aligned: copied
    tl = torch.cat((table, table), 1).long()[:, :table.shape[1]]  # int64, rows further apart
    n = torch.tensor(lens).cuda()
    compare(c.attention(q, tl, n), q.cpu(), kv, [1] * 3, c, True)
    compare(c.attention(odd, table, n.int()), odd.cpu(), kv, [1] * 3, c, True)
    wide_table = torch.full((3, 40), -1).int().cuda()
    wide_table[:, :table.shape[1]] = table
    compare(c.attention(q, wide_table[:, :table.shape[1]], n), q.cpu(), kv, [1] * 3, c, True)


def test_rows_behind_the_last_sequence(ipex):
    """Zeros from the operator; left as they were by the C entry, which writes to its caller's tensor."""
    c = cache_of(10, 2, 64, 16, 32, BF)
    kv, table = fill(c, [20, 9], 100)
    q = randn(103, 9, 4, 64).to(BF)
    starts = torch.tensor([1, 3, 6]).int().cuda()
    lens = torch.tensor([20, 9]).int().cuda()
    got = c.attention(q.cuda(), table, lens, starts)
    compare(got[1:6], q[1:6], kv, [2, 3], c, True)
    assert (got[:1] == 0).all() and (got[6:] == 0).all()
    import ctypes

    from ipex_b200 import _capi

    d = _capi.Kv4Desc(10, 2, 64, 16, 32, _capi.T_BF16)
    L = _capi.lib()
    ws = torch.zeros(L.woq_b200_kv4_attention_workspace_bytes(ctypes.byref(d), 2, 9, 4), dtype=torch.uint8, device="cuda")
    out, qg = torch.full((9, 4, 64), 3.0, device="cuda", dtype=BF), q.cuda()
    args = (ctypes.byref(d), c.tensor.data_ptr(), qg.data_ptr(), 256, 64, 4, table.data_ptr(), table.stride(0), table.shape[1],
            lens.data_ptr(), starts.data_ptr(), 2, 9, 64 ** -0.5, 1, out.data_ptr(), 256, 64, ws.data_ptr())
    assert L.woq_b200_kv4_attention(*args, ws.numel() - 1, None) == 4
    torch.cuda.synchronize()
    assert L.woq_b200_kv4_attention(*args, ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[1:6], got[1:6]) and (out[:1] == 3).all() and (out[6:] == 3).all()
    assert (ws[:L.woq_b200_workspace_header_bytes()] == 0).all()


def test_pages_that_the_cache_does_not_have(ipex):
    """Their keys are left out and the status says so; nothing outside the cache is read."""
    c = cache_of(10, 1, 64, 16, 32, BF)
    kv, table = fill(c, [64, 30], 110)
    q = randn(113, 2, 4, 64).to(BF)
    torch.ops.torch_ipex.woq_check_status()
    bad = table.clone()
    bad[0, 1], bad[0, 3] = 10, -1
    got = c.attention(q.cuda(), bad, torch.tensor([64, 30]).int().cuda())
    k, v = kv[0]
    keep = torch.tensor([i for i in range(64) if i // 16 not in (1, 3)])
    compare(got, q, [(k[keep], v[keep]), kv[1]], [1, 1], c, False)
    with pytest.raises(RuntimeError, match="page"):
        torch.ops.torch_ipex.woq_check_status()
    torch.ops.torch_ipex.woq_check_status()
    # lengths beyond the table are cut, negative ones are none
    got = c.attention(q.cuda(), table[:, :2].contiguous(), torch.tensor([1 << 30, -5]).int().cuda())
    compare(got, q, [(k[:32], v[:32]), (k[:0], v[:0])], [1, 1], c, False)
    torch.ops.torch_ipex.woq_check_status()


def test_same_bits_every_time(ipex):
    c = cache_of(700, 2, 128, 16, 64, BF)
    lens = [5000, 33, 3000, 700]
    kv, table = fill(c, lens, 120)
    q, n = randn(123, 4, 8, 128).to(BF).cuda(), torch.tensor(lens).int().cuda()
    first = c.attention(q, table, n)
    for _ in range(50):
        assert torch.equal(c.attention(q, table, n), first)


def test_captured_step_follows_its_tensors(ipex):
    """Append and attention in a graph, replayed with other tokens, slots, lengths and pages; two graphs, and eager calls of
    another size beside them on another stream."""
    heads, d = 4, 128
    c = cache_of(64, 2, d, 16, 64, BF, fill=0xff)
    lens = [37, 160, 5]
    kv, table = fill(c, lens, 130)
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    cs = _IPEXPagedKv4Cache.rotary_table(400, d)
    big = torch.full((3, 20), -1).int().cuda()
    big[:, :table.shape[1]] = table
    used = set(table[table >= 0].tolist())
    spare = [p for p in range(64) if p not in used]
    for b in range(3):  # room to grow
        first = -(-lens[b] // 16)
        for i in range(first, first + 2):
            big[b, i] = spare.pop()
    qkv = torch.zeros(3, (2 * heads + 4) * d, dtype=BF, device="cuda")
    slots, pos, n = (torch.zeros(3, dtype=torch.int64, device="cuda") for _ in range(3))

    def step():
        q, k, v = qkv.view(3, -1, d).split([2 * heads, 2, 2], 1)
        q = c.append(k, v, slots, q, pos, cs)
        return q, c.attention(q, big, n.int())

    slots.fill_(-1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    other = cache_of(700, 1, 64, 16, 32, FP)
    okv, otable = fill(other, [9000], 140)
    oq = randn(143, 1, 4, 64).to(FP)
    for i in range(20):
        x = randn(200 + i, 3, (2 * heads + 4) * d).to(BF)
        qkv.copy_(x)
        pos.copy_(torch.tensor(lens))
        slots.copy_(torch.tensor([int(big[b, lens[b] // 16]) * 16 + lens[b] % 16 for b in range(3)]))
        n.copy_(torch.tensor(lens) + 1)
        torch.cuda.synchronize()
        graphs[i % 2][0].replay()
        with torch.cuda.stream(side):
            beside = other.attention(oq.cuda(), otable, torch.tensor([9000]).int().cuda())
        torch.cuda.synchronize()
        compare(beside, oq, okv, [1], other, True)
        q, o = graphs[i % 2][1]
        new = c.read(slots)
        for b in range(3):
            kv[b] = tuple(torch.cat((old, now[b:b + 1].cpu().double())) for old, now in zip(kv[b], new))
            lens[b] += 1
        compare(o, q.cpu(), kv, [1] * 3, c, True)


def test_pages_far_into_a_large_cache(ipex):
    """Byte offsets beyond 2^32."""
    page_bytes = 2 * 16 * 2304
    pages = (5 << 30) // page_bytes
    c = cache_of(1, 2, 128, 256, 64, BF)
    c.tensor = torch.empty(pages, 2, 16, 2304, dtype=torch.uint8, device="cuda")
    c.num_pages = pages
    n = 600
    where = torch.tensor([pages - 1, 0, pages // 2])
    slots = where[torch.arange(n) // 256] * 256 + torch.arange(n) % 256
    k, v, q = randn(1, n, 2, 128).to(BF), randn(2, n, 2, 128).to(BF), randn(3, 1, 8, 128).to(BF)
    c.append(k.cuda(), v.cuda(), slots.cuda())
    kq, vq = R.quantise(k, 64)[0], R.quantise(v, 64)[0]
    kk, vv = c.read(slots.cuda())
    assert torch.equal(kk.cpu().double(), kq) and torch.equal(vv.cpu().double(), vq)
    got = c.attention(q.cuda(), where[None].int().cuda(), torch.tensor([n]).int().cuda())
    compare(got, q, [(kq, vq)], [1], c, True)


def test_refusals(ipex):
    ops = torch.ops.torch_ipex
    c = cache_of(4, 2, 128, 16, 64, BF)
    x, s = torch.zeros(3, 2, 128, dtype=BF, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    table, lens = torch.zeros(3, 1).int().cuda(), torch.zeros(3).int().cuda()
    for call in (
            lambda: ops.kv4_cache_append(c.tensor, x.float(), x.float(), s),
            lambda: ops.kv4_cache_append(c.tensor, x, x[:2], s),
            lambda: ops.kv4_cache_append(c.tensor, x[:, :1], x[:, :1], s),
            lambda: ops.kv4_cache_append(c.tensor, x[..., :64], x[..., :64], s),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s[:2]),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s.float()),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s.cpu()),
            lambda: ops.kv4_cache_append(c.tensor[:, :, :, :2000], x, x, s),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s, x, s),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s, x, s, torch.zeros(4, 24, device="cuda")),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s, x, s, torch.zeros(4, 144, device="cuda")),
            lambda: ops.kv4_cache_append(c.tensor, x, x, s, x.half(), s, torch.zeros(4, 128, device="cuda")),
            lambda: ops.kv4_cache_read(c.tensor, s, 64, BF),
            lambda: ops.kv4_cache_read(c.tensor, s, 128, torch.float32),
            lambda: ops.kv4_cache_attention(x[:, :1], c.tensor, table, lens),
            lambda: ops.kv4_cache_attention(x, c.tensor, table, lens[:2]),
            lambda: ops.kv4_cache_attention(x[:2], c.tensor, table, lens),
            lambda: ops.kv4_cache_attention(x, c.tensor, table, lens, lens),
            lambda: ops.kv4_cache_attention(x, c.tensor, table.cpu(), lens),
            lambda: ops.kv4_cache_attention(x, c.tensor, table, lens, None, float("nan")),
            lambda: c.attention(x.half(), table, lens),
            lambda: c.append(x.half(), x.half(), s)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    for bad in ((4, 2, 96), (4, 2, 128, 24), (4, 0, 128), (-1, 2, 128), (4, 2, 64, 16, 128), (4, 2, 128, 16, 64, torch.float32)):
        with pytest.raises(ValueError):
            _IPEXPagedKv4Cache(*bad)
    # nothing to do
    assert c.append(x[:0], x[:0], s[:0], x[:0]).shape == (0, 2, 128)
    assert c.attention(x[:0], table[:0], lens[:0]).shape == (0, 2, 128)
    assert c.attention(x[:0], table, lens, torch.zeros(4).int().cuda()).shape == (0, 2, 128)
    assert c.read(s[:0])[0].shape == (0, 2, 128)
