"""Every route of attention over the 4-bit cache: each instance of both kernels, the rare branches of the prompt kernel, and
calls that mix prompts with single tokens."""
import pytest
import torch

from tests import kv4_reference as R
from tests.test_gpu_kv4_cache import BF, FP, SHAPES, cache_of, check, compare, fill, ipex, randn  # noqa: F401 (ipex: the fixture)

pytestmark = pytest.mark.gpu


# ---- instances ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, group", SHAPES)
@pytest.mark.parametrize("new", [[3, 2, 3], [6, 8, 4], [150, 77, 1]])
def test_every_instance(ipex, t, d, group, new):  # noqa: F811
    """Tiles of 16 rows, of 32 (heads of 64) and of 128; the prompt kernel takes the last."""
    c = cache_of(40, 2, d, 32, group, t, fill=0xff)
    check(c, [300, 77, 140], new, 4, 11)


# ---- prompts -----------------------------------------------------------------------------------------------------
def ramp(c, lens, table, step):
    """Replaces the keys of all sequences: token j has every element step * j (j from the end for a negative step)."""
    page, kv = c.page_size, []
    for b, n in enumerate(lens):
        j = torch.arange(n, dtype=torch.float64)
        k = (step * j if step > 0 else -step * (n - 1 - j))[:, None, None].expand(n, c.kv_heads, c.head_dim).to(c.dtype)
        v = randn(20 + b, n, c.kv_heads, c.head_dim).to(c.dtype)
        slots = table[b].cpu().long()[torch.arange(n) // page] * page + torch.arange(n) % page
        c.append(k.cuda(), v.cuda(), slots.cuda())
        kv.append((R.quantise(k, c.group_size)[0], R.quantise(v, c.group_size)[0]))
    return kv


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, heads, lens, new", [(64, 4, [700, 300], [100, 300]), (128, 4, [900], [150]), (256, 2, [400, 130], [90, 140]),
                                                 (128, 2, [5000], [64])])
@pytest.mark.parametrize("step", [0.002, -0.002, 0.0001])
def test_prompts_whose_scores_grow(ipex, t, d, heads, lens, new, step):  # noqa: F811
    """By more than 15 (log2) from one tile of keys to the next, so that sums in tensor memory are rescaled at every tile; falling
    instead, never; growing slowly, seldom.  Rows that see nothing and CTAs that share the keys among them."""
    c = cache_of(100, 2, d, 64, 32, t, fill=0xff)
    _, table = fill(c, lens, 12)
    kv = ramp(c, lens, table, step)
    q = (0.75 + 0.5 * torch.rand(sum(new), 2 * heads, d, generator=torch.Generator().manual_seed(13))).to(t)
    starts = torch.tensor([0] + new).cumsum(0).int().cuda()
    for causal in (True, False):
        got = c.attention(q.cuda(), table, torch.tensor(lens).int().cuda(), starts, 64 / d, causal)
        compare(got, q, kv, new, c, causal, 64 / d)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, lens, new", [(128, [300, 170], [100, 170]), (64, [400], [70]), (256, [2000], [80])])
@pytest.mark.parametrize("scale, wide", [(0.0, 1.0), (-0.3, 1.0), (1.0, 4.0), (-1.0, 4.0), (1e-30, 1.0)])
def test_prompts_with_scores_of_any_size(ipex, t, d, lens, new, scale, wide):  # noqa: F811
    c = cache_of(50, 1, d, 64, 64, t, fill=0xff)
    for causal in (True, False):
        check(c, lens, new, 4, 14, causal=causal, scale=scale, wide=wide)


@pytest.mark.parametrize("page", [16, 48, 80, 256])
@pytest.mark.parametrize("d, group", [(64, 32), (128, 128), (256, 64)])
def test_prompts_on_pages_of_any_size(ipex, page, d, group):  # noqa: F811
    c = cache_of(60, 2, d, page, group, BF, fill=0xff)
    check(c, [300, 90, 257], [100, 90, 130], 4, 15)


@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, length, new, scale", [(64, 320, 100, None), (128, 320, 100, 0.0), (128, 320, 100, -0.3), (256, 160, 70, None),
                                                   (128, 4000, 70, None)])
def test_prompts_with_pages_that_the_cache_does_not_have(ipex, t, d, length, new, scale):  # noqa: F811
    """Left out and reported; all the more in a tile that has no other page; pages that stand twice count twice."""
    page = 16
    c = cache_of(length // page + 6, 1, d, page, 32, t, fill=0xff)
    kv, table = fill(c, [length, 90], 16)
    q = randn(17, new + 50, 4, d).to(t)
    starts, lens = torch.tensor([0, new, new + 50]).int().cuda(), torch.tensor([length, 90]).int().cuda()
    torch.ops.torch_ipex.woq_check_status()
    missing = [1, 3, (length - new) // page - 1] + ([20 + i for i in range(64)] if length > 1000 else [])
    twice = 4  # holds page 2's keys
    bad = table.clone()
    for i, p in enumerate(missing):
        bad[0, p] = (c.num_pages, -1, 1 << 30)[i % 3]
    bad[0, twice] = bad[0, 2]  # (also where it was to be a missing one)
    missing = [p for p in missing if p != twice]
    at = [i for i in range(length) if i // page not in missing]
    at = [i - 2 * page if i // page == twice else i for i in at]
    k, v = kv[0]
    for causal in (True, False):
        got = c.attention(q.cuda(), bad, lens, starts, scale, causal)
        with pytest.raises(RuntimeError, match="page"):
            torch.ops.torch_ipex.woq_check_status()
        # (they stand before the new tokens, so that every row sees all the others up to its own)
        compare(got, q, [(k[at], v[at]), kv[1]], [new, 50], c, causal, scale)
    torch.ops.torch_ipex.woq_check_status()


@pytest.mark.parametrize("t", [BF, FP])
def test_a_captured_prompt_follows_its_tensors(ipex, t):  # noqa: F811
    """Lengths, starts and pages are read at every replay; two graphs in turn on different streams."""
    c = cache_of(64, 2, 128, 32, 64, t, fill=0xff)
    sets = [([200, 90, 300], [100, 90, 10]), ([40, 300, 250], [1, 150, 49]), ([10, 0, 333], [20, 0, 180])]
    table, q = torch.full((3, 12), -1).int().cuda(), torch.zeros(200, 8, 128, dtype=t, device="cuda")
    lens, starts = torch.zeros(3).int().cuda(), torch.zeros(4).int().cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.attention(q, table, lens, starts)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = c.attention(q, table, lens, starts)
        graphs.append((g, out))
    for i in range(6):
        n, new = sets[i % 3]
        kv, pages = fill(c, n, 18 + i)
        fresh = randn(19 + i, 200, 8, 128).to(t)
        q.copy_(fresh)
        table.fill_(-1)
        table[:, :pages.shape[1]] = pages
        lens.copy_(torch.tensor(n))
        starts.copy_(torch.tensor([0] + new).cumsum(0))
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        with torch.cuda.stream((side, torch.cuda.current_stream())[i // 2 % 2]):
            g.replay()
        torch.cuda.synchronize()
        compare(out, fresh, kv, new, c, True)
        assert (out[sum(new):] == 0).all()


# ---- prompts and single tokens in one call -----------------------------------------------------------------------
@pytest.mark.parametrize("t", [BF, FP])
@pytest.mark.parametrize("d, kv_heads, singles, prompt", [(128, 2, 63, 1500), (64, 2, 30, 700), (256, 1, 20, 500),  # many rows on average
                                                          (128, 2, 200, 900), (64, 3, 150, 600), (256, 1, 120, 300)])  # few
@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_prompt_among_single_tokens(ipex, t, d, kv_heads, singles, prompt, at):  # noqa: F811
    """The sequences of a call go to one kernel together, by their rows on average: single tokens to the prompt kernel, or a prompt
    to the other.  The prompt first, in the middle or last; drafts of three tokens and sequences without rows beside it."""
    lens = [(37 * i) % 200 for i in range(singles)]
    new = [(1, 1, 3, 1, 0)[i % 5] for i in range(singles)]
    where = (0, singles // 2, singles)[at]
    lens.insert(where, prompt + 45)
    new.insert(where, prompt)
    c = cache_of(sum(-(-n // 16) for n in lens) + 1, kv_heads, d, 16, 32, t, fill=0xff)
    check(c, lens, new, 4, 21)
