"""The 4-bit key/value cache where its arithmetic and its arguments are at their edges."""
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
