"""Sizes of the 4-bit cache that its numbers cannot hold: refused on the host, before any CUDA call."""
import ctypes

import pytest

FAKE = 4096  # a pointer that is never followed: the call is refused


@pytest.fixture(scope="module")
def capi():
    from ipex_b200 import _capi

    _capi.lib()
    return _capi


def desc(capi, **over):
    d = dict(num_pages=4, kv_heads=1, head_dim=64, page_size=16, group_size=64, dtype=capi.T_BF16)
    d.update(over)
    return ctypes.byref(capi.Kv4Desc(**d))


@pytest.mark.parametrize("pages, page_size", [(511, 16 * 262657), ((1 << 27) - 1, 16), (1, (1 << 31) - 16), (1, (1 << 31) - 1008)])
def test_tables_whose_tokens_do_not_leave_room_for_a_tile(capi, pages, page_size):
    """Lengths are rounded up to units of 32 keys and tiles of 128 in 31 bits: a table may hold 2^31 - 1024 tokens at most."""
    assert 2 ** 31 - 1024 < pages * page_size < 2 ** 31
    d = desc(capi, page_size=page_size)
    for starts in (None, FAKE):
        assert capi.lib().woq_b200_kv4_attention(d, FAKE, FAKE, 256, 64, 4, FAKE, pages, pages, FAKE, starts, 1, 1, 0.1, 1, FAKE,
                                                 256, 64, FAKE, 1 << 40, None) == 2


def test_rows_that_do_not_leave_room_for_a_tile(capi):
    tokens = ((1 << 31) - 1) // 4
    assert capi.lib().woq_b200_kv4_attention(desc(capi), FAKE, FAKE, 0, 64, 4, FAKE, 4, 4, FAKE, FAKE, 1, tokens, 0.1, 1, FAKE,
                                             0, 64, FAKE, 1 << 40, None) == 2


@pytest.mark.parametrize("over", [dict(num_pages=1 << 57), dict(num_pages=1 << 62), dict(num_pages=1 << 40, kv_heads=65535, page_size=1 << 20)])
def test_caches_whose_bytes_pass_63_bits(capi, over):
    """A size that wrapped round would be taken for the bytes to allocate."""
    d, L = desc(capi, **over), capi.lib()
    assert L.woq_b200_kv4_bytes(d) == 0
    assert L.woq_b200_kv4_read(d, FAKE, FAKE, 1, FAKE, FAKE, None) == 1
    assert L.woq_b200_kv4_append(d, FAKE, None, 0, 0, 0, FAKE, 64, 64, FAKE, 64, 64, FAKE, None, None, 0, 0, 0, 1, None, None) == 1
    assert L.woq_b200_kv4_attention(d, FAKE, FAKE, 256, 64, over.get("kv_heads", 1), FAKE, 1, 1, FAKE, None, 1, 1, 0.1, 1, FAKE, 256,
                                    64, FAKE, 1 << 40, None) == 1


def test_a_cache_of_the_most_bytes_there_can_be(capi):
    pages = ((1 << 63) - 1) // 1152
    assert capi.lib().woq_b200_kv4_bytes(desc(capi, num_pages=pages)) == pages * 1152
    assert capi.lib().woq_b200_kv4_bytes(desc(capi, num_pages=pages + 1)) == 0
