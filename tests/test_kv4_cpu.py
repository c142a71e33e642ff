"""The 4-bit key/value cache and the norm behind a residual without a GPU: refusals happen on the host, before any CUDA
call, and the plain reference of the tests agrees with itself."""
import ctypes

import pytest
import torch

from tests import kv4_reference as R

FAKE = 4096  # a pointer that is never followed: the call is refused


@pytest.fixture(scope="module")
def capi():
    from ipex_b200 import _capi

    _capi.lib()
    return _capi


def desc(capi, **over):
    d = dict(num_pages=4, kv_heads=2, head_dim=128, page_size=32, group_size=64, dtype=capi.T_BF16)
    d.update(over)
    return ctypes.byref(capi.Kv4Desc(**d))


@pytest.mark.parametrize("over, code", [
    (dict(dtype=1), 2), (dict(head_dim=96), 2), (dict(group_size=16), 2), (dict(head_dim=64, group_size=128), 2),
    (dict(page_size=24), 1), (dict(page_size=0), 1), (dict(kv_heads=0), 1), (dict(num_pages=-1), 1)])
def test_descriptions_that_are_refused(capi, over, code):
    L = capi.lib()
    d = desc(capi, **over)
    assert L.woq_b200_kv4_bytes(d) == 0
    assert L.woq_b200_kv4_read(d, FAKE, FAKE, 1, FAKE, FAKE, None) == code
    assert L.woq_b200_kv4_append(d, FAKE, None, 0, 0, 0, FAKE, 128, 128, FAKE, 128, 128, FAKE, None, None, 0, 0, 0, 1, None,
                                 None) == code
    assert L.woq_b200_kv4_attention(d, FAKE, FAKE, 256, 128, 2, FAKE, 1, 1, FAKE, None, 1, 1, 1.0, 1, FAKE, 256, 128, FAKE,
                                    1 << 30, None) == code
    assert len(L.woq_b200_last_error()) > 10


@pytest.mark.parametrize("d, g", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_size_of_a_cache(capi, d, g):
    # codes of keys and values and a pair of 16-bit parameters per group of each
    per_token = d // 2 * 2 + 2 * (d // g) * 4
    assert capi.lib().woq_b200_kv4_bytes(desc(capi, head_dim=d, group_size=g)) == 4 * 2 * 32 * per_token
    assert capi.lib().woq_b200_kv4_bytes(desc(capi, head_dim=d, group_size=g, num_pages=0)) == 0


def append(capi, d=None, cache=FAKE, q=FAKE, q_tok=512, q_head=128, q_heads=4, k=FAKE, k_tok=256, k_head=128, v=FAKE, v_tok=256,
           v_head=128, slots=FAKE, positions=FAKE, cos_sin=FAKE, max_pos=10, rot=128, tokens=1, q_out=FAKE):
    return capi.lib().woq_b200_kv4_append(d or desc(capi), cache, q, q_tok, q_head, q_heads, k, k_tok, k_head, v, v_tok, v_head,
                                          slots, positions, cos_sin, max_pos, rot, 0, tokens, q_out, None)


@pytest.mark.parametrize("bad, code", [
    (dict(cache=None), 1), (dict(cache=FAKE + 8), 1), (dict(slots=None), 1), (dict(k=None), 1), (dict(v=FAKE + 2), 1),
    (dict(k_tok=252), 1), (dict(q_head=4), 1), (dict(q=None), 1), (dict(q_out=None), 1), (dict(positions=None), 1),
    (dict(cos_sin=None), 1), (dict(cos_sin=FAKE + 4), 1), (dict(max_pos=0), 1), (dict(rot=8), 2), (dict(rot=144), 2), (dict(rot=-16), 2),
    (dict(tokens=-1), 1), (dict(q_heads=-1), 1), (dict(tokens=1 << 31), 1)])
def test_appends_that_are_refused(capi, bad, code):
    assert append(capi, **bad) == code


def test_appending_nothing_is_fine(capi):
    assert append(capi, tokens=0, cache=None, slots=None, k=None, v=None, q=None) == 0


def attention(capi, d=None, cache=FAKE, q=FAKE, q_tok=512, q_head=128, q_heads=4, table=FAKE, table_ld=4, max_pages=4, lens=FAKE,
              starts=None, batch=2, tokens=2, scale=0.1, causal=1, out=FAKE, o_tok=512, o_head=128, ws=FAKE, ws_bytes=1 << 40):
    return capi.lib().woq_b200_kv4_attention(d or desc(capi), cache, q, q_tok, q_head, q_heads, table, table_ld, max_pages, lens,
                                             starts, batch, tokens, scale, causal, out, o_tok, o_head, ws, ws_bytes, None)


@pytest.mark.parametrize("bad, code", [
    (dict(cache=None), 1), (dict(q=None), 1), (dict(q=FAKE + 4), 1), (dict(q_tok=508), 1), (dict(q_heads=3), 1),
    (dict(q_heads=0), 1), (dict(table=None), 1), (dict(table_ld=3), 1), (dict(lens=None), 1), (dict(batch=3), 1),
    (dict(batch=-1), 1), (dict(tokens=-1), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(out=None), 1), (dict(o_head=100), 1), (dict(ws=None), 1), (dict(ws=FAKE + 8), 1), (dict(max_pages=-1), 1),
    (dict(max_pages=1 << 27, table_ld=1 << 27), 2),
    (dict(tokens=(1 << 31) - 1, batch=(1 << 31) - 1), 2)])
def test_attention_calls_that_are_refused(capi, bad, code):
    assert attention(capi, **bad) == code


def test_numbers_of_rows_that_no_launch_can_take(capi):
    """Tiles of rows are numbered in 31 bits: many sequences for a few rows pass them as many rows do."""
    assert attention(capi, starts=FAKE, batch=(1 << 31) - 1, tokens=1) == 2
    assert attention(capi, starts=FAKE, batch=1, tokens=1 << 25, max_pages=1 << 23, table_ld=1 << 23) == 2


def test_attention_of_nothing_is_fine(capi):
    assert attention(capi, batch=0, tokens=0, q=None, out=None, ws=None) == 0


@pytest.mark.parametrize("bad, code", [
    (dict(x=None), 1), (dict(r=None), 1), (dict(sum=None), 1), (dict(qa=FAKE + 8), 1), (dict(k=24), 1), (dict(k=0), 1),
    (dict(ldx=56), 1), (dict(ldr=68), 1), (dict(lds=66), 1), (dict(mode=4), 2), (dict(mode=2, zpa=None), 1),
    (dict(k=131088, ldx=131088, ldr=131088, lds=131088), 2), (dict(m=-1), 1)])
def test_norms_behind_a_residual_that_are_refused(capi, bad, code):
    a = dict(x=FAKE, ldx=64, r=FAKE, ldr=64, gamma=FAKE, m=1, k=64, mode=6, sum=FAKE, lds=64, qa=FAKE, sa=FAKE, zpa=FAKE)
    a.update(bad)
    assert capi.lib().woq_b200_add_rmsnorm_quant(a["x"], a["ldx"], a["r"], a["ldr"], a["gamma"], 1e-5, a["m"], a["k"], a["mode"],
                                                 a["sum"], a["lds"], a["qa"], a["sa"], a["zpa"], None) == code


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_reference_quantiser_is_within_half_a_step(t):
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).to(t)
    y, s = R.quantise(x, 32)
    step = s.repeat_interleave(32, -1)
    # half a step, up to 15 steps of a scale that is one rounding too small, and the value's own rounding
    assert ((y - x.double()).abs() <= step * (0.5 + 15 * R.EPS[t]) + y.abs() * R.EPS[t] / 2).all()
    assert (R.quantise(torch.full((2, 64), 3.0).to(t), 64)[0] == 3.0).all()
