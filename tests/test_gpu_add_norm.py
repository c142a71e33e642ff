"""The residual's addition with RMS norm and 8-bit codes against a plain 64-bit implementation."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import ipex_b200

    ipex_b200.load_ops()
    return torch.ops.torch_ipex


def check(x, r, g, got, asym):
    """The sum exactly.  Codes: y's 32-bit value is off by at most 4 units of 2^-24 (the sum of squares is a sum of
    positive terms in 32 bits: k 2^-24 relative at worst, far less in practice, halved by the root), so y may be rounded
    to the other neighbour in bf16: 2^-8 of itself, in the element and in the ends of the range.  Half a code, and that."""
    h, qa, sa, zpa = (t.cpu() for t in got)
    k = x.shape[-1]
    want = (x.cpu().float() + r.cpu().float()).bfloat16()
    assert torch.equal(h, want)
    hd = want.double().reshape(-1, k)
    y = hd * (hd.square().mean(-1, keepdim=True) + EPS).rsqrt() * g.cpu().double()
    qa, s = qa.reshape(-1, k), sa.double()[:, None]
    top = y.abs().amax(-1, keepdim=True)
    if asym:
        codes = qa.view(torch.uint8).double() - zpa.double()[:, None]
        step = (y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)) / 255
    else:
        assert zpa.numel() == 0
        codes, step = qa.double(), top / 127
    assert ((s - step).abs() <= step * 2.0 ** -22 + top * 2.0 ** -7 / (127 if not asym else 127.5)).all()
    # asymmetric codes are rounded together with a rounded zero point: a whole code
    half = 1.0 if asym else 0.5
    assert ((codes * s - y).abs() <= half * s * (1 + 2.0 ** -16) + y.abs() * 2.0 ** -8 + top * 2.0 ** -7).all()
    # and exactly the definition, from the rounded y, wherever its rounding is not in doubt: y's 32-bit value is within
    # 2^-18 (chains of fewer than 100 additions, halved by the root, and four roundings).  The quotient is a 32-bit one, as
    # the definition says: an element of half the maximum gives 63.5 in 32 bits, a tie that goes to the even code, where
    # 64 bits still show that the scale was rounded.
    y16 = y.bfloat16().double()
    ulp = 2.0 ** (y.abs().clamp_min(1e-30).log2().floor() - 7)
    sure = ((y - y16).abs() - ulp / 2).abs() > y.abs() * 2.0 ** -18
    if not asym:
        c = (y16.float() / s.float()).round().clamp(-128, 127).double()
        assert (c == codes)[sure].all() and sure.double().mean() > 0.99


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("rows, k", [(1, 16), (1, 4096), (3, 2048), (5, 2064), (128, 8192), (129, 8192), (129, 4112), (7, 14336),
                                     (130, 14336), (2, 16400), (131, 20000), (2, 131072), (1000, 64)])
def test_against_the_definition(ops, rows, k, asym):
    gen = torch.Generator().manual_seed(rows * k)
    x, r = torch.randn(rows, k, generator=gen).bfloat16().cuda(), (3 * torch.randn(rows, k, generator=gen)).bfloat16().cuda()
    g = (1 + 0.3 * torch.randn(k, generator=gen)).bfloat16().cuda()
    check(x, r, g, ops.woq_add_rmsnorm_quant(x, r, g, EPS, 2 if asym else 6), asym)


@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("rows, k", [(37, 6160), (38, 6160), (37, 6144), (1, 8192), (37, 16384), (38, 8208), (296, 14336), (297, 14336)])
def test_around_the_changes_of_the_split(ops, rows, k, asym):
    gen = torch.Generator().manual_seed(rows + k)
    x, r = torch.randn(rows, k, generator=gen).bfloat16().cuda(), (3 * torch.randn(rows, k, generator=gen)).bfloat16().cuda()
    g = (1 + 0.3 * torch.randn(k, generator=gen)).bfloat16().cuda()
    check(x, r, g, ops.woq_add_rmsnorm_quant(x, r, g, EPS, 2 if asym else 6), asym)


def test_strides_shapes_and_types(ops):
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(2, 3, 100, generator=gen).bfloat16().cuda()[..., 4:84]      # not aligned: copied
    r = torch.randn(6, 160, generator=gen).bfloat16().cuda()[:, :80].view(6, 80).unflatten(0, (2, 3))
    g = torch.rand(80, generator=gen).cuda() + 0.5                              # fp32 weight: rounded to bf16
    got = ops.woq_add_rmsnorm_quant(x, r, g, EPS, 6)
    assert got[0].shape == got[1].shape == (2, 3, 80) and got[2].shape == (6,)
    check(x, r, g.bfloat16(), got, False)
    broadcast = torch.randn(1, 80, generator=gen).bfloat16().cuda().expand(6, 80)
    check(r.reshape(6, 80), broadcast, g.bfloat16(), ops.woq_add_rmsnorm_quant(r.reshape(6, 80), broadcast, g, EPS, 6), False)
    empty = ops.woq_add_rmsnorm_quant(x[:0], r[:0], g, EPS, 2)
    assert empty[0].shape == (0, 3, 80) and empty[3].shape == (0,)


def test_rows_of_zeros_and_rows_that_are_not_finite(ops):
    x = torch.zeros(4, 64, device="cuda").bfloat16()
    r = torch.ones(4, 64, device="cuda").bfloat16()
    r[0], r[1, 3], r[2, 5] = 0, float("inf"), float("nan")
    g = torch.ones(64, device="cuda").bfloat16()
    for mode in (2, 6):
        h, qa, sa, zpa = ops.woq_add_rmsnorm_quant(x, r, g, EPS, mode)
        assert torch.equal(h.view(torch.int16)[[0, 3]], r.view(torch.int16)[[0, 3]])
        assert sa[0] == 0 and (qa[0] == 0).all() and sa[1].isnan() and sa[2].isnan() and sa[3].isfinite()


def test_matches_the_norm_without_a_residual(ops):
    """On the sum, woq_rmsnorm_quant adds the squares in another order: codes one apart at most, and seldom."""
    gen = torch.Generator().manual_seed(6)
    x, r = torch.randn(50, 4096, generator=gen).bfloat16().cuda(), torch.randn(50, 4096, generator=gen).bfloat16().cuda()
    g = torch.rand(4096, generator=gen).bfloat16().cuda()
    h, qa, sa, _ = ops.woq_add_rmsnorm_quant(x, r, g, EPS, 6)
    qb, sb, _ = ops.woq_rmsnorm_quant(h, g, EPS, 6)
    same = sa == sb
    assert same.float().mean() > 0.9
    d = (qa[same].int() - qb[same].int()).abs()
    assert d.max() <= 1 and (d > 0).float().mean() < 1e-2


def test_module_with_a_residual_in_a_graph(ops):
    """_IPEXRmsNormQuantLinears(x, residual) is its linears on the norm of the sum, and returns the sum; captured too."""
    import ipex_b200 as ipex
    from ipex_b200.transformers.fusions.norm_quant import _IPEXRmsNormQuantLinears

    q = ipex.quantization
    qm = q.get_weight_only_quant_qconfig_mapping(weight_dtype=q.WoqWeightDtype.INT8, lowp_mode=q.WoqLowpMode.INT8,
                                                 act_quant_mode=q.WoqActQuantMode.PER_BATCH_SYM)
    holder = torch.nn.Module()
    for i, n in enumerate((512, 128)):
        torch.manual_seed(i)
        setattr(holder, f"l{i}", torch.nn.Linear(512, n, bias=False))
    holder = ipex.llm.optimize(holder, quantization_config=qm)
    norm = torch.nn.RMSNorm(512, eps=EPS).cuda().bfloat16()
    fused = _IPEXRmsNormQuantLinears(norm, [holder.l0, holder.l1])
    x, r = torch.randn(2, 3, 512, device="cuda").bfloat16(), torch.randn(2, 3, 512, device="cuda").bfloat16()
    outs, h = fused(x, r)
    assert torch.equal(h, x + r)
    codes, scales = ops.woq_add_rmsnorm_quant(x, r, norm.weight, EPS, 6)[1:3]
    for got, mod in zip(outs, (holder.l0, holder.l1)):
        want = ops.woq_linear_prequant(codes, scales, torch.empty(0, dtype=torch.int32, device="cuda"),
                                       mod._op_context.get_data_handle(), 0, [])
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fused(x, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        caught, hc = fused(x, r)
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    fresh, hf = fused(x, r)
    assert torch.equal(hc, hf) and all(torch.equal(a, b) for a, b in zip(caught, fresh))


def test_refusals(ops):
    x, g = torch.zeros(2, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda").bfloat16()
    for call in (lambda: ops.woq_add_rmsnorm_quant(x.half(), x.half(), g, EPS, 6),
                 lambda: ops.woq_add_rmsnorm_quant(x, x[:1], g, EPS, 6), lambda: ops.woq_add_rmsnorm_quant(x, x.float(), g, EPS, 6),
                 lambda: ops.woq_add_rmsnorm_quant(x, x, g[:32], EPS, 6), lambda: ops.woq_add_rmsnorm_quant(x, x, g, EPS, 4),
                 lambda: ops.woq_add_rmsnorm_quant(x[:, :24], x[:, :24], g[:24], EPS, 6),
                 lambda: ops.woq_add_rmsnorm_quant(x, x.cpu(), g, EPS, 6)):
        with pytest.raises(RuntimeError):
            call()
