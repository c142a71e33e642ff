"""The operators between the linears together, as a decoder layer uses them: residual + norm + codes, the projections on
them, append, attention, output projection; for a prompt, then token by token, and through the decode stack's layer."""
import pytest
import torch

from tests import kv4_reference as R

pytestmark = pytest.mark.gpu
HID, HQ, HK, D, PAGE, G = 512, 8, 2, 64, 16, 32


@pytest.fixture(scope="module")
def ipex():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import ipex_b200

    ipex_b200.load_ops()
    yield ipex_b200
    torch.ops.torch_ipex.woq_check_status()


@torch.no_grad()
def test_a_layer_for_a_prompt_and_then_tokens(ipex):
    """INT8 linears behind the fused norm, a 4-bit cache between them.  Every stage against the plain form of it on what the
    stage before gave."""
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache
    from ipex_b200.transformers.fusions.norm_quant import _IPEXRmsNormQuantLinears

    q = ipex.quantization
    qm = q.get_weight_only_quant_qconfig_mapping(weight_dtype=q.WoqWeightDtype.INT8, lowp_mode=q.WoqLowpMode.INT8,
                                                 act_quant_mode=q.WoqActQuantMode.PER_BATCH_SYM)
    holder = torch.nn.Module()
    torch.manual_seed(1)
    holder.q, holder.k, holder.v, holder.o = (torch.nn.Linear(i, o, bias=False) for i, o in (
        (HID, HQ * D), (HID, HK * D), (HID, HK * D), (HQ * D, HID)))
    holder = ipex.llm.optimize(holder, quantization_config=qm)
    norm = torch.nn.RMSNorm(HID, eps=1e-5).cuda().bfloat16()
    project = _IPEXRmsNormQuantLinears(norm, [holder.q, holder.k, holder.v])
    cache = _IPEXPagedKv4Cache(12, HK, D, PAGE, G)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(2)).view(2, 6).int().cuda()
    cs = _IPEXPagedKv4Cache.rotary_table(100, D)
    lens, held = [0, 0], [[None, None], [None, None]]
    for new in ([37, 61], [1, 1], [1, 1], [2, 5], [1, 1]):
        n = sum(new)
        x, r = torch.randn(n, HID, device="cuda").bfloat16(), torch.randn(n, HID, device="cuda").bfloat16()
        (qq, kk, vv), total = project(x, r)
        assert torch.equal(total, x + r)
        qq, kk, vv = qq.view(n, HQ, D), kk.view(n, HK, D), vv.view(n, HK, D)
        pos = torch.cat([torch.arange(a, a + m) for a, m in zip(lens, new)])
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(new))
        slots = table.cpu().long()[seq, pos // PAGE] * PAGE + pos % PAGE
        turned = cache.append(kk, vv, slots.cuda(), qq, pos.cuda(), cs)
        want = R.rotate(qq.cpu(), pos, cs.cpu(), False)
        assert ((turned.cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all()
        stored = [t.cpu().double() for t in cache.read(slots.cuda())]
        assert torch.equal(stored[1], R.quantise(vv.cpu(), G)[0])
        lens = [a + m for a, m in zip(lens, new)]
        starts = None if new == [1, 1] else torch.tensor([0, new[0], n]).int().cuda()
        out = cache.attention(turned, table, torch.tensor(lens).int().cuda(), starts)
        row = 0
        for b, m in enumerate(new):
            for i in range(2):
                part = stored[i][row:row + m]
                held[b][i] = part if held[b][i] is None else torch.cat((held[b][i], part))
            ref, tol = R.attend(turned[row:row + m].cpu().double(), held[b][0], held[b][1], D ** -0.5, True)
            assert ((out[row:row + m].cpu().double() - ref).abs() <= tol(R.EPS[torch.bfloat16])).all()
            row += m
        y = holder.o(out.reshape(n, HQ * D))
        assert y.shape == (n, HID) and y.isfinite().all()


def test_the_decode_stack_runs_on_the_4_bit_cache(ipex):
    """One layer of the stack, a prompt and two decode steps, the second from a graph: the same rows as the eager step."""
    import bench_stack as B
    from ipex_b200.transformers.fusions.kv4_cache import _IPEXPagedKv4Cache

    q = ipex.quantization
    qm = q.get_weight_only_quant_qconfig_mapping(weight_dtype=q.WoqWeightDtype.INT4, lowp_mode=q.WoqLowpMode.BF16,
                                                 group_size=B.GROUP)
    dev = torch.device("cuda:0")
    layer = B.DecoderLayer(dev)
    torch.manual_seed(3)
    for p in layer.parameters():
        if p.dim() == 2:
            p.data.normal_(0.0, 0.02)
    layer = ipex.llm.optimize(layer, dtype=torch.bfloat16, quantization_config=qm, inplace=True, device=dev)
    cache = _IPEXPagedKv4Cache(6, B.KV_HEADS, B.HEAD_DIM, B.PAGE, B.KV_GROUP)
    table = torch.arange(6).view(2, 3).int().cuda()
    cs = _IPEXPagedKv4Cache.rotary_table(192, B.HEAD_DIM, B.THETA)
    pos = torch.arange(100, device=dev)
    first = torch.arange(2, device=dev)[:, None] * 192
    seqs = B.Kv4Sequences((first + pos).flatten(), pos.repeat(2), cs, table, torch.tensor([100, 100]).int().cuda(),
                          torch.tensor([0, 100, 200]).int().cuda())
    with torch.no_grad():
        y = layer(torch.randn(2, 100, B.HIDDEN, device=dev).bfloat16(), seqs, cache, None, None, None, None)
        assert y.shape == (2, 100, B.HIDDEN) and y.isfinite().all()
        x, at = torch.randn(2, 1, B.HIDDEN, device=dev).bfloat16(), torch.full((1,), 100, device=dev)

        def step():
            s = B.Kv4Sequences(first[:, 0] + at, at.expand(2), cs, table, (at + 1).int().expand(2).contiguous())
            return layer(x, s, cache, None, None, None, None)

        eager = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            caught = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(caught, eager) and eager.isfinite().all()
        at.add_(1)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(caught, step())
