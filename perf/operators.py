"""What the operators between a decoder layer's weight-only-quantised linears are timed on, through
`torch.ops.torch_ipex`: the residual's addition with RMS norm and 8-bit codes for the INT8-compute linears,
appending rotated keys and values to a paged 4-bit cache, and attention over that cache.

Head counts and widths are those of the 8B and 70B decode stacks that the benchmark runs (32 or 64 query heads over
8 key/value heads of 128), and generic ones beside them.

The cache is a uint8 tensor [pages, key/value heads, page size / 16, block bytes].  A block holds 16 tokens of one head:
the codes of the keys, those of the values (D / 2 bytes a token each), then {scale, lowest value} pairs for the keys
[token][group], then for the values, in the type of the keys.  Which byte of a block holds which code: `_places`.
"""
import math
import os
import sys

import torch

own = False
EPS, THETA = 1e-5, 5e5


def _ops():
    root = os.path.join(os.getcwd(), "intel-extension-for-pytorch_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import ipex_b200

    ipex_b200.load_ops()
    return torch.ops.torch_ipex


# ---- cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of an 8B model between two linears: the smallest call
        dict(name="norm_1", op="norm", rows=1, k=4096, asym=False),
        # a mid-sized decode batch with the asymmetric recipe
        dict(name="norm_asym_37", op="norm", rows=37, k=8192, asym=True),
        # a long prompt of a 70B model
        dict(name="norm_4096", op="norm", rows=4096, k=8192, asym=False),
        # one decode step of eight sequences of an 8B model, keys and values as slices of the concatenated projection
        dict(name="append_8", op="append", tokens=8, q_heads=32, kv_heads=8, d=128, group=64, page=64, dtype="bf16",
             rot=128, interleaved=False),
        # fp16, narrow heads, a rotation of half the head in neighbouring pairs, an odd number of tokens
        dict(name="append_fp16_1001", op="append", tokens=1001, q_heads=25, kv_heads=5, d=64, group=32, page=16, dtype="fp16",
             rot=32, interleaved=True),
        # a long prompt of a 70B model
        dict(name="append_8000", op="append", tokens=8000, q_heads=64, kv_heads=8, d=128, group=64, page=64, dtype="bf16",
             rot=128, interleaved=False),
        # one user's decode step after the stack's prompt: the smallest attention call
        dict(name="attend_1", op="attend", batch=1, past_lo=1024, past_hi=1024, new_lo=1, new_hi=1, q_heads=32, kv_heads=8,
             d=128, group=64, page=64, dtype="bf16", causal=True),
        # the decode stack's largest batch
        dict(name="attend_32", op="attend", batch=32, past_lo=1024, past_hi=1151, new_lo=1, new_hi=1, q_heads=32, kv_heads=8,
             d=128, group=64, page=64, dtype="bf16", causal=True),
        # continuous batching on a 70B model: lengths from one token to long ones, small pages
        dict(name="attend_64_ragged", op="attend", batch=64, past_lo=0, past_hi=8191, new_lo=1, new_hi=1, q_heads=64,
             kv_heads=8, d=128, group=64, page=16, dtype="bf16", causal=True),
        # two long documents, fp16, one scale for a whole head
        dict(name="attend_long_2", op="attend", batch=2, past_lo=99999, past_hi=100001, new_lo=1, new_hi=1, q_heads=40,
             kv_heads=8, d=128, group=128, page=256, dtype="fp16", causal=True),
        # a few drafted tokens for each of 16 sequences, wide heads
        dict(name="attend_draft_16", op="attend", batch=16, past_lo=30, past_hi=4001, new_lo=3, new_hi=6, q_heads=16,
             kv_heads=4, d=256, group=32, page=32, dtype="bf16", causal=True),
        # two prompts of an 8B model, one behind a cached prefix: the largest case
        dict(name="attend_prompt", op="attend", batch=2, past_lo=0, past_hi=777, new_lo=3000, new_hi=4096, q_heads=32,
             kv_heads=8, d=128, group=64, page=64, dtype="bf16", causal=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "append", "one", "one", "few", "prompt"])
    if kind == "norm":
        k = 16 * _log(rng, 16, 1024)
        return dict(op="norm", rows=_log(rng, 1, (4096 * 8192) // k), k=k, asym=rng.random() < 0.5)
    d = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 64, 128) if g <= d])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    common = dict(q_heads=q_heads, kv_heads=kv_heads, d=d, group=group, page=rng.choice([16, 16, 32, 64, 64, 128, 256]),
                  dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "append":
        most = max(1, (8000 * 80 * 128) // ((q_heads + 2 * kv_heads) * d))
        return dict(op="append", tokens=_log(rng, 1, most), rot=rng.choice([d, d, d // 2, d // 4]),
                    interleaved=rng.random() < 0.3, **common)
    if kind == "one":
        batch = _log(rng, 1, 128)
        # tokens of the cache that the largest decode case holds
        most = max(1, (64 * 4096 * 8 * 128) // (batch * kv_heads * d * max(1, q_heads // (8 * kv_heads))))
        hi = _log(rng, 1, min(most, 120000))
        return dict(op="attend", batch=batch, past_lo=rng.randint(0, hi), past_hi=hi, new_lo=1, new_hi=1, causal=True, **common)
    if kind == "few":
        batch, new = _log(rng, 1, 32), rng.randint(2, 12)
        most = max(1, (64 * 4096 * 8 * 128) // (batch * q_heads * d))
        hi = _log(rng, 1, min(most, 30000))
        return dict(op="attend", batch=batch, past_lo=rng.randint(0, hi), past_hi=hi, new_lo=rng.randint(1, new), new_hi=new,
                    causal=rng.random() < 0.9, **common)
    batch = rng.randint(1, 4)
    most = int(math.sqrt((2 * 3500 * 4000 * 32 * 128) / (batch * q_heads * d)))
    new = _log(rng, min(64, most), max(64, min(6000, most // 2 + 1)))
    past = rng.randint(0, max(0, most - new)) if rng.random() < 0.5 else 0
    return dict(op="attend", batch=batch, past_lo=past // 2, past_hi=past, new_lo=(new + 1) // 2, new_hi=new,
                causal=rng.random() < 0.9, **common)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi in a mixed order; the largest first where there is one."""
    return [hi] if n == 1 else [lo + (hi - lo) * ((n - 1 - i * 7 % n) if math.gcd(7, n) == 1 else n - 1 - i) // (n - 1) for i in range(n)]


def _lengths(case):
    """Per sequence: new tokens, and cached tokens with the new ones."""
    b = case["batch"]
    new = _spread(case["new_lo"], case["new_hi"], b)
    past = list(reversed(_spread(case["past_lo"], case["past_hi"], b)))
    return new, [p + n for p, n in zip(past, new)]


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


# ---- the cache's layout -----------------------------------------------------------------------------------------
def _places(d, device):
    """Byte within a block and shift within the byte of the codes of token r and element i, [16, d]: of keys, of values."""
    r, i = torch.arange(16, device=device)[:, None], torch.arange(d, device=device)[None]
    w = min(d, 128)  # wider heads: 128 elements after 128
    half, j, words = i // w, i % w, w // 32
    # a key's row: 32-bit words [j / 8 % 4][j / 32]; a word's low half holds the even ones of 8 neighbours
    nib = j % 8 // 2 + 4 * (j % 2)
    k_byte = r * (d // 2) + half * (w // 2) + (j // 8 % 4 * words + j // 32) * 4 + nib // 2
    # values: words [j % 8][pair of tokens][j / 32], the first token of a pair in the low half
    swap = j % 2 * 4 if w == 128 else j // 2 % 2 * 4
    vn = j // 8 % 4
    v_byte = 8 * d + half * (w * 8) + (j % 8 * 8 + (r // 2 ^ swap)) * (words * 4) + j // 32 * 4 + r % 2 * 2 + vn // 2
    return (k_byte, nib % 2 * 4 + 0 * r), (v_byte, vn % 2 * 4 + 0 * r)


def _block_bytes(d, group):
    return 16 * d + 128 * (d // group)


def _codes(x, group):
    """Codes and {scale, lowest} of x [..., d] in its type."""
    t = x.dtype
    g = x.double().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    want = (hi - lo) / 15
    s = want.to(t)
    s = (s.view(torch.int16) - (s.double() > want).to(torch.int16)).view(t)  # toward zero
    sd = s.double()
    c = torch.where(sd[..., None] > 0, ((g - lo[..., None]) / sd[..., None].clamp_min(1e-300)).round().clamp(0, 15), 0.0)
    return c.flatten(-2).to(torch.uint8), torch.stack((s, lo.to(t)), -1)


def _values(codes, params):
    """What codes [..., d] and {scale, lowest} [..., d / group, 2] stand for: one rounding to the parameters' type."""
    p = params.float()
    g = codes.float().unflatten(-1, (params.shape[-2], -1))
    return (g * p[..., 0:1] + p[..., 1:2]).flatten(-2).to(params.dtype)


def _pack(k, v, group):
    """Blocks uint8 [n, block bytes] of k, v [n, 16, d]."""
    d = k.shape[-1]
    out = []
    for x, (byte, shift) in zip((k, v), _places(d, k.device)):
        c, p = _codes(x, group)
        order = (byte * 2 + shift // 4).flatten().argsort()  # the elements in the order of their nibbles
        c = c.flatten(1)[:, order]
        out.append((c[:, 0::2] | c[:, 1::2] << 4, p.flatten(1).view(torch.uint8)))
    return torch.cat((out[0][0], out[1][0], out[0][1], out[1][1]), 1)


def _unpack(blocks, d, group, dtype):
    """Keys and values [n, 16, d] that blocks [n, block bytes] stand for."""
    pb = 64 * (d // group)
    (kb, ks), (vb, vs) = _places(d, blocks.device)
    kp = blocks[:, 16 * d:16 * d + pb].contiguous().view(dtype).view(-1, 16, d // group, 2)
    vp = blocks[:, 16 * d + pb:].contiguous().view(dtype).view(-1, 16, d // group, 2)
    return (_values((blocks[:, kb] >> ks.to(torch.uint8)) & 15, kp), _values((blocks[:, vb] >> vs.to(torch.uint8)) & 15, vp))


# ---- inputs -----------------------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _table(positions, rot):
    inv = 1.0 / (THETA ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv[None]
    return torch.cat((a.cos(), a.sin()), 1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "norm":
        rows, k = case["rows"], case["k"]
        spread = (0.5 * _randn(gen, k)).exp()  # some channels of a residual stream are larger than others
        return dict(case=case, x=_randn(gen, rows, k).bfloat16(), residual=(3 * _randn(gen, rows, k) * spread).bfloat16(),
                    gamma=(1 + 0.2 * _randn(gen, k)).bfloat16())
    t, hq, hk, d, page, group = _type(case), case["q_heads"], case["kv_heads"], case["d"], case["page"], case["group"]
    spread = (0.5 * _randn(gen, hk, d)).exp()  # keys have wide channels
    if case["op"] == "append":
        n = case["tokens"]
        qkv = _randn(gen, n, (hq + 2 * hk) * d)
        qkv[:, hq * d:(hq + hk) * d] *= spread.flatten()
        pages = -(-n // page) + 3
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(n, device="cuda")
        past = int(torch.randint(0, 5000, (1,), device="cuda", generator=gen))
        return dict(case=case, qkv=qkv.to(t), cache=torch.zeros(pages, hk, page // 16, _block_bytes(d, group), dtype=torch.uint8, device="cuda"),
                    slots=order[at // page] * page + at % page, positions=past + at, cos_sin=_table(past + n, case["rot"]))
    new, lens = _lengths(case)
    b = len(new)
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1) + 1
    pages = sum(need) + 2
    cache = torch.empty(pages, hk, page // 16, _block_bytes(d, group), dtype=torch.uint8, device="cuda")
    flat = cache.view(pages * hk * (page // 16), -1)
    chunk = max(1, (1 << 24) // (16 * d))
    heads = torch.arange(pages * hk * (page // 16), device="cuda") // (page // 16) % hk
    for at in range(0, flat.shape[0], chunk):
        n = min(chunk, flat.shape[0] - at)
        scale = spread[heads[at:at + n]][:, None]
        flat[at:at + n] = _pack((_randn(gen, n, 16, d) * scale).to(t), _randn(gen, n, 16, d).to(t), group)
    order = torch.randperm(pages, device="cuda", generator=gen)
    ends = torch.tensor([0] + need, device="cuda").cumsum(0)
    j = torch.arange(width, device="cuda")[None]
    table = torch.where(j < (ends[1:] - ends[:-1])[:, None], order[(ends[:-1, None] + j).clamp_max(pages - 1)], -1).int()
    starts = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    return dict(case=case, q=_randn(gen, sum(new), hq, d).to(t), cache=cache, table=table, new=new, lens=lens,
                seq_lens=torch.tensor(lens, device="cuda", dtype=torch.int32),
                starts=starts if case["new_hi"] > 1 else None, scale=d ** -0.5)


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _norm(x, residual, gamma, asym):
    h = (x.float() + residual.float()).bfloat16()
    hd = h.double()
    y = (hd * (hd.square().mean(-1, keepdim=True) + EPS).rsqrt() * gamma.double()).bfloat16().double()
    if asym:
        lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
        s = ((hi - lo) / 255).float().double()
        z = -(lo / s).round()
        return h, (((y / s + z).round().clamp(0, 255) - z) * s).bfloat16()
    s = (y.abs().amax(-1, keepdim=True) / 127).float().double()
    return h, ((y / s).round().clamp(-128, 127) * s).bfloat16()


def _rotate(x, positions, cos_sin, interleaved):
    """x [tokens, heads, d]: the first `rot` elements rotated, in 64 bits (they decide codes), rounded once."""
    rot = cos_sin.shape[1]
    cs = cos_sin[positions].double()[:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    r = x[..., :rot].double()
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r.to(x.dtype), x[..., rot:]), -1)


def _attend(st):
    case, q = st["case"], st["q"]
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["d"], case["page"]
    b, longest, rows, g = case["batch"], max(st["lens"]), max(st["new"]), hq // hk
    lens = st["seq_lens"].long()
    starts = st["starts"].long() if st["starts"] is not None else torch.arange(b + 1, device=q.device)
    new = starts[1:] - starts[:-1]
    nblk = -(-longest // 16)
    blk = torch.arange(nblk, device=q.device)
    pages = st["table"].long()[:, blk * 16 // page].clamp_min(0)
    blocks = st["cache"][pages, :, blk % (page // 16)]  # [b, nblk, hk, bytes]
    k, v = _unpack(blocks.flatten(0, 2), d, case["group"], q.dtype)
    fold = lambda x: x.view(b, nblk, hk, 16, d).permute(0, 2, 1, 3, 4).reshape(b, hk, nblk * 16, d).float()  # noqa: E731
    k, v = fold(k), fold(v)
    j, i = torch.arange(nblk * 16, device=q.device), torch.arange(rows, device=q.device)
    live = i[None] < new[:, None]
    at = (starts[:-1, None] + i[None]).clamp_max(q.shape[0] - 1)
    qp = q[at].float().view(b, rows, hk, g, d).permute(0, 2, 3, 1, 4)  # [b, hk, g, rows, d]
    sees = lens[:, None] - (new[:, None] - 1 - i[None] if case["causal"] else 0 * i[None])
    seen = j < sees[..., None]  # [b, rows, keys]
    s = torch.matmul(qp.flatten(2, 3), k.transpose(-1, -2)).view(b, hk, g, rows, -1) * st["scale"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    v = v.masked_fill(~(j < lens[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.flatten(2, 3), v).view(b, hk, g, rows, d).permute(0, 3, 1, 2, 4).reshape(b, rows, hq, d)
    return o[live].to(q.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        if own:
            mode = 2 if case["asym"] else 6
            h, codes, scales, zeros = _ops().woq_add_rmsnorm_quant(state["x"], state["residual"], state["gamma"], EPS, mode)
            values = torch.empty_like(h)
            if case["asym"]:
                codes = torch.sub(codes.view(torch.uint8), zeros[:, None])
            torch.mul(codes, scales[:, None], out=values)
        else:
            h, values = _norm(state["x"], state["residual"], state["gamma"], case["asym"])
        return {"sum": h, "values": values}
    if case["op"] == "append":
        hq, hk, d = case["q_heads"], case["kv_heads"], case["d"]
        q, k, v = state["qkv"].view(-1, hq + 2 * hk, d).split([hq, hk, hk], 1)
        if own:
            q = _ops().kv4_cache_append(state["cache"], k, v, state["slots"], q, state["positions"], state["cos_sin"],
                                        case["interleaved"])
            k, v = _ops().kv4_cache_read(state["cache"], state["slots"], d, q.dtype)
        else:
            q = _rotate(q, state["positions"], state["cos_sin"], case["interleaved"])
            k = _values(*_codes(_rotate(k, state["positions"], state["cos_sin"], case["interleaved"]), case["group"]))
            v = _values(*_codes(v, case["group"]))
        return {"query": q, "keys": k, "values": v}
    if own:
        return _ops().kv4_cache_attention(state["q"], state["cache"], state["table"], state["seq_lens"], state["starts"],
                                          state["scale"], case["causal"])
    return _attend(state)


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["k"]
        # x, residual read; sum and the codes' values written
        return {"bytes": 8 * n + 2 * case["k"], "flops": 10 * n}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["d"]
    row = 2 * hk * (d // 2 + 4 * (d // case["group"]))  # a token's keys and values in the cache
    if case["op"] == "append":
        n = case["tokens"]
        # q, k, v and the angles read; q, the cache's rows and what they stand for written
        return {"bytes": n * (2 * (hq + 2 * hk) * d + 4 * case["rot"] + 16 + 2 * (hq + 2 * hk) * d + row), "flops": n * (6 * (hq + hk) * d + 8 * hk * d)}
    new, lens = _lengths(case)
    seen = sum(n * (m - n) + n * (n + 1) // 2 if case["causal"] else n * m for n, m in zip(new, lens))
    return {"bytes": sum(lens) * row + 4 * sum(new) * hq * d, "flops": 4 * d * hq * seen}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        total = st["x"].double() + st["residual"].double()
        h = total.to(torch.bfloat16).to(torch.float64)
        root = torch.sqrt(torch.sum(h * h, 1) / h.shape[1] + EPS)
        y = (h / root[:, None] * st["gamma"].double()).to(torch.bfloat16).to(torch.float64)
        if case["asym"]:
            low, top = torch.min(y, 1).values, torch.max(y, 1).values
            step = ((top - low) / 255.0).float().double()
            zero = -torch.round(low / step)
            c = torch.clamp(torch.round(y / step[:, None] + zero[:, None]), 0, 255) - zero[:, None]
        else:
            step = (torch.max(torch.abs(y), 1).values / 127.0).float().double()
            c = torch.clamp(torch.round(y / step[:, None]), -128, 127)
        return {"sum": total, "values": c * step[:, None]}
    t, hq, hk, d, group, page = _type(case), case["q_heads"], case["kv_heads"], case["d"], case["group"], case["page"]
    if case["op"] == "append":
        if case["tokens"] * (hq + 2 * hk) * d > 90_000_000:
            return None
        x = st["qkv"].double().reshape(-1, hq + 2 * hk, d)
        half = case["rot"] // 2
        table = st["cos_sin"].double().index_select(0, st["positions"])
        z = torch.complex(table[:, :half], table[:, half:])[:, None]
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        turned = x[:, :hq + hk].clone()
        w = torch.complex(turned[..., first], turned[..., second]) * z
        turned[..., first], turned[..., second] = w.real.contiguous(), w.imag.contiguous()
        out = []
        for y in (turned[:, hq:].to(t).double(), x[:, hq + hk:]):
            y = y.reshape(-1, hk, d // group, group)
            low, top = torch.aminmax(y, dim=-1, keepdim=True)
            step = (top - low) / 15
            bits = 8 if t == torch.bfloat16 else 11  # digits of the scale; kept toward zero
            unit = torch.exp2(torch.clamp(torch.floor(torch.log2(step.clamp_min(1e-300))), min=-126.0 if bits == 8 else -14.0) - (bits - 1))
            step = torch.floor(step / unit) * unit
            c = torch.where(step > 0, torch.clamp(torch.round((y - low) / step), 0, 15), torch.zeros_like(y))
            out.append((c * step + low).reshape(-1, hk, d))
        return {"query": turned[:, :hq], "keys": out[0], "values": out[1]}
    new, lens = _lengths(case)
    if sum(n * m for n, m in zip(new, lens)) * hq * d > 3e12:
        return None
    out, at = [], 0
    for b, (n, m) in enumerate(zip(new, lens)):
        token = torch.arange(m, device="cuda")
        block = st["cache"][st["table"][b].long()[token // page], :, token % page // 16]  # [m, hk, bytes]
        pair = []
        for (byte, shift), p0 in zip(_places(d, "cuda"), (16 * d, 16 * d + 64 * (d // group))):
            r = token % 16
            c = torch.gather(block, 2, byte[r][:, None].expand(m, hk, d)).to(torch.int64) // (2 ** shift[r])[:, None] % 16
            every = block[:, :, p0:p0 + 64 * (d // group)].contiguous().view(t).view(m, hk, 16, d // group, 2)
            p = every[torch.arange(m, device="cuda"), :, r].double().repeat_interleave(group, 2)
            pair.append((c * p[..., 0] + p[..., 1]).to(t).double())
        k, v = pair
        rows = torch.arange(n, device="cuda")
        for h0 in range(hk):
            g = hq // hk
            qq = st["q"][at:at + n, h0 * g:(h0 + 1) * g].double().permute(1, 0, 2)
            s = torch.einsum("gnd,md->gnm", qq, k[:, h0]) * st["scale"]
            if case["causal"]:
                s = s.masked_fill(token[None, None] > (m - n + rows)[None, :, None], -math.inf)
            out.append(torch.einsum("gnm,md->ngd", torch.softmax(s, -1), v[:, h0]))
        at += n
        out[-hk:] = [torch.cat(out[-hk:], 1)]
    return torch.cat(out)
