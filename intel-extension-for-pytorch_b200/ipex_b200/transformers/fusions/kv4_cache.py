"""Paged key/value cache in 4 bits, between the q / k / v linears of a decoder layer and its output projection.

With 4-bit weights a decode step reads about as many bytes of a 16-bit cache as of weights once a batch holds some tens
of thousands of tokens; here a token and head take D + 8 D / group_size bytes instead of 4 D.  Keys are rotated on the
way in, and attention multiplies by the values that the cache stands for.  The reference's caches hold the activations'
type (csrc/cpu/aten/kernels/PagedAttentionKrnl.cpp); this one has no counterpart there."""
import torch

from ..._ops import load_ops


class _IPEXPagedKv4Cache:
    """`tensor`: uint8 [num_pages, kv_heads, page_size / 16, block bytes].  A slot is page * page_size + position in the
    page.  Which pages belong to a sequence is the caller's book-keeping (`block_table`).

    append(key, value, slots, ...) stores tokens, rotating keys (and returning rotated queries) by `positions` through
    `cos_sin` (fp32 [positions, rot]: rot / 2 cosines, then as many sines; `rotary_table` makes one).
    attention(query, block_table, seq_lens, ...) attends to the first seq_lens[b] tokens of every sequence.
    read(slots) gives back the keys and values that the cache stands for."""

    def __init__(self, num_pages, kv_heads, head_dim, page_size=64, group_size=64, dtype=torch.bfloat16, device="cuda"):
        load_ops()
        if head_dim not in (64, 128, 256) or group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError(f"the 4-bit cache has heads of 64, 128 or 256 elements and groups of 32, 64 or 128 within a "
                             f"head, got {head_dim} and {group_size}")
        if page_size <= 0 or page_size % 16 or num_pages < 0 or kv_heads < 1:
            raise ValueError(f"the 4-bit cache needs pages of a multiple of 16 tokens, num_pages >= 0 and a head, got "
                             f"{page_size}, {num_pages}, {kv_heads}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"the 4-bit cache stands for bf16 or fp16 values, got {dtype}")
        self.num_pages, self.kv_heads, self.head_dim = num_pages, kv_heads, head_dim
        self.page_size, self.group_size, self.dtype = page_size, group_size, dtype
        block = 16 * head_dim + 128 * (head_dim // group_size)
        self.tensor = torch.zeros(num_pages, kv_heads, page_size // 16, block, dtype=torch.uint8, device=device)

    @staticmethod
    def rotary_table(max_positions, rot, theta=10000.0, device="cuda"):
        """fp32 [max_positions, rot]; the angles are computed in 64 bits."""
        inv = theta ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
        angle = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * inv[None]
        return torch.cat((angle.cos(), angle.sin()), 1).float()

    def _check(self, t, what):
        if t.dtype != self.dtype or t.dim() != 3 or t.shape[2] != self.head_dim:
            raise ValueError(f"{what} must be [tokens, heads, {self.head_dim}] of {self.dtype}, got {list(t.shape)} of {t.dtype}")

    def append(self, key, value, slots, query=None, positions=None, cos_sin=None, interleaved=False):
        """Returns the rotated query, or None without one."""
        self._check(key, "key")
        q = torch.ops.torch_ipex.kv4_cache_append(self.tensor, key, value, slots, query, positions, cos_sin, interleaved)
        return None if query is None else q

    def attention(self, query, block_table, seq_lens, query_starts=None, scale=None, causal=True):
        self._check(query, "query")
        return torch.ops.torch_ipex.kv4_cache_attention(query, self.tensor, block_table, seq_lens, query_starts, scale, causal)

    def read(self, slots):
        return torch.ops.torch_ipex.kv4_cache_read(self.tensor, slots, self.head_dim, self.dtype)
