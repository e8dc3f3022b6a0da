"""The 8-bit key/value cache: paged e4m3 codes with one scale per block of tokens and head, and the operators on it.

A value is its code times the scale of its block and head. Scales are powers of two, 2^(e - 7) for a block whose largest magnitude
lies in [2^e, 2^(e+1)) and at least 2^-60 (0: nothing but zeros). e4m3 is a floating format, so a power of two costs no precision,
a block whose scale grows keeps its older codes bit for bit down to its smallest normal value, and codes move between blocks
exactly. NaN is stored as NaN; infinities count as the largest finite bf16 value. Attention takes blocks whose value scales lie up to
2^100 apart in one row (those of zeros count as 2^-80).

Sequences are given as everywhere in ``ops``: ``block_table`` int32 [sequences, blocks], ``ctx_lens`` int32 the tokens a sequence
holds with the call's rows, ``cu_q`` int32 [sequences + 1] bounds of its rows, which are the last of its tokens. On CUDA every
call enqueues on the current stream, takes its scratch from the allocator (calls on other streams and captured graphs share none)
and checks shapes, types and devices; what is wrong with them raises ValueError. What lies in tensors is checked by the kernels, which
record it in the workspace's status word: table entries outside the cache are not followed, attention leaves out a sequence whose rows or
length do not fit the call or its table and adds nothing to sums that are shorter than the length, eviction takes a length only as far as
table and sums reach. CPU tensors run the float32 forms of ``ops.reference``, where such a length raises ValueError.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import reference as _ref
from . import sm100 as _sm


class Kv8Cache:
    """``k`` float8_e4m3fn [blocks, kv heads, page, head size], ``v`` likewise with its own head size, ``k_scale`` and ``v_scale``
    float32 [blocks, kv heads], powers of two or 0."""

    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, n_blocks: int, page: int, kv_heads: int, dk: int, dv: Optional[int] = None, device="cpu") -> "Kv8Cache":
        def codes(d):
            return torch.zeros(n_blocks, kv_heads, page, d, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        s = torch.zeros(2, n_blocks, kv_heads, device=device)
        return cls(codes(dk), codes(dv or dk), s[0], s[1])

    @property
    def page(self) -> int:
        return self.k.shape[2]

    def copy_blocks(self, src, dst):
        """Blocks ``src`` (int64) to blocks ``dst``."""
        for t in (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale):
            t[dst] = t[src]

    def bytes_per_block(self) -> int:
        return self.k[0].numel() + self.v[0].numel() + 8 * self.k.shape[1]


def _check(cache: Kv8Cache, who: str):
    k, v = cache.k, cache.v
    if k.is_cuda:
        raise ValueError(f"{who}: tensors on different devices")
    if k.dim() != 4 or v.dim() != 4 or k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn or k.shape[:3] != v.shape[:3]:
        raise ValueError(f"{who}: codes are float8_e4m3fn [blocks, kv heads, page, head size]")
    for s in (cache.k_scale, cache.v_scale):
        if s.dtype != torch.float32 or s.shape != k.shape[:2]:
            raise ValueError(f"{who}: scales are float32 [blocks, kv heads]")


def _sizes(cache: Kv8Cache, rows, block_table, who: str):
    """(sequences, table width, kv heads, page, dk, dv) and the sizes of ``rows``: what the front ends rely on. The extension checks
    the rest."""
    try:
        n, width = block_table.shape
        _, kv, page, dk = cache.k.shape
        _, _, _, dv = cache.v.shape
        _, heads, cols = rows.shape
    except ValueError:
        raise ValueError(f"{who}: codes are [blocks, kv heads, page, head size], block tables [sequences, blocks], rows or sums have three "
                         "dimensions") from None
    if kv < 1 or page < 1 or heads < 1:
        raise ValueError(f"{who}: a cache and rows without heads or cells")
    return n, width, kv, page, dk, dv, heads, cols


def _check_lengths(cache: Kv8Cache, block_table, ctx_lens, has_rows, weights, who: str):
    n = int(torch.where(has_rows, ctx_lens, torch.zeros_like(ctx_lens)).amax()) if ctx_lens.numel() else 0
    if n > block_table.shape[1] * cache.page:
        raise ValueError(f"{who}: lengths beyond the block table")
    if weights is not None and n > weights.shape[2]:
        raise ValueError(f"{who}: lengths beyond the sums of weights")


def _check_weights(w, cache: Kv8Cache, block_table, who: str):
    if w.dim() != 3 or w.dtype != torch.float32 or w.shape[:2] != (block_table.shape[0], cache.k.shape[1]):
        raise ValueError(f"{who}: sums of weights are float32 [sequences, kv heads, keys]")


def kv8_append(cache: Kv8Cache, k, v, block_table, ctx_lens, cu_q, max_q_len: int) -> None:
    """Writes the rows' keys and values (``k`` [T, kv heads, dk], ``v`` [T, kv heads, dv], rows and heads may lie apart) to the
    cache. A block that gets its first cell begins anew: its other cells become zero. In others the scale grows where a new value
    needs it, and the older codes are rounded to it. A block that gets tokens belongs to one sequence of the call. Rows at positions
    that the table has no block for are left out."""
    if k.is_cuda or cache.k.is_cuda:
        _sm.ext().kv8_append(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, block_table, ctx_lens, cu_q, max_q_len,
                             _sm.Workspace.get(cache.k.device).status)
        return
    _check(cache, "kv8_append")
    if k.dim() != 3 or v.dim() != 3 or k.shape[:2] != v.shape[:2] or k.shape[1:] != cache.k.shape[1::2] or v.shape[1:] != cache.v.shape[1::2]:
        raise ValueError("kv8_append: rows [T, kv heads, head size] do not fit the cache")
    _ref.kv8_append(cache, k, v, block_table, ctx_lens, cu_q)


@functools.lru_cache(maxsize=4096)
def _prompt_splits(n: int, kv_heads: int, rows: int, row_tile: int, tiles: int) -> int:
    """Parts of a prompt call's keys: as many as make the waves of CTAs times their tiles (and what a part costs beside them)
    least."""
    ctas = n * kv_heads * -(-rows // row_tile)
    best, cost = 1, None
    for s in range(1, min(32, tiles) + 1):
        c = -(-ctas * s // _sm.NUM_SMS) * (-(-tiles // s) + (4 if s == 1 else 7))
        if cost is None or c < cost:
            best, cost = s, c
    return best


def kv8_attention(q, cache: Kv8Cache, block_table, ctx_lens, cu_q, max_q_len: int, scale: float, window: int = 0, softcap: float = 0.0,
                  sink=None, weights=None, observe: int = 0, max_ctx: Optional[int] = None, out=None):
    """Causal attention of the query rows ``q`` [T, heads, dk] over the cache; returns [T, heads, dv] (``out`` takes it; its rows
    may lie apart). ``window`` > 0: the last that many keys are visible; ``softcap`` > 0: scores become softcap * tanh(score /
    softcap); ``sink`` [heads] float32: exp(sink) joins the denominator. A row that sees no key is zero. ``max_q_len`` == 1 selects
    the decode kernel. ``max_ctx``: bound of the lengths, for the split over the keys (None: the table's).

    ``weights`` float32 [sequences, kv heads, >= longest context]: every key's softmax weight, summed over the query heads that
    share its head and over the sequence's last ``observe`` rows (0: all of the call), is added to its sum: what ``kv8_evict`` goes
    by. The sums do not depend on the order of anything but the rows. A decode call with sums takes 4 bytes of scratch per row, head
    and key up to ``max_ctx``."""
    n, width, kv, page, dk, dv, heads, cols = _sizes(cache, q, block_table, "kv8_attention")
    if not q.is_cuda:
        _check(cache, "kv8_attention")
        if cols != dk or heads % kv:
            raise ValueError("kv8_attention: queries [T, heads, head size] do not fit the cache")
        if window < 0 or softcap < 0:
            raise ValueError("kv8_attention: window and soft cap are not negative")
        if weights is not None:
            _check_weights(weights, cache, block_table, "kv8_attention")
            if observe < 0:
                raise ValueError("kv8_attention: observed rows are not negative")
        _check_lengths(cache, block_table, ctx_lens, cu_q[1:] > cu_q[:-1], weights, "kv8_attention")
        o = _ref.kv8_attention(q, cache, block_table, ctx_lens, cu_q, scale, window, softcap, sink, weights, observe)
        return o if out is None else out.copy_(o)
    if out is None:
        out = torch.empty(q.shape[0], heads, dv, dtype=q.dtype, device=q.device)
    tiles = max(1, -(-min(max_ctx or 1 << 30, width * page) // 128))
    if window > 0 and max_q_len == 1:
        tiles = min(tiles, -(-window // 128) + 1)
    group = heads // kv
    if max_q_len == 1:
        splits = min(_sm.NUM_SMS, n * kv * -(-group // (8 if group <= 8 else 16)) * tiles)      # CTAs
    else:
        rows = 256 if dk <= 128 and dv <= 128 else 128
        splits = _prompt_splits(n, kv, max_q_len * group, rows, tiles if window <= 0 else min(tiles, (window + max_q_len) // 128 + 1))
    _sm.ext().kv8_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, ctx_lens, cu_q, max_q_len, scale, window,
                            softcap, sink, splits, out, _sm.Workspace.get(q.device).status, weights, observe, tiles)
    # kernels beside the attention's own: the join of the parts, the sums (of prompt rows: their records first)
    _sm.LAUNCHES["n"] += (splits > 1) + (0 if weights is None else 1 if max_q_len == 1 else 2)
    return out


def kv8_evict(cache: Kv8Cache, block_table, ctx_lens, weights, budget: int, dst_table, keep_first: int = 0, keep_last: int = 0):
    """Keeps ``budget`` tokens of every sequence and kv head: the first ``keep_first``, the last ``keep_last`` and, of those between,
    the ones with the largest ``weights`` (as ``kv8_attention`` sums them up; equal ones: the earlier). They move in order to the
    blocks of ``dst_table`` int32 [sequences, >= budget / page], which no table of the call reads; a sequence that holds no more
    than the budget moves as it is. Keys keep the rotary positions that they were cached with.

    Returns (lengths int32 [sequences], the kept tokens' places before int32 [sequences, kv heads, budget], -1 behind the last, and
    their sums float32 likewise, 0 behind the last)."""
    B, _, kv, page, _, _, _, _ = _sizes(cache, weights, block_table, "kv8_evict")
    if budget < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget or dst_table.dim() != 2 \
            or dst_table.shape[0] != B or dst_table.shape[1] * page < budget:
        raise ValueError("kv8_evict: the budget holds the first and last tokens that stay, the blocks of the result hold the budget")
    if not weights.is_cuda:
        _check(cache, "kv8_evict")
        _check_weights(weights, cache, block_table, "kv8_evict")
        _check_lengths(cache, block_table, ctx_lens, torch.ones_like(ctx_lens, dtype=torch.bool), weights, "kv8_evict")
        return _ref.kv8_evict(cache, block_table, ctx_lens, weights, budget, dst_table, keep_first, keep_last)
    dev = weights.device
    lens = torch.empty(B, dtype=torch.int32, device=dev)
    kept = torch.empty(B, kv, budget, dtype=torch.int32, device=dev)
    sums = torch.empty(B, kv, budget, device=dev)
    _sm.ext().kv8_evict(cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, ctx_lens, weights, budget, keep_first, keep_last,
                        dst_table, lens, kept, sums, _sm.Workspace.get(dev).status)
    return lens, kept, sums
