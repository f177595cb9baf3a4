"""A paged key / value cache in 8 bits for serving MoBA models (no counterpart in the reference, which has no cache).

A page holds `page_size` consecutive tokens of one sequence and is the chunk that the gate selects.  Keys and values are held as
float8_e4m3fn or int8 with a scale for each (page, key head), a power of two; beside them lie what the gate scores, the mean of the
page's keys, and the attention weight that the page has received, by which pages are let go.  The kernels are those of csrc/kv_*.hip.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from flash_moba import flash_moba_hip as flash_moba_gpu
from flash_moba.rotary import flash_moba_rotary_func, rotary_form


class MobaKVCache(NamedTuple):
    """The tensors of a cache (all layers' caches are their own).  k and v may have any strides that are multiples of 16 with a
    dense last dimension, the others are dense.  Contents before a page's first token do not matter."""
    k: torch.Tensor                  # (pages, heads_k, page_size, head_size) float8_e4m3fn or int8
    v: torch.Tensor
    k_scale: torch.Tensor            # (pages, heads_k) fp32
    v_scale: torch.Tensor
    k_sum: torch.Tensor              # (pages, heads_k, head_size) fp32: sum of the page's keys, as they were given
    k_mean: torch.Tensor             # the same shape, fp16 / bf16 (the dtype of q, k and v): that sum over the page's tokens
    weight: Optional[torch.Tensor]   # (pages, heads_k) int64: attention weight received, in units of 2^-32; None: not kept

    @classmethod
    def allocate(cls, num_pages, page_size, num_heads_k, head_size, dtype=torch.bfloat16, cache_dtype=torch.float8_e4m3fn, device="cuda",
                 keep_weight=True):
        """An empty cache: page_size a multiple of 64 up to 1024, head_size of 16 up to 256, dtype that of q, k and v."""
        if dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError("FlashMoBA only supports fp16 and bf16 data types")
        if cache_dtype not in (torch.float8_e4m3fn, torch.int8):
            raise RuntimeError("a cache holds float8_e4m3fn or int8")
        if page_size < 64 or page_size > 1024 or page_size % 64 != 0:
            raise RuntimeError("page_size must be a multiple of 64 up to 1024")
        if head_size < 16 or head_size > 256 or head_size % 16 != 0:
            raise RuntimeError("head_size must be a multiple of 16 up to 256")
        rows, one = (num_pages, num_heads_k, head_size), (num_pages, num_heads_k)
        held = (num_pages, num_heads_k, page_size, head_size)
        return cls(torch.zeros(held, dtype=torch.int8, device=device).view(cache_dtype), torch.zeros(held, dtype=torch.int8, device=device).view(cache_dtype),
                   torch.ones(one, dtype=torch.float32, device=device), torch.ones(one, dtype=torch.float32, device=device),
                   torch.zeros(rows, dtype=torch.float32, device=device), torch.zeros(rows, dtype=dtype, device=device),
                   torch.zeros(one, dtype=torch.int64, device=device) if keep_weight else None)


# --------------------------------------------------------------------------------------
# custom ops, for traced graphs (eager calls go to the host module directly)
# --------------------------------------------------------------------------------------
@torch.library.custom_op("flash_moba::_cache_append", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale", "k_sum", "k_mean", "weight"), device_types="cuda")
def _cache_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k_sum: torch.Tensor,
                  k_mean: torch.Tensor, weight: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                  max_seqlen: int, seqlens_k: torch.Tensor, block_table: torch.Tensor) -> None:
    flash_moba_gpu.host_module().cache_append_op(k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight, k, v, cu_seqlens, max_seqlen, seqlens_k, block_table)


@torch.library.register_fake("flash_moba::_cache_append")
def _cache_append_fake(k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight, k, v, cu_seqlens, max_seqlen, seqlens_k, block_table):
    return None


@torch.library.custom_op("flash_moba::_cache_attn", mutates_args=("weight",), device_types="cuda")
def _cache_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k_sum: torch.Tensor,
                k_mean: torch.Tensor, weight: Optional[torch.Tensor], cu_seqlens_q: torch.Tensor, max_seqlen_q: int, seqlens_k: torch.Tensor,
                max_seqlen_k: int, block_table: torch.Tensor, topk: int, softmax_scale: Optional[float], add_weight: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return flash_moba_gpu.host_module().cache_attn_op(q, k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight, cu_seqlens_q, max_seqlen_q, seqlens_k,
                                                      max_seqlen_k, block_table, topk, softmax_scale, add_weight)


@torch.library.register_fake("flash_moba::_cache_attn")
def _cache_attn_fake(q, k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, topk,
                     softmax_scale, add_weight):
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


@torch.library.custom_op("flash_moba::_cache_evict", mutates_args=(), device_types="cuda")
def _cache_evict(weight: torch.Tensor, seqlens_k: torch.Tensor, block_table: torch.Tensor, page_size: int, keep: int, sink: int,
                 recent: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(flash_moba_gpu.host_module().cache_evict_op(weight, seqlens_k, block_table, page_size, keep, sink, recent))


@torch.library.register_fake("flash_moba::_cache_evict")
def _cache_evict_fake(weight, seqlens_k, block_table, page_size, keep, sink, recent):
    return (block_table.new_empty(block_table.shape), seqlens_k.new_empty(seqlens_k.shape), block_table.new_empty(block_table.shape),
            seqlens_k.new_empty(seqlens_k.shape))


# --------------------------------------------------------------------------------------
# public functions
# --------------------------------------------------------------------------------------
def flash_moba_cache_append_func(cache, k, v, cu_seqlens, max_seqlen, seqlens_k, block_table):
    """Writes new keys and values into the pages of a cache, in place, rounded to 8 bits.

    k, v: (tokens, num_heads_k, head_size) of the dtype of cache.k_mean, any strides; cu_seqlens: (batch + 1,) int32, which of them are whose;
    max_seqlen: the most that a sequence gets; seqlens_k: (batch,) int32, tokens of every sequence WITH the new ones, which are its
    last; block_table: (batch, n) int32, page of the tokens i * page_size and on of a sequence at [b, i].  A page may get
    tokens of one sequence only, and has one place in its table.

    The scale of a page and head is the least power of two (2^-64 to 2^64) that brings the largest finite magnitude among its tokens to
    448 (e4m3) or 127 (int8) at most; infinities are held as that, NaN as NaN (int8: 0).  Where a later token needs a larger scale, the
    page's earlier tokens are rounded again.  Places behind the end of a sequence, tokens before its beginning and table entries
    that are no page (outside [0, pages)) are left alone.  A page's first token starts its sum and its weight anew.

    Tokens are taken back (drafts that were refused) by smaller lengths: what is appended next lies over them.  k_sum of a page that had
    tokens before them still has them, though, as nothing says how many it has summed: put back what cache.k_sum[page] was before they
    came, and append again those of them that stay.  (The page's scale stays as large as they made it.)
    """
    if not torch.compiler.is_compiling() and flash_moba_gpu.host_module().cache_append(cache, k, v, cu_seqlens, max_seqlen, seqlens_k, block_table):
        return
    torch.ops.flash_moba._cache_append(*cache, k, v, cu_seqlens, max_seqlen, seqlens_k, block_table)


def flash_moba_cache_attn_func(q, cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, softmax_scale=None,
                               add_weight=False, return_lse=False):
    """MoBA attention of the last tokens of every sequence over a cache: decode steps, drafts, parts of prompts, whole prompts.

    q: (tokens, num_heads, head_size) of the dtype of cache.k_mean, any strides, num_heads a multiple of the cache's heads;
    cu_seqlens_q: (batch + 1,) int32; max_seqlen_q: the most rows of a sequence; seqlens_k, block_table: as for
    flash_moba_cache_append_func (the rows' own keys are in the cache already); max_seqlen_k: at least the longest of seqlens_k.

    Row i of a sequence has position seqlens_k - rows + i.  It sees, up to its position, the keys of its own page and of the
    moba_topk - 1 (at most 63) pages before it whose mean key has the largest product with it, decided as in 64 bits, of equals the
    later page; a product that is NaN or -inf selects nothing, and neither does a table entry that is no page.
    softmax_scale defaults to head_size ** -0.5.  Rows that see no key produce 0 (and a log-sum-exp of +inf).  A value that is NaN makes
    its feature NaN for every row that sees it, whatever its weight.

    With add_weight=True the part of a row's softmax that a page holds is added to cache.weight (64-bit integers in units of 2^-32, so that
    the sums do not depend on an order), which flash_moba_cache_evict_func chooses by.

    Returns out, like q; with return_lse=True (out, softmax_lse (num_heads, tokens) fp32).  No backward pass.
    """
    res = None
    if not torch.compiler.is_compiling():
        res = flash_moba_gpu.host_module().cache_attn(q, cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, softmax_scale, add_weight)
    if res is None:
        res = torch.ops.flash_moba._cache_attn(q, *cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, softmax_scale, add_weight)
    return res if return_lse else res[0]


def flash_moba_with_cache_func(q, k, v, cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, positions=None,
                               sections=None, base=10000.0, rotary_dim=None, interleaved=False, softmax_scale=None, add_weight=False,
                               return_lse=False):
    """A serving step end to end: rotary positions on q and k (with `positions`, as flash_moba_rotary_func), the keys and values of the
    tokens into the cache (as flash_moba_cache_append_func), attention of the tokens over it (as flash_moba_cache_attn_func).  An eager
    call on ordinary tensors that is refused, for want of memory too, has left the cache as it was."""
    if positions is not None:
        positions, sections, rotary_dim = rotary_form(q, positions, sections, rotary_dim)
    if not torch.compiler.is_compiling():
        res = flash_moba_gpu.host_module().cache_step(q, k, v, cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, positions,
                                                      sections or (), base, rotary_dim or 0, interleaved, softmax_scale, add_weight)
        if res is not None:
            return res if return_lse else res[0]
    if q.shape[0] != k.shape[0]:
        raise RuntimeError("q, k and v must be of the same tokens")
    if positions is not None:
        q, k = flash_moba_rotary_func(q, k, positions, sections, base, rotary_dim, interleaved)
    flash_moba_cache_append_func(cache, k, v, cu_seqlens_q, max_seqlen_q, seqlens_k, block_table)
    return flash_moba_cache_attn_func(q, cache, cu_seqlens_q, max_seqlen_q, seqlens_k, max_seqlen_k, block_table, moba_topk, softmax_scale, add_weight, return_lse)


def flash_moba_cache_evict_func(weight, seqlens_k, block_table, page_size, keep_pages, sink_pages=1, recent_pages=1):
    """Which pages every sequence keeps when it has more than `keep_pages`: the first `sink_pages`, the last `recent_pages` (at
    least 1, the page that is being filled), and of the others those that received most attention weight (cache.weight, summed over
    heads; of equals the first).  Sequences with fewer pages keep all.  A table entry that is no page has no weight, and is
    let go as it stands.

    Returns (block_table, seqlens_k, freed, num_freed): the table of the pages kept, in order, and -1 behind them; the tokens
    that are left; the pages let go in the same form, and how many they are.  The cache itself stays as it is: the freed pages can be given out again
    at once.  Keys keep the positions that they were turned by, so rotary positions go on counting from the sequence's own length.
    """
    if not torch.compiler.is_compiling():
        res = flash_moba_gpu.host_module().cache_evict(weight, seqlens_k, block_table, page_size, keep_pages, sink_pages, recent_pages)
        if res is not None:
            return res
    return torch.ops.flash_moba._cache_evict(weight, seqlens_k, block_table, page_size, keep_pages, sink_pages, recent_pages)
