"""What one form of the attention has no launch grid for takes the other, and what neither has is known before anything runs."""
import ctypes

import pytest
import torch

import cache_reference as R
import flash_moba
from flash_moba import flash_moba_hip as H
from test_gpu_kv_append import cache_struct
from test_gpu_kv_attn import check, setup

gpu = pytest.mark.gpu


def attn_args(cache, **kw):
    a = H.CacheAttnArgs()
    a.cache = cache
    a.q = a.out = a.softmax_lse = a.cu_seqlens_q = a.seqlens_k = a.block_table = a.workspace = 4096
    a.batch, a.total_q, a.heads, a.max_seqlen_q, a.max_seqlen_k, a.max_pages, a.topk, a.table_stride = 2, 16, 4, 8, 500, 8, 3, 8
    a.softmax_scale, a.workspace_bytes = 0.1, 1 << 50
    for n in ("q_row_stride", "q_head_stride", "o_row_stride", "o_head_stride"):
        setattr(a, n, 64)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_the_check_says_what_the_call_would():
    lib = H.load_library()
    ok = lambda **kw: lib.fmoba_cache_attn_check(ctypes.byref(attn_args(cache_struct(heads_k=kw.pop("heads_k", 2)), **kw)))  # noqa: E731
    assert lib.fmoba_cache_attn_check(None) != 0
    assert ok() == 0 and ok(total_q=0) == 0
    for kw, message in [(dict(topk=65), b"moba_topk"), (dict(heads=3), b"divide"), (dict(workspace=4100), b"workspace"),
                        (dict(batch=8400, heads_k=1, heads=64, total_q=8400 * 16, max_seqlen_q=16, max_seqlen_k=64 * 2000, max_pages=2000), b"rows times heads for the launch grid"),
                        (dict(batch=3000, heads_k=32, heads=32, total_q=3000, max_seqlen_q=1, max_seqlen_k=64 * 33000, max_pages=33000), b"sequences times heads, for the launch grid")]:
        assert ok(**kw) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
        assert lib.fmoba_cache_attn(ctypes.byref(attn_args(cache_struct(heads_k=kw.pop("heads_k", 2)), **kw)), None) != 0
    # 131072 rows of 128 sequences, 32 heads of their own, the longest of 262144 tokens: a workgroup a page would be 2^32 threads, so a row and head each
    big = dict(batch=128, heads_k=32, heads=32, total_q=131072, max_seqlen_q=131072, max_seqlen_k=262144, max_pages=4096, topk=8)
    assert ok(**big) == 0
    # and 300000 rows of 64 heads, which are 2^33 threads of a workgroup each: shared pages, though a page is selected twice on average
    assert ok(batch=1, heads_k=64, heads=64, total_q=300000, max_seqlen_q=300000, max_seqlen_k=64 * 30000, max_pages=30000, topk=1) == 0


@gpu
def test_where_a_workgroup_a_page_does_not_fit_the_grid_rows_read_their_own():
    """More sequences times pages than 2^32 threads, with rows enough for the form that shares pages: only a few pages are there."""
    batch, heads, dim, P, cols = 8400, 8, 16, 64, 2000
    lens_q = [0] * (batch - 3) + [300000, 1, 2]
    cache, _, q, _ = setup(heads, 1, dim, P, [300003], [P * 8], torch.bfloat16, torch.int8)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((batch, cols), -1, **i32)
    table[-3:, -8:] = torch.arange(8, **i32)
    cu = torch.tensor([0] + lens_q, **i32).cumsum(0, dtype=torch.int32)
    lens = torch.full((batch,), cols * P, **i32)
    args = (cu, 300000, lens, cols * P, table, 64)
    rows = [0, 150000, 299599, 299999, 300000, 300002]
    out, lse = flash_moba.flash_moba_cache_attn_func(q, cache, *args, return_lse=True)
    s = R.state(cache)
    for t in rows:
        length = cols * P if t >= 300000 else cols * P - (299999 - t)
        length -= 1 if t == 300001 else 0
        want, want_lse, _, sizes = R.attention(s, q[t:t + 1].cpu(), [0, 1], [length], [table[-1].tolist()], 64)
        check(out[t:t + 1], lse[:, t:t + 1], want, want_lse, sizes, False)
