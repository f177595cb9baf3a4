"""A serving step that is refused leaves the cache as it was, and what one form of the attention has no launch grid for takes the other."""
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
                        (dict(batch=1, heads_k=1, heads=1, total_q=(1 << 30) + (1 << 20), max_seqlen_q=(1 << 30) + (1 << 20)), b"too many rows"),
                        (dict(batch=3000, heads_k=32, heads=32, total_q=3000, max_seqlen_q=1, max_seqlen_k=64 * 33000, max_pages=33000), b"sequences times heads, for the launch grid")]:
        assert ok(**kw) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
        assert lib.fmoba_cache_attn(ctypes.byref(attn_args(cache_struct(heads_k=kw.pop("heads_k", 2)), **kw)), None) != 0
    # 131072 rows of 128 sequences, 32 heads of their own, the longest of 262144 tokens: a workgroup a page would be 2^32 threads, so a row and head each
    big = dict(batch=128, heads_k=32, heads=32, total_q=131072, max_seqlen_q=131072, max_seqlen_k=262144, max_pages=4096, topk=8)
    assert ok(**big) == 0
    # and 300000 rows of 64 heads, which are 2^33 threads of a workgroup each: shared pages, though a page is selected twice on average
    assert ok(batch=1, heads_k=64, heads=64, total_q=300000, max_seqlen_q=300000, max_seqlen_k=64 * 30000, max_pages=30000, topk=1) == 0


def test_the_largest_length_is_a_length():
    lib = H.load_library()
    need = [lib.fmoba_cache_attn_workspace_bytes(ctypes.byref(attn_args(cache_struct(), total_q=4096, max_seqlen_q=4096, max_seqlen_k=n))) for n in (64 * 8, 2 ** 31 - 1)]
    assert need[0] == need[1] > 0


def step_inputs(batch, rows, heads, cols, positions):
    """Sequences of cols pages of 64, of which the table has the last page only."""
    P, dim = 64, 16
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = flash_moba.MobaKVCache.allocate(4, P, 1, dim)
    cache.k_sum.normal_()
    cache.weight.random_(0, 1 << 40)
    table = torch.full((batch, cols), -1, **i32)
    table[0, -1] = 2
    q = torch.randn((batch * rows, heads, dim), device="cuda", dtype=torch.bfloat16)
    k = torch.randn((batch * rows, 1, dim), device="cuda", dtype=torch.bfloat16)
    cu = torch.arange(batch + 1, **i32) * rows
    lens = torch.full((batch,), cols * P - 5, **i32)
    pos = torch.arange(batch * rows, device="cuda") if positions else None
    return cache, (q, k, k, cache, cu, rows, lens, cols * P, table, 1), dict(positions=pos, add_weight=True)


def unchanged(cache, before):
    return all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, before))


@gpu
@pytest.mark.parametrize("rows,heads,positions", [(16, 64, False), (16, 64, True), (8, 128, True)])
def test_a_step_refused_for_its_launch_grid_leaves_the_cache(rows, heads, positions):
    cache, args, kw = step_inputs(8400, rows, heads, 2000, positions)
    before = [t.clone() for t in cache]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="launch grid"):
            flash_moba.flash_moba_with_cache_func(*args, **kw)
    torch.cuda.synchronize()
    assert unchanged(cache, before)


@gpu
@pytest.mark.parametrize("rows,heads,positions", [(8192, 64, False), (4096, 64, True)])
def test_a_step_without_memory_leaves_the_cache_and_can_be_made_again(rows, heads, positions):
    cache, args, kw = step_inputs(1, rows, heads, 200, positions)
    args = args[:-1] + (64,)  # (top-k: a visit has a place in the workspace)
    flash_moba.flash_moba_cache_append_func(cache, args[1][:30], args[1][:30], torch.tensor([0, 30], dtype=torch.int32, device="cuda"), 30,
                                            torch.tensor([200 * 64 - 20], dtype=torch.int32, device="cuda"), args[8])
    before = [t.clone() for t in cache]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (96 << 20)) / total)
        with pytest.raises(torch.OutOfMemoryError):
            flash_moba.flash_moba_with_cache_func(*args, **kw)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    torch.cuda.synchronize()
    assert unchanged(cache, before)
    twin = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    out = flash_moba.flash_moba_with_cache_func(*args, **kw)
    q, k = args[:2]
    if positions:
        q, k = flash_moba.flash_moba_rotary_func(q, k, kw["positions"])
    flash_moba.flash_moba_cache_append_func(twin, k, args[2], *args[4:7], args[8])
    assert torch.equal(out, flash_moba.flash_moba_cache_attn_func(q, twin, *args[4:], add_weight=True))
    assert unchanged(cache, twin)


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


@gpu
@pytest.mark.parametrize("pages", [6, 2100])
@pytest.mark.parametrize("rows", [3, 2100])
def test_rows_that_are_all_padding(rows, pages):
    """No sequence has a row, and max_seqlen_q says so: both forms, and the scores' own launch, would have an empty grid."""
    P, dim = 64, 32
    cache, table, q, _ = setup(4, 2, dim, P, [rows], [P * pages], torch.bfloat16, torch.int8)
    before = [t.clone() for t in cache]
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (torch.tensor([0, 0], **i32), 0, torch.tensor([P * pages], **i32), P * pages, torch.tensor(table, **i32), 3)
    out, lse = flash_moba.flash_moba_cache_attn_func(q, cache, *args, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isposinf(lse).all())
    out, lse = flash_moba.flash_moba_with_cache_func(q, q[:, :2], q[:, :2], cache, *args, positions=torch.arange(rows, device="cuda"), add_weight=True, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isposinf(lse).all()) and unchanged(cache, before)


def test_scratch_of_many_rows_is_bounded_by_what_rows_leave_behind():
    """The gate's scores are a gigabyte, however many rows there are: what a prompt needs more are its visits and a bit for every row and page."""
    lib = H.load_library()

    def scratch(rows, length, batch=1):
        pages = length // 128
        a = attn_args(cache_struct(page_size=128, heads_k=8, head_dim=128), batch=batch, heads=32, total_q=rows, max_seqlen_q=rows // batch, max_seqlen_k=length, max_pages=pages, topk=8)
        visits = rows * 32 * (8 * (128 * 2 + 8) + 8 * 4)
        bits = 32 * (rows // 32 + batch) * pages * 4
        return lib.fmoba_cache_attn_workspace_bytes(ctypes.byref(a)) - visits - bits

    for rows, length, batch in ((262144, 262144, 1), (524288, 524288, 1), (8192, 1 << 20, 1), (131072, 1 << 22, 1), (65536, 262144, 4)):
        assert 0 < scratch(rows, length, batch) <= (1 << 30) + (1 << 24), (rows, length)
    assert 0 <= scratch(65536, 131072) < 1 << 12  # 1024 pages: in LDS


@gpu
@pytest.mark.parametrize("pages,rows,heads", [(1100, [5300, 700], 24), (3000, [4000], 24)])
def test_blocks_of_rows_that_share_a_place_for_their_scores(pages, rows, heads):
    """More blocks of rows than workgroups of the gate."""
    P, dim = 64, 16
    lens = [P * pages - 3, P * 1040][:len(rows)]
    cache, table, q, cu = setup(heads, 1, dim, P, rows, lens, torch.bfloat16, torch.int8)
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (torch.tensor(cu, **i32), max(rows), torch.tensor(lens, **i32), max(lens), torch.tensor(table, **i32), 4)
    out, lse = flash_moba.flash_moba_cache_attn_func(q, cache, *args, return_lse=True)
    s = R.state(cache)
    for b, n in enumerate(rows):
        for first in (0, n // 2 // 32 * 32, n - 33):  # some blocks of every stretch
            t = slice(cu[b] + first, cu[b] + first + 33)
            want, want_lse, _, sizes = R.attention(s, q[t].cpu(), [0, 33], [lens[b] - n + first + 33], [table[b]], 4)
            check(out[t], lse[:, t], want, want_lse, sizes, True)
    whole = out.clone()
    assert torch.equal(whole, flash_moba.flash_moba_cache_attn_func(q, cache, *args))


@gpu
@pytest.mark.parametrize("traced", [False, True])
@pytest.mark.parametrize("positions", [False, True])
def test_a_step_has_the_keys_of_its_queries(positions, traced):
    """More or fewer keys than queries would be written at other positions than the queries have."""
    cache, args, kw = step_inputs(1, 5, 4, 6, positions)
    before = [t.clone() for t in cache]
    for n in (4, 6):
        k = torch.ones((n, 1, 16), device="cuda", dtype=torch.bfloat16)
        step = torch.compile(flash_moba.flash_moba_with_cache_func, backend="aot_eager") if traced else flash_moba.flash_moba_with_cache_func
        with pytest.raises(Exception, match="same tokens"):
            step(args[0], k, k, *args[3:], **kw)
    assert unchanged(cache, before)


@gpu
@pytest.mark.parametrize("start,draft,stay", [(70, 4, 2), (62, 4, 1), (62, 6, 3), (64, 3, 0), (1, 1, 0)])
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
def test_drafts_that_were_refused_are_taken_back(held, start, draft, stay):
    """Within a page, across a page's end, from a page's beginning: as if the refused tokens had never come."""
    P, dim = 64, 32
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[3, 0, 2]], **i32)
    g = torch.Generator(device="cuda").manual_seed(start)
    k, v, refused = (torch.rand((100, 2, dim), generator=g, device="cuda").bfloat16() + 1 for _ in range(3))
    caches = [flash_moba.MobaKVCache.allocate(4, P, 2, dim, cache_dtype=held) for _ in range(2)]

    def append(cache, k, v, length):
        flash_moba.flash_moba_cache_append_func(cache, k, v, torch.tensor([0, len(k)], **i32), len(k), torch.tensor([length], **i32), table)

    for cache in caches:
        append(cache, k[:start], v[:start], start)
    drafted, plain = caches
    page = table[0, (start - 1) // P]
    was = drafted.k_sum[page].clone()
    append(drafted, torch.cat([k[start:start + stay], refused[:draft - stay]]), torch.cat([v[start:start + stay], refused[:draft - stay]]), start + draft)
    drafted.k_sum[page] = was
    if stay:
        append(drafted, k[start:start + stay], v[start:start + stay], start + stay)
        append(plain, k[start:start + stay], v[start:start + stay], start + stay)
    for cache in caches:
        append(cache, k[start + stay:start + stay + 9], v[start + stay:start + stay + 9], start + stay + 9)
    end = start + stay + 9
    for c in range((end + P - 1) // P):
        n, at = min(P, end - c * P), table[0, c]
        for name in ("k", "v"):
            # the same, or at a scale that the refused ones enlarged: each is rounded once more at most, half a step of int8 or 2^-4 of it
            a, b = ((getattr(cache, name)[at, :, :n].double(), getattr(cache, name + "_scale")[at].double()[:, None, None]) for cache in caches)
            assert bool((a[1] >= b[1]).all())
            step = torch.where(a[1] == b[1], 0.0, (b[1] + a[1] / 2).expand_as(a[0]) if held == torch.int8 else 3 * 2.0 ** -4 * a[0].abs() * a[1])
            assert bool(((a[0] * a[1] - b[0] * b[1]).abs() <= step).all()), name
        for name in ("k_sum", "k_mean"):
            assert torch.equal(getattr(drafted, name)[at], getattr(plain, name)[at]), name


@gpu
@pytest.mark.parametrize("rows,pages", [(2, 20), (1100, 20), (2, 2100), (1100, 1100)])
def test_lengths_may_be_said_to_be_anything(rows, pages):
    """max_seqlen_k (and max_seqlen_q) of 2^31 - 1, as a program that captures its steps once for all lengths says."""
    P, dim, most = 64, 32, 2 ** 31 - 1
    cache, table, q, cu = setup(2, 1, dim, P, [rows], [P * pages - 9], torch.bfloat16, torch.int8)
    i32 = dict(dtype=torch.int32, device="cuda")
    args = torch.tensor(cu, **i32), torch.tensor([P * pages - 9], **i32), torch.tensor(table, **i32)
    k, v = (torch.randn((rows, 1, dim), device="cuda").bfloat16() for _ in range(2))
    twin = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    want, want_lse = flash_moba.flash_moba_with_cache_func(q, k, v, cache, args[0], rows, args[1], P * pages, args[2], 5, add_weight=True, return_lse=True)
    out, lse = flash_moba.flash_moba_with_cache_func(q, k, v, twin, args[0], most, args[1], most, args[2], 5, add_weight=True, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and unchanged(cache, twin) and bool((want != 0).any())
