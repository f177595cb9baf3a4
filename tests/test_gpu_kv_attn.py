"""flash_moba_cache_attn_func (and the whole step) against its definition in 64 bits.

Which pages a row reads is decided as in 64 bits, so nothing is left out of the comparison for near-ties.  Error of an output: a score of D
products in 32 bits is off by at most (D + 8) 2^-24 of scale sum |q| |k| (8: the scales, the change of base and the exponential's argument), the exponential
by 2^-22, a sum of n weights by n 2^-24; weights are off by twice the first two, relatively, and an output by that times sum p |v|, and by half a
step of its type.  Where many rows share a page, its weights are rounded to fp16 (2^-11; weights below 2^-14 by 2^-25 of the largest), and its part of an
output to 32767ths of its largest feature: half a step of each of the parts, whose weights add up to 1, is up to max |v| 2^-16."""
import ctypes
import math

import pytest
import torch

import cache_reference as R
import flash_moba
from flash_moba import flash_moba_hip as H
from test_gpu_kv_append import BAD_CACHES, cache_struct, random_cache, tables

gpu = pytest.mark.gpu


def check(got, lse, want, want_lse, sizes, parts):
    size, dot, most, count = sizes
    D = got.shape[2]
    delta = ((D + 8) * 2.0 ** -24 * dot + 2.0 ** -22)
    weights = (2 * delta + count * 2.0 ** -24 + (2.0 ** -11 if parts else 0.0)).t()[:, :, None]
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 * 1.01 + size * weights + (((2.0 ** -25 * count + 2.0 ** -16 * 1.01) * most).t()[:, :, None] if parts else 0.0) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.float().cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"out {(err - tol).max().item():.3e} over, largest error {err.max().item():.3e}"
    lse = lse.cpu().double()
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    fine = torch.isfinite(want_lse)
    assert bool(((lse - want_lse).abs()[fine] <= (delta + count * 2.0 ** -24 + 2.0 ** -22 * want_lse.abs().clamp_min(1.0))[fine]).all()), (lse - want_lse).abs()[fine].max()


def filled_cache(pages, heads_k, P, dim, dtype, held, seed, layout="heads"):
    """Pages with means of their own, so that rows choose by them."""
    c = random_cache(pages, heads_k, P, dim, dtype, held, seed, layout)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    c.k_scale.copy_(torch.rand(c.k_scale.shape, generator=g, device="cuda") * 0.02 + 0.002)  # (not only powers of two)
    c.v_scale.copy_(torch.rand(c.k_scale.shape, generator=g, device="cuda") * 0.1 + 0.001)
    c.k_mean.normal_(generator=g)
    return c


def setup(heads, heads_k, dim, P, lens_q, lens_k, dtype, held, seed=1, layout="heads", spare=2):
    pages = sum((n + P - 1) // P for n in lens_k) + spare
    cache = filled_cache(pages, heads_k, P, dim, dtype, held, seed, layout)
    table = tables(lens_k, P, pages, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    q = torch.randn((sum(lens_q), heads, dim), generator=g, device="cuda").to(dtype)
    cu = [0]
    for n in lens_q:
        cu.append(cu[-1] + n)
    return cache, table, q, cu


def call(cache, table, q, cu, lens_k, topk, **kw):
    i32 = dict(dtype=torch.int32, device="cuda")
    lens_q = [b - a for a, b in zip(cu, cu[1:])]
    return flash_moba.flash_moba_cache_attn_func(q, cache, torch.tensor(cu, **i32), kw.pop("max_q", max(lens_q)), torch.tensor(lens_k, **i32), kw.pop("max_k", max(max(lens_k), 1)),
                                                 torch.tensor(table, **i32), topk, return_lse=True, **kw)


CASES = [  # heads, heads_k, dim, page, lens_q, lens_k, topk
    (1, 1, 16, 64, [1], [1], 1),
    (4, 1, 128, 128, [1, 1, 1], [1, 128, 1000], 3),
    (8, 8, 64, 64, [1, 0, 2], [700, 5, 641], 4),
    (6, 2, 80, 64, [3, 8], [129, 1500], 5),
    (4, 2, 256, 64, [5], [900], 64),
    (2, 1, 96, 1024, [2], [3000], 2),
    (2, 2, 48, 192, [1, 7], [64 * 40, 192 * 3], 7),
    (4, 4, 128, 128, [8], [8], 8),                   # a prompt of a few tokens
    (4, 2, 64, 64, [300], [300], 2),                 # whole prompts
    (4, 1, 128, 128, [70, 1, 0, 33], [500, 300, 9, 33], 3),
    (2, 2, 80, 64, [65, 64], [1000, 64], 9),
    (3, 3, 256, 128, [40], [700], 4),
    (8, 1, 32, 256, [50], [900], 1),                 # its own page alone
    (4, 2, 112, 64, [20, 9], [64 * 30, 64 * 21 + 1], 64),
    # 2048 rows times heads and more, whose pages are shared
    (4, 2, 64, 64, [600], [600], 2),
    (4, 1, 128, 128, [700, 1, 0, 33], [900, 300, 9, 33], 3),
    (2, 2, 80, 64, [1030, 64], [1500, 64], 9),
    (3, 3, 256, 128, [700], [1400], 4),
    (3, 1, 192, 64, [699], [700], 5),
    (8, 1, 32, 256, [300], [900], 1),
    (4, 2, 112, 64, [500, 30], [64 * 30, 64 * 21 + 1], 64),
    (16, 8, 64, 320, [130], [1500], 3),
    (32, 2, 128, 1024, [66], [3000], 2),
    (7, 1, 48, 192, [290, 7], [64 * 40, 192 * 3], 7),
    (2, 1, 16, 64, [5, 1100, 0, 40], [0, 1101, 77, 39], 17),
    (4, 2, 96, 384, [40, 500], [384 * 4, 901], 3),
    # and more steps of their pages than the last launch has places for
    (1, 1, 32, 256, [2200], [256 * 40 + 10], 40),
    (4, 1, 128, 1024, [3, 550], [1000, 1024 * 9 + 5], 9),
    (4, 4, 256, 128, [530], [128 * 34 - 1], 33),
]


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,heads_k,dim,P,lens_q,lens_k,topk", CASES)
def test_outputs_are_the_definitions(held, dtype, heads, heads_k, dim, P, lens_q, lens_k, topk):
    cache, table, q, cu = setup(heads, heads_k, dim, P, lens_q, lens_k, dtype, held, layout="tokens" if heads_k == 2 else "heads")
    s, before = R.state(cache), cache.weight.clone()
    out, lse = call(cache, table, q, cu, lens_k, topk, add_weight=True)
    want, want_lse, weight, sizes = R.attention(s, q.cpu(), cu, lens_k, table, topk)
    many = max(lens_q) > 8
    check(out, lse, want, want_lse, sizes, many)
    # weights: relatively as the outputs' weights, and half a unit for every visit
    got = (cache.weight - before).cpu().double() * 2.0 ** -32
    D = dim
    rel = 2 * ((D + 8) * 2.0 ** -24 * sizes[1].max().item() + 2.0 ** -22) + sizes[3].max().item() * 2.0 ** -24 + 2.0 ** -22
    rows = sum(lens_q) * heads
    assert bool(((got - weight).abs() <= weight * rel + rows * (P // 64) * 2.0 ** -33).all()), (got - weight).abs().max()
    # the same without weights, and once more: no bit differs
    out2, lse2 = call(cache, table, q, cu, lens_k, topk)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    w = cache.weight.clone()
    call(cache, table, q, cu, lens_k, topk, add_weight=True)
    assert torch.equal(cache.weight - w, w - before)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 40, 1100])
def test_long_contexts_with_many_pages(rows):
    """More pages than registers (256) and LDS (2048, 1024 where rows share pages) hold; few are read."""
    for n in (300, 2049, 2050, 5000) if rows <= 5 else (300, 1100, 2100):
        lens_k = [64 * n - 7]
        cache, table, q, cu = setup(2, 1, 16, 64, [rows], lens_k, torch.bfloat16, torch.int8, seed=n)
        out, lse = call(cache, table, q, cu, lens_k, 6)
        want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, table, 6)
        check(out, lse, want, want_lse, sizes, rows > 8)


@gpu
@pytest.mark.parametrize("n", [32768, 33000])
def test_the_longest_tables(n):
    """The most pages that rows share, and more, chosen by many rows (most of them are the same page, and worth nothing), and a bound on the rows that says nothing."""
    P, dim, rows = 64, 16, 2100
    cache, _, q, cu = setup(1, 1, dim, P, [rows], [P * 200], torch.bfloat16, torch.float8_e4m3fn)
    g = torch.Generator().manual_seed(8)
    table = [[200] * n]
    for i, c in enumerate(torch.randperm(n - 40, generator=g)[:160].tolist()):
        table[0][c] = i
    table[0][-40:] = list(range(160, 200))
    q.abs_()
    cache.k_mean.abs_()
    cache.k_mean[200] = -1.0
    cache.k[200] = 0
    lens_k = [P * n - 5]
    out, lse = call(cache, table, q, cu, lens_k, 64)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, table, 64)
    check(out, lse, want, want_lse, sizes, True)
    few, few_lse = call(cache, table, q[-2:], [0, 2], lens_k, 64, max_q=2 ** 31 - 1)
    check(few, few_lse, want[-2:], want_lse[:, -2:], tuple(x[-2:] if x.dim() == 3 else x[:, -2:] for x in sizes), False)


@gpu
@pytest.mark.parametrize("rows", [1, 20, 1100])
def test_ties_and_near_ties_are_decided_as_in_64_bits(rows):
    """Means that differ in the last bits of a sum: in 32 bits the order of its terms would decide.  Equal ones: the later page."""
    P, dim, n = 64, 64, 40
    cache, table, q, cu = setup(2, 1, dim, P, [rows], [P * n], torch.bfloat16, torch.float8_e4m3fn)
    base = torch.randn(dim, device="cuda").bfloat16()
    cache.k_mean[:] = base
    for c in range(0, n, 2):  # every other page: one feature by one step
        page, d = table[0][c], c % dim
        cache.k_mean[page, 0, d] = base[d].float() * (1 + 2.0 ** -7)
    # terms of very different sizes: 2^-10 to 2^10, products of 16 bits, 64 of them: 42 bits, so that 64-bit sums are exact
    q[:] = q[:1, :1] * 2.0 ** torch.linspace(-10, 10, dim, device="cuda").round()
    q[:, 1] = 0  # all scores equal
    kw = dict(softmax_scale=2.0 ** -30)  # every key of the pages chosen weighs the same
    w = cache.weight.clone()
    out, lse = call(cache, table, q, cu, [P * n], 5, add_weight=True, **kw)
    want, want_lse, weight, sizes = R.attention(R.state(cache), q.cpu(), cu, [P * n], table, 5, scale=2.0 ** -30)
    check(out, lse, want, want_lse, sizes, rows > 8)
    assert torch.equal((cache.weight > w).cpu(), weight > 0)


@gpu
@pytest.mark.parametrize("P", [64, 256])
@pytest.mark.parametrize("rows", [1, 33, 260])
def test_what_lies_behind_a_row_is_not_seen(rows, P):
    """NaN in places behind a sequence's end and behind a row, in pages that are no one's, and table entries that are no page."""
    dim = 64
    lens_k = [P * 5 + 40, 70]
    cache, table, q, cu = setup(4, 2, dim, P, [rows, rows], lens_k, torch.bfloat16, torch.float8_e4m3fn, spare=3)
    s = R.state(cache)
    want, want_lse, _, sizes = R.attention(s, q.cpu(), cu, lens_k, table, 3)
    out, lse = call(cache, table, q, cu, lens_k, 3)
    check(out, lse, want, want_lse, sizes, rows > 8)
    nan = float("nan")
    for b, n in enumerate(lens_k):
        for t in (cache.k, cache.v):
            t.view(torch.int8)[table[b][n // P], :, n % P:] = 0x7F
    used = {p for row in table for p in row}
    for page in set(range(cache.k.shape[0])) - used:
        cache.k.view(torch.int8)[page], cache.v.view(torch.int8)[page] = 0x7F, 0x7F
        cache.k_scale[page] = cache.v_scale[page] = cache.k_mean[page] = nan
    out2, lse2 = call(cache, table, q, cu, lens_k, 3)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # the last key of a sequence: its earlier rows do not see it
    last = lens_k[0] - 1
    cache.v.view(torch.int8)[table[0][last // P], :, last % P] = 0x7F
    cache.k.view(torch.int8)[table[0][last // P], :, last % P] = 0x7F
    out3, _ = call(cache, table, q, cu, lens_k, 3)
    assert torch.equal(out3[:rows - 1], out[:rows - 1]) and torch.equal(out3[rows:], out[rows:]) and bool(out3[rows - 1].isnan().all())
    # entries that are no page: not selected
    holes = [list(row) for row in table]
    holes[0][1], holes[0][3], holes[1][0] = -1, cache.k.shape[0], 1 << 30
    out4, lse4 = call(cache, holes, q[:, :], cu, lens_k, 3)
    cache.v.view(torch.int8)[table[0][last // P], :, last % P] = 0
    cache.k.view(torch.int8)[table[0][last // P], :, last % P] = 0
    out4, lse4 = call(cache, holes, q, cu, lens_k, 3)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, holes, 3)
    check(out4, lse4, want, want_lse, sizes, rows > 8)


@gpu
@pytest.mark.parametrize("heads", [2, 160])
def test_rows_that_see_nothing_and_lengths_that_do_not_fit(heads):
    P, dim = 64, 32
    cache, table, q, cu = setup(heads, 1, dim, P, [1, 12, 1], [1, 200, 64], torch.float16, torch.int8)
    lens = [0, 5, -3]  # no token, fewer tokens than rows, less than none
    out, lse = call(cache, table, q, cu, lens, 4, max_k=200)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens, table, 4)
    check(out, lse, want, want_lse, sizes, True)
    assert bool((out[:1] == 0).all()) and bool(torch.isinf(lse[:, 0]).all()) and bool((out[1:8] == 0).all())
    # rows, tables and lengths beyond what the call says: nothing outside is read, what fits is right
    a = call(cache, table, q, cu, [1, 200, 64], 4)
    b = call(cache, table, q, cu, [1, 10 ** 6, 64], 4, max_k=200)
    assert torch.equal(a[0][:1], b[0][:1]) and torch.equal(a[0][13:], b[0][13:])
    c = call(cache, table, q, cu, [1, 200, 64], 4, max_q=3)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, [1, 200, 64], table, 4)
    check(c[0][:4], c[1][:, :4], want[:4], want_lse[:, :4], tuple(x[:4] if x.dim() == 3 else x[:, :4] for x in sizes), heads > 2)  # (160 heads are 2240 rows and heads: pages are shared)
    assert bool((c[0][4:13] == 0).all())
    call(cache, table, q, [0, 100, 7, 900], [9, 200, 64], 4, max_k=200, max_q=12)
    call(cache, table, q, [-5, 3, 8, 14], [9, 200, 64], 4, max_k=200, max_q=12)
    torch.cuda.synchronize()
    i32 = dict(dtype=torch.int32, device="cuda")
    none = flash_moba.flash_moba_cache_attn_func(q[:0], cache, torch.tensor([0, 0], **i32), 0, torch.tensor([9], **i32), 9, torch.tensor([[0]], **i32), 4)
    assert none.shape == (0, heads, 32)
    empty = flash_moba.MobaKVCache.allocate(0, P, 1, dim, torch.float16, torch.int8)
    out, lse = call(empty, [[0], [0], [0]], q, cu, [1, 12, 1], 4)
    assert bool((out == 0).all()) and bool(torch.isinf(lse).all())
    out, lse = call(cache, [[], [], []], q, cu, [1, 12, 1], 4)
    assert bool((out == 0).all()) and bool(torch.isinf(lse).all())


@gpu
@pytest.mark.parametrize("rows,pages", [(2, 6), (30, 6), (1030, 30)])
def test_values_that_are_no_ordinary_numbers(rows, pages):
    P, dim = 64, 32
    cache, table, q, cu = setup(2, 2, dim, P, [rows], [64 * pages], torch.bfloat16, torch.float8_e4m3fn)
    q[0, 0, 0], q[1, 1, 3] = float("nan"), float("inf")
    cache.k_mean[table[0][2], 0, 5] = float("nan")   # selects nothing
    cache.k_mean[table[0][1], 0] = -float("inf")
    out, lse = call(cache, table, q, cu, [64 * pages], 3)
    assert bool(out[0, 0].isnan().all()) and bool(lse[0, 0].isnan())
    assert not bool(out[0, 1].isnan().any())
    clean = [i for i in range(rows) if i > 1]
    s = R.state(cache)
    s["k_mean"][table[0][1], 0] = -1e30  # (as a finite score below all others: five pages or more before a row, so it is never among the best 2)
    s["k_mean"][table[0][2], 0] = float("nan")
    qs = q.clone()
    qs[0], qs[1] = 0, 0
    qa = qs.abs()  # with it the product with -1e30 is negative, as with -inf
    out, lse = call(cache, table, qa, cu, [64 * pages], 3)
    want, want_lse, _, sizes = R.attention(s, qa.cpu(), cu, [64 * pages], table, 3)
    pick = lambda x: x[clean] if x.dim() == 3 else x[:, clean]  # noqa: E731
    if clean:
        check(out[clean], lse[:, clean], pick(want), pick(want_lse), tuple(map(pick, sizes)), rows > 8)


@gpu
@pytest.mark.parametrize("P", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40, 520])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales_of_any_sign_and_pages_without_any(scale, rows, P):
    cache, table, q, cu = setup(4, 2, 64, P, [rows], [P * 5 + 30], torch.bfloat16, torch.float8_e4m3fn)
    cache.k_scale[table[0][2]] = 0.0
    cache.v_scale[table[0][3]] = 0.0
    out, lse = call(cache, table, q, cu, [P * 5 + 30], 4, softmax_scale=scale)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, [P * 5 + 30], table, 4, scale=scale)
    check(out, lse, want, want_lse, sizes, rows > 8)


@gpu
def test_strides_scales_and_broadcast():
    P, dim = 128, 64
    lens_q, lens_k = [1, 2], [300, 1000]
    cache, table, q, cu = setup(4, 2, dim, P, lens_q, lens_k, torch.bfloat16, torch.int8)
    want, lse = call(cache, table, q, cu, lens_k, 3, softmax_scale=0.3)
    ref, ref_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, table, 3, scale=0.3)
    check(want, lse, ref, ref_lse, sizes, False)
    qkv = torch.zeros((3, 3, 4, dim), dtype=q.dtype, device="cuda")
    qkv[:, 0] = q
    assert torch.equal(call(cache, table, qkv[:, 0], cu, lens_k, 3, softmax_scale=0.3)[0], want)
    assert torch.equal(call(cache, table, q.transpose(1, 2).contiguous().transpose(1, 2), cu, lens_k, 3, softmax_scale=0.3)[0], want)
    wide = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    wide[:, :len(table[0])] = torch.tensor(table)
    i32 = dict(dtype=torch.int32, device="cuda")
    got = flash_moba.flash_moba_cache_attn_func(q, cache, torch.tensor(cu, **i32), 2, torch.tensor(lens_k, **i32), 10 ** 6, wide[:, :len(table[0]) + 1], 3, softmax_scale=0.3)
    assert torch.equal(got, want)
    moved = cache._replace(k=cache.k.transpose(1, 2).contiguous().transpose(1, 2), v=cache.v.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3))
    assert torch.equal(call(moved, table, q, cu, lens_k, 3, softmax_scale=0.3)[0], want)
    # a page of a shared beginning, in two sequences' tables
    table[1][0] = table[0][0]
    out, lse = call(cache, table, q, cu, lens_k, 3)
    ref, ref_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, table, 3)
    check(out, lse, ref, ref_lse, sizes, False)


@gpu
def test_a_cache_whose_offsets_pass_32_bits():
    """Pages strided so that the last ones lie more than 2^32 bytes away."""
    P, dim, pages = 64, 128, 9
    cache = filled_cache(pages, 1, P, dim, torch.bfloat16, torch.int8, 3)
    stride = 1 << 29
    big = torch.empty((pages - 1) * stride + P * dim, dtype=torch.int8, device="cuda")
    far = cache._replace(k=big.as_strided((pages, 1, P, dim), (stride, P * dim, dim, 1)), v=big.as_strided((pages, 1, P, dim), (stride, P * dim, dim, 1)))
    far.k.copy_(cache.k)
    near = cache._replace(v=cache.k.clone())
    q = torch.randn((1 + 30, 4, dim), device="cuda").bfloat16()
    table = [[8, 1, 0, 7], [6, 2, 5, 8]]
    a = call(far, table, q, [0, 1, 31], [250, 256], 3)
    b = call(near, table, q, [0, 1, 31], [250, 256], 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    many = torch.randn((1 + 600, 4, dim), device="cuda").bfloat16()  # (rows that share pages; the first ones see nothing)
    a = call(far, table, many, [0, 1, 601], [250, 256], 3)
    b = call(near, table, many, [0, 1, 601], [250, 256], 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and bool((a[0][400:] != 0).any())
    k = torch.randn((5, 1, dim), device="cuda").bfloat16() * 100
    i32 = dict(dtype=torch.int32, device="cuda")
    for c in (far, near):
        c = flash_moba.MobaKVCache(c.k, torch.empty((pages, 1, P, dim), dtype=torch.int8, device="cuda"), *[t.clone() for t in c[2:]])
        flash_moba.flash_moba_cache_append_func(c, k, k, torch.tensor([0, 5], **i32), 5, torch.tensor([250], **i32), torch.tensor([[1, 2, 3, 8]], **i32))
    assert torch.equal(far.k[8], near.k[8])


@gpu
@pytest.mark.parametrize("rows", [1, 12, 300])
def test_a_step_replays_from_graphs_that_run_side_by_side(rows):
    """Positions, append, attention and weights captured twice (two graphs of the same call share nothing but the cache of each) and replayed while tokens come."""
    P, dim, heads, heads_k = 64, 64, 4, 2
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = [200, 130]
    most = 400 + 4 * rows
    table = torch.tensor(tables([most, most], P, most // 25 + 4, 4), **i32)
    caches = [filled_cache(most // 25 + 4, heads_k, P, dim, torch.bfloat16, torch.float8_e4m3fn, 5) for _ in range(3)]
    cu = torch.tensor([0, rows, 2 * rows], **i32)
    seqlens = torch.tensor(lens, **i32)
    q, k, v = (torch.randn((2 * rows, h, dim), device="cuda").bfloat16() for h in (heads, heads_k, heads_k))
    positions = torch.arange(2 * rows, device="cuda")[None]

    def step(cache):
        return flash_moba.flash_moba_with_cache_func(q, k, v, cache, cu, rows, seqlens, most, table, 3, positions=positions, add_weight=True)

    torch.cuda.synchronize()
    graphs, held = [], []
    for cache in caches[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(cache))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for x in (q, k, v):
            x.normal_()
        positions += rows
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        want = step(caches[2])
        torch.cuda.synchronize()
        for out, cache in zip(held, caches):
            assert torch.equal(out, want), turn
            assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, caches[2])), turn
        seqlens += rows


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("sections", [None, (8, 12, 12)])
def test_a_program_that_serves(held, sections):
    """A prompt in two parts, decode steps, eviction, more decode steps, with the freed pages given out again: every step against the definition."""
    P, dim, heads, heads_k, topk = 64, 64, 8, 2, 3
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = flash_moba.MobaKVCache.allocate(12, P, heads_k, dim, torch.bfloat16, held)
    s, free, table, length, position = R.state(cache), list(range(12)), [], 0, 0
    g = torch.Generator(device="cuda").manual_seed(6)
    for rows in (150, 300, 1, 1, 60, "evict", 1, 1, 2, 70):  # 512 tokens, 8 pages, when 4 are kept
        if rows == "evict":
            got = flash_moba.flash_moba_cache_evict_func(cache.weight, torch.tensor([length], **i32), torch.tensor([table], **i32), P, 4, sink_pages=1, recent_pages=2)
            kept, lens, freed = R.evict(cache.weight.cpu(), [length], [table], P, 4, 1, 2)
            n = got[3].item()
            assert got[0][0, :len(kept[0])].tolist() == kept[0] and got[2][0, :n].tolist() == freed[0] and n == 4 and got[1].item() == lens[0]
            table, length, free = kept[0], lens[0], freed[0] + free
            continue
        length, position = length + rows, position + rows
        while len(table) * P < length:
            table.append(free.pop(0))
        q, k, v = (torch.randn((rows, h, dim), generator=g, device="cuda").bfloat16() for h in (heads, heads_k, heads_k))
        at = torch.arange(position - rows, position, device="cuda")
        at = at if sections is None else torch.stack([at, at % 7, at // 3])
        args = (torch.tensor([0, rows], **i32), rows, torch.tensor([length], **i32), length, torch.tensor([table], **i32), topk)
        out, lse = flash_moba.flash_moba_with_cache_func(q, k, v, cache, *args, positions=at, sections=sections, add_weight=True, return_lse=True)
        q, k = flash_moba.flash_moba_rotary_func(q, k, at, sections)
        R.append(s, k.cpu(), v.cpu(), [0, rows], [length], [table])
        for name in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(cache, name).float().cpu().double(), s[name]), name
        s["k_mean"] = cache.k_mean.float().cpu().double()  # (rounded to 16 bits: what the gate reads)
        want, want_lse, weight, sizes = R.attention(s, q.cpu(), [0, rows], [length], [table], topk)
        check(out, lse, want, want_lse, sizes, rows > 8)
        s["weight"] = s["weight"] + (weight * 2.0 ** 32).round().long()
    assert bool(((cache.weight.cpu() - s["weight"]).abs() <= s["weight"].abs().double() * 1e-4 + 2.0 ** 12).all())


@gpu
@pytest.mark.parametrize("dtype,held", [(torch.bfloat16, torch.int8), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("dim,rotary_dim,sections,interleaved", [(64, None, None, False), (64, 40, None, False), (128, 64, (8, 12, 12), False), (256, None, None, True), (96, 48, (4, 20), True),
                                                                 (16, 8, None, False)])
def test_a_step_is_its_parts(dtype, held, dim, rotary_dim, sections, interleaved):
    """Positions on the way into the cache: the bits of the three functions one after the other; tokens across a page's end, of no sequence, and before a sequence's beginning."""
    P, heads, heads_k = 64, 6, 2
    i32 = dict(dtype=torch.int32, device="cuda")
    new, lens_k = [1, 8, 0, 3, 5, 1], [1, 131, 70, 66, 3, 128]
    cache, table, q, cu = setup(heads, heads_k, dim, P, new + [2], lens_k, dtype, held)
    cu = cu[:-1]
    other = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    g = torch.Generator(device="cuda").manual_seed(11)
    kv = torch.randn((sum(new) + 2, 2, heads_k, dim), generator=g, device="cuda").to(dtype)  # (strided: both in one tensor)
    k, v = kv[:, 0], kv[:, 1]
    at = torch.randint(0, 10 ** 6, (len(sections) if sections else 1, sum(new) + 2), generator=g, device="cuda")
    turn = dict(sections=sections, base=5e5, rotary_dim=rotary_dim, interleaved=interleaved)
    for positions in (at, at.int()):
        args = (torch.tensor(cu, **i32), 8, torch.tensor(lens_k, **i32), max(lens_k), torch.tensor(table, **i32), 3)
        out, lse = flash_moba.flash_moba_with_cache_func(q, k, v, cache, *args, positions=positions, add_weight=True, return_lse=True, **turn)
        tq, tk = flash_moba.flash_moba_rotary_func(q, k, positions, sections, 5e5, rotary_dim, interleaved)
        flash_moba.flash_moba_cache_append_func(other, tk, v, args[0], 8, args[2], args[4])
        want, want_lse = flash_moba.flash_moba_cache_attn_func(tq, other, *args, add_weight=True, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, other))


@gpu
def test_step_and_attention_from_traced_graphs():
    P, dim = 64, 32
    cache, table, q, cu = setup(4, 2, dim, P, [3], [200], torch.bfloat16, torch.int8)
    other = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.randn((3, 2, dim), device="cuda").bfloat16()
    pos = torch.arange(3, device="cuda")
    args = (torch.tensor(cu, **i32), 3, torch.tensor([200], **i32), 200, torch.tensor(table, **i32), 3)

    def step(q, k, *tensors):
        return flash_moba.flash_moba_with_cache_func(q, k, k, flash_moba.MobaKVCache(*tensors), *args, positions=pos, add_weight=True, return_lse=True)

    got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, *cache)
    want = step(q, k, *other)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(a, b) for a, b in zip(cache, other))


@gpu
@pytest.mark.parametrize("change,message", [
    (dict(q=lambda q: q.half()), "dtype"), (dict(q=lambda q: q[:, :3]), "divide"), (dict(q=lambda q: q[..., :16]), "head size"), (dict(q=lambda q: q.clone().requires_grad_(True)), "no backward"),
    (dict(topk=0), "moba_topk"), (dict(topk=65), "moba_topk"), (dict(max_k=-1), "out of range"), (dict(cache=lambda c: c._replace(weight=None)), "keeps no weight"),
    (dict(cache=lambda c: c._replace(k=c.k.cpu(), v=c.v.cpu())), ""), (dict(table=lambda t: t.float()), "block_table"), (dict(lens=lambda t: t[:0]), "seqlens_k"),
])
def test_refusals(change, message):
    cache = flash_moba.MobaKVCache.allocate(3, 64, 2, 32)
    i32 = dict(dtype=torch.int32, device="cuda")
    a = dict(q=torch.zeros((4, 4, 32), dtype=torch.bfloat16, device="cuda"), lens=torch.tensor([4], **i32), table=torch.tensor([[0]], **i32), cache=cache)
    a = {n: change[n](t) if n in change else t for n, t in a.items()}
    args = (torch.tensor([0, 4], **i32), 4, a["lens"], change.get("max_k", 4), a["table"], change.get("topk", 3))
    with pytest.raises(RuntimeError, match=message):
        flash_moba.flash_moba_cache_attn_func(a["q"], a["cache"], *args, add_weight=True)
    # and the whole step leaves the cache as it was
    k = torch.ones((4, 2, 32), dtype=torch.bfloat16, device="cuda")
    before = [t.clone() for t in cache]
    with pytest.raises(RuntimeError, match=message):
        flash_moba.flash_moba_with_cache_func(a["q"], k, k, a["cache"], *args, add_weight=True)
    assert all(torch.equal(x.view(torch.int8), y.view(torch.int8)) for x, y in zip(cache, before))


def test_the_entry_point_refuses_without_a_gpu():
    lib = H.load_library()
    assert lib.fmoba_cache_attn(None, None) != 0 and lib.fmoba_cache_attn_workspace_bytes(None) == 0

    def args(cache, **kw):
        a = H.CacheAttnArgs()
        a.cache = cache
        a.q = a.out = a.softmax_lse = a.cu_seqlens_q = a.seqlens_k = a.block_table = a.workspace = 4096
        a.batch, a.total_q, a.heads, a.max_seqlen_q, a.max_seqlen_k, a.max_pages, a.topk, a.table_stride = 2, 16, 4, 8, 500, 8, 3, 8
        a.softmax_scale, a.workspace_bytes = 0.1, 1 << 40
        for n in ("q_row_stride", "q_head_stride", "o_row_stride", "o_head_stride"):
            setattr(a, n, 64)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    for kw, message in BAD_CACHES:
        assert lib.fmoba_cache_attn(ctypes.byref(args(cache_struct(**kw))), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
    for kw, message in [(dict(batch=0), b"batch"), (dict(total_q=-1), b"sizes"), (dict(heads=3), b"divide"), (dict(topk=0), b"moba_topk"), (dict(topk=65), b"moba_topk"), (dict(q=0), b"null"),
                        (dict(softmax_lse=0), b"null"), (dict(block_table=0), b"null"), (dict(q_row_stride=4), b"strides"), (dict(out=4100), b"aligned"), (dict(workspace_bytes=16, total_q=4096), b"workspace"),
                        (dict(workspace=4100), b"workspace"), (dict(total_q=1 << 30, heads=8), b"launch grid"),
                        (dict(batch=65535, total_q=1 << 22, max_seqlen_k=65536, max_pages=1024), b"launch grid"),              # a workgroup a row and head
                        (dict(batch=65535, total_q=1 << 26, max_seqlen_k=65536, max_pages=1024), b"times pages for the launch grid")]:
        assert lib.fmoba_cache_attn(ctypes.byref(args(cache_struct(), **kw)), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
    assert lib.fmoba_cache_attn(ctypes.byref(args(cache_struct(weight=0), add_weight=1)), None) != 0
    assert b"no weight" in lib.fmoba_last_error()
    assert lib.fmoba_cache_attn(ctypes.byref(args(cache_struct(), total_q=0)), None) == 0
