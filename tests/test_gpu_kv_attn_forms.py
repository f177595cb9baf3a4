"""The two forms of flash_moba_cache_attn_func, each where it runs: what a caller sees of a value must not depend on how many rows a call has.

The row form is held to the bound of test_gpu_kv_attn.py.  Of the form for many rows: a weight goes to the second product as two fp16 numbers, of which the second is what the
first cuts off (2^-10) and is cut off itself (2^-10 of that), and less than 2^-14 of 2^-15 is a multiple of 2^-39: 2^-20 of a weight and 2^-39 a key of max |v|; sums of n weights and of n products
are off by n 2^-24 each; a visit's output is off by half a step of 32767ths of its largest feature, which is at most max |v|, and the visits' weights add up to 1: 2^-16 of it."""
import ctypes
import math

import pytest
import torch

import cache_reference as R
import flash_moba
from flash_moba import flash_moba_hip as H
from test_gpu_kv_attn import CASES, call, check, setup
from test_gpu_kv_append import cache_struct

gpu = pytest.mark.gpu


def shares_pages(heads, heads_k, dim, P, lens_q, lens_k, topk, max_pages):
    """Whether a call is of the form for many rows: it alone has a workspace for tables of up to 2049 pages."""
    a = H.CacheAttnArgs()
    a.cache = cache_struct(page_size=P, heads_k=heads_k, head_dim=dim)
    a.batch, a.total_q, a.heads, a.max_seqlen_q, a.max_seqlen_k, a.max_pages, a.topk = len(lens_q), sum(lens_q), heads, max(lens_q), max(lens_k), max_pages, topk
    assert min(-(-max(lens_k) // P), max_pages) <= 2049
    return H.load_library().fmoba_cache_attn_workspace_bytes(ctypes.byref(a)) > 0


def check_form(got, lse, want, want_lse, sizes, parts):
    if not parts:
        return check(got, lse, want, want_lse, sizes, False)
    size, dot, most, count = sizes
    delta = (got.shape[2] + 8) * 2.0 ** -24 * dot + 2.0 ** -22
    weights = (2 * delta + 2 * count * 2.0 ** -24 + 2.0 ** -20).t()[:, :, None]
    tol = want.abs() * torch.finfo(got.dtype).eps / 2 * 1.01 + size * weights + ((2.0 ** -39 * count + 2.0 ** -16 * 1.01) * most).t()[:, :, None] + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.float().cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"out {(err - tol).max().item():.3e} over, largest error {err.max().item():.3e}"
    check(got, lse, want, want_lse, sizes, True)  # (and the log-sum-exp)


def check_with_nans(out, lse, want, want_lse, sizes, parts):
    assert torch.equal(out.isnan().cpu(), want.isnan())
    check_form(out.nan_to_num(0.0), lse, want.nan_to_num(0.0), want_lse, sizes, parts)


@gpu
@pytest.mark.parametrize("heads,heads_k,dim,P,rows,length,topk,parts", [
    (1, 1, 32, 256, 2200, 256 * 40 + 10, 40, True),     # a page of several steps, all of it in LDS
    (2, 1, 64, 192, 1100, 192 * 30 - 1, 24, True),
    (4, 1, 128, 1024, 550, 1024 * 9 + 5, 9, True),      # and 64 keys of it at a time
    (4, 2, 256, 128, 520, 128 * 34, 33, True),
    (4, 2, 64, 64, 600, 900, 5, True),                  # a page of one step
    (4, 2, 128, 256, 600, 2000, 5, True),               # pages of several columns
    (4, 2, 128, 128, 20, 2000, 5, False),
])
def test_a_row_has_the_nans_of_the_values_that_it_sees(heads, heads_k, dim, P, rows, length, topk, parts):
    cache, table, q, cu = setup(heads, heads_k, dim, P, [rows], [length], torch.bfloat16, torch.float8_e4m3fn)
    assert shares_pages(heads, heads_k, dim, P, [rows], [length], topk, len(table[0])) == parts
    used = (length + P - 1) // P
    for c, place, hk, e in ((0, 3, 0, 5), (used // 2, P - 1, heads_k - 1, dim - 1), (used - 1, (length - 1) % P // 2, 0, 0), (used - 2, 70 % P, 0, dim // 2)):
        cache.v.view(torch.int8)[table[0][c], hk, place, e] = -1 if c & 1 else 0x7F  # (of either sign)
    out, lse = call(cache, table, q, cu, [length], topk)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, [length], table, topk)
    assert bool(want.isnan().any()) and not bool(want.isnan().all())
    check_with_nans(out, lse, want, want_lse, sizes, parts)


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,heads_k,dim,P,lens_q,lens_k,topk", CASES)
def test_every_call_keeps_the_bound_of_its_form(held, dtype, heads, heads_k, dim, P, lens_q, lens_k, topk):
    cache, table, q, cu = setup(heads, heads_k, dim, P, lens_q, lens_k, dtype, held, seed=21)
    out, lse = call(cache, table, q, cu, lens_k, topk)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, lens_k, table, topk)
    check_form(out, lse, want, want_lse, sizes, shares_pages(heads, heads_k, dim, P, lens_q, lens_k, topk, len(table[0])))


@gpu
@pytest.mark.parametrize("P", [64, 256])
@pytest.mark.parametrize("rows,parts", [(1, False), (40, False), (1100, True)])
def test_a_nan_under_a_weight_that_vanishes(rows, parts, P):
    """The row form multiplies every value that a row sees; where rows share pages a visit whose weights vanish beside the others' counts as much."""
    dim, length = 64, P * 3 + max(rows, 20)
    cache, table, q, cu = setup(2, 1, dim, P, [rows], [length], torch.bfloat16, torch.float8_e4m3fn)
    topk = len(table[0])
    assert shares_pages(2, 1, dim, P, [rows], [length], topk, topk) == parts
    q.abs_()
    q += 0.5
    cache.k_scale.fill_(0.25)
    cache.k.copy_(torch.ones(cache.k.shape, device="cuda").to(cache.k.dtype))
    cache.k[table[0][1]] = torch.full(cache.k.shape[1:], -448.0, device="cuda").to(cache.k.dtype)  # scores 400 and more below the others: their exponential is 0
    cache.v.view(torch.int8)[table[0][1], 0, 7, 11] = 0x7F
    out, lse = call(cache, table, q, cu, [length], topk)
    want, want_lse, _, sizes = R.attention(R.state(cache), q.cpu(), cu, [length], table, topk)
    assert bool(want[:, :, 11].isnan().all()) and want.isnan().sum().item() == rows * 2
    check_with_nans(out, lse, want, want_lse, sizes, parts)


@gpu
@pytest.mark.parametrize("rows,parts", [(3, False), (1100, True)])
@pytest.mark.parametrize("power", [-62, -66, -70, -90])
def test_scores_too_small_for_32_bits_are_decided_as_in_64(power, rows, parts):
    """Queries and means whose products are subnormal in 32 bits, or nothing: every page has another score all the same."""
    P, dim, n, topk = 64, 64, 40, 5
    cache, table, q, cu = setup(2, 1, dim, P, [rows], [P * n], torch.bfloat16, torch.float8_e4m3fn)
    assert shares_pages(2, 1, dim, P, [rows], [P * n], topk, len(table[0])) == parts
    q *= 2.0 ** power
    cache.k_mean.mul_(2.0 ** power)
    q[-1, 1] = 0  # (equal scores: the later pages)
    assert bool((q[:-1] != 0).any(-1).all())
    w = cache.weight.clone()
    out, lse = call(cache, table, q, cu, [P * n], topk, add_weight=True)
    want, want_lse, weight, sizes = R.attention(R.state(cache), q.cpu(), cu, [P * n], table, topk)
    check_form(out, lse, want, want_lse, sizes, parts)
    assert torch.equal((cache.weight > w).cpu(), weight > 0)


@gpu
@pytest.mark.parametrize("rows,parts", [(3, False), (1100, True)])
def test_subnormal_features_count(rows, parts):
    """fp16: the only normal feature of a row says the opposite of the others, which are subnormal."""
    P, dim, n, topk = 64, 64, 40, 5
    cache, table, q, cu = setup(2, 1, dim, P, [rows], [P * n], torch.float16, torch.int8)
    assert shares_pages(2, 1, dim, P, [rows], [P * n], topk, len(table[0])) == parts
    q[:] = 2.0 ** -15
    q[:, :, 0] = 2.0 ** -14
    for c in range(n):
        cache.k_mean[table[0][c]] = (c - 16) * 2.0 ** -6
        cache.k_mean[table[0][c], :, 0] = (16 - c) * 2.0 ** -6
    w = cache.weight.clone()
    out, lse = call(cache, table, q, cu, [P * n], topk, add_weight=True)
    want, want_lse, weight, sizes = R.attention(R.state(cache), q.cpu(), cu, [P * n], table, topk)
    check_form(out, lse, want, want_lse, sizes, parts)
    assert torch.equal((cache.weight > w).cpu(), weight > 0)
