"""flash_moba_cache_append_func against its definition in 64 bits.  What is held and its scales have to be the same: scales are powers of two, so nothing but the
rounding to 8 bits itself rounds.  A sum of n keys in 32 bits is off by at most n 2^-24 of the sum of their magnitudes, a mean by that and
half a step of its type."""
import ctypes

import pytest
import torch

import cache_reference as R
import flash_moba
from flash_moba import flash_moba_hip as H

gpu = pytest.mark.gpu


def random_cache(pages, heads_k, P, dim, dtype, held, seed, layout="heads"):
    """A cache whose pages are full of what was there before."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = flash_moba.MobaKVCache.allocate(pages, P, heads_k, dim, dtype, held)
    if layout == "tokens":  # (pages, page_size, heads, head_size) in memory
        c = c._replace(k=torch.zeros((pages, P, heads_k, dim), dtype=torch.int8, device="cuda").view(held).transpose(1, 2),
                       v=torch.zeros((pages, P, heads_k, dim), dtype=torch.int8, device="cuda").view(held).transpose(1, 2))
    for t in (c.k, c.v):
        t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 40).clamp(-120, 120).to(held))
    c.k_scale.copy_(2.0 ** torch.randint(-8, -3, c.k_scale.shape, generator=g, device="cuda"))
    c.v_scale.copy_(2.0 ** torch.randint(-8, -3, c.k_scale.shape, generator=g, device="cuda"))
    c.k_sum.normal_(generator=g)
    c.k_mean.copy_(c.k_sum / P)
    c.weight.random_(0, 1 << 40, generator=g)
    return c


def tables(lens, P, pages, seed, width=None):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max((n + P - 1) // P for n in lens) + 1
    rows = []
    for n in lens:
        used = (n + P - 1) // P
        rows.append([order.pop() for _ in range(used)] + [-1] * (width - used))
    return rows


def check(cache, s, count):
    """count: the most keys of a sum"""
    for name in ("k", "v"):
        got = getattr(cache, name).float().cpu().double()
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(s[name], nan=1e9)), name
        assert torch.equal(getattr(cache, name + "_scale").cpu().double(), s[name + "_scale"]), name
    size = s["size"]
    assert bool(((cache.k_sum.cpu().double() - s["k_sum"]).abs() <= count * 2.0 ** -24 * size).all())
    mean_tol = s["k_mean"].abs() * torch.finfo(cache.k_mean.dtype).eps / 2 + count * 2.0 ** -24 * size + 2.0 ** -25
    assert bool(((cache.k_mean.float().cpu().double() - s["k_mean"]).abs() <= mean_tol).all())
    assert torch.equal(cache.weight.cpu(), s["weight"])


def run(cache, k, v, lens_new, lens_after, table, s=None):
    cu = [0]
    for n in lens_new:
        cu.append(cu[-1] + n)
    s = R.state(cache) if s is None else s
    s.setdefault("size", s["k_sum"].abs())
    R.append(s, k.cpu(), v.cpu(), cu, lens_after, table)
    s["size"] = s["size"] + k.abs().float().nan_to_num(posinf=0).sum(0).max().item()
    i32 = dict(dtype=torch.int32, device="cuda")
    flash_moba.flash_moba_cache_append_func(cache, k, v, torch.tensor(cu, **i32), max(lens_new), torch.tensor(lens_after, **i32), torch.tensor(table, **i32))
    return s


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads_k,dim,P,lens_new,lens_after,layout", [
    (1, 16, 64, [1], [1], "heads"),
    (2, 128, 128, [1, 1, 1, 1], [1, 128, 129, 300], "heads"),
    (3, 80, 64, [200, 0, 1, 63], [200, 77, 65, 126], "tokens"),   # 25 rows a pass, a page filled to its last place but one
    (1, 256, 256, [600, 5], [700, 261], "heads"),                 # rows read twice
    (2, 64, 1024, [1500], [2049], "tokens"),
    (2, 96, 64, [129, 64], [129, 64], "heads"),
])
def test_pages_are_the_definitions(held, dtype, heads_k, dim, P, lens_new, lens_after, layout):
    pages = sum((n + P - 1) // P for n in lens_after) + 2
    cache = random_cache(pages, heads_k, P, dim, dtype, held, 1, layout)
    g = torch.Generator(device="cuda").manual_seed(2)
    n = sum(lens_new)
    kv = torch.randn((n, 2, heads_k, dim), generator=g, device="cuda").to(dtype)  # (strided)
    kv[:, 1] *= torch.exp2(torch.randint(-6, 7, (n, heads_k, 1), generator=g, device="cuda").float()).to(dtype)
    table = tables(lens_after, P, pages, 3)
    s = run(cache, kv[:, 0], kv[:, 1], lens_new, lens_after, table)
    check(cache, s, P + 2)


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
def test_a_page_filled_token_by_token_and_its_growing_scale(held):
    P, dim, dtype = 64, 32, torch.bfloat16
    cache = random_cache(5, 2, P, dim, dtype, held, 4)
    table, s, length = [[3, 1, 4]], None, 60
    g = torch.Generator(device="cuda").manual_seed(5)
    cache.k_scale[3] = cache.v_scale[3] = 2.0 ** -10
    for step in (1, 1, 1, 2, 1, 3, 1):  # across a page's end
        length += step
        k, v = (torch.randn((step, 2, dim), generator=g, device="cuda").to(dtype) * 2.0 ** (length - 61) for _ in range(2))
        s = run(cache, k, v, [step], [length], table, s)
    check(cache, s, 2 * P)


@gpu
@pytest.mark.parametrize("held", [torch.float8_e4m3fn, torch.int8])
def test_values_that_are_no_ordinary_numbers(held):
    P, dim, dtype = 64, 16, torch.bfloat16
    cache = random_cache(6, 1, P, dim, dtype, held, 6)
    k = torch.ones((6, 1, dim), dtype=dtype, device="cuda")
    k[0, 0, 1], k[0, 0, 2], k[0, 0, 3] = float("inf"), -float("inf"), float("nan")
    k[1] = 0                      # nothing but zeros: the least scale
    k[2] *= 2.0 ** -100
    k[3] *= 2.0 ** 120            # beyond the largest scale: cut off
    k[4] = float("nan")
    k[5] = torch.tensor([448.0, 449.0, 127.0, 127.5, 17.0, 19.0, 0.5, 1.5, 2.5, -0.5, -1.5, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -0.0, 1.0], device="cuda")
    s = R.state(cache)
    cu = list(range(7))
    lens = [1] * 6
    table = [[i] for i in range(6)]
    R.append(s, k.cpu(), k.cpu(), cu, lens, table)
    i32 = dict(dtype=torch.int32, device="cuda")
    flash_moba.flash_moba_cache_append_func(cache, k, k, torch.tensor(cu, **i32), 1, torch.tensor(lens, **i32), torch.tensor(table, **i32))
    for name in ("k", "v"):
        got = getattr(cache, name).float().cpu().double()
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(s[name], nan=1e9))
        assert torch.equal(getattr(cache, name + "_scale").cpu().double(), s[name + "_scale"])
    assert torch.equal(cache.k_sum.cpu().double().nan_to_num(nan=7.0), s["k_sum"].nan_to_num(nan=7.0))  # one key each: no rounding


@gpu
def test_what_is_no_page_or_no_token_is_left_alone():
    P, dim = 64, 32
    cache = random_cache(4, 1, P, dim, torch.float16, torch.int8, 7)
    before = [t.clone() for t in cache]
    k = torch.randn((300, 1, dim), device="cuda").half()
    i32 = dict(dtype=torch.int32, device="cuda")
    args = lambda cu, lens, table: (torch.tensor(cu, **i32), 300, torch.tensor(lens, **i32), torch.tensor(table, **i32))  # noqa: E731
    # no page of the cache; a sequence shorter than its new tokens (the first of them have no place), and a table that ends too early
    for cu, lens, table in ([[0, 100], [100], [[-1, 4]]], [[0, 100], [0], [[0, 1]]], [[0, 300], [-5], [[0, 1]]], [[0, 0], [64], [[0, 1]]]):
        flash_moba.flash_moba_cache_append_func(cache, k, k, *args(cu, lens, table))
        assert all(torch.equal(a, b) for a, b in zip(cache, before)), (cu, lens, table)
    flash_moba.flash_moba_cache_append_func(cache, k[:0], k[:0], torch.tensor([0, 0], **i32), 0, torch.tensor([9], **i32), torch.tensor([[0]], **i32))
    s = R.state(cache)
    R.append(s, k.cpu(), k.cpu(), [0, 300], [130], [[2, 0]])
    flash_moba.flash_moba_cache_append_func(cache, k, k, *args([0, 300], [130], [[2, 0]]))
    assert torch.equal(cache.k.cpu().double(), s["k"]) and torch.equal(cache.weight.cpu(), s["weight"])
    # offsets that are no offsets: nothing outside of k is read
    flash_moba.flash_moba_cache_append_func(cache, k, k, *args([290, 2000], [2000], [[3] * 40]))
    torch.cuda.synchronize()


@gpu
def test_append_replays_from_a_graph_and_runs_on_other_streams():
    P, dim, lens = 64, 64, [65, 300]
    g = torch.Generator(device="cuda").manual_seed(9)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor(tables([600, 600], P, 30, 9), **i32)
    cu, seqlens = torch.tensor([0, 2, 5], **i32), torch.tensor(lens, **i32)
    k, v = (torch.randn((5, 2, dim), generator=g, device="cuda").bfloat16() for _ in range(2))
    cache = random_cache(30, 2, P, dim, torch.bfloat16, torch.float8_e4m3fn, 10)
    eager = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flash_moba.flash_moba_cache_append_func(cache, k, v, cu, 3, seqlens, table)
    side, here = torch.cuda.Stream(), seqlens.clone()
    for step in range(4):
        k.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            flash_moba.flash_moba_cache_append_func(eager, k, v, cu, 3, here, table)
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, eager)), step
        seqlens += torch.tensor([2, 3], **i32)
        here += torch.tensor([2, 3], **i32)


@gpu
def test_append_from_a_traced_graph():
    P, dim = 64, 32
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = random_cache(4, 1, P, dim, torch.bfloat16, torch.int8, 11)
    other = flash_moba.MobaKVCache(*[t.clone() for t in cache])
    k = torch.randn((70, 1, dim), device="cuda").bfloat16()
    args = (torch.tensor([0, 70], **i32), 70, torch.tensor([100], **i32), torch.tensor([[2, 0]], **i32))

    def step(k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight, k):
        flash_moba.flash_moba_cache_append_func(flash_moba.MobaKVCache(k_cache, v_cache, k_scale, v_scale, k_sum, k_mean, weight), k, k, *args)
        return k

    torch.compile(step, backend="aot_eager", fullgraph=True)(*cache, k)
    flash_moba.flash_moba_cache_append_func(other, k, k, *args)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))


@gpu
@pytest.mark.parametrize("change,message", [
    (dict(k=lambda k: k.float()), "dtype"), (dict(k=lambda k: k[:, :1]), "k and v must be"), (dict(cu=lambda t: t.long()), "cu_seqlens"), (dict(cu=lambda t: t[:1]), "cu_seqlens"),
    (dict(lens=lambda t: t.long()), "seqlens_k"), (dict(table=lambda t: t[0]), "block_table"), (dict(table=lambda t: t.long()), "block_table"),
    (dict(cache=lambda c: c._replace(k=c.k.float())), "float8_e4m3fn or int8"), (dict(cache=lambda c: c._replace(v=c.v[:1])), "one shape"),
    (dict(cache=lambda c: c._replace(k_scale=c.k_scale.double())), "k_scale"), (dict(cache=lambda c: c._replace(k_sum=c.k_sum[:1])), "k_sum"),
    (dict(cache=lambda c: c._replace(k_mean=c.k_mean.float())), "fp16 and bf16"), (dict(cache=lambda c: c._replace(weight=c.weight.int())), "weight"),
    (dict(cache=lambda c: c._replace(k=c.k[:, :, :32], v=c.v[:, :, :32])), "page_size"), (dict(cache=lambda c: tuple(c)[:3]), "MobaKVCache"),
    (dict(k=lambda k: k.clone().requires_grad_(True)), "no backward"), (dict(max_seqlen=-1), "out of range"),
])
def test_refusals(change, message):
    cache = flash_moba.MobaKVCache.allocate(3, 64, 2, 32)
    i32 = dict(dtype=torch.int32, device="cuda")
    a = dict(k=torch.zeros((4, 2, 32), dtype=torch.bfloat16, device="cuda"), cu=torch.tensor([0, 4], **i32), lens=torch.tensor([4], **i32), table=torch.tensor([[0]], **i32), cache=cache)
    v = a["k"].clone()
    a = {n: change[n](t) if n in change else t for n, t in a.items()}
    with pytest.raises(RuntimeError, match=message):
        flash_moba.flash_moba_cache_append_func(a["cache"], a["k"], v, a["cu"], change.get("max_seqlen", 4), a["lens"], a["table"])


def cache_struct(**kw):
    c = H.KVCache()
    c.k = c.v = c.k_scale = c.v_scale = c.k_sum = c.k_mean = c.weight = 4096
    c.num_pages, c.page_size, c.heads_k, c.head_dim, c.format, c.dtype = 8, 64, 2, 64, 0, 1
    for n in ("k_page_stride", "k_head_stride", "k_token_stride", "v_page_stride", "v_head_stride", "v_token_stride"):
        setattr(c, n, 64)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


BAD_CACHES = [(dict(dtype=2), b"fp16 and bf16"), (dict(format=2), b"e4m3 or int8"), (dict(page_size=32), b"page_size"), (dict(page_size=96), b"page_size"), (dict(page_size=2048), b"page_size"),
              (dict(head_dim=24), b"head_size"), (dict(head_dim=272), b"head_size"), (dict(head_dim=0), b"head_size"), (dict(num_pages=-1), b"pages"), (dict(heads_k=0), b"heads"),
              (dict(k=0), b"null"), (dict(k_mean=0), b"null"), (dict(v_token_stride=8), b"strides"), (dict(k=4104), b"aligned")]


def test_the_entry_point_refuses_without_a_gpu():
    lib = H.load_library()
    assert lib.fmoba_cache_append(None, None) != 0

    def args(cache, **kw):
        a = H.CacheAppendArgs()
        a.cache = cache
        a.k = a.v = a.cu_seqlens = a.seqlens_k = a.block_table = 4096
        a.batch, a.total_new, a.max_seqlen_new, a.max_pages, a.table_stride = 2, 16, 8, 4, 4
        for n in ("k_row_stride", "k_head_stride", "v_row_stride", "v_head_stride"):
            setattr(a, n, 64)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    for kw, message in BAD_CACHES:
        assert lib.fmoba_cache_append(ctypes.byref(args(cache_struct(**kw))), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
    for kw, message in [(dict(batch=0), b"batch"), (dict(total_new=-1), b"sizes"), (dict(k=0), b"null"), (dict(block_table=0), b"null"), (dict(k_row_stride=4), b"strides"), (dict(v=4100), b"aligned"),
                        (dict(total_new=2 ** 31 - 1, max_seqlen_new=2 ** 31 - 1, max_pages=1 << 26), b"launch grid")]:
        assert lib.fmoba_cache_append(ctypes.byref(args(cache_struct(), **kw)), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
    assert lib.fmoba_cache_append(ctypes.byref(args(cache_struct(), total_new=0)), None) == 0

    def turn(**kw):
        r = H.RotaryArgs()
        r.total, r.heads, r.heads_k, r.head_dim, r.rotary_dim, r.axes, r.log2_base, r.dtype = 16, 4, 2, 64, 64, 1, 13.0, 1
        r.sections[0] = 32
        r.q = r.k = r.q_out = r.positions = 4096
        r.k_row_stride = r.k_head_stride = 64
        for n, v in kw.items():
            setattr(r, n, v)
        return r

    assert lib.fmoba_cache_append_turned(ctypes.byref(args(cache_struct())), None, None) != 0 and lib.fmoba_cache_append_turned(None, ctypes.byref(turn()), None) != 0
    for kw, r, message in [(dict(max_seqlen_new=9), {}, b"up to 8"), (dict(total_new=15), {}, b"not the keys"), ({}, dict(heads_k=1), b"not the keys"), ({}, dict(k=8192), b"not the keys"),
                           ({}, dict(k_row_stride=128), b"not the keys"), ({}, dict(dtype=0), b"not the keys"), ({}, dict(q_out=0), b"null"), ({}, dict(rotary_dim=128), b"rotary_dim"),
                           (dict(v=0), {}, b"null"), (dict(batch=0), {}, b"batch")]:
        assert lib.fmoba_cache_append_turned(ctypes.byref(args(cache_struct(), **kw)), ctypes.byref(turn(**r)), None) != 0, (kw, r)
        assert message in lib.fmoba_last_error(), (kw, r, lib.fmoba_last_error())
    assert lib.fmoba_cache_append(ctypes.byref(args(cache_struct(num_pages=0, k=0))), None) == 0


def test_a_cache_is_not_allocated_in_forms_that_the_kernels_do_not_take():
    allocate = flash_moba.MobaKVCache.allocate
    for args, kw in [((4, 32, 1, 64), {}), ((4, 2048, 1, 64), {}), ((4, 64, 1, 40), {}), ((4, 64, 1, 512), {}), ((4, 64, 1, 64), dict(dtype=torch.float32)),
                     ((4, 64, 1, 64), dict(cache_dtype=torch.float8_e5m2))]:
        with pytest.raises(RuntimeError):
            allocate(*args, device="cpu", **kw)
    c = allocate(4, 64, 2, 48, device="cpu", keep_weight=False)
    assert c.weight is None and c.k.shape == (4, 2, 64, 48) and c.k_mean.shape == (4, 2, 48)
