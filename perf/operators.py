"""The operators of a serving step over a paged 8-bit cache, and the rotary positions in front of every attention here.

A case is a dict of plain values; `op` says which operator it calls:

    rotary   flash_moba_rotary_func: tokens, heads, heads_k, dim, rotary_dim, sections (pairs of every axis), far (positions below
             it), interleaved, packed (q and k are slices of one projection), train (with its backward)
    append   flash_moba_cache_append_func: new tokens of every sequence (lens_q) behind those of before (lens_k counts both)
    attn     flash_moba_cache_attn_func: the last lens_q rows of sequences of lens_k tokens; weight: their attention weights are
             added up per page
    evict    flash_moba_cache_evict_func: keep, sink, recent pages of every sequence
    step     flash_moba_with_cache_func: rotary, append and attention of one step

    page     tokens of a page: the gate's chunk, and what shares a scale per key head
    bits     what the cache holds: "e4m3" or "int8"
"""
import math
import random
import sys

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
_HELD = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_MOST = {"e4m3": 448.0, "int8": 127.0}
_LEAST_SCALE, _LARGEST_SCALE = 2.0 ** -64, 2.0 ** 64
_UNIT = 2.0 ** -32  # of an attention weight


def _api():
    if "flash-moba_amd" not in sys.path:
        sys.path.insert(0, "flash-moba_amd")
    import flash_moba

    return flash_moba


def _text(values):
    return ",".join(map(str, values))


def _ints(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------------------------------------------------------ cases
def _rotary(tokens, heads, heads_k, dim, sections, far, dtype="bf16", rotary_dim=None, interleaved=False, packed=False, train=False):
    return {"op": "rotary", "tokens": tokens, "heads": heads, "heads_k": heads_k, "dim": dim, "rotary_dim": rotary_dim or dim,
            "sections": _text(sections), "far": far, "dtype": dtype, "interleaved": interleaved, "packed": packed, "train": train}


def _cached(op, lens_q, lens_k, heads, heads_k, dim, page, topk, bits="e4m3", dtype="bf16", weight=False):
    return {"op": op, "lens_q": _text(lens_q), "lens_k": _text(lens_k), "heads": heads, "heads_k": heads_k, "dim": dim, "page": page,
            "topk": topk, "bits": bits, "dtype": dtype, "weight": weight}


def _evict(lens_k, heads_k, page, keep, sink, recent):
    return {"op": "evict", "lens_k": _text(lens_k), "heads_k": heads_k, "page": page, "keep": keep, "sink": sink, "recent": recent}


def listed():
    r = random.Random(20)
    decode_k = [int(512 * 2 ** r.uniform(0, 6)) for _ in range(16)]
    return [
        # q and k of one decode step of 16 requests, far into their contexts: latency
        dict(_rotary(16, 32, 8, 128, [64], 262144), name="rotary_decode"),
        # a training step on frames (time, height, width), q and k from one projection, with the gradients
        dict(_rotary(24571, 16, 16, 128, [16, 24, 24], 8192, packed=True, train=True), name="rotary_frames_train"),
        # the new tokens of 16 requests written into the cache: latency
        dict(_cached("append", [1] * 16, decode_k, 32, 8, 128, 128, 8), name="append_decode"),
        # prompts written into the cache, one of them behind what it holds already
        dict(_cached("append", [8192, 5003, 1077], [8192, 5003, 9301], 32, 8, 128, 64, 8, bits="int8", dtype="fp16"), name="append_prompts"),
        # a serving step: one new token for each of 16 requests with 512 to 32768 tokens so far, grouped heads
        dict(_cached("attn", [1] * 16, decode_k, 32, 8, 128, 128, 8), name="attn_decode"),
        # few requests, very long contexts, narrow heads of their own, weights kept for eviction
        dict(_cached("attn", [1] * 4, [262144, 100003, 200000, 65537], 16, 16, 64, 128, 16, bits="int8", dtype="fp16", weight=True), name="attn_decode_long"),
        # drafts of four tokens to be verified, a head dimension between the powers of two
        dict(_cached("attn", [4] * 8, [4099, 777, 12037, 2048, 9000, 63, 5000, 16001], 16, 4, 96, 64, 8), name="attn_drafts"),
        # the next 1024 tokens of long prompts against the cache so far
        dict(_cached("attn", [1024, 1024, 777], [9216, 33000, 20000], 32, 8, 128, 128, 8), name="attn_chunked_prefill"),
        # a whole prompt, with weights
        dict(_cached("attn", [8191], [8191], 16, 16, 128, 128, 8, weight=True), name="attn_prompt"),
        # requests that are over their budget by a few pages
        dict(_evict([n * 3 for n in decode_k], 8, 128, 64, 1, 2), name="evict_few"),
        # many requests with very long contexts
        dict(_evict([262144 - 1021 * i for i in range(64)], 8, 64, 1024, 4, 16), name="evict_many"),
        # all of a serving step: positions, cache, attention
        dict(_cached("step", [1] * 16, decode_k, 32, 8, 128, 128, 8, weight=True), name="step_decode"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """Serving and training over the ranges of the listed cases."""
    while True:
        op = rng.choice(["rotary", "append", "attn", "attn", "attn", "evict", "step"])
        dtype, bits = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "int8"])
        dim, page = rng.choice([128, 128, 128, 64, 64, 96, 80, 256]), rng.choice([64, 128, 128, 256])
        heads = rng.choice([8, 16, 32])
        heads_k = rng.choice([heads, heads // 4, heads // 8])
        if op == "rotary":
            rotary_dim = rng.choice([dim, dim, dim // 2])
            pairs, axes = rotary_dim // 2, rng.choice([1, 1, 2, 3])
            cuts = sorted(rng.sample(range(1, pairs), axes - 1))
            sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
            return _rotary(_log(rng, 1, 32768), heads, heads_k, dim, sections, _log(rng, 1024, 2 ** 20), dtype, rotary_dim, rng.random() < 0.3,
                           heads == heads_k and rng.random() < 0.5, rng.random() < 0.5)
        if op == "evict":
            lens = [_log(rng, 64, 262144) for _ in range(_log(rng, 1, 64))]
            sink, recent = rng.randrange(0, 5), rng.randrange(1, 17)
            return _evict(lens, heads_k, page, sink + recent + _log(rng, 1, 512), sink, recent)
        rows = rng.choice(["one", "one", "few", "part", "whole"]) if op != "step" else "one"
        if rows in ("one", "few"):
            batch = _log(rng, 1, 64)
            lens_q = [1 if rows == "one" else rng.randrange(1, 9) for _ in range(batch)]
            lens_k = [n + _log(rng, 256, 65536) for n in lens_q]
        elif rows == "part":
            batch = _log(rng, 1, 4)
            lens_q = [_log(rng, 9, 1500) for _ in range(batch)]
            lens_k = [n + _log(rng, 256, 32768) for n in lens_q]
        else:
            lens_k = lens_q = [_log(rng, 64, 8191) for _ in range(_log(rng, 1, 3))]
        # the plain form's scores and the cache fit the card several times over
        if max(lens_q) * max(lens_k) * len(lens_q) * heads > 3.3e9 or max(lens_k) * len(lens_k) * heads_k * dim > 1.5e9:
            continue
        return _cached(op, lens_q, lens_k, heads, heads_k, dim, page, _log(rng, 2, 32), bits, dtype, rng.random() < 0.4)


# ----------------------------------------------------------------------------------------------------------------- inputs
def _offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def _power_of_two(amax, most):
    """The least power of two that brings amax to `most` or below, within the limits of a scale."""
    mantissa, exponent = torch.frexp(amax.double() / most)
    least = torch.ldexp(torch.ones_like(mantissa), exponent - (mantissa == 0.5).to(exponent.dtype))
    return least.clamp(_LEAST_SCALE, _LARGEST_SCALE).float()


def _held(x, bits):
    """x (in units of its scale) as it is held: rounded to nearest, ties to even."""
    x = x.clamp(-_MOST[bits], _MOST[bits])
    return x.to(torch.float8_e4m3fn) if bits == "e4m3" else x.round().to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    s = dict(case)
    if case["op"] == "rotary":
        dtype, n, heads, heads_k, dim = _DTYPE[case["dtype"]], case["tokens"], case["heads"], case["heads_k"], case["dim"]
        sections = _ints(case["sections"])
        if case["packed"]:
            s["q"], s["k"], _ = normal(n, 3, heads, dim).to(dtype).unbind(1)
        else:
            s["q"], s["k"] = normal(n, heads, dim).to(dtype), normal(n, heads_k, dim).to(dtype)
        s["positions"] = torch.randint(0, case["far"], (len(sections), n), generator=g, device="cuda", dtype=torch.int32)
        s["sections"] = tuple(sections)
        if case["train"]:
            s["dq"], s["dk"] = normal(n, heads, dim).to(dtype), normal(n, heads_k, dim).to(dtype)
            s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
        return s
    page, heads_k, lens_k = case["page"], case["heads_k"], _ints(case["lens_k"])
    used = [(n + page - 1) // page for n in lens_k]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens_k), max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s["block_table"] = table
    s["seqlens_k"] = torch.tensor(lens_k, dtype=torch.int32, device="cuda")
    s["num_weights"] = pages
    # weights of heavy hitters: a few pages have most
    s["weights"] = (normal(pages, heads_k).mul(2).exp() * 1e9).to(torch.int64)
    if case["op"] == "evict":
        return s
    dtype, dim, bits, lens_q = _DTYPE[case["dtype"]], case["dim"], case["bits"], _ints(case["lens_q"])
    s["cu_seqlens_q"], s["max_q"], s["max_k"] = _offsets(lens_q), max(lens_q), max(lens_k)
    total = sum(lens_q)
    s["q"] = normal(total, case["heads"], dim).to(dtype)
    if case["op"] != "attn":
        s["k"], s["v"] = normal(total, heads_k, dim).to(dtype), normal(total, heads_k, dim).to(dtype)
    if case["op"] == "step":
        s["positions"] = (s["seqlens_k"] - 1)[None].contiguous()
    # pages as they are met: full of keys with a part that a page shares, the places behind a sequence's end hold what was there before
    cache = []
    for x in (normal(pages, heads_k, page, dim) + 0.5 * normal(pages, heads_k, 1, dim), normal(pages, heads_k, page, dim)):
        x = x.to(dtype)
        scale = _power_of_two(x.abs().amax((2, 3)), _MOST[bits])
        cache.append((_held(x.float() / scale[:, :, None, None], bits), scale, x))
    s["k_cache"], s["k_scale"], k = cache[0]
    s["v_cache"], s["v_scale"], _ = cache[1]
    # the keys' sums: of all of a page's, and of those that the last page of a sequence has (before the call that adds some)
    before = [n - (m if case["op"] != "attn" else 0) for n, m in zip(lens_k, lens_q)]
    k_sum, count = k.float().sum(2), torch.full((pages,), page, device="cuda", dtype=torch.float32)
    for b, n in enumerate(before):
        if n % page:
            p = int(table[b, n // page])
            k_sum[p], count[p] = k[p, :, :n % page].float().sum(1), n % page
    s["k_sum"], s["k_mean"] = k_sum, (k_sum / count[:, None, None]).to(dtype)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _rotate_plain(x, cos, sin, rotary_dim, interleaved):
    """x (tokens, heads, dim), cos and sin (tokens, 1, rotary_dim / 2)"""
    f, half = x.float(), rotary_dim // 2
    r = f.clone()
    a, b = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, half), slice(half, rotary_dim))
    r[..., a] = f[..., a] * cos - f[..., b] * sin
    r[..., b] = f[..., a] * sin + f[..., b] * cos
    return r.to(x.dtype)


def _turns(positions, sections, rotary_dim, base=10000.0):
    pairs = rotary_dim // 2
    axis = torch.repeat_interleave(torch.arange(len(sections), device="cuda"), torch.tensor(sections, device="cuda"), output_size=pairs)
    freq = base ** (-2.0 * torch.arange(pairs, device="cuda", dtype=torch.float64) / rotary_dim)
    angle = positions[axis].double().t() * freq
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_rotary(s):
    cos, sin = _turns(s["positions"], s["sections"], s["rotary_dim"])
    with torch.no_grad():
        res = {"q": _rotate_plain(s["q"], cos, sin, s["rotary_dim"], s["interleaved"]), "k": _rotate_plain(s["k"], cos, sin, s["rotary_dim"], s["interleaved"])}
        if s["train"]:
            res["dq"] = _rotate_plain(s["dq"], cos, -sin, s["rotary_dim"], s["interleaved"])
            res["dk"] = _rotate_plain(s["dk"], cos, -sin, s["rotary_dim"], s["interleaved"])
    return res


def _plain_append(s, k, v):
    P, bits, cu, table = s["page"], s["bits"], s["cu_seqlens_q"].long(), s["block_table"].long()
    batch, heads_k = table.shape[0], k.shape[1]
    new = cu[1:] - cu[:-1]
    start = s["seqlens_k"].long() - new
    seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), new)
    pos = start[seq] + torch.arange(k.shape[0], device="cuda") - cu[seq]
    # the pages that get tokens: (sequence, place in its table)
    first, last = start // P, (s["seqlens_k"].long() - 1) // P
    width = s["max_q"] // P + 2
    place = first[:, None] + torch.arange(width, device="cuda")
    b_of, j_of = torch.nonzero((place <= last[:, None]) & (new[:, None] > 0), as_tuple=True)
    slot = place[b_of, j_of]
    pages = table[b_of, slot]
    row = torch.zeros((batch, width), dtype=torch.long, device="cuda")
    row[b_of, j_of] = torch.arange(len(pages), device="cuda")
    where = row[seq, pos // P - first[seq]]
    old = (start[b_of] - slot * P).clamp(0, P)  # tokens that a page has before
    filled = (s["seqlens_k"].long()[b_of] - slot * P).clamp(0, P)
    fresh = (old == 0)[:, None]
    is_old = (torch.arange(P, device="cuda") < old[:, None])[:, None, :, None]
    grid = torch.zeros((len(pages), P, heads_k, k.shape[2]), device="cuda")
    got = torch.zeros((len(pages), P), dtype=torch.bool, device="cuda")
    got[where, pos % P] = True
    got = got[:, None, :, None]

    def write(x, held, scales):
        grid.zero_()
        grid[where, pos % P] = x.float()
        new_x = grid.transpose(1, 2)
        amax = torch.where(torch.isfinite(new_x), new_x.abs(), 0.0).amax((2, 3))
        was = scales[pages]
        scale = _power_of_two(amax, _MOST[bits])
        scale = torch.where(fresh, scale, torch.maximum(scale, was))
        kept = held[pages]
        again = _held(kept.float() * (was / scale)[:, :, None, None], bits)
        there = _held(new_x / scale[:, :, None, None], bits)
        held[pages] = torch.where(got, there.view(torch.int8), torch.where(is_old, again.view(torch.int8), kept.view(torch.int8))).view(held.dtype)
        scales[pages] = scale
        return new_x.sum(2)

    sums = write(k, s["k_cache"], s["k_scale"])
    sums = torch.where(fresh[:, :, None], sums, s["k_sum"][pages] + sums)
    s["k_sum"][pages] = sums
    s["k_mean"][pages] = (sums / filled[:, None, None]).to(s["k_mean"].dtype)
    s["weights"][pages] = torch.where(fresh, 0, s["weights"][pages])
    write(v, s["v_cache"], s["v_scale"])


def _plain_attn(s, q):
    P, heads, dim = s["page"], q.shape[1], q.shape[2]
    cu, table = s["cu_seqlens_q"].long(), s["block_table"].long()
    batch, heads_k, cols = table.shape[0], s["k_cache"].shape[1], table.shape[1]
    G, R, K = heads // heads_k, s["max_q"], cols * P
    len_q, len_k = cu[1:] - cu[:-1], s["seqlens_k"].long()
    rows = torch.arange(R, device="cuda")
    there = rows < len_q[:, None]
    src = torch.where(there, cu[:-1, None] + rows, 0)
    # (sequences, key heads, heads of the group, rows, features)
    qs = q[src].float().view(batch, R, heads_k, G, dim).permute(0, 2, 3, 1, 4)
    pos = torch.where(there, (len_k - len_q)[:, None] + rows, -1)
    at = table.clamp_min(0)
    mean = s["k_mean"][at].double().permute(0, 2, 1, 3)
    score = torch.matmul(qs.double().flatten(2, 3), mean.transpose(2, 3)).view(batch, heads_k, G, R, cols)
    own_page = (pos // P)[:, None, None, :, None]
    col = torch.arange(cols, device="cuda")
    score = torch.where((col < own_page) & (score == score), score, -math.inf)
    # best first, of equals the higher page first
    value, order = torch.sort(score.flip(-1), dim=-1, descending=True, stable=True)
    best = min(s["topk"] - 1, cols)
    order = torch.where(value[..., :best] > -math.inf, cols - 1 - order[..., :best], cols)
    chosen = torch.zeros(score.shape[:-1] + (cols + 1,), dtype=torch.bool, device="cuda").scatter_(-1, order, True)[..., :cols]
    chosen |= (col == own_page) & (pos >= 0)[:, None, None, :, None]
    seen = (torch.arange(K, device="cuda") <= pos[..., None])[:, None, None].unflatten(-1, (cols, P)) & chosen[..., None]
    k = (s["k_cache"][at].float() * s["k_scale"][at][..., None, None]).permute(0, 2, 1, 3, 4).reshape(batch, heads_k, K, dim)
    p = torch.matmul(qs.flatten(2, 3) * dim ** -0.5, k.transpose(2, 3)).view(batch, heads_k, G, R, cols, P)
    del k
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax((-2, -1), keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum((-2, -1), keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    live = torch.arange(K, device="cuda") < len_k[:, None]  # what lies behind a sequence's end is not looked at
    v = (s["v_cache"][at].float() * s["v_scale"][at][..., None, None]).permute(0, 2, 1, 3, 4).reshape(batch, heads_k, K, dim)
    v = torch.where(live[:, None, :, None], v, 0.0)
    out = torch.matmul(p.view(batch, heads_k, G * R, K), v).view(batch, heads_k, G, R, dim)
    lse = torch.where(total > 0, top + total.log(), math.inf)[..., 0, 0]
    res = {"out": out.permute(0, 3, 1, 2, 4).reshape(batch, R, heads, dim)[there].to(q.dtype),
           "lse": lse.permute(0, 3, 1, 2).reshape(batch, R, heads)[there].t().contiguous()}
    if s["weight"]:
        part = torch.round(p.sum(-1).double() / _UNIT).to(torch.int64).sum((2, 3))  # (sequences, key heads, pages)
        s["weights"].index_add_(0, at.flatten(), torch.where(table[:, :, None] >= 0, part.transpose(1, 2), 0).flatten(0, 1))
        res["weights"] = s["weights"] * _UNIT
    return res


def _plain_evict(s):
    P, table, n_k = s["page"], s["block_table"].long(), s["seqlens_k"].long()
    cols = table.shape[1]
    pages = (n_k + P - 1) // P
    col = torch.arange(cols, device="cuda")
    valid = col < pages[:, None]
    score = s["weights"][table.clamp_min(0)].sum(-1)
    stays = (col < s["sink"]) | (col >= pages[:, None] - s["recent"])
    score = torch.where(valid, torch.where(stays, torch.iinfo(torch.int64).max, score), -1)
    _, order = torch.sort(score, dim=1, descending=True, stable=True)
    kept = torch.zeros_like(valid).scatter_(1, order[:, :s["keep"]], True) & valid
    gone = valid & ~kept

    def listed_first(mask):
        _, order = torch.sort((~mask).to(torch.int8), dim=1, stable=True)
        return torch.where(col < mask.sum(1)[:, None], table.gather(1, order), -1).to(torch.int32)

    dropped = gone.sum(1)
    return {"block_table": listed_first(kept), "seqlens_k": (n_k - dropped * P).to(torch.int32), "freed": listed_first(gone), "num_freed": dropped.to(torch.int32)}


def _state(s):
    return {"k": s["k_cache"], "v": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"],
            "k_sum": s["k_sum"], "k_mean": s["k_mean"]}


def _plain(s):
    if s["op"] == "rotary":
        return _plain_rotary(s)
    if s["op"] == "evict":
        return _plain_evict(s)
    if s["op"] == "attn":
        return _plain_attn(s, s["q"])
    if s["op"] == "append":
        _plain_append(s, s["k"], s["v"])
        return _state(s)
    cos, sin = _turns(s["positions"], (s["dim"] // 2,), s["dim"])
    q, k = _rotate_plain(s["q"], cos, sin, s["dim"], False), _rotate_plain(s["k"], cos, sin, s["dim"], False)
    _plain_append(s, k, s["v"])
    return {**_plain_attn(s, q), **_state(s)}


# -------------------------------------------------------------------------------------------------------------------- own
def _own(s):
    api = _api()
    if s["op"] == "rotary":
        if not s["train"]:
            q, k = api.flash_moba_rotary_func(s["q"], s["k"], s["positions"], s["sections"], rotary_dim=s["rotary_dim"], interleaved=s["interleaved"])
            return {"q": q, "k": k}
        with torch.enable_grad():
            q, k = api.flash_moba_rotary_func(s["q"], s["k"], s["positions"], s["sections"], rotary_dim=s["rotary_dim"], interleaved=s["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if s["op"] == "evict":
        table, seqlens, freed, num_freed = api.flash_moba_cache_evict_func(s["weights"], s["seqlens_k"], s["block_table"], s["page"], s["keep"],
                                                                           sink_pages=s["sink"], recent_pages=s["recent"])
        return {"block_table": table, "seqlens_k": seqlens, "freed": freed, "num_freed": num_freed}
    cache = api.MobaKVCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["k_sum"], s["k_mean"], s["weights"])
    if s["op"] == "append":
        api.flash_moba_cache_append_func(cache, s["k"], s["v"], s["cu_seqlens_q"], s["max_q"], s["seqlens_k"], s["block_table"])
        return _state(s)
    if s["op"] == "attn":
        out, lse = api.flash_moba_cache_attn_func(s["q"], cache, s["cu_seqlens_q"], s["max_q"], s["seqlens_k"], s["max_k"], s["block_table"], s["topk"],
                                                  add_weight=s["weight"], return_lse=True)
        res = {"out": out, "lse": lse}
    else:
        out, lse = api.flash_moba_with_cache_func(s["q"], s["k"], s["v"], cache, s["cu_seqlens_q"], s["max_q"], s["seqlens_k"], s["max_k"], s["block_table"],
                                                  s["topk"], positions=s["positions"], add_weight=s["weight"], return_lse=True)
        res = {"out": out, "lse": lse, **_state(s)}
    if s["weight"]:
        res["weights"] = s["weights"] * _UNIT
    return res


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Inputs and outputs once each; of the cache what the rows can need: the means of the pages in front, the selected pages."""
    if case["op"] == "rotary":
        n, pairs = case["tokens"], case["rotary_dim"] // 2
        one = n * (case["heads"] + case["heads_k"]) * case["dim"] * 4  # read and written, 2 bytes each
        times = 2 if case["train"] else 1
        return {"bytes": times * one + n * 4 * len(_ints(case["sections"])), "flops": times * 6 * n * (case["heads"] + case["heads_k"]) * pairs}
    P, heads_k, lens_k = case["page"], case["heads_k"], _ints(case["lens_k"])
    used = [(n + P - 1) // P for n in lens_k]
    if case["op"] == "evict":
        return {"bytes": sum(used) * (heads_k * 8 + 4 + 4) + len(used) * max(used) * 4 + len(used) * 12, "flops": sum(used) * heads_k}
    dim, heads, lens_q = case["dim"], case["heads"], _ints(case["lens_q"])
    size = flops = 0
    if case["op"] != "attn":
        touched = sum((n - 1) // P - (n - m) // P + 1 for n, m in zip(lens_k, lens_q))
        size += sum(lens_q) * heads_k * dim * 2 * (2 + 1) + touched * heads_k * (dim * (4 + 4 + 2) + 4 * 4)
        flops += sum(lens_q) * heads_k * dim * 2 * 4
    if case["op"] == "step":
        size += sum(lens_q) * (heads + heads_k) * dim * 4
        flops += 3 * sum(lens_q) * (heads + heads_k) * dim
    if case["op"] != "append":
        G, pairs, scores = heads // heads_k, 0, 0
        for m, n in zip(lens_q, lens_k):
            pos = np.arange(n - m, n, dtype=np.int64)
            page = pos // P
            seen = int((np.minimum(case["topk"] - 1, page) * P + pos % P + 1).sum())
            pairs += seen
            scores += int(page.sum())
            size += ((n - 1) // P) * heads_k * dim * 2 + min(n, seen * G) * heads_k * (2 * dim + 8 / P)
        size += sum(lens_q) * heads * (dim * 4 + 4)
        if case["weight"]:
            size += sum(used) * heads_k * 16
        flops += heads * dim * (2 * scores + 4 * pairs)
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------ exact
def _exact_rotary(q, positions, sections, rotary_dim, interleaved, sign=1.0):
    """Pairs as complex numbers, turned by exp(i angle)."""
    x = q.detach().double()
    n, heads, dim = x.shape
    turn = []
    j = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            turn.append(positions[axis].double() * math.exp(-2.0 * j / rotary_dim * math.log(10000.0)))
            j += 1
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), sign * torch.stack(turn, 1))[:, None]
    body = x[..., :rotary_dim]
    z = torch.view_as_complex(body.reshape(n, heads, -1, 2).contiguous() if interleaved else
                              body.reshape(n, heads, 2, -1).transpose(2, 3).contiguous()) * turn
    z = torch.view_as_real(z)
    z = z.reshape(n, heads, rotary_dim) if interleaved else z.transpose(2, 3).reshape(n, heads, rotary_dim)
    return torch.cat([z, x[..., rotary_dim:]], -1)


def _exact_held(x, bits):
    """The nearest value that 8 bits hold, of two the even one, by its exponent."""
    x = x.clamp(-_MOST[bits], _MOST[bits])
    if bits == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    return torch.round(x * torch.exp2(3 - e)) * torch.exp2(e - 3)


def _exact_append(s, k, v):
    P, bits = s["page"], s["bits"]
    table, lens, cu = s["block_table"].tolist(), s["seqlens_k"].tolist(), s["cu_seqlens_q"].tolist()
    e = {"k": s["k_cache"].double(), "v": s["v_cache"].double(), "k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double(),
         "k_sum": s["k_sum"].double(), "k_mean": s["k_mean"].double(), "weights": s["weights"].clone()}
    for b in range(len(lens)):
        start, end = lens[b] - (cu[b + 1] - cu[b]), lens[b]
        for slot in range(start // P, (end - 1) // P + 1 if end > start else 0):
            lo, hi, page = max(start, slot * P), min(end, (slot + 1) * P), table[b][slot]
            old = lo - slot * P
            for name, x in (("k", k), ("v", v)):
                x = x[cu[b] + lo - start:cu[b] + hi - start].double().transpose(0, 1)
                need = (x.abs().amax((1, 2)) / _MOST[bits]).clamp_min(_LEAST_SCALE)
                scale = torch.exp2(torch.ceil(torch.log2(need)))
                if old:
                    scale = torch.maximum(scale, e[name + "_scale"][page])
                    e[name][page, :, :old] = _exact_held(e[name][page, :, :old] * (e[name + "_scale"][page] / scale)[:, None, None], bits)
                e[name][page, :, old:hi - slot * P] = _exact_held(x / scale[:, None, None], bits)
                e[name + "_scale"][page] = scale
                if name == "k":
                    e["k_sum"][page] = x.sum(1) + (e["k_sum"][page] if old else 0.0)
                    e["k_mean"][page] = e["k_sum"][page] / (hi - slot * P)
                    if not old:
                        e["weights"][page] = 0
    return e


def _exact_attn(s, q, e):
    """Sequence by sequence and key head by key head; q in the type that the gate and the attention read."""
    P, heads_k, dim = s["page"], e["k"].shape[1], q.shape[2]
    G, topk = q.shape[1] // heads_k, s["topk"]
    cu, lens, table = s["cu_seqlens_q"].tolist(), s["seqlens_k"].tolist(), s["block_table"].long()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((q.shape[1], q.shape[0]), math.inf, dtype=torch.float64, device="cuda")
    weights = e["weights"].double() * _UNIT
    for b in range(len(lens)):
        rows, n = slice(cu[b], cu[b + 1]), lens[b]
        R = cu[b + 1] - cu[b]
        if R == 0 or n == 0:
            continue
        cols = (n + P - 1) // P
        pages = table[b, :cols]
        pos = torch.arange(n - R, n, device="cuda")
        own_page = pos // P
        tri = torch.arange(cols, device="cuda")[None] < own_page[:, None]
        causal = torch.arange(n, device="cuda")[None] <= pos[:, None]
        for hk in range(heads_k):
            mean = e["k_mean"][pages, hk].to(s["k_mean"].dtype).double()
            kk = (e["k"][pages, hk] * e["k_scale"][pages, hk][:, None, None]).reshape(-1, dim)[:n]
            vv = (e["v"][pages, hk] * e["v_scale"][pages, hk][:, None, None]).reshape(-1, dim)[:n]
            for h in range(hk * G, hk * G + G):
                qh = q[rows, h].double()
                score = (qh @ mean.t()).masked_fill(~tri, -math.inf)
                pick = torch.zeros((R, cols), dtype=torch.bool, device="cuda")
                pick[torch.arange(R, device="cuda"), own_page] = True
                count = min(topk - 1, cols)
                if count:
                    value, idx = score.topk(count, dim=1)
                    pick.scatter_(1, idx, pick.gather(1, idx) | (value > -math.inf))
                seen = pick.repeat_interleave(P, 1)[:, :n] & causal
                w = ((qh @ kk.t()) / math.sqrt(dim)).masked_fill(~seen, -math.inf)
                lse[h, rows] = torch.logsumexp(w, 1)
                w = torch.softmax(w, 1)
                out[rows, h] = w @ vv
                if s["weight"]:
                    part = torch.zeros(cols * P, dtype=torch.float64, device="cuda")
                    part[:n] = w.sum(0)
                    weights[pages, hk] += part.view(cols, P).sum(1)
    res = {"out": out, "lse": lse}
    if s["weight"]:
        res["weights"] = weights
    return res


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        args = (s["positions"], s["sections"], s["rotary_dim"], s["interleaved"])
        res = {"q": _exact_rotary(s["q"], *args), "k": _exact_rotary(s["k"], *args)}
        if case["train"]:
            res["dq"], res["dk"] = _exact_rotary(s["dq"], *args, sign=-1.0), _exact_rotary(s["dk"], *args, sign=-1.0)
        return res
    if case["op"] == "evict":
        return None  # whole numbers
    if case["op"] == "attn":
        e = {"k": s["k_cache"].double(), "v": s["v_cache"].double(), "k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double(),
             "k_mean": s["k_mean"].double(), "weights": s["weights"]}
        return _exact_attn(s, s["q"], e)
    if case["op"] == "append":
        e = _exact_append(s, s["k"], s["v"])
        del e["weights"]
        return e
    # what a step's attention reads was rounded on the way: positions to 16 bits, the cache to 8
    args = (s["positions"], (s["dim"] // 2,), s["dim"], False)
    q, k = (_exact_rotary(x, *args).to(x.dtype) for x in (s["q"], s["k"]))
    e = _exact_append(s, k, s["v"])
    res = _exact_attn(s, q, e)
    del e["weights"]
    return {**res, **e}
