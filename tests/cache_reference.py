"""The paged 8-bit cache in 64 bits on the CPU, written from its definition: a dict of tensors like MobaKVCache's fields, and what the functions do to it."""
import itertools
import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def state(cache):
    s = {n: getattr(cache, n).detach().cpu() for n in ("k_scale", "v_scale", "k_sum", "weight") if getattr(cache, n) is not None}
    s = {n: (t.double() if n != "weight" else t.clone()) for n, t in s.items()}
    for n in ("k", "v", "k_mean"):
        s[n] = getattr(cache, n).detach().float().cpu().double()
    s["held"], s["dtype"] = cache.k.dtype, cache.k_mean.dtype
    return s


def rounded(x, held):
    """Nearest value that `held` has, ties to even; x in units of the scale."""
    x = x.clamp(-MOST[held], MOST[held])
    if held == torch.int8:
        return torch.nan_to_num(torch.round(x))
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -9))).clamp_min(-6.0) - 3)
    return torch.round(x / step) * step


def scale_of(x, held):
    finite = x[torch.isfinite(x)]
    amax = finite.abs().max().item() if finite.numel() else 0.0
    e = -64
    while e < 64 and amax > MOST[held] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(s, k, v, cu, seqlens_k, table):
    """In place; returns the (page, place) pairs written."""
    held, P, pages = s["held"], s["k"].shape[2], s["k"].shape[0]
    written = set()
    for b in range(len(seqlens_k)):
        n, end = cu[b + 1] - cu[b], seqlens_k[b]
        for slot in range(len(table[b])):
            lo, hi, page = max(end - n, slot * P, 0), min(end, (slot + 1) * P), table[b][slot]
            if lo >= hi or not 0 <= page < pages:
                continue
            old = lo - slot * P
            for h in range(s["k"].shape[1]):
                for name, x in (("k", k), ("v", v)):
                    x = x[cu[b] + lo - (end - n):cu[b] + hi - (end - n), h].double()
                    scale = scale_of(x, held)
                    if old:
                        was = s[name + "_scale"][page, h].item()
                        if scale > was:
                            s[name][page, h, :old] = rounded(s[name][page, h, :old] * (was / scale), held)
                        scale = max(scale, was)
                    s[name + "_scale"][page, h] = scale
                    s[name][page, h, old:old + len(x)] = rounded(x / scale, held)
                    if name == "k":
                        s["k_sum"][page, h] = x.sum(0) + (s["k_sum"][page, h] if old else 0.0)
                        s["k_mean"][page, h] = s["k_sum"][page, h] / (old + len(x))
                if not old and "weight" in s:
                    s["weight"][page, h] = 0
            written |= {(page, old + i) for i in range(hi - lo)}
    return written


def attention(s, q, cu, seqlens_k, table, topk, scale=None):
    """out, lse, weight of every page and head in units of one, and what errors are relative to: sum of p |v| (rows, heads, features),
    largest sum of scale |q| |k| (heads, rows), largest |v| (heads, rows) and number of keys (heads, rows)."""
    P, dim, heads = s["k"].shape[2], q.shape[2], q.shape[1]
    G = heads // s["k"].shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((heads, q.shape[0]), math.inf, dtype=torch.float64)
    size, dot, most, count = torch.zeros_like(out), torch.zeros((heads, q.shape[0])).double(), torch.zeros((heads, q.shape[0])).double(), torch.zeros((heads, q.shape[0])).double()
    weight = torch.zeros(s["k_scale"].shape, dtype=torch.float64)
    for b in range(len(seqlens_k)):
        n = min(-(-max(seqlens_k[b], 0) // P), len(table[b]))
        if n == 0:
            continue
        pages = torch.tensor(table[b][:n])
        there = (pages >= 0) & (pages < s["k"].shape[0])
        pages = pages.where(there, torch.zeros_like(pages))
        for h, i0 in itertools.product(range(heads), range(cu[b], cu[b + 1], 128)):
            hk, rows = h // G, torch.arange(i0, min(i0 + 128, cu[b + 1]))
            x, pos = q[rows, h].double(), seqlens_k[b] - (cu[b + 1] - rows)
            own = torch.arange(n) == pos[:, None] // P
            score = x @ s["k_mean"][pages, hk].T
            score = score.where((torch.arange(n) < pos[:, None] // P) & there & (score > -math.inf), torch.tensor(-math.inf).double())
            best = n - 1 - score.flip(1).argsort(dim=1, descending=True, stable=True)[:, :topk - 1]  # of equals the later page
            chosen = torch.zeros_like(own).scatter(1, best, score.gather(1, best) > -math.inf) | (own & there)
            seen = chosen.repeat_interleave(P, 1) & (torch.arange(n * P) <= pos[:, None])
            used = chosen.any(0)  # (of the other pages nothing is needed)
            seen, chosen = seen[:, used.repeat_interleave(P)], chosen[:, used]
            k = (s["k"][pages[used], hk] * s["k_scale"][pages[used], hk][:, None, None]).reshape(-1, dim)
            v = (s["v"][pages[used], hk] * s["v_scale"][pages[used], hk][:, None, None]).reshape(-1, dim)
            some = seen.any(1)
            if not bool(some.any()):
                continue
            rows, x, seen = rows[some], x[some], seen[some]
            w = (x @ k.T * scale).where(seen, torch.tensor(-math.inf).double())
            lse[h, rows] = torch.logsumexp(w, 1)
            p = torch.softmax(w, 1)
            no_number = seen.double() @ v.isnan().double() > 0  # (a NaN that a row does not see is none of it)
            fine = v.nan_to_num(0.0)
            out[rows, h] = (p @ fine).masked_fill(no_number, math.nan)
            size[rows, h] = p @ fine.abs()
            most[h, rows] = fine.abs().amax(1).where(seen, torch.tensor(0.0).double()).amax(1)
            dot[h, rows] = (x.abs() @ k.abs().T).where(seen, torch.tensor(0.0).double()).amax(1) * abs(scale)
            count[h, rows] = seen.sum(1).double()
            weight[:, hk].index_add_(0, pages[used], p.view(len(rows), -1, P).sum((0, 2)))
    return out, lse, weight, (size, dot, most, count)


def evict(weight, seqlens_k, table, P, keep, sink, recent):
    kept, lens, freed = [], [], []
    for b, length in enumerate(seqlens_k):
        pages = table[b][:(length + P - 1) // P]
        n = len(pages)
        stay = set(range(n))
        if n > keep:
            fixed = set(range(min(sink, n))) | set(range(max(n - recent, 0), n))
            others = sorted((i for i in range(n) if i not in fixed), key=lambda i: (-int(weight[pages[i]].sum()) if 0 <= pages[i] < len(weight) else 0, i))
            stay = fixed | set(others[:keep - len(fixed)])
        kept.append([pages[i] for i in range(n) if i in stay])
        freed.append([pages[i] for i in range(n) if i not in stay])
        lens.append(length - P * len(freed[-1]))
    return kept, lens, freed
