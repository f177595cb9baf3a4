"""The paged 8-bit cache in 64 bits on the CPU, written from its definition: a dict of tensors like MobaKVCache's fields, and what the functions do to it."""
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
        for i in range(cu[b], cu[b + 1]):
            pos = seqlens_k[b] - (cu[b + 1] - i)
            if pos < 0:
                continue
            for h in range(heads):
                hk, x = h // G, q[i, h].double()
                there = [c for c in range(pos // P + 1) if 0 <= table[b][c] < s["k"].shape[0]]
                score = [((x @ s["k_mean"][table[b][c], hk]).item(), c) for c in there if c < pos // P]
                score = sorted(e for e in score if e[0] > -math.inf)[::-1]
                chosen = [c for _, c in score[:topk - 1]] + [c for c in there if c == pos // P]
                parts, vs = [], []
                for c in chosen:
                    page, n = table[b][c], min(P, pos + 1 - c * P)
                    k = s["k"][page, hk, :n] * s["k_scale"][page, hk]
                    parts.append(k @ x * scale)
                    dot[h, i] = max(dot[h, i].item(), (k.abs() @ x.abs()).max().item() * abs(scale))
                    vs.append(s["v"][page, hk, :n] * s["v_scale"][page, hk])
                if not chosen:
                    continue
                w = torch.cat(parts)
                lse[h, i] = torch.logsumexp(w, 0)
                p = torch.softmax(w, 0)
                vs = torch.cat(vs)
                out[i, h], size[i, h], most[h, i], count[h, i] = p @ vs, p @ vs.abs(), vs.abs().max(), len(w)
                for c, part in zip(chosen, p.split([len(x) for x in parts])):
                    weight[table[b][c], hk] += part.sum()
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
