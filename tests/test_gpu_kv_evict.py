"""flash_moba_cache_evict_func against a sort on the CPU: whole numbers, so everything has to be the same."""
import ctypes

import pytest
import torch

import cache_reference as R
import flash_moba
from flash_moba import flash_moba_hip as H

gpu = pytest.mark.gpu


def compare(weight, lens, table, P, keep, sink, recent):
    i32 = dict(dtype=torch.int32, device="cuda")
    t = torch.tensor(table, **i32)
    got = flash_moba.flash_moba_cache_evict_func(weight.cuda(), torch.tensor(lens, **i32), t, P, keep, sink_pages=sink, recent_pages=recent)
    kept, left, freed = R.evict(weight, lens, table, P, keep, sink, recent)
    width = t.shape[1]
    pad = lambda rows: [r + [-1] * (width - len(r)) for r in rows]  # noqa: E731
    assert got[0].tolist() == pad(kept)
    assert got[1].tolist() == left
    assert got[2].tolist() == pad(freed)
    assert got[3].tolist() == [len(f) for f in freed]


def tables(lens, P, pages, seed):
    g = torch.Generator().manual_seed(seed)
    width = max((n + P - 1) // P for n in lens) + 2
    return [torch.randperm(pages, generator=g)[:width].tolist() for _ in lens]


@gpu
@pytest.mark.parametrize("kind", ["any", "few values", "none", "huge", "one byte"])
@pytest.mark.parametrize("lens,P,heads_k,keep,sink,recent", [
    ([1], 64, 1, 1, 0, 1),
    ([0, 64, 65, 640, 641, 5000], 64, 2, 10, 1, 2),
    ([64 * 63 + 1, 100, 4096], 64, 8, 7, 3, 4),      # no place for others
    ([128 * 2500, 128 * 1024 - 5, 128 * 1025], 128, 3, 1000, 0, 1),
    ([64 * 1024], 64, 4, 1023, 1, 1),                # one goes
])
def test_pages_kept_are_those_of_a_sort(kind, lens, P, heads_k, keep, sink, recent):
    g = torch.Generator().manual_seed(len(lens) + keep)
    pages = 3000
    most = {"any": 1 << 40, "few values": 3, "none": 1, "huge": 1 << 59, "one byte": 256}[kind]
    weight = torch.randint(0, most, (pages, heads_k), generator=g, dtype=torch.int64)
    compare(weight, lens, tables(lens, P, pages, keep), P, keep, sink, recent)


@gpu
def test_more_pages_than_the_shared_memory_holds_and_entries_that_are_no_page():
    g = torch.Generator().manual_seed(3)
    weight = torch.randint(0, 1 << 20, (20000, 2), generator=g, dtype=torch.int64)
    lens = [64 * 17001 - 9, 64 * 8192, 64 * 8193]
    table = tables(lens, 64, 20000, 4)
    table[0][100] = table[1][7] = -1
    table[2][50] = 20000
    compare(weight, lens, table, 64, 4000, 2, 3)
    # a sequence that is longer than its table keeps what the table has
    i32 = dict(dtype=torch.int32, device="cuda")
    got = flash_moba.flash_moba_cache_evict_func(weight.cuda(), torch.tensor([64 * 9], **i32), torch.tensor([[5, 6, 7]], **i32), 64, 2, sink_pages=0, recent_pages=1)
    assert got[3].tolist() == [1] and got[0][0, 1].item() == 7


@gpu
def test_evict_replays_from_a_graph_and_leaves_its_inputs():
    i32 = dict(dtype=torch.int32, device="cuda")
    weight = torch.randint(0, 1 << 30, (500, 2), dtype=torch.int64, device="cuda")
    lens, table = torch.tensor([64 * 200, 64 * 30 - 3], **i32), torch.tensor(tables([64 * 200, 64 * 30], 64, 500, 5), **i32)
    was = table.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = flash_moba.flash_moba_cache_evict_func(weight, lens, table, 64, 20)
    for _ in range(3):
        weight.random_(0, 1 << 30)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = flash_moba.flash_moba_cache_evict_func(weight, lens, table, 64, 20)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert torch.equal(table, was)
    traced = torch.compile(lambda w: flash_moba.flash_moba_cache_evict_func(w, lens, table, 64, 20), backend="aot_eager", fullgraph=True)(weight)
    assert all(torch.equal(a, b) for a, b in zip(traced, want))


@gpu
@pytest.mark.parametrize("change,message", [(dict(keep=2), "fewer pages to keep"), (dict(recent=0), "being filled"), (dict(sink=-1), "sink"), (dict(P=0), "page_size"),
                                            (dict(weight=torch.float32), "weight must be"), (dict(keep=1 << 40), "below 2"), (dict(lens=2), "block_table")])
def test_refusals(change, message):
    i32 = dict(dtype=torch.int32, device="cuda")
    weight = torch.zeros((4, 2), dtype=change.get("weight", torch.int64), device="cuda")
    with pytest.raises(RuntimeError, match=message):
        flash_moba.flash_moba_cache_evict_func(weight, torch.zeros(change.get("lens", 1), **i32), torch.zeros((1, 3), **i32), change.get("P", 64), change.get("keep", 8),
                                               sink_pages=change.get("sink", 1), recent_pages=change.get("recent", 2))


def test_the_entry_point_refuses_without_a_gpu():
    lib = H.load_library()
    assert lib.fmoba_cache_evict(None, None) != 0
    assert lib.fmoba_cache_evict_workspace_bytes(4, 1024) == 0 and lib.fmoba_cache_evict_workspace_bytes(4, 1025) == 4 * 1025 * 8

    def args(**kw):
        a = H.CacheEvictArgs()
        a.weight = a.seqlens_k = a.block_table = a.new_table = a.new_seqlens = a.freed = a.num_freed = 4096
        a.batch, a.max_pages, a.num_pages, a.heads_k, a.page_size, a.keep, a.sink, a.recent, a.table_stride = 2, 16, 64, 2, 64, 8, 1, 1, 16
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    for kw, message in [(dict(batch=0), b"batch"), (dict(heads_k=0), b"heads"), (dict(page_size=0), b"page_size"), (dict(recent=0), b"being filled"), (dict(sink=-1), b"sink"), (dict(keep=1), b"fewer"),
                        (dict(weight=0), b"null"), (dict(freed=0), b"null"), (dict(max_pages=9000), b"workspace")]:
        assert lib.fmoba_cache_evict(ctypes.byref(args(**kw)), None) != 0, kw
        assert message in lib.fmoba_last_error(), (kw, lib.fmoba_last_error())
