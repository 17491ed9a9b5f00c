"""GPU: paged_extend with the count of free pages updated in place.  Its CTAs are then one cluster, and the count is written when
all of them have read it: sizes of 1, 2, 4 and 8 CTAs, few and many threads, more than 48 KB of shared memory, again and
again, and replayed."""
import pytest
import torch

from test_paged_cache_gpu import Account, ints, tensors

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1, 1), (30, 8, 200, 9), (200, 16, 513, 3), (300, 16, 1500, 5), (1023, 16, 3000, 4), (1025, 32, 5000, 6), (5000, 3, 9000, 3),
         (1025, 32, 20000, 40), (16384, 16, 16384, 1)]


def book(B, page, new_hi, pages=60000):
    a = Account(pages, page, B, max(1, (new_hi + 60) // page + 1), seed=B)
    a.lengths = [a.rng.randint(0, 50) for _ in range(B)]
    for b in range(B):
        for c in range(a.need(a.lengths[b])):
            a.table[b][c] = a.free.pop()
    return a


@pytest.mark.parametrize("B,page,rows,new_hi", SIZES)
def test_sizes(pkg, cuda, B, page, rows, new_hi):
    a = book(B, page, new_hi)
    new = [a.rng.randint(0, new_hi) for _ in range(B)]
    table, lengths, free, count = tensors(cuda, a)
    before, table0, added = count.clone(), table.clone(), ints(cuda, new)
    start, granted, maps = a.extend(new, rows)
    made = pkg.paged_extend(table.clone(), lengths, added, free, before, rows=rows, page_size=page)
    out = made._replace(free_count=count)
    for _ in range(20):
        count.copy_(before)
        table.copy_(table0)
        r = pkg.paged_extend(table, lengths, added, free, count, rows=rows, page_size=page, out=out)
        assert r.free_count is count and count.item() == len(a.free)
        assert r.row_start.tolist() == start and r.granted.tolist() == granted and torch.equal(table, ints(cuda, a.table))
        assert torch.equal(torch.stack((r.request, r.position, r.slot), 1), ints(cuda, maps))


@pytest.mark.parametrize("B,page,rows,new_hi", [(30, 8, 200, 9), (300, 16, 1500, 5), (5000, 3, 9000, 3)])
def test_replayed(pkg, cuda, B, page, rows, new_hi):
    """Steps of a captured extend and keep, the count in place in both."""
    a = book(B, page, new_hi)
    new = [a.rng.randint(0, new_hi) for _ in range(B)]
    table, lengths, free, count = tensors(cuda, a)
    added, kept = ints(cuda, new), ints(cuda, [0] * B)
    out = pkg.paged_extend(table.clone(), lengths, added, free, count.clone(), rows=rows, page_size=page)._replace(free_count=count)

    def step():
        pkg.paged_extend(table, lengths, added, free, count, rows=rows, page_size=page, out=out)
        pkg.paged_keep(table, lengths, out.granted, kept, free, count, page_size=page, lengths_out=lengths, free_count_out=count)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        new = [a.rng.randint(0, new_hi) for _ in range(B)]
        keep = [a.rng.choice([-1, 0, 1, new_hi]) if i % 2 else a.rng.randint(-1, 2) for _ in range(B)]
        added.copy_(ints(cuda, new))
        kept.copy_(ints(cuda, keep))
        start, granted, maps = a.extend(new, rows)
        a.keep(granted, keep)
        graph.replay()
        torch.cuda.synchronize()
        assert out.granted.tolist() == granted and out.row_start.tolist() == start and lengths.tolist() == a.lengths
        assert count.item() == len(a.free) and free[:len(a.free)].tolist() == a.free
        assert torch.equal(torch.stack((out.request, out.position, out.slot), 1), ints(cuda, maps))


def test_an_abandoned_step(pkg, cuda):
    """With the count in place a step that is given up gives its pages back by a keep of nothing; with a count of its own it costs nothing."""
    a = book(40, 8, 20, pages=900)
    table, lengths, free, count = tensors(cuda, a)
    new, before, left = [20] * 40, len(a.free), sorted(a.free)
    r = pkg.paged_extend(table, lengths, ints(cuda, new), free, count, rows=800, page_size=8)
    assert r.free_count.item() < before and count.item() == before
    r = pkg.paged_extend(table, lengths, ints(cuda, new), free, count, rows=800, page_size=8, out=r._replace(free_count=count))
    assert count.item() < before
    pkg.paged_keep(table, lengths, r.granted, ints(cuda, [0] * 40), free, count, page_size=8, lengths_out=lengths, free_count_out=count)
    assert count.item() == before and lengths.tolist() == a.lengths and sorted(free[:before].tolist()) == left
