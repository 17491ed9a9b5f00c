"""GPU: the page tables and maps of a paged cache, and what follows a verification, against a plain account in Python."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(cuda, values):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Account:
    """The same books kept in Python lists."""

    def __init__(self, pages, page, requests, columns, seed=0):
        self.page, self.columns, self.rng = page, columns, random.Random(seed)
        self.free = list(range(pages))
        self.rng.shuffle(self.free)
        self.pages = pages
        self.table = [[-9] * columns for _ in range(requests)]
        self.lengths = [0] * requests

    def need(self, tokens):
        return -(-tokens // self.page)

    def extend(self, new, rows):
        start, granted, maps, wanted, end, taken = [0], [], [(-1, -1, -1)] * rows, 0, 0, 0
        count = len(self.free)
        for b, n in enumerate(new):
            n = max(n, 0)
            end += n
            L = self.lengths[b]
            fits = 0 <= L and L + n <= self.columns * self.page and end <= rows
            need = self.need(L + n) - self.need(L) if fits else 0
            wanted += need
            served = fits and (need == 0 or wanted <= count)
            if served:
                for i in range(need):
                    self.table[b][self.need(L) + i] = self.free.pop()
                for j in range(n):
                    p = L + j
                    maps[start[-1] + j] = (b, p, self.table[b][p // self.page] * self.page + p % self.page)
            granted.append(n if served else 0)
            start.append(min(end, rows))
        return start, granted, maps

    def keep(self, granted, kept, path=None):
        moves = []
        for b, (n, k) in enumerate(zip(granted, kept)):
            L = self.lengths[b]
            good = min(k, n)
            if path is not None and good > 0:
                good, last = min(good, len(path[b])), -1
                for j in range(good):
                    if not last < path[b][j] < n:
                        good = j
                        break
                    last = path[b][j]
                    moves.append((b, L + path[b][j], L + j))
            after = 0 if k < 0 else L + good
            for c in range(self.need(after), self.need(L + n)):
                self.free.append(self.table[b][c])
            self.lengths[b] = after
        return moves


def tensors(cuda, a):
    free = torch.full((a.pages,), -3, dtype=torch.int32, device=cuda)
    free[:len(a.free)] = ints(cuda, a.free)
    return ints(cuda, a.table), ints(cuda, a.lengths), free, ints(cuda, [len(a.free)])


def test_a_run_of_steps(pkg, cuda):
    """Prompts, trees, refusals for want of pages, ends of requests, all in place, as a server's loop has it."""
    B, page, pages, rows = 37, 8, 60, 300
    a = Account(pages, page, B, 20, seed=3)
    table, lengths, free, count = tensors(cuda, a)
    step_count = torch.empty_like(count)
    out = None
    short = 0
    for step in range(40):
        new = [a.rng.choice([0, 1, 1, 3, 8, 17]) if step else 5 for _ in range(B)]
        new[a.rng.randrange(B)] = -2
        start, granted, maps = a.extend(new, rows)
        r = pkg.paged_extend(table, lengths, ints(cuda, new), free, count, rows=rows, page_size=page, out=out)
        out = r._replace(free_count=step_count)       # (from the second step on, into the same tensors)
        assert r.row_start.tolist() == start and r.granted.tolist() == granted
        assert list(zip(r.request.tolist(), r.position.tolist(), r.slot.tolist())) == maps
        assert r.free_count.item() == len(a.free) and table.tolist() == a.table
        short += granted != [max(n, 0) for n in new]
        width = 9
        path = [sorted(a.rng.sample(range(20), width)) if a.rng.random() < 0.8 else [a.rng.randrange(-2, 9) for _ in range(width)] for _ in range(B)]
        kept = [-1 if a.rng.random() < 0.05 else a.rng.randint(0, 12) for _ in range(B)]
        a.keep(granted, kept, path)
        pool = torch.zeros(pages, page, 1, 8, dtype=torch.float16, device=cuda)
        got, c = pkg.paged_keep(table, lengths, r.granted, ints(cuda, kept), free, r.free_count, page_size=page, path=ints(cuda, path), k_pages=pool,
                                v_pages=pool.clone(), lengths_out=lengths, free_count_out=count)
        assert got is lengths and c is count
        assert lengths.tolist() == a.lengths and count.item() == len(a.free) and free[:len(a.free)].tolist() == a.free
    assert short > 3


@pytest.mark.parametrize("B,page,rows,new_hi", [(1, 1, 1, 1), (1, 16, 5000, 5000), (3, 7, 40, 9), (1023, 16, 3000, 4), (1025, 32, 20000, 40),
                                                (5000, 3, 9000, 3), (16384, 16, 16384, 1)])
def test_sizes(pkg, cuda, B, page, rows, new_hi):
    a = Account(60000, page, B, max(1, (new_hi + 60) // page + 1), seed=B)
    a.lengths = [a.rng.randint(0, 50) for _ in range(B)]
    for b in range(B):
        for c in range(a.need(a.lengths[b])):
            a.table[b][c] = a.free.pop()
    new = [a.rng.randint(0, new_hi) for _ in range(B)]
    table, lengths, free, count = tensors(cuda, a)
    start, granted, maps = a.extend(new, rows)
    r = pkg.paged_extend(table, lengths, ints(cuda, new), free, count, rows=rows, page_size=page)
    assert r.row_start.tolist() == start and r.granted.tolist() == granted and r.free_count.item() == len(a.free)
    assert r.request.tolist() == [m[0] for m in maps] and r.position.tolist() == [m[1] for m in maps] and r.slot.tolist() == [m[2] for m in maps]
    assert torch.equal(table, ints(cuda, a.table))
    kept = [a.rng.randint(-1, new_hi) for _ in range(B)]
    a.keep(granted, kept)
    after, left = pkg.paged_keep(table, lengths, r.granted, ints(cuda, kept), free, r.free_count, page_size=page)
    assert after.tolist() == a.lengths and left.item() == len(a.free) and torch.equal(free[:len(a.free)], ints(cuda, a.free))


def test_the_table_of_a_wider_one_and_empty_batches(pkg, cuda):
    wide = torch.full((4, 30), -9, dtype=torch.int32, device=cuda)
    free = torch.arange(50, dtype=torch.int32, device=cuda)
    r = pkg.paged_extend(wide[:, 3:13], ints(cuda, [0, 0, 0, 0]), ints(cuda, [1, 20, 0, 3]), free, ints(cuda, [50]), rows=24, page_size=4)
    assert wide[:, 3:9].tolist() == [[49, -9, -9, -9, -9, -9], [48, 47, 46, 45, 44, -9], [-9] * 6, [43, -9, -9, -9, -9, -9]]
    assert (wide[:, :3] == -9).all() and (wide[:, 13:] == -9).all() and r.free_count.item() == 43
    none = pkg.paged_extend(wide[:0], ints(cuda, []), ints(cuda, []), free, ints(cuda, [50]), rows=3, page_size=4)
    assert none.row_start.tolist() == [0] and none.slot.tolist() == [-1] * 3 and none.free_count.item() == 50
    none = pkg.paged_extend(wide, ints(cuda, [0] * 4), ints(cuda, [1] * 4), free, ints(cuda, [50]), rows=0, page_size=4)
    assert none.granted.tolist() == [0] * 4 and none.row_start.tolist() == [0] * 5
    lengths, count = pkg.paged_keep(wide[:0], ints(cuda, []), ints(cuda, []), ints(cuda, []), free, ints(cuda, [50]), page_size=4)
    assert lengths.numel() == 0 and count.item() == 50


@pytest.mark.parametrize("layers,heads,size,page,dtype", [(1, 1, 8, 4, torch.bfloat16), (5, 3, 80, 16, torch.float16), (2, 4, 256, 64, torch.bfloat16),
                                                          (30, 8, 128, 8, torch.bfloat16)])
@pytest.mark.parametrize("width", [1, 7, 40])
def test_accepted_drafts_close_up(pkg, cuda, layers, heads, size, page, dtype, width):
    B = 11
    a = Account(80 + B * 60 // page + 1, page, B, 70 // page + 10, seed=width)
    table, lengths, free, count = tensors(cuda, a)
    r = pkg.paged_extend(table, lengths, ints(cuda, [5 + 2 * b for b in range(B)]), free, count, rows=400, page_size=page)
    a.extend([5 + 2 * b for b in range(B)], 400)
    a.keep([5 + 2 * b for b in range(B)], [5 + 2 * b for b in range(B)])
    lengths = ints(cuda, a.lengths)
    new = [a.rng.randint(0, 41) for _ in range(B)]
    _, granted, _ = a.extend(new, 600)
    r = pkg.paged_extend(table, lengths, ints(cuda, new), free, r.free_count, rows=600, page_size=page)
    assert granted == new
    # one cache by layers, one whose heads come before its tokens
    k = torch.randn(layers, a.pages, page, heads, size, device=cuda).to(dtype)
    v = torch.randn(layers, a.pages, heads, page, size, device=cuda).to(dtype).transpose(2, 3)
    path = [sorted(a.rng.sample(range(42), width)) for _ in range(B)]
    path[3] = [i for i in range(width)]                        # nothing moves
    kept = [a.rng.randint(0, width) for _ in range(B)]
    kept[5] = -1
    want_k, want_v = k.clone(), v.clone()
    slot = lambda b, p: (a.table[b][p // page], p % page)
    before_k, before_v = k.clone(), v.clone()
    for b, s, t in a.keep(granted, kept, path):
        want_k[:, slot(b, t)[0], slot(b, t)[1]] = before_k[:, slot(b, s)[0], slot(b, s)[1]]
        want_v[:, slot(b, t)[0], slot(b, t)[1]] = before_v[:, slot(b, s)[0], slot(b, s)[1]]
    after, left = pkg.paged_keep(table, lengths, r.granted, ints(cuda, kept), free, r.free_count, page_size=page, path=ints(cuda, path),
                                 k_pages=k, v_pages=v)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    assert after.tolist() == a.lengths and left.item() == len(a.free) and free[:len(a.free)].tolist() == a.free


def test_numbers_outside_their_ranges(pkg, cuda):
    """Whatever the tensors on the GPU hold, nothing is written outside (the guards around them stay as they are)."""
    B, page, pages = 4, 8, 12
    whole = torch.full((6, 10), 77, dtype=torch.int32, device=cuda)
    table = whole[1:5, 2:7]
    table.copy_(ints(cuda, [[0, 1, -4, 2 ** 30, 5], [2 ** 31 - 1] * 5, [3, 4, 5, 6, 7], [-1] * 5]))
    extra = torch.full((pages + 8,), 55, dtype=torch.int32, device=cuda)
    free = extra[4:4 + pages].copy_(torch.arange(pages, device=cuda) * 3 - 9)
    pools = torch.full((2, pages + 2, page, 2, 16), 1.0, dtype=torch.bfloat16, device=cuda)
    for lengths, new, count, kept, path in (
            ([-1, 2 ** 31 - 1, 30, 3], [5, 5, 2 ** 31 - 1, -3], 2 ** 31 - 1, [3, 2 ** 31 - 1, 2, -1], [[0, 1, 2]] * 4),
            ([20, 17, 40, 0], [2, 9, 1, 40], -7, [2, 9, 1, 40], [[1, 3, 2 ** 31 - 1], [0, 8, 9], [-1, 0, 1], [5, 6, 39]])):
        r = pkg.paged_extend(table, ints(cuda, lengths), ints(cuda, new), free, ints(cuda, [count]), rows=20, page_size=page)
        assert 0 <= r.free_count.item() <= pages and r.row_start.min() >= 0 and r.row_start.max() <= 20
        assert (r.slot < pages * page).all()
        granted = r.granted if count < 0 else ints(cuda, [2 ** 31 - 1, 5, -4, 9])
        after, left = pkg.paged_keep(table, ints(cuda, lengths), granted, ints(cuda, kept), free, ints(cuda, [count]), page_size=page,
                                     path=ints(cuda, path), k_pages=pools[0, 1:-1], v_pages=pools[1, 1:-1])
        assert 0 <= left.item() <= pages and after.min() >= 0
    assert (whole[0] == 77).all() and (whole[5] == 77).all() and (whole[:, :2] == 77).all() and (whole[:, 7:] == 77).all()
    assert (extra[:4] == 55).all() and (extra[4 + pages:] == 55).all() and (pools == 1.0).all()


def test_refusals(pkg, cuda):
    table, lengths, new = torch.zeros(2, 5, dtype=torch.int32, device=cuda), ints(cuda, [3, 4]), ints(cuda, [1, 1])
    free, count = torch.arange(9, dtype=torch.int32, device=cuda), ints(cuda, [9])
    n0 = pkg.launch_count()

    def refused(status, fn, *a, **k):
        with pytest.raises(pkg.IxkError) as e:
            fn(*a, **k)
        assert e.value.status == status, str(e.value)

    bad, un = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED
    extend = lambda t=table, l=lengths, n=new, f=free, c=count, rows=4, page=16, **k: pkg.paged_extend(t, l, n, f, c, rows=rows, page_size=page, **k)
    refused(bad, extend, table.long())
    refused(bad, extend, table.t())
    refused(bad, extend, l=lengths[:1])
    refused(bad, extend, n=new.float())
    refused(bad, extend, c=ints(cuda, [1, 2]))
    refused(bad, extend, page=0)
    refused(bad, extend, rows=-1)
    refused(un, extend, page=2 ** 29)
    refused(bad, extend, f=free[:0])
    refused(bad, extend, table[:, :0])
    refused(un, extend, torch.zeros(20000, 1, dtype=torch.int32, device=cuda), torch.zeros(20000, dtype=torch.int32, device=cuda),
            torch.zeros(20000, dtype=torch.int32, device=cuda))
    good = pkg.PagedRows(*(torch.zeros(n, dtype=torch.int32, device=cuda) for n in (3, 2, 4, 4, 4, 1)))
    refused(bad, extend, out=good._replace(granted=new))
    refused(bad, extend, out=good._replace(slot=good.slot[:3]))
    refused(pkg.IXK_NO_DEVICE, extend, n=new.cpu())
    pool = torch.zeros(9, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    path = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    keep = lambda **k: pkg.paged_keep(table, lengths, new, new.clone(), free, count, page_size=16, **k)
    refused(bad, keep, path=path)
    refused(bad, keep, k_pages=pool, v_pages=pool)
    refused(bad, keep, path=path[:1], k_pages=pool, v_pages=pool)
    refused(bad, keep, path=path, k_pages=pool, v_pages=pool[:8])
    refused(bad, keep, path=path, k_pages=pool[:8], v_pages=pool[:8])
    refused(bad, keep, path=path[:, :0], k_pages=pool, v_pages=pool)
    refused(un, keep, path=path, k_pages=pool.float(), v_pages=pool.float())
    refused(un, keep, path=path, k_pages=pool[..., :60], v_pages=pool[..., :60])
    refused(un, keep, path=torch.zeros(2, 2000, dtype=torch.int32, device=cuda), k_pages=pool, v_pages=pool)
    refused(bad, keep, lengths_out=new)
    refused(bad, keep, path=path, k_pages=pool, v_pages=pool)           # the same memory twice: moved twice
    assert pkg.launch_count() == n0


def test_replayed_on_another_stream_and_without_native_calls(pkg, cuda, monkeypatch):
    """A captured step that keeps its books in place: three replays are three steps."""
    def state():
        a = Account(200, 4, 6, 30, seed=1)
        return a, *tensors(cuda, a)

    a, table, lengths, free, count = state()
    new, kept, path = ints(cuda, [3, 4, 5, 1, 0, 9]), ints(cuda, [2, 4, 1, 0, 0, 3]), ints(cuda, [[0, 2, 8, 9]] * 6)
    pool, values = torch.randn(2, 200, 4, 1, 8, device=cuda).half()
    step_count = torch.zeros_like(count)
    out = pkg.PagedRows(*(torch.zeros(n, dtype=torch.int32, device=cuda) for n in (7, 6, 25, 25, 25)), step_count)

    def step(stream=None):
        r = pkg.paged_extend(table, lengths, new, free, count, rows=25, page_size=4, out=out, stream=stream)
        pkg.paged_keep(table, lengths, r.granted, kept, free, r.free_count, page_size=4, path=path, k_pages=pool, v_pages=values, lengths_out=lengths,
                       free_count_out=count, stream=stream)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(side)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    graph.replay()
    monkeypatch.setattr(pkg, "_NATIVE", None)
    step()
    for _ in range(5):
        _, granted, _ = a.extend(new.tolist(), 25)
        a.keep(granted, kept.tolist(), path.tolist())
    assert lengths.tolist() == a.lengths and count.item() == len(a.free) and free[:len(a.free)].tolist() == a.free


def test_paths_that_name_an_entry_twice_or_go_back(pkg, cuda):
    """Such a path ends before the entry; what it kept so far moves."""
    table, lengths, free, count = ints(cuda, [[0, 1], [2, 3], [4, 5]]), ints(cuda, [3, 0, 2]), ints(cuda, [-1] * 6), ints(cuda, [0])
    granted, kept, path = ints(cuda, [5, 5, 5]), ints(cuda, [4, 4, 4]), ints(cuda, [[1, 1, 2, 3], [0, 3, 2, 4], [2, 3, 5, 4]])
    k, v = torch.randn(2, 2, 6, 4, 1, 8, device=cuda).half()
    flat = [t.clone().view(2, 24, 8) for t in (k, v)]
    for t, before in zip(flat, [t.clone() for t in flat]):
        for to, source in ((3, 4), (9, 11), (18, 20), (19, 21)):
            t[:, to] = before[:, source]
    after, left = pkg.paged_keep(table, lengths, granted, kept, free, count, page_size=4, path=path, k_pages=k, v_pages=v)
    assert after.tolist() == [4, 2, 4] and torch.equal(k.view(2, 24, 8), flat[0]) and torch.equal(v.view(2, 24, 8), flat[1])
    assert left.item() == 3 and free.tolist() == [1, 3, 5, -1, -1, -1]


def test_a_cache_of_more_than_2_to_the_31_elements(pkg, cuda):
    """Norm and rotation into its last page, and a move there."""
    pages, page = 2 ** 31 // (16 * 8 * 64) + 40, 16
    k = torch.empty(pages, page, 8, 64, dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    q, kk, vv = (torch.randn(3, n, 64, device=cuda).bfloat16() for n in (8, 8, 8))
    cos, sin = torch.ones(20, 8, device=cuda), torch.zeros(20, 8, device=cuda)
    last = pages - 1
    slots = ints(cuda, [last * page + i for i in (9, 11, 14)])
    pkg.qk_norm_rotary_forward(q, kk, cos=cos, sin=sin, positions=ints(cuda, [9, 11, 14]), v=vv, slots=slots, k_pages=k, v_pages=v)
    _, dense = pkg.qk_norm_rotary_forward(q, kk, cos=cos, sin=sin, positions=ints(cuda, [9, 11, 14]))
    assert torch.equal(k[last, [9, 11, 14]], dense) and torch.equal(v[last, [9, 11, 14]], vv)
    after, left = pkg.paged_keep(ints(cuda, [[last]]), ints(cuda, [9]), ints(cuda, [7]), ints(cuda, [3]), torch.zeros(pages, dtype=torch.int32, device=cuda),
                                 ints(cuda, [0]), page_size=page, path=ints(cuda, [[0, 2, 5]]), k_pages=k, v_pages=v)
    assert after.item() == 12 and left.item() == 0
    assert torch.equal(k[last, 9:12], dense) and torch.equal(v[last, 9:12], vv)
