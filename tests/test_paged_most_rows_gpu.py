"""GPU: page tables, maps and free lists of almost 2^31 entries: a thread's next index lies behind 2^31."""
import pytest
import torch

pytestmark = pytest.mark.gpu

MOST = 0x7fffffff - 65536      # the most rows of a call


def room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip("not enough memory free")


def ints(cuda, *values):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def is_all(t, value):
    low, high = t.aminmax()
    return low.item() == value == high.item()


def test_maps(pkg, cuda):
    room(40)
    guard = 1 << 20
    whole = torch.full((3 * (MOST + 1) + guard,), 77, dtype=torch.int32, device=cuda)
    maps = [whole[guard + i * (MOST + 1):][:MOST] for i in range(3)]
    table, lengths, free, count = ints(cuda, *[-1] * 8).view(2, 4), ints(cuda, 3, 0), ints(cuda, *range(9)), ints(cuda, 9)
    table[0, 0] = 8
    out = pkg.PagedRows(ints(cuda, 0, 0, 0), ints(cuda, 0, 0), *maps, ints(cuda, 0))
    pkg.paged_extend(table, lengths, ints(cuda, 5, 3), free, count, rows=MOST, page_size=4, out=out)
    assert out.row_start.tolist() == [0, 5, 8] and out.granted.tolist() == [5, 3] and out.free_count.item() == 7
    assert maps[0][:8].tolist() == [0] * 5 + [1] * 3 and maps[1][:8].tolist() == [3, 4, 5, 6, 7, 0, 1, 2]
    assert maps[2][:8].tolist() == [35, 32, 33, 34, 35, 28, 29, 30]
    for i, m in enumerate(maps):
        assert is_all(m[8:], -1) and whole[guard + i * (MOST + 1) + MOST].item() == 77
    assert is_all(whole[:guard], 77)
    del whole, maps, m, out
    torch.cuda.empty_cache()


def test_pages(pkg, cuda):
    """One request takes almost 2^31 pages of one token, and gives them back."""
    room(60)
    pages = 0x7fffffff
    free = torch.arange(pages, dtype=torch.int32, device=cuda)
    table = torch.full((1, pages), -1, dtype=torch.int32, device=cuda)
    lengths, count = ints(cuda, 0), ints(cuda, pages)
    r = pkg.paged_extend(table, lengths, ints(cuda, MOST), free, count, rows=MOST, page_size=1)
    assert r.granted.item() == MOST and r.free_count.item() == pages - MOST and is_all(r.request, 0)
    # the i-th token takes the i-th page from the list's end
    assert r.position[0].item() == 0 and is_all(r.position[1:] - r.position[:-1], 1)
    assert is_all(r.slot.add_(r.position), pages - 1)
    assert is_all(table[0, :MOST].add_(r.position), pages - 1) and is_all(table[0, MOST:], -1)
    del r
    table[0, :MOST] = torch.arange(MOST, dtype=torch.int32, device=cuda)
    left = ints(cuda, pages - MOST)
    pkg.paged_keep(table, lengths, ints(cuda, MOST), ints(cuda, -1), free, left, page_size=1, lengths_out=lengths, free_count_out=count)
    assert lengths.item() == 0 and count.item() == pages
    assert free[pages - MOST].item() == 0 and is_all(free[pages - MOST + 1:] - free[pages - MOST:-1], 1)
    assert is_all(free[:pages - MOST] - torch.arange(pages - MOST, dtype=torch.int32, device=cuda), 0)
    del free, table
    torch.cuda.empty_cache()
