"""GPU: attention of packed rows over a paged cache against the definition in 64 bits.

Tolerance.  With weights w = p / sum p, rounding each p by at most u = eps / 2 of the type and dividing by the sum of the
rounded ones gives o' - o = sum w d (v - o) / (1 + sum w d), |d| <= u: at most u / (1 - u) of sum w |v - o| <= sum w |v| + |o|.
Scores: H products summed in fp32 (each addition cuts at most 2^-23 of the sum of their sizes), the factor and 2^x at a few
2^-23 more: an error e of the exponent changes a weight by e.  The result itself is rounded once, by u |o|.  The sums of
the weights and of P.V are of up to T terms in fp32, and positive or bounded by sum w |v|: below 2^-14 of it for the lengths here."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(cuda, lengths, new, heads, kv_heads, size, page, dtype, seed=0, columns=None, layout="tokens", stale=float("nan")):
    """A cache whose every place that no token holds is `stale`, pages in random order."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    B, total = len(lengths), [a + b for a, b in zip(lengths, new)]
    used = [-(-t // page) for t in total]
    columns = columns or max(max(used), 1)
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=cuda).int()
    table = torch.full((B, columns), -7, dtype=torch.int32, device=cuda)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n

    def cache():
        if layout == "tokens":
            c = torch.empty(pages, page, kv_heads, size, dtype=dtype, device=cuda)
        elif layout == "heads":
            c = torch.empty(pages, kv_heads, page, size, dtype=dtype, device=cuda).transpose(1, 2)
        else:       # a slice of something wider
            c = torch.empty(pages, page, kv_heads + 1, size + 24, dtype=dtype, device=cuda)[:, :, 1:, 16:16 + size]
        c.fill_(stale)
        for b in range(B):
            for i in range(used[b]):
                n = min(page, total[b] - i * page)
                c[table[b, i], :n] = torch.randn(n, kv_heads, size, generator=g, device=cuda).to(dtype)
        return c

    rows = sum(new)
    return {"q": torch.randn(rows, heads, size, generator=g, device=cuda).mul_(1.5).to(dtype), "k": cache(), "v": cache(), "table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=cuda), "granted": torch.tensor(new, dtype=torch.int32, device=cuda),
            "row_start": torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=cuda), "scale": size ** -0.5, "mask": None}


def random_mask(s, words, seed=1, share=0.5):
    """Any pattern of bits, those behind the drafts too."""
    g = torch.Generator(device=s["q"].device).manual_seed(seed)
    bits = torch.rand(s["q"].shape[0], words, 32, generator=g, device=s["q"].device) < share
    v = (bits.long() << torch.arange(32, device=bits.device)).sum(2)
    return torch.where(v >= 2 ** 31, v - 2 ** 32, v).int()


def call(pkg, s, **more):
    return pkg.fmha_paged_forward(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["row_start"], s["granted"], scale=s["scale"],
                                  mask=s["mask"], with_lse=True, **more)


def seen(s, b, r0, n, L):
    """[n, L + n]: what each row sees."""
    dev = s["q"].device
    if s["mask"] is None:
        drafts = torch.ones(n, n, dtype=torch.bool, device=dev).tril()
    else:
        i = torch.arange(n, device=dev)
        words = s["mask"][r0:r0 + n].long()
        inside = i < 32 * words.shape[1]
        drafts = (words[:, torch.where(inside, i, 0) // 32] >> (i % 32) & 1 > 0) & inside
    return torch.cat((torch.ones(n, L, dtype=torch.bool, device=dev), drafts), 1)


def expected(s):
    """(row of q, out, lse, tolerance of out, of lse) of every request, in 64 bits."""
    page, H = s["k"].shape[1], s["q"].shape[2]
    u = torch.finfo(s["q"].dtype).eps / 2
    group = s["q"].shape[1] // s["k"].shape[2]
    for b, (L, n, r0) in enumerate(zip(s["lengths"].tolist(), s["granted"].tolist(), s["row_start"].tolist())):
        if n == 0:
            continue
        ids = s["table"][b, :-(-(L + n) // page)].long()
        k = s["k"][ids].flatten(0, 1)[:L + n].double().repeat_interleave(group, 1).transpose(0, 1)
        v = s["v"][ids].flatten(0, 1)[:L + n].double().repeat_interleave(group, 1).transpose(0, 1)
        q = s["q"][r0:r0 + n].double().transpose(0, 1)
        hidden = ~seen(s, b, r0, n, L)
        z = (q @ k.transpose(1, 2) * s["scale"]).masked_fill(hidden, -math.inf)
        lse = torch.logsumexp(z, 2)
        w = torch.where(torch.isfinite(lse)[..., None], torch.exp(z - lse[..., None]), torch.zeros_like(z))
        w = w.masked_fill(hidden, 0.0)
        o = w @ v
        sizes = (q.abs() @ k.abs().transpose(1, 2) * abs(s["scale"])).masked_fill(hidden, 0.0).amax(2)
        e = (H + 8) * 2.0 ** -23 * sizes + 2.0 ** -20
        spread = w @ v.abs() + o.abs()
        tol = u * o.abs() + (u / (1 - u) + e[..., None] + 2.0 ** -14) * spread + 1e-30
        yield r0, o.transpose(0, 1), lse.t(), tol.transpose(0, 1), (e + 2.0 ** -20 + lse.abs().nan_to_num(posinf=0.0) * 2.0 ** -22).t()


def check(s, out, lse):
    for r0, o, e, tol, tol_lse in expected(s):
        n = o.shape[0]
        bad = (out[r0:r0 + n].double() - o).abs() > tol
        assert not bad.any() and out[r0:r0 + n].isfinite().all(), f"row {r0}: {int(bad.sum())} of {bad.numel()} off, worst " \
            f"{((out[r0:r0 + n].double() - o).abs() / tol).max():.2f} of the tolerance"
        none = e == -math.inf
        assert torch.equal(lse[r0:r0 + n] == -math.inf, none)
        assert ((lse[r0:r0 + n].double() - e).masked_fill(none, 0.0).abs() <= tol_lse).all()


CASES = [
    # lengths, new tokens, heads, kv heads, head size, page, type, mask words (0: chain)
    ([0], [1], 1, 1, 64, 8, "bf16", 0),
    ([63], [1], 4, 1, 128, 16, "bf16", 0),
    ([63], [2], 4, 2, 128, 16, "fp16", 0),
    ([64, 65, 1, 0], [1, 1, 1, 1], 8, 8, 128, 64, "bf16", 0),
    ([700], [5], 16, 4, 128, 16, "bf16", 0),
    ([128, 0, 300, 5], [3, 7, 0, 64], 6, 2, 80, 32, "fp16", 2),
    ([1, 2, 3, 130, 257], [4, 40, 33, 17, 2], 5, 1, 256, 16, "bf16", 2),
    ([20000], [1], 8, 1, 128, 128, "bf16", 0),
    ([9000, 3], [16, 48], 20, 5, 256, 16, "fp16", 2),
    ([500, 77], [48, 20], 24, 3, 64, 256, "bf16", 0),         # more rows than a tile: 8 x 48
    ([500, 77], [48, 20], 24, 3, 64, 256, "bf16", 2),
    ([100], [300], 4, 4, 128, 64, "bf16", 0),                 # a stretch of prompt
    ([100], [300], 4, 4, 128, 64, "fp16", 4),                 # drafts behind the mask's last word are not seen
    ([2500] * 3, [64] * 3, 16, 2, 128, 32, "bf16", 2),
    ([3, 200], [5, 6], 3, 1, 8, 8, "bf16", 1),
    ([90, 1000], [2, 9], 7, 1, 40, 8, "fp16", 1),
    ([60, 40], [9, 70], 2, 2, 192, 16, "bf16", 3),
    ([250], [5], 128, 1, 64, 64, "bf16", 1),                  # 128 query heads to a key head
    ([250], [3], 67, 1, 128, 64, "fp16", 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"L{c[0][0]}x{len(c[0])}n{c[1][0]}N{c[2]}K{c[3]}H{c[4]}P{c[5]}{c[6]}w{c[7]}")
def test_against_the_definition(pkg, cuda, case):
    lengths, new, heads, kv, size, page, dtype, words = case
    s = make(cuda, lengths, new, heads, kv, size, page, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype], seed=len(lengths) + size)
    if words:
        s["mask"] = random_mask(s, words)
    check(s, *call(pkg, s))


@pytest.mark.parametrize("size,page", [(64, 16), (128, 8), (256, 32)])
def test_many_requests_of_all_short_lengths(pkg, cuda, size, page):
    lengths, new = list(range(0, 330)), [1 + i % 5 for i in range(330)]
    new[7] = new[200] = 0
    s = make(cuda, lengths, new, 4, 2, size, page, torch.bfloat16, seed=size)
    s["mask"] = random_mask(s, 1, share=0.7)
    check(s, *call(pkg, s))


@pytest.mark.parametrize("layout", ["heads", "slice"])
def test_strides(pkg, cuda, layout):
    s = make(cuda, [300, 17], [4, 9], 6, 2, 72, 16, torch.float16, layout=layout)
    wide = torch.randn(13, 3, 10, 88, device=cuda).half()
    s["q"] = wide[:, 1, 2:8, 8:80]
    out = torch.zeros(13, 6, 104, dtype=torch.float16, device=cuda)[:, :, 24:96]
    got, lse = call(pkg, s, out=out)
    assert got is out
    check(s, out, lse)


def test_rows_that_see_nothing(pkg, cuda):
    s = make(cuda, [0, 0, 70], [3, 1, 2], 4, 2, 128, 16, torch.bfloat16)
    s["mask"] = torch.tensor([[0b010], [0], [0b111], [0], [-2 ** 31], [0b11]], dtype=torch.int32, device=cuda)
    out, lse = call(pkg, s)
    assert (out[[1, 3]] == 0).all() and (lse[[1, 3]] == -math.inf).all()
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,words", [(0, 1), (61, 1), (200, 1), (61, 0), (4000, 1)])
def test_values_that_are_no_numbers_reach_only_rows_that_see_them(pkg, cuda, dtype, L, words):
    n, page = 9, 16
    s = make(cuda, [5, L, 30], [1, n, 2], 4, 2, 128, page, dtype, seed=L)
    if words:
        s["mask"] = random_mask(s, 1)
    want, want_lse = call(pkg, s)
    hurt = {2: (0, 3, math.inf), 4: (1, 127, math.nan), 8: (0, 64, -math.inf)}
    for i, (head, column, value) in hurt.items():
        t = L + i
        s["v"][s["table"][1, t // page], t % page, head, column] = value
        s["k"][s["table"][1, t // page], t % page, head, column] = math.nan if i == 4 else 1.0
    # (of the keys, one that nobody may see: its own scores are NaN)
    out, lse = call(pkg, s)
    sees = seen(s, 1, 1, n, L)[:, L:]
    for j in range(n):
        for i, (head, column, value) in hurt.items():
            for h in range(4):
                x = out[1 + j, h, column].item()
                if h // 2 != head:
                    continue
                if not sees[j, i]:
                    assert math.isfinite(x) or (i != 4 and head == 0 and any(sees[j, k] for k in (2, 8))), (j, i, h)
                elif i == 4:
                    assert math.isnan(x)
                elif not math.isnan(x):
                    assert x == value or any(sees[j, k] and hurt[k][1] == column for k in hurt if k != i)
    # rows of other requests, and rows that see none of the three, are as they were
    plain = [0] + [1 + j for j in range(n) if not any(sees[j, k] for k in hurt)] + [n + 1, n + 2]
    assert torch.equal(out[plain], want[plain]) and torch.equal(lse[plain], want_lse[plain])


def test_rows_of_nobody_are_left_alone(pkg, cuda):
    s = make(cuda, [40, 100, 7], [3, 4, 5], 4, 2, 64, 8, torch.bfloat16)
    want, want_lse = call(pkg, s)
    # room for more rows, and a request that was granted fewer than it has rows
    s["q"] = torch.cat((s["q"], torch.full((6, 4, 64), math.nan, device=cuda).bfloat16()))
    s["granted"] = torch.tensor([3, 0, 5], dtype=torch.int32, device=cuda)
    out, lse = torch.full_like(s["q"], 3.0), torch.full(s["q"].shape[:2], 5.0, device=cuda)
    call(pkg, s, out=out, lse=lse)
    mine = [0, 1, 2, 7, 8, 9, 10, 11]
    rest = [3, 4, 5, 6, *range(12, 18)]
    assert (out[rest] == 3.0).all() and (lse[rest] == 5.0).all()
    check(s, out, lse)
    assert torch.allclose(out[mine].float(), want[mine].float(), atol=0.05)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 30.0])
def test_scales(pkg, cuda, scale):
    s = make(cuda, [200, 50], [3, 6], 4, 2, 128, 16, torch.float16)
    s["scale"] = scale
    check(s, *call(pkg, s))


def test_large_scores_that_rise_from_unit_to_unit(pkg, cuda):
    """The running maximum moves all the time: O is rescaled in every unit."""
    s = make(cuda, [1000], [4], 4, 1, 128, 16, torch.bfloat16)
    t = torch.arange(1004, device=cuda)
    s["q"] = torch.ones_like(s["q"])
    s["k"][s["table"][0, t // 16].long(), t % 16] = (t[:, None, None] * 0.01).bfloat16().expand(-1, 1, 128)
    check(s, *call(pkg, s))


def test_numbers_outside_their_ranges(pkg, cuda):
    """Page numbers outside the cache read as zeros; lengths, counts and row starts are cut to what the buffers hold."""
    s = make(cuda, [100, 50], [2, 3], 4, 2, 64, 16, torch.bfloat16)
    good_out, good_lse = call(pkg, s)
    s["table"][0, 1], s["table"][0, 3] = -5, 2 ** 30
    ids = s["table"][0].clone()
    out, lse = call(pkg, s)
    assert torch.equal(out[2:], good_out[2:])
    zeros = s["k"].new_zeros(1, *s["k"].shape[1:])
    t = dict(s, k=torch.cat((s["k"], zeros)), v=torch.cat((s["v"], zeros)), table=s["table"].clone())
    t["table"][0] = torch.where((ids < 0) | (ids >= len(s["k"])), len(s["k"]), ids)
    check(t, out, lse)
    # more tokens than the table has places for, rows outside q, negative numbers
    for lengths, start, granted in (([2 ** 31 - 1, -4], [0, 2, 5], [2, 3]), ([100, 50], [-3, 4, 5], [2, 9]), ([100, 50], [2 ** 31 - 1, 0, 5], [2 ** 31 - 1, -1])):
        s["lengths"], s["row_start"], s["granted"] = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in (lengths, start, granted))
        out = torch.zeros_like(s["q"])
        call(pkg, s, out=out)
    torch.cuda.synchronize()


def test_a_cache_of_more_than_2_to_the_31_elements(pkg, cuda):
    pages = 2 ** 31 // (256 * 2 * 128) + 40
    big = torch.zeros(pages, 256, 2, 128, dtype=torch.bfloat16, device=cuda)
    s = make(cuda, [700, 300], [4, 2], 4, 2, 128, 256, torch.bfloat16, stale=0.0)
    small = s["table"].long()
    far = pages - 1 - small
    for name in ("k", "v"):
        t = s[name]
        if name == "k":
            big[far.clamp(max=pages - 1)] = t[small.clamp(min=0)]
            s["k"] = big
        else:
            near = torch.zeros_like(big[:1]).expand(pages, -1, -1, -1)
            s["v"] = big       # (keys and values are the same tensor)
    s["table"] = torch.where(small >= 0, far, -7).int()
    out, lse = call(pkg, s)
    check(s, out, lse)


def test_repeated_replayed_and_on_another_stream(pkg, cuda):
    s = make(cuda, [3000, 40, 900, 0], [8, 1, 5, 3], 8, 2, 128, 16, torch.bfloat16)
    want, want_lse = call(pkg, s)
    for _ in range(3):
        out, lse = call(pkg, s)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = call(pkg, s, stream=side)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # a graph follows the numbers on the GPU: other lengths, the same launches
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call(pkg, s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    s["lengths"].copy_(torch.tensor([100, 39, 17, 0], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(s, out, lse)


def test_workspace_of_a_call_may_serve_the_next(pkg, cuda):
    """What a call leaves in the scratch says nothing to the next one, of other lengths."""
    a = make(cuda, [20000], [2], 8, 2, 128, 16, torch.bfloat16)
    b = make(cuda, [10, 3000], [1, 1], 8, 2, 128, 16, torch.bfloat16)
    ws = torch.full((pkg.fmha_paged_workspace_bytes(a["q"], a["k"]),), 0xff, dtype=torch.uint8, device=cuda)
    for s in (a, b, a, b):
        check(s, *call(pkg, s, workspace=ws))


def test_refusals(pkg, cuda):
    s = make(cuda, [30], [2], 4, 2, 64, 16, torch.bfloat16)
    n0 = pkg.launch_count()

    def refused(status, **change):
        t = dict(s, **{k: v for k, v in change.items() if k in s})
        with pytest.raises(pkg.IxkError) as e:
            call(pkg, t, **{k: v for k, v in change.items() if k not in s})
        assert e.value.status == status, str(e.value)

    bad, un = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED
    refused(bad, q=s["q"].half())
    refused(un, q=s["q"].float(), k=s["k"].float(), v=s["v"].float())
    refused(bad, q=s["q"][:, :3])
    refused(bad, q=torch.zeros(2, 4, 72, device=cuda).bfloat16())
    refused(bad, table=s["table"].long())
    refused(bad, lengths=s["lengths"].long())
    refused(bad, row_start=s["row_start"][:1])
    refused(bad, granted=s["granted"][:0])
    refused(bad, mask=torch.zeros(3, 1, dtype=torch.int32, device=cuda))
    refused(bad, mask=torch.zeros(2, 0, dtype=torch.int32, device=cuda))
    refused(bad, scale=math.nan)
    refused(bad, out=torch.zeros(2, 4, 64, device=cuda))
    refused(bad, lse=torch.zeros(2, 4, device=cuda).half())
    refused(un, k=s["k"][:, :12], v=s["v"][:, :12])                                    # page size 12
    refused(un, k=s["k"][:, :4], v=s["v"][:, :4])
    refused(un, out=torch.zeros(2, 4, 68, device=cuda).bfloat16()[:, :, :64])
    refused(bad, v=s["v"][:-1])
    refused(pkg.IXK_WORKSPACE_TOO_SMALL, workspace=torch.empty(64, dtype=torch.uint8, device=cuda))
    refused(pkg.IXK_NO_DEVICE, lengths=s["lengths"].cpu())
    assert pkg.launch_count() == n0
    # nothing to do
    none = dict(s, q=s["q"][:0])
    assert call(pkg, none)[0].shape == (0, 4, 64)


def test_native_and_python_calls_agree(pkg, cuda, monkeypatch):
    s = make(cuda, [300, 20], [3, 4], 4, 2, 128, 16, torch.bfloat16)
    s["mask"] = random_mask(s, 1)
    want, want_lse = call(pkg, s)
    monkeypatch.setattr(pkg, "_NATIVE", None)
    out, lse = call(pkg, s)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("size,lengths", [(128, [300, 20000, 7] + [40] * 50), (256, [9000] + [200, 3] * 40), (64, [30000, 30000] + [5] * 60), (128, [8000])])
def test_one_long_request_among_short_ones(pkg, cuda, size, lengths):
    """Tiles in parts of many workers beside tiles that one worker does whole."""
    s = make(cuda, lengths, [3] * len(lengths), 8, 2, size, 16, torch.bfloat16, seed=4)
    check(s, *call(pkg, s))


@pytest.mark.parametrize("lengths", [[70, 2000, 9, 0], [40] * 90])
def test_the_result_in_the_place_of_q(pkg, cuda, lengths):
    s = make(cuda, lengths, [5] * len(lengths), 12, 4, 128, 16, torch.bfloat16, seed=2)
    out, lse = call(pkg, s)
    q = s["q"].clone()
    again, lse2 = call(pkg, dict(s, q=q), out=q)
    assert again is q and torch.equal(q, out) and torch.equal(lse, lse2)
    with pytest.raises(pkg.IxkError):
        wide = torch.zeros(q.shape[0], 24, 128, dtype=q.dtype, device=cuda)
        call(pkg, dict(s, q=wide[:, :12]), out=wide[:, ::2])


@pytest.mark.parametrize("layout", ["tokens", "heads"])
@pytest.mark.parametrize("size,page", [(128, 8), (256, 8), (256, 16), (256, 32), (192, 8)])
def test_small_pages(pkg, cuda, size, page, layout):
    """Copies of 8 keys over all of a head's columns, or (heads that do not follow one another) of a page's keys of 64 columns; ends of
    requests at every place of a group of 8."""
    lengths = [0, 3, 61, 64, 100, 127, 700] + list(range(40, 56))
    s = make(cuda, lengths, [1 + i % 9 for i in range(len(lengths))], 6, 2, size, page, torch.float16, seed=3, layout=layout)
    s["mask"] = random_mask(s, 1)
    check(s, *call(pkg, s))


@pytest.mark.parametrize("size,page", [(128, 8), (256, 8), (256, 16)])
@pytest.mark.parametrize("L", [0, 5, 61, 203])
def test_values_that_are_no_numbers_in_small_pages(pkg, cuda, size, page, L):
    """Drafts whose values are no numbers reach the rows that see them, and only those."""
    s = make(cuda, [L, 30], [13, 2], 4, 2, size, page, torch.bfloat16, seed=6)
    s["mask"] = random_mask(s, 1)
    bad = (2, 7, 8, 12)
    for d in bad:
        p = L + d
        s["v"][s["table"][0, p // page].long(), p % page, :, d * 3] = float("inf") if d % 2 else float("nan")
    out, _ = call(pkg, s)
    clean = dict(s, v=torch.where(s["v"].isfinite(), s["v"], torch.zeros_like(s["v"])))
    want, _ = call(pkg, clean)
    for j in range(13):
        for d in bad:
            sees = bool(s["mask"][j, 0] >> d & 1)
            assert bool(out[j, :, d * 3].isfinite().all()) != sees, (j, d)
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[:13, :, [d * 3 for d in bad]] = True
    assert torch.equal(out[~odd], want[~odd])
