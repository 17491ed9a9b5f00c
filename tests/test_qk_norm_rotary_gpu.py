"""GPU: norm and rotation of query and key heads in one pass, and the gradient, against the formulas in 64 bits.

Tolerance.  A result is rounded once, by u = eps / 2 of its type (times its size).  Before that fp32: a head's sum of squares
is H terms, at most (H + 8) 2^-24 off, its root half that; the products and their sum are a few 2^-24 of r (|x w cos| + |x' w' sin|).
Backward: mean(h x) likewise is H terms, and enters with |x| r^3 mean |h x|.  The gains' gradients are sums of n = tokens * heads
fp32 terms: at most n 2^-24 of the sum of their sizes, and their own errors as above."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def tables(places, rotary, cuda, base=10000.0):
    angle = torch.arange(places, dtype=torch.float64, device=cuda)[:, None] * base ** (-torch.arange(rotary // 2, dtype=torch.float64, device=cuda) * 2 / rotary)
    return angle.cos().float(), angle.sin().float()


def turn(x, cos, sin, rotary, half, sign=1.0):
    """x [T, N, H] in 64 bits; cos, sin [T, rotary / 2]."""
    c, s = cos.double()[:, None], sin.double()[:, None] * sign
    if half:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        return torch.cat((a * c - b * s, b * c + a * s, x[..., rotary:]), -1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), x[..., rotary:]), -1)


def sizes(x, cos, sin, rotary, half):
    """The sum of the sizes of what turn() adds up."""
    c, s = cos.abs(), sin.abs()
    x = x.abs()
    if half:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        return torch.cat((a * c[:, None] + b * s[:, None], b * c[:, None] + a * s[:, None], x[..., rotary:]), -1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    return torch.cat((torch.stack((a * c[:, None] + b * s[:, None], b * c[:, None] + a * s[:, None]), -1).flatten(-2), x[..., rotary:]), -1)


def forward(x, w, eps, cos, sin, rotary, half):
    x = x.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r * w
    return turn(u, cos, sin, rotary, half), sizes(u, cos, sin, rotary, half)


def backward(g, x, w, eps, cos, sin, rotary, half):
    """(dx, the size of what it is made of, dgain, the sum of its terms' sizes)"""
    x, H = x.double(), x.shape[-1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    gt, gs = turn(g.double(), cos, sin, rotary, half, -1.0), sizes(g.double(), cos, sin, rotary, half)
    h = gt * w
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    size = r * (gs * w.abs() + x.abs() * r * r * (gs * w.abs() * x.abs()).mean(-1, keepdim=True))
    return dx, size, (gt * x * r).sum((0, 1)), (gs * x.abs() * r).sum((0, 1))


def inputs(cuda, T, N, NK, H, dtype, param, rotary, places=4096, seed=0, positions=torch.int32):
    g = torch.Generator(device=cuda).manual_seed(seed)
    qkv = (torch.randn(T, N + 2 * NK, H, generator=g, device=cuda) * torch.rand(T, N + 2 * NK, 1, generator=g, device=cuda).mul(3).exp()).to(dtype)
    s = {"q": qkv[:, :N], "k": qkv[:, N:N + NK], "v": qkv[:, N + NK:]}
    s["q_gain"], s["k_gain"] = (torch.randn(H, generator=g, device=cuda).mul(0.3).add(1).to(param) for _ in range(2))
    s["cos"], s["sin"] = tables(places, rotary, cuda)
    s["positions"] = None if positions is None else torch.randint(0, places, (T,), generator=g, device=cuda).to(positions)
    s["grad_q"], s["grad_k"] = (torch.randn(T, n, H, generator=g, device=cuda).to(dtype) for n in (N, NK))
    return s


def angles(s, T):
    p = torch.arange(T, device=s["cos"].device) % len(s["cos"]) if s["positions"] is None else s["positions"].long()
    return s["cos"][p], s["sin"][p]


def close(got, want, size, H, extra=0):
    u = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * u * 2      # (a step among the subnormal numbers)
    tol = u * want.abs() * (1 + 2.0 ** -10) + (2 * H + 64 + extra) * E * size + tiny
    bad = (got.double() - want).abs() > tol
    assert got.isfinite().all() and not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got.double() - want).abs() / tol).max():.2f} of the tolerance"


BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
CASES = [
    # tokens, heads, kv heads, head size, type, gains' type, rotary, half split, positions' type, gain_offset
    (1, 1, 1, 8, BF, BF, 8, False, torch.int32, 0.0),
    (1, 4, 1, 64, BF, BF, 64, True, torch.int64, 1.0),
    (5, 7, 3, 80, HF, HF, 32, False, torch.int32, 0.0),
    (3, 16, 4, 128, BF, F32, 128, True, None, 0.0),
    (65, 9, 2, 96, F32, F32, 96, True, torch.int64, 1.0),
    (130, 5, 5, 256, HF, F32, 64, True, torch.int32, 0.0),
    (257, 16, 16, 256, BF, F32, 256, False, torch.int32, 0.0),
    (1000, 33, 1, 40, BF, BF, 16, True, torch.int32, 0.0),
    (3000, 8, 2, 128, HF, HF, 128, True, torch.int32, 1.0),
    (411, 2, 1, 248, F32, F32, 248, False, None, 0.0),
    (200, 3, 3, 72, BF, BF, 48, True, torch.int64, 0.0),
]
IDS = [f"T{c[0]}N{c[1]}K{c[2]}H{c[3]}{str(c[4])[6:]}r{c[6]}{'h' if c[7] else 'i'}" for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_and_backward(pkg, cuda, case):
    T, N, NK, H, dtype, param, rotary, half, positions, offset = case
    s = inputs(cuda, T, N, NK, H, dtype, param, rotary, seed=T, positions=positions)
    common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], gain_offset=offset, eps=1e-5, cos=s["cos"], sin=s["sin"], positions=s["positions"],
                  half_split=half)
    q, k = pkg.qk_norm_rotary_forward(s["q"], s["k"], **common)
    grads = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common)
    cos, sin = angles(s, T)
    for i, (name, y) in enumerate((("q", q), ("k", k))):
        w = s[name + "_gain"].double() + offset
        close(y, *forward(s[name], w, 1e-5, cos, sin, rotary, half), H)
        dx, size, dgain, terms = backward(s["grad_" + name], s[name], w, 1e-5, cos, sin, rotary, half)
        close(grads[i], dx, size, H, extra=2 * H)
        close(grads[2 + i], dgain, terms, H, extra=T * s[name].shape[1])


@pytest.mark.parametrize("half", [True, False])
def test_gradients_against_differences(pkg, cuda, half):
    """Central differences of the formula in 64 bits along random directions, step 1e-5: their own error is below 1e-8."""
    T, N, NK, H, rotary = 17, 3, 2, 64, 32
    s = inputs(cuda, T, N, NK, H, F32, F32, rotary, seed=5)
    cos, sin = angles(s, T)
    dq, dk, dqg, dkg = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], q_gain=s["q_gain"], k_gain=s["k_gain"], eps=1e-5,
                                                   cos=s["cos"], sin=s["sin"], positions=s["positions"], half_split=half)
    for x, w, g, dx, dw in ((s["q"], s["q_gain"], s["grad_q"], dq, dqg), (s["k"], s["k_gain"], s["grad_k"], dk, dkg)):
        def f(x, w):
            return (forward(x, w, 1e-5, cos, sin, rotary, half)[0] * g.double()).sum()

        for seed in range(3):
            r = torch.Generator(device=cuda).manual_seed(seed)
            d, e, step = torch.randn(x.shape, generator=r, device=cuda).double(), torch.randn(H, generator=r, device=cuda).double(), 1e-5
            x64, w64 = x.double(), w.double()
            along_x = (f(x64 + step * d, w64) - f(x64 - step * d, w64)) / (2 * step)
            along_w = (f(x64, w64 + step * e) - f(x64, w64 - step * e)) / (2 * step)
            # fp32 gradients, (4 H + 64) 2^-24 off at most in each of x.numel() terms (of a size below 2 |dx|), see the head of the file
            size = backward(g, x, w64, 1e-5, cos, sin, rotary, half)
            assert (along_x - (dx.double() * d).sum()).abs() <= ((4 * H + 64) * E * size[1] * d.abs()).sum() + 1e-6 * along_x.abs() + 1e-6
            assert (along_w - (dw.double() * e).sum()).abs() <= ((4 * H + 64 + T * N) * E * size[3] * e.abs()).sum() + 1e-6 * along_w.abs() + 1e-6


@pytest.mark.parametrize("layout", ["tokens", "heads"])
@pytest.mark.parametrize("T,N,NK,H,page,dtype", [(1, 4, 1, 128, 16, BF), (70, 6, 2, 80, 8, HF), (900, 16, 4, 128, 64, BF), (33, 8, 8, 256, 5, BF)])
def test_into_the_pages(pkg, cuda, T, N, NK, H, page, dtype, layout):
    s = inputs(cuda, T, N, NK, H, dtype, dtype, H // 32 * 32, seed=T)
    pages = T // page + 4
    make = lambda: (torch.full((pages, page, NK, H), 7.0, device=cuda).to(dtype) if layout == "tokens" else
                    torch.full((pages, NK, page, H), 7.0, device=cuda).to(dtype).transpose(1, 2))
    k_pages, v_pages = make(), make()
    slots = torch.randperm(pages * page, device=cuda)[:T].int()
    skip = [i for i in range(T) if i % 7 == 3]
    slots[skip] = torch.tensor([(-1, pages * page, 2 ** 31 - 1)[i % 3] for i in skip], dtype=torch.int32, device=cuda)
    common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], eps=1e-6, cos=s["cos"], sin=s["sin"], positions=s["positions"])
    dense_q, dense_k = pkg.qk_norm_rotary_forward(s["q"], s["k"], **common)
    q, none = pkg.qk_norm_rotary_forward(s["q"], s["k"], v=s["v"], slots=slots, k_pages=k_pages, v_pages=v_pages, **common)
    assert none is None and torch.equal(q, dense_q)
    want_k, want_v = make(), make()
    for t in range(T):
        if t not in skip:
            at = (slots[t].item() // page, slots[t].item() % page)
            want_k[at], want_v[at] = dense_k[t], s["v"][t]
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


def test_tokens_outside_the_tables_are_left_out(pkg, cuda):
    T, N, NK, H = 50, 5, 2, 64
    for dtype in (torch.int32, torch.int64):
        s = inputs(cuda, T, N, NK, H, BF, F32, H, places=100, positions=dtype)
        out = [t for t in range(T) if t % 5 == 2]
        s["positions"][out] = torch.tensor([(-1, 100, 2 ** 31 - 1, -2 ** 31)[t % 4] for t in out], device=cuda).to(dtype)
        s["q"][out[0]], s["grad_k"][out[1]] = float("nan"), float("inf")
        q_out, k_out = torch.full_like(s["grad_q"], 3.0), torch.full_like(s["grad_k"], 3.0)
        # (eps 0: a row that is left out has no root)
        common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], eps=0.0, cos=s["cos"], sin=s["sin"], positions=s["positions"])
        pkg.qk_norm_rotary_forward(s["q"], s["k"], q_out=q_out, k_out=k_out, **common)
        inside = [t for t in range(T) if t not in out]
        assert (q_out[out] == 3.0).all() and (k_out[out] == 3.0).all()
        few = dict(common, positions=s["positions"][inside])
        q, k = pkg.qk_norm_rotary_forward(s["q"][inside], s["k"][inside], **few)
        assert torch.equal(q_out[inside], q) and torch.equal(k_out[inside], k)
        got = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common)
        want = pkg.qk_norm_rotary_backward(s["grad_q"][inside], s["grad_k"][inside], s["q"][inside], s["k"][inside], **few)
        for g, w in zip(got[:2], want[:2]):
            assert (g[out] == 0).all() and torch.equal(g[inside], w)
        for g, w, n in zip(got[2:], want[2:], (N, NK)):
            assert torch.allclose(g, w, rtol=0, atol=float(T * n * E * (w.abs().max() + 100)))


def test_in_place_without_gains_and_views(pkg, cuda):
    s = inputs(cuda, 300, 6, 2, 128, HF, HF, 128, seed=9)
    common = dict(cos=s["cos"], sin=s["sin"], positions=s["positions"], half_split=False, eps=1e-6)
    q, k = pkg.qk_norm_rotary_forward(s["q"], s["k"], **common)
    cos, sin = angles(s, 300)
    one = torch.ones(128, dtype=torch.float64, device=cuda)
    close(q, *forward(s["q"], one, 1e-6, cos, sin, 128, False), 128)
    gq, gk = s["grad_q"].clone(), s["grad_k"].clone()
    want = pkg.qk_norm_rotary_backward(gq, gk, s["q"], s["k"], **common)
    assert want[2] is None and want[3] is None
    got = pkg.qk_norm_rotary_backward(gq, gk, s["q"], s["k"], dq=gq, dk=gk, **common)
    assert got[0] is gq and torch.equal(gq, want[0]) and torch.equal(gk, want[1])
    # into slices of one tensor, as the gradient of the fused projection is
    fused = torch.zeros(300, 10, 128, dtype=HF, device=cuda)
    pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], dq=fused[:, :6], dk=fused[:, 6:8], **common)
    assert torch.equal(fused[:, :6], want[0]) and torch.equal(fused[:, 6:8], want[1]) and (fused[:, 8:] == 0).all()
    got = pkg.qk_norm_rotary_forward(s["q"], s["k"], q_out=s["q"], k_out=s["k"], **common)
    assert got[0] is s["q"] and torch.equal(s["q"], q) and torch.equal(s["k"], k)
    # one gain, not the other; a head that all tokens share
    gain = torch.full((128,), 2.0, device=cuda).half()
    shared = s["grad_q"][:1, :1].expand(300, 3, 128)
    a, _ = pkg.qk_norm_rotary_forward(shared, s["k"], q_gain=gain, **common)
    b, _ = pkg.qk_norm_rotary_forward(shared.contiguous(), s["k"], q_gain=gain, **common)
    assert torch.equal(a, b)
    r = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], k_gain=gain, **common)
    assert r[2] is None and r[3].shape == (128,)


def test_empty_calls_and_long_ones(pkg, cuda):
    s = inputs(cuda, 0, 4, 2, 64, BF, F32, 64)
    common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"], positions=s["positions"])
    q, k = pkg.qk_norm_rotary_forward(s["q"], s["k"], **common)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    r = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common)
    assert (r[2] == 0).all() and (r[3] == 0).all()
    # more than 2^31 elements between the first and the last token
    wide = torch.empty(33000, 2 ** 16 + 8, dtype=BF, device=cuda)
    x = wide[:, 8:8 + 128].unflatten(1, (2, 64))
    x.copy_(torch.randn(33000, 2, 64, device=cuda))
    cos, sin = tables(33000, 64, cuda)
    a, _ = pkg.qk_norm_rotary_forward(x, x[:, :1], cos=cos, sin=sin)
    b, _ = pkg.qk_norm_rotary_forward(x.contiguous(), x[:, :1].contiguous(), cos=cos, sin=sin)
    assert torch.equal(a, b)


def test_same_bits_again_in_a_graph_on_another_stream_and_through_python(pkg, cuda, monkeypatch):
    s = inputs(cuda, 700, 9, 3, 128, BF, BF, 64, seed=2)
    common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"], positions=s["positions"])

    def both(**more):
        return (*pkg.qk_norm_rotary_forward(s["q"], s["k"], **common, **more),
                *pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common, **more))

    want = both()
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))
    assert same(both())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(stream=side)
    side.synchronize()
    assert same(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    graph.replay()
    torch.cuda.synchronize()
    assert same(got)
    monkeypatch.setattr(pkg, "_NATIVE", None)
    assert same(both())


def test_refusals(pkg, cuda):
    s = inputs(cuda, 10, 4, 2, 64, BF, F32, 64)
    n0 = pkg.launch_count()
    base = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"], positions=s["positions"])

    def refused(status, q=s["q"], k=s["k"], **change):
        with pytest.raises(pkg.IxkError) as e:
            pkg.qk_norm_rotary_forward(q, k, **dict(base, **change))
        assert e.value.status == status, str(e.value)

    bad, un = pkg.IXK_INVALID_ARGUMENT, pkg.IXK_UNIMPLEMENTED
    refused(bad, k=s["k"][:9])
    refused(bad, k=s["k"].half())
    refused(un, q=s["q"].double(), k=s["k"].double())
    refused(bad, q_gain=s["q_gain"][:32])
    refused(bad, k_gain=s["k_gain"].bfloat16())
    refused(bad, cos=s["cos"].half())
    refused(bad, cos=s["cos"][:, :30].contiguous(), sin=s["sin"][:, :30].contiguous())       # 60 elements
    refused(bad, cos=torch.zeros(9, 40, device=cuda), sin=torch.zeros(9, 40, device=cuda))      # more than the head
    refused(bad, positions=s["positions"][:9])
    refused(bad, positions=s["positions"].float())
    refused(bad, eps=-1.0)
    refused(bad, q_out=torch.zeros(10, 4, 64, device=cuda))
    refused(bad, q_out=torch.zeros(10, 1, 64, device=cuda).bfloat16().expand(10, 4, 64))
    refused(bad, q=torch.zeros(10, 4, 68, device=cuda).bfloat16()[..., :64])
    refused(bad, slots=torch.zeros(10, dtype=torch.int32, device=cuda))
    pool = torch.zeros(5, 8, 2, 64, device=cuda).bfloat16()
    cache = dict(v=s["v"], slots=torch.zeros(10, dtype=torch.int32, device=cuda), k_pages=pool, v_pages=pool)
    refused(bad, **dict(cache, slots=cache["slots"].long()))
    refused(bad, **dict(cache, k_pages=pool[:, :, :1], v_pages=pool[:, :, :1]))
    refused(bad, **dict(cache, k_out=s["grad_k"]))
    refused(bad, **dict(cache, v=s["v"][:, :1]))
    refused(pkg.IXK_NO_DEVICE, positions=s["positions"].cpu())
    with pytest.raises(pkg.IxkError) as e:
        pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], workspace=torch.empty(16, dtype=torch.uint8, device=cuda), **base)
    assert e.value.status == pkg.IXK_WORKSPACE_TOO_SMALL
    assert pkg.launch_count() == n0


MORE = [(40, 3, 2, H, dtype, F32, rotary, half, torch.int32, 0.5)
        for dtype in (HF, F32) for H, rotary, half in ((64, 24, False), (64, 40, False), (80, 72, False), (128, 56, False), (128, 72, False), (136, 136, False),
                                                       (160, 80, True), (200, 16, True), (256, 136, False), (256, 240, True), (16, 8, False), (24, 16, True))]
# just below and above whole turns of a token a warp (148 multiprocessors x 4 blocks x 4 warps), and last turns that several warps share
MORE += [(T, 2, 1, 64, BF, BF, 64, True, torch.int64, 0.0) for T in (1183, 1184, 1185, 2367, 2368, 2369, 2400, 4736, 4737, 7200)]
MORE += [(T, 9, 5, 128, HF, HF, 128, False, None, 0.0) for T in (2, 300, 2369, 2960, 5000)]


@pytest.mark.parametrize("case", MORE, ids=[f"T{c[0]}N{c[1]}K{c[2]}H{c[3]}{str(c[4])[6:]}r{c[6]}{'h' if c[7] else 'i'}" for c in MORE])
def test_parts_of_heads_and_turns(pkg, cuda, case):
    test_forward_and_backward(pkg, cuda, case)


@pytest.mark.parametrize("half", [True, False])
def test_fp32_between_sectors(pkg, cuda, half):
    """Tensors that begin in the middle of a 32-byte sector: the same bits."""
    s = inputs(cuda, 70, 3, 1, 96, F32, F32, 96, seed=8)
    common = dict(q_gain=s["q_gain"], k_gain=s["k_gain"], cos=s["cos"], sin=s["sin"], positions=s["positions"], half_split=half)
    off = lambda t: torch.full((t.numel() + 8,), 7.0, device=cuda)[4:-4].view(t.shape)  # noqa: E731
    moved = {n: off(s[n]).copy_(s[n]) for n in ("q", "k", "grad_q", "grad_k")}
    assert moved["q"].data_ptr() % 32 == 16
    want = pkg.qk_norm_rotary_forward(s["q"], s["k"], **common)
    out = [off(t) for t in want]
    pkg.qk_norm_rotary_forward(moved["q"], moved["k"], q_out=out[0], k_out=out[1], **common)
    grads = pkg.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common)
    d = [off(t) for t in grads[:2]]
    again = pkg.qk_norm_rotary_backward(moved["grad_q"], moved["grad_k"], moved["q"], moved["k"], dq=d[0], dk=d[1], **common)
    for a, b in zip((*want, *grads), (*out, *again)):
        assert torch.equal(a, b)
    for t in out + d:
        whole = torch.as_strided(t, (t.numel() + 8,), (1,), t.storage_offset() - 4)
        assert (whole[:4] == 7.0).all() and (whole[-4:] == 7.0).all()
