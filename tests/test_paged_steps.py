"""Steps of a decoder over a paged cache (layers.paged_step, layers.paged_accept_): prompts, single tokens, drafted chains and trees of
several requests together, some accepted, some ended, some refused for want of pages, against the same text recomputed whole."""
import importlib
import math
import os
import random
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

LAYERS, HIDDEN, HEADS, KV, HD, FFN, ROTARY, PLACES = 2, 128, 6, 2, 64, 256, 64, 512


class PlainOps:
    """Only the products; everything else is the layers' plain form."""

    def gemm(self, x, w, *, bias=None, c=None, beta=0.0, epilogue="DEFAULT", out=None):
        y = x.float() @ w.float() + (0 if c is None else beta * c.float())
        return (torch.nn.functional.gelu(y, approximate="tanh") if epilogue == "GELU" else y).to(x.dtype)


def weights(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(dtype)  # noqa: E731
    return [dict(wqkv=r(HIDDEN, (HEADS + 2 * KV) * HD), wo=r(HEADS * HD, HIDDEN), wgate=r(HIDDEN, FFN), wup=r(HIDDEN, FFN), wdown=r(FFN, HIDDEN),
                 norm_attn=r(HIDDEN), norm_mlp=r(HIDDEN), norm_q=r(HD), norm_k=r(HD)) for _ in range(LAYERS)]


def whole_text(full, x, places, seen):
    """The decoder in 64 bits over a text x [tokens, HIDDEN] at places [tokens], seen [tokens, tokens]."""
    x = x.double()
    norm = lambda t, w: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * (1 + w.double())  # noqa: E731
    angle = places.double()[:, None] * 10000.0 ** (-torch.arange(0, ROTARY, 2).double() / ROTARY)
    c, s = angle.cos()[:, None], angle.sin()[:, None]

    def turn(t):
        a, b = t[..., :ROTARY // 2], t[..., ROTARY // 2:ROTARY]
        return torch.cat((a * c - b * s, b * c + a * s, t[..., ROTARY:]), -1)

    for w in full:
        d = {k: v.double() for k, v in w.items()}
        qkv = (norm(x, d["norm_attn"]) @ d["wqkv"]).view(len(x), HEADS + 2 * KV, HD)
        q, k = turn(norm(qkv[:, :HEADS], d["norm_q"])), turn(norm(qkv[:, HEADS:HEADS + KV], d["norm_k"]))
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, qkv[:, HEADS + KV:]))
        z = torch.where(seen, torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(HD), -math.inf)
        x = x + torch.einsum("hij,jhd->ihd", torch.softmax(z, -1), v).reshape(len(x), -1) @ d["wo"]
        h = norm(x, d["norm_mlp"])
        x = x + (torch.nn.functional.gelu(h @ d["wgate"], approximate="tanh") * (h @ d["wup"])) @ d["wdown"]
    return x


def a_tree(rng, n):
    """Parents (-1: the committed text), ascending; depth and ancestors of every draft."""
    parent = [rng.randint(max(-1, j - 4), j - 1) for j in range(n)]
    line = []
    for j in range(n):
        line.append((line[parent[j]] if parent[j] >= 0 else []) + [j])
    return [len(a) - 1 for a in line], line


class Server:
    """A batch of requests and what each has read so far."""

    def __init__(self, layers, dtype, device, requests=5, pages=14, page=8, seed=0):
        self.layers, self.device, self.dtype, self.rng = layers, device, dtype, random.Random(seed)
        self.g = torch.Generator().manual_seed(seed + 1)
        self.cache = layers.PagedCache.empty(LAYERS, pages, page, KV, HD, requests, 200, dtype=dtype, device=device)
        self.rope = layers.rotary_tables(torch.arange(PLACES, device=device), ROTARY)
        self.text = [torch.zeros(0, HIDDEN, dtype=dtype) for _ in range(requests)]

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def draw(self, rows, most):
        """(x, new, positions, mask, lines): a step with a tree for every request."""
        new, lines, positions = [], [], [-1] * rows
        mask = torch.zeros(rows, 2, dtype=torch.int64)
        at = 0
        for t in self.text:
            n = self.rng.choice((0, 1, 1, 3, most)) if len(t) else self.rng.randint(1, most)
            depth, line = a_tree(self.rng, n)
            for j in range(n):
                positions[at + j] = len(t) + depth[j]
                for i in line[j]:
                    mask[at + j, i // 32] |= 1 << (i % 32)
            at += n
            new.append(n)
            lines.append(line)
        assert at <= rows
        x = torch.randn(rows, HIDDEN, generator=self.g).to(self.dtype)
        mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
        return x, new, positions, mask, lines

    def choose(self, lines, granted):
        """kept and path: the way down to a random draft, or part of it; now and then a request ends."""
        kept, path = [], torch.zeros(len(lines), 48, dtype=torch.int32)
        for b, line in enumerate(lines):
            if self.rng.random() < 0.12:
                kept.append(-1)
                continue
            way = self.rng.choice(line) if granted[b] and line else []
            kept.append(len(way))
            path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        return kept, path

    def read(self, x, start, granted, kept, path):
        for b, k in enumerate(kept):
            if k < 0:
                self.text[b] = self.text[b][:0]
            elif granted[b]:
                self.text[b] = torch.cat((self.text[b], x[start[b] + path[b, :k].long()]))


def expected_rows(server, full, x, b, r0, line):
    old, n = server.text[b], len(line)
    L = len(old)
    places = torch.cat((torch.arange(L), torch.tensor([L + len(a) - 1 for a in line])))
    seen = torch.ones(L + n, L + n).tril().bool()
    seen[L:, L:] = False
    for j, a in enumerate(line):
        seen[L + j, torch.tensor(a) + L] = True
    return whole_text(full, torch.cat((old, x[r0:r0 + n])), places, seen)[L:]


def run(pkg, device, dtype, make_ops, rtol, atol, seed, steps=9):
    layers = importlib.import_module(pkg.__name__ + ".layers")
    ops = make_ops(layers)
    full = weights(dtype)
    ws = [layers.GroupedLayerWeights.shard({k: v.to(device) for k, v in w.items()}, HEADS, KV, HD, 0, 1) for w in full]
    server = Server(layers, dtype, device, seed=seed)
    refused = ended = 0
    for i in range(steps):
        x, new, positions, mask, lines = server.draw(203, 40)
        y, step = layers.paged_step(x.to(device), ws, server.cache, server.ints(new), ops, rope=server.rope, positions=server.ints(positions),
                                    mask=mask.to(device))
        granted, start = step.granted.tolist(), step.row_start.tolist()
        y = y.cpu()
        assert bool(torch.isfinite(y).all())
        for b, line in enumerate(lines):
            assert granted[b] in (0, new[b])
            refused += granted[b] < new[b]
            if granted[b]:
                want = expected_rows(server, full, x, b, start[b], line)
                got = y[start[b]:start[b] + new[b]].double()
                assert bool(((got - want).abs() <= atol + rtol * want.abs()).all()), (i, b, float((got - want).abs().max()))
        kept, path = server.choose(lines, granted)
        ended += sum(k < 0 for k in kept)
        layers.paged_accept_(server.cache, step, server.ints(kept), ops, path=path.to(device))
        server.read(x, start, granted, kept, path)
        lengths = server.cache.lengths.tolist()
        assert lengths == [len(t) for t in server.text]
        page = server.cache.page_size
        held = [p for b, L in enumerate(lengths) for p in server.cache.page_table[b, :-(-L // page)].tolist()]
        free = server.cache.free_pages[:int(server.cache.free_count)].tolist()
        assert sorted(held + free) == list(range(server.cache.k_pages.shape[1]))      # every page once, held or free
    return refused, ended


def test_steps_in_plain_form(pkg):
    """fp32 throughout, sums of at most a few hundred terms of order 1 in two layers: 1e-4 has room."""
    refused, ended = run(pkg, "cpu", torch.float32, lambda layers: PlainOps(), 1e-4, 1e-4, seed=0, steps=16)
    assert refused and ended


def test_a_chain_is_a_tree_without_branches(pkg):
    layers = importlib.import_module(pkg.__name__ + ".layers")
    ws = [layers.GroupedLayerWeights.shard(w, HEADS, KV, HD, 0, 1) for w in weights(torch.float32)]
    x = torch.randn(9, HIDDEN, generator=torch.Generator().manual_seed(5))
    new = torch.tensor([4, 0, 3], dtype=torch.int32)
    results = []
    for mask in (None, torch.tensor([[1], [3], [7], [15], [1], [3], [7], [0], [0]], dtype=torch.int32)):
        server = Server(layers, torch.float32, "cpu", requests=3)
        y, step = layers.paged_step(x, ws, server.cache, new, PlainOps(), rope=server.rope, mask=mask)
        layers.paged_accept_(server.cache, step, torch.tensor([3, 0, -1], dtype=torch.int32), PlainOps())
        assert server.cache.lengths.tolist() == [3, 0, 0] and int(server.cache.free_count) == 13
        results.append(y[:7])
    assert torch.equal(*results)


def _rank(rank, world, port, queue):
    import __graft_entry__ as entry
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        layers = importlib.import_module(entry.load_package().__name__ + ".layers")
        full, x, new = weights(torch.float32), torch.randn(11, HIDDEN, generator=torch.Generator().manual_seed(5)), [6, 5]
        results = []
        for r, n in ((rank, world), (0, 1)):
            ws = [layers.GroupedLayerWeights.shard(w, HEADS, KV, HD, r, n) for w in full]
            cache = layers.PagedCache.empty(LAYERS, 10, 4, KV // n, HD, 2, 40, dtype=torch.float32)
            rope = layers.rotary_tables(torch.arange(PLACES), ROTARY)
            reduce = None if n > 1 else lambda t, group=None: t
            results.append(layers.paged_step(x, ws, cache, torch.tensor(new, dtype=torch.int32), PlainOps(), rope=rope, reduce=reduce)[0])
        queue.put((rank, float((results[0] - results[1]).abs().max())))
    finally:
        dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_heads_over_two_ranks():
    """The sharded step is the whole one, but for the order of sums: 1e-4 as above."""
    with socket.socket() as sock:
        sock.bind(("127.0.0.1", 0))
        port = sock.getsockname()[1]
    context = mp.get_context("spawn")
    queue = context.Queue()
    ranks = [context.Process(target=_rank, args=(r, 2, port, queue)) for r in range(2)]
    for p in ranks:
        p.start()
    errors = [queue.get(timeout=240) for _ in ranks]
    for p in ranks:
        p.join(60)
        assert p.exitcode == 0
    assert max(e for _, e in errors) < 1e-4, errors


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 1])
def test_steps_on_the_gpu(pkg, cuda, seed):
    """Activations of order 1, stored in bf16 between kernels: the bounds of the other layer tests."""
    refused, ended = run(pkg, cuda, torch.bfloat16, lambda layers: layers.KernelOps(pkg), 2e-2, 6e-2, seed=seed, steps=16)
    assert refused and ended


@pytest.mark.gpu
def test_captured_steps(pkg, cuda):
    """A step and its end in one graph, replayed over changing inputs: the bits of the same steps launched one by one."""
    layers = importlib.import_module(pkg.__name__ + ".layers")
    ops = layers.KernelOps(pkg)
    ws = [layers.GroupedLayerWeights.shard({k: v.to(cuda) for k, v in w.items()}, HEADS, KV, HD, 0, 1) for w in weights(torch.bfloat16)]
    eager, captured = (Server(layers, torch.bfloat16, cuda, seed=3) for _ in range(2))
    rows = 203
    held = dict(x=torch.zeros(rows, HIDDEN, dtype=torch.bfloat16, device=cuda), new=eager.ints([0] * 5), positions=eager.ints([-1] * rows),
                mask=torch.zeros(rows, 2, dtype=torch.int32, device=cuda), kept=eager.ints([0] * 5), path=eager.ints([[0] * 48] * 5))

    def work(server, x, new, positions, mask, kept, path):
        y, step = layers.paged_step(x, ws, server.cache, new, ops, rope=server.rope, positions=positions, mask=mask)
        layers.paged_accept_(server.cache, step, kept, ops, path=path)
        return y, step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(captured, **held)                       # (no request has new tokens: nothing changes)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y_held, step_held = work(captured, **held)
    for _ in range(8):
        x, new, positions, mask, lines = eager.draw(rows, 40)
        kept, path = eager.choose(lines, new)        # (of those that turn out to be refused nothing is there to be kept)
        now = dict(x=x.to(cuda), new=eager.ints(new), positions=eager.ints(positions), mask=mask.to(cuda), kept=eager.ints(kept), path=path.to(cuda))
        y, step = work(eager, **now)
        for name, t in now.items():
            held[name].copy_(t)
        graph.replay()
        for a, b in zip((y, *step), (y_held, *step_held)):
            assert torch.equal(a, b)
        for name in ("page_table", "lengths", "free_count"):
            assert torch.equal(getattr(eager.cache, name), getattr(captured.cache, name))
        eager.read(x, step.row_start.tolist(), step.granted.tolist(), kept, path)
        assert eager.cache.lengths.tolist() == [len(t) for t in eager.text]


@pytest.mark.gpu
def test_two_servers_at_once(pkg, cuda):
    """Two batches on two streams, their steps on the GPU at one time: the bits of each alone."""
    layers = importlib.import_module(pkg.__name__ + ".layers")
    ops = layers.KernelOps(pkg)
    ws = [layers.GroupedLayerWeights.shard({k: v.to(cuda) for k, v in w.items()}, HEADS, KV, HD, 0, 1) for w in weights(torch.bfloat16)]

    def steps(seed):
        server = Server(layers, torch.bfloat16, cuda, seed=seed, pages=90)
        work = []
        for _ in range(6):
            x, new, positions, mask, lines = server.draw(203, 40)
            kept, path = server.choose(lines, new)
            start = [sum(new[:b]) for b in range(len(new))]
            work.append((x.to(cuda), server.ints(new), server.ints(positions), mask.to(cuda), server.ints(kept), path.to(cuda)))
            server.read(x, start, new, kept, path)
        return server, work

    def go(server, work):
        results = []
        for x, new, positions, mask, kept, path in work:
            y, step = layers.paged_step(x, ws, server.cache, new, ops, rope=server.rope, positions=positions, mask=mask)
            layers.paged_accept_(server.cache, step, kept, ops, path=path)
            results += [y, step.slot, server.cache.lengths.clone()]
        return results

    alone = [go(*steps(seed)) for seed in (1, 2)]
    both = [steps(seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        results = []
        for server, _ in both:
            server.cache.lengths.zero_()
            server.cache.free_count.fill_(90)
            server.cache.free_pages.copy_(torch.arange(89, -1, -1))
            server.cache.page_table.fill_(-1)
        torch.cuda.synchronize()
        for s, (server, work) in zip(streams, both):
            with torch.cuda.stream(s):
                torch.cuda._sleep(6000000)           # (both streams' work is there before either begins)
                results.append(go(server, work))
        torch.cuda.synchronize()
        for one, other in zip(alone, results):
            for a, b in zip(one, other):
                assert torch.equal(a, b)
