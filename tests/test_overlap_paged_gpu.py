"""GPU: the kernels of a paged cache and of norm and rotation of heads start while their predecessor runs and wait for it in front of
their first access.

Chains of calls, each fed by the last, on the same buffers and scratch: eagerly and as a graph replay they give the bits of
the same chain in a process in which every launch waits for the one before (CUDA_LAUNCH_BLOCKING)."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def steps_chain(pkg, dev, lengths, new, heads, kv_heads, size, page, tree, in_place, dtype=torch.bfloat16):
    """Steps over two layers: tables and maps, norm and rotation into the pages, attention, whose result is the next layer's
    projection, and what follows the verification; every call reads what the one in front of it has written."""
    B, layers, steps = len(lengths), 2, 4
    g = torch.Generator(device=dev).manual_seed(B + size)
    most = max(lengths) + steps * new + new
    columns = -(-most // page)
    pages = sum(-(-(n + steps * new + new) // page) for n in lengths) + 2
    kv0 = torch.randn(2, layers, pages, page, kv_heads, size, generator=g, device=dev).to(dtype)
    ints = dict(dtype=torch.int32, device=dev)
    table0, free0, at = torch.full((B, columns), -1, **ints), torch.arange(pages, **ints), pages
    for b, n in enumerate(lengths):
        c = -(-n // page)
        table0[b, :c] = free0[at - c:at].flip(0)
        at -= c
    lengths0, count0, added = torch.tensor(lengths, **ints), torch.tensor([at], **ints), torch.full((B,), new, **ints)
    rows = B * new
    x0 = torch.randn(rows, heads + 2 * kv_heads, size, generator=g, device=dev).to(dtype)
    gains = [torch.randn(size, generator=g, device=dev).to(dtype) for _ in range(2)]
    angle = torch.rand(most, size // 2, generator=g, device=dev) * 6
    cos, sin = angle.cos(), angle.sin()
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, 1), generator=g, device=dev).int() | 1 if tree else None
    path = torch.arange(0, 2 * new, 2, **ints).expand(B, -1).contiguous() if tree else None
    kept = torch.randint(0, new + 1, (B,), generator=g, device=dev).int()
    ws = torch.empty(pkg.fmha_paged_workspace_bytes(x0[:, :heads], kv0[0, 0]), dtype=torch.uint8, device=dev)
    step_count = torch.empty_like(count0)

    def run():
        kv, table, free, length, count, x, got = kv0.clone(), table0.clone(), free0.clone(), lengths0.clone(), count0.clone(), x0.clone(), []
        for _ in range(steps):
            r = pkg.paged_extend(table, length, added, free, count, rows=rows, page_size=page)
            if in_place:
                pkg.paged_extend(table, length, added, free, count, rows=rows, page_size=page, out=r._replace(free_count=count))
            else:
                pkg.paged_extend(table, length, added, free, count, rows=rows, page_size=page, out=r._replace(free_count=step_count))
            for layer in range(layers):
                q, k, v = x.split((heads, kv_heads, kv_heads), 1)
                pkg.qk_norm_rotary_forward(q, k, q_gain=gains[0], k_gain=gains[1], cos=cos, sin=sin, positions=r.position, v=v, slots=r.slot,
                                           k_pages=kv[0, layer], v_pages=kv[1, layer], q_out=q)
                out, lse = pkg.fmha_paged_forward(q, kv[0, layer], kv[1, layer], table, length, r.row_start, r.granted, scale=size ** -0.5,
                                                  mask=mask, with_lse=True, workspace=ws)
                x = torch.cat((out, v, k), 1)
                got += [out, lse, x]
            pkg.paged_keep(table, length, r.granted, kept, free, count if in_place else step_count, page_size=page, path=path,
                           k_pages=kv[0] if tree else None, v_pages=kv[1] if tree else None, lengths_out=length, free_count_out=count)
            got += [r.granted.clone(), r.slot.clone(), length.clone()]
        # (a list's free end and pages of nobody hold what the order of earlier steps left there: of the results only what counts)
        return got + [kv, table, count]
    return run


def gradients_chain(pkg, dev, T, N, K, H, dtype, half):
    """Forward and backward of norm and rotation, each step's inputs the last one's gradients, the scratch shared by all."""
    g = torch.Generator(device=dev).manual_seed(T)
    x0 = torch.randn(T, N + K, H, generator=g, device=dev).to(dtype)
    # (fp32 gains for fp16 heads: their gradients are sums over 48000 heads, beyond fp16's range)
    gains = [torch.randn(H, generator=g, device=dev).to(torch.bfloat16 if dtype == torch.bfloat16 else torch.float32) for _ in range(2)]
    angle = torch.rand(500, H // 4, generator=g, device=dev) * 6
    common = dict(cos=angle.cos(), sin=angle.sin(), half_split=half)
    ws = torch.empty(pkg.qk_norm_rotary_backward_workspace_bytes(x0[:, :N], x0[:, N:], common["cos"]), dtype=torch.uint8, device=dev)

    def run():
        x, (wq, wk), got = x0, gains, []
        for _ in range(4):
            q, k = pkg.qk_norm_rotary_forward(x[:, :N], x[:, N:], q_gain=wq, k_gain=wk, **common)
            dq, dk, dwq, dwk = pkg.qk_norm_rotary_backward(q, k, x[:, :N], x[:, N:], q_gain=wq, k_gain=wk, workspace=ws, **common)
            x, wq, wk = torch.cat((q + dq, k + dk), 1), wq + 1e-6 * dwq, wk + 1e-6 * dwk
            got += [q, k, dq, dk, dwq, dwk]
        return got
    return run


CHAINS = {
    "tree": lambda pkg, dev: steps_chain(pkg, dev, [900, 30, 0, 64, 411], 8, 8, 2, 128, 16, True, False),
    "tree in place": lambda pkg, dev: steps_chain(pkg, dev, [40] * 300, 5, 4, 4, 64, 8, True, True, torch.float16),
    "chain": lambda pkg, dev: steps_chain(pkg, dev, [5000, 200, 3], 4, 10, 2, 256, 32, False, False),
    "single": lambda pkg, dev: steps_chain(pkg, dev, [20000], 1, 8, 1, 128, 64, False, True),
    "prompt": lambda pkg, dev: steps_chain(pkg, dev, [0, 100], 300, 4, 2, 96, 16, False, False),
    "gradients": lambda pkg, dev: gradients_chain(pkg, dev, 1371, 7, 1, 128, torch.bfloat16, True),
    "gradients, few": lambda pkg, dev: gradients_chain(pkg, dev, 9, 3, 2, 64, torch.float32, False),
    "gradients, many": lambda pkg, dev: gradients_chain(pkg, dev, 6000, 8, 8, 256, torch.float16, True),
}


def main(path):
    """Every chain, each launch after the end of the one before."""
    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    pkg, dev = entry.load_package(), torch.device("cuda:0")
    results = {}
    for name, make in CHAINS.items():
        run = make(pkg, dev)
        run()
        assert torch.cuda.current_stream().query()      # nothing is in flight when a call returns
        results[name] = [t.cpu() for t in run()]
    assert pkg.device_status() == 0
    torch.save(results, path)


@pytest.fixture(scope="module")
def one_at_a_time(cuda, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("chains") / "results.pt")
    r = subprocess.run([sys.executable, os.path.abspath(__file__), path], env={**os.environ, "CUDA_LAUNCH_BLOCKING": "1"},
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    return torch.load(path)


@pytest.mark.parametrize("name", list(CHAINS))
def test_chains_overlap_without_changing_a_bit(pkg, cuda, one_at_a_time, name):
    want = [t.to(cuda) for t in one_at_a_time[name]]
    assert all(t.float().isnan().sum() == 0 for t in want)
    run = CHAINS[name](pkg, cuda)

    def check(got):
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    for _ in range(5):
        check(run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        check(got)
    del graph


if __name__ == "__main__":
    main(sys.argv[1])
