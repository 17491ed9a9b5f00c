"""The operators of a decoding step over a paged key/value cache, as cases that can be timed and compared.

Four families, each entered the way a program enters it:

  extend   `paged_extend`: pages for the new tokens of every request from a free list, and the row, position and slot maps,
           all from lengths that live on the GPU
  qk       `qk_norm_rotary_forward` / `qk_norm_rotary_backward`: RMSNorm of every query and key head and the position
           rotation in one pass; mode "cache" writes keys and values into their pages, "dense" returns the keys, "train" is a
           forward and a backward call
  tree     `fmha_paged_forward`: attention of the new tokens (a tree of drafted ones, a chain, or one a request) over the pages
  keep     `paged_keep`: after the drafts are verified, the keys and values of the accepted ones move together, lengths grow,
           unused pages go back

Request lengths are spread between two numbers, evenly in their logarithm, and dealt to the requests by the seed; the cache's
pages lie in random order.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0


def _extend(name, requests, lo, hi, new_lo, new_hi, page, short=0.0, spare_rows=0):
    return {"name": name, "family": "extend", "requests": requests, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "page": page,
            "short": short, "spare_rows": spare_rows}


def _qk(name, tokens, heads, kv_heads, size, mode, dtype="bf16", rotary=0, half=True, param="same", page=64):
    return {"name": name, "family": "qk", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "size": size, "mode": mode, "dtype": dtype,
            "rotary": rotary or size, "half": half, "param": param, "page": page}


def _tree(name, requests, lo, hi, new_lo, new_hi, heads, kv_heads, size, page, kind, dtype="bf16", lse=False, spare_rows=0):
    return {"name": name, "family": "tree", "requests": requests, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "heads": heads,
            "kv_heads": kv_heads, "size": size, "page": page, "kind": kind, "dtype": dtype, "lse": lse, "spare_rows": spare_rows}


def _keep(name, requests, lo, hi, new_lo, new_hi, layers, kv_heads, size, page, dtype="bf16"):
    return {"name": name, "family": "keep", "requests": requests, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "layers": layers,
            "kv_heads": kv_heads, "size": size, "page": page, "dtype": dtype}


def listed():
    return [
        # a decoding step's maps for a batch of 64, one token each: the call's latency
        _extend("extend_decode_64", 64, 1, 4096, 1, 1, 16),
        # a busy server: prompts and drafts of 1500 requests at once, and too few pages for all of them
        _extend("extend_mixed_1500", 1500, 1, 9000, 1, 200, 32, short=0.1, spare_rows=77),
        # a decoding step of 64 tokens, grouped heads, into the pages: the call's latency
        _qk("qk_decode_64", 64, 16, 4, 128, "cache", page=16),
        # a prompt of 16384 tokens through a wide model, into the pages
        _qk("qk_prompt_16384", 16384, 32, 8, 128, "cache"),
        # training on the GPT-J-shaped block (16 heads of 256), four sequences of 2048 tokens
        _qk("qk_train_8192x256", 8192, 16, 16, 256, "train", param="fp32"),
        # a ragged batch in fp16, odd head counts, the first 32 elements of a head rotated in interleaved pairs
        _qk("qk_train_odd", 1371, 7, 1, 80, "train", dtype="fp16", rotary=32, half=False),
        # one request verifies a chain of five drafts: the call's latency
        _tree("tree_chain_1x5", 1, 700, 700, 5, 5, 16, 4, 128, 16, "chain"),
        # 64 requests verify trees of 16 drafts
        _tree("tree_verify_64x16", 64, 1024, 4096, 16, 16, 16, 4, 128, 64, "tree"),
        # the larger heads of the Gemma-shaped block, fp16, wide trees on ragged contexts, some rows of the batch unused
        _tree("tree_ragged_h256", 24, 100, 12000, 1, 48, 20, 5, 256, 16, "tree", dtype="fp16", lse=True, spare_rows=9),
        # plain decoding of eight long contexts, eight query heads to a key head
        _tree("decode_long_8", 8, 30000, 65000, 1, 1, 32, 4, 128, 128, "chain"),
        # after a small verification: two layers
        _keep("keep_small", 8, 100, 3000, 6, 6, 2, 4, 128, 16),
        # after the verification of 128 trees: every layer's cache at once
        _keep("keep_tree_128", 128, 50, 4000, 8, 32, 24, 4, 128, 64),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    """One more case of the same ranges; none costs more than the largest listed one."""
    family = rng.choice(["extend", "qk", "qk", "tree", "tree", "tree", "keep"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if family == "extend":
        new_hi = _log_int(rng, 1, 400)
        requests = max(1, min(_log_int(rng, 1, 2000), 150000 // new_hi))
        c = _extend("", requests, _log_int(rng, 1, 50), _log_int(rng, 50, 9000), rng.randint(0, min(3, new_hi)), new_hi, page,
                    rng.choice([0.0, 0.0, 0.1, 0.5]), rng.choice([0, 0, 5, 300]))
    elif family == "qk":
        size = rng.choice([64, 80, 96, 128, 128, 160, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 7]) if kv_heads < 8 else kv_heads * rng.choice([1, 2])
        mode = rng.choice(["cache", "cache", "dense", "train", "train"])
        tokens = min(_log_int(rng, 1, 16384), int(6e7 / ((heads + kv_heads) * size)))
        c = _qk("", max(1, tokens), heads, kv_heads, size, mode, rng.choice(["bf16", "bf16", "fp16"] + (["fp32"] if mode != "cache" else [])),
                rng.choice([size, size, size // 32 * 16]), rng.random() < 0.6, rng.choice(["same", "fp32"]), page)
    elif family == "tree":
        size = rng.choice([64, 80, 128, 128, 192, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
        new_hi = rng.choice([1, 1, 4, 8, 16, 33, 64])
        lo, hi = _log_int(rng, 1, 4000), _log_int(rng, 4000, 65000)
        most = min(4e8 / (kv_heads * size), 2e8 / (heads * new_hi))       # tokens of a padded batch: the plain form has to hold them
        hi = min(hi, int(most) - new_hi)
        requests = max(1, min(_log_int(rng, 1, 128), int(most / (hi + new_hi))))
        c = _tree("", requests, min(lo, hi), hi, 1 if requests > 1 else new_hi, new_hi, heads, kv_heads, size, page,
                  "chain" if new_hi == 1 else rng.choice(["tree", "tree", "chain"]), rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.3,
                  rng.choice([0, 0, 7]))
    else:
        new_hi = rng.randint(2, 48)
        requests = _log_int(rng, 1, 128)
        c = _keep("", requests, _log_int(rng, 1, 100), _log_int(rng, 100, 4000), rng.randint(1, new_hi), new_hi, rng.choice([1, 2, 8, 24]),
                  rng.choice([1, 3, 4]), rng.choice([64, 80, 128]), page, rng.choice(["bf16", "fp16"]))
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------- preparation

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread in the logarithm (of the number and one)."""
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    t = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    return t.mul_(scale) if scale != 1.0 else t


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _dealt(g, values):
    return torch.tensor(values, device="cuda")[torch.randperm(len(values), generator=g, device="cuda")].int()


def _requests(c, g, spare_pages=0):
    """Lengths, new tokens, and a cache whose pages lie in random order: the table of the pages that hold the lengths (and, where
    `spare_pages` is negative, the new tokens as well) and the free list behind them."""
    B, S = c["requests"], c["page"]
    lengths, new = _dealt(g, _spread(c["lo"], c["hi"], B)), _dealt(g, _spread(c["new_lo"], c["new_hi"], B))
    # (what lies in the table's unused places is any page)
    with_new = (lengths + new + S - 1) // S
    used = with_new if spare_pages < 0 else (lengths + S - 1) // S
    columns = (c["hi"] + c["new_hi"] + S - 1) // S
    # (one number of pages however the lengths are dealt)
    total = sum(-(-v // S) for v in _spread(c["lo"], c["hi"], B)) + max(spare_pages, sum(-(-v // S) for v in _spread(c["new_lo"], c["new_hi"], B))) + 8
    order = torch.randperm(total, generator=g, device="cuda").int()
    place = (used.cumsum(0) - used)[:, None] + torch.arange(columns, device="cuda")
    held = torch.arange(columns, device="cuda") < used[:, None]
    table = torch.where(held, order[torch.where(held, place, 0)], 0).int()
    free = torch.zeros(total, dtype=torch.int32, device="cuda")
    count = total - int(used.sum())
    free[:count] = order[total - count:]
    return lengths, new, table, total, free, torch.tensor([count], dtype=torch.int32, device="cuda")


def _pages(g, c, pages, dt, layers=None):
    shape = (pages, c["page"], c["kv_heads"], c["size"])
    shape = shape if layers is None else (layers,) + shape
    return _randn(g, *shape, dtype=dt), _randn(g, *shape, dtype=dt)


def prepare(case, seed):
    """What the program holds when it makes the call."""
    c, g = case, _generator(seed)
    s = {"case": c}
    if c["family"] == "extend":
        new = _spread(c["new_lo"], c["new_hi"], c["requests"])
        need = sum(new) // c["page"] + c["requests"]
        s["lengths"], s["new"], s["table"], s["pages"], s["free"], s["count"] = _requests(c, g, need)
        if c["short"]:      # the list runs out before all requests have their pages
            wanted = int(((s["lengths"] + s["new"] + c["page"] - 1) // c["page"] - (s["lengths"] + c["page"] - 1) // c["page"]).sum())
            s["count"] = torch.tensor([int(wanted * (1.0 - c["short"]))], dtype=torch.int32, device="cuda")
        s["rows"] = sum(new) + c["spare_rows"]
        return s
    dt = DTYPES[c["dtype"]]
    if c["family"] == "qk":
        T, H, N, NK = c["tokens"], c["size"], c["heads"], c["kv_heads"]
        pt = torch.float32 if c["param"] == "fp32" else dt
        # slices of one fused projection; every head has its own size, as projections have
        qkv = _randn(g, T, N + 2 * NK, H).mul_((_randn(g, N + 2 * NK, 1) * 0.5).exp_()).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :N], qkv[:, N:N + NK], qkv[:, N + NK:]
        s["offset"] = 0.0 if c["half"] else 1.0
        s["q_gain"] = (_randn(g, H, scale=0.1) + (1.0 - s["offset"])).to(pt)
        s["k_gain"] = (_randn(g, H, scale=0.1) + (1.0 - s["offset"])).to(pt)
        places = 32768
        half = c["rotary"] // 2
        angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # a packed batch: runs of consecutive positions that begin anywhere
        start = _ints(g, 0, places - 2048, T // 512 + 1)
        t = torch.arange(T, device="cuda")
        s["positions"] = (start[t // 512] + t % 512).int()
        if c["mode"] == "cache":
            pages = (T + c["page"] - 1) // c["page"] + 3
            s["slots"] = torch.randperm(pages * c["page"], generator=g, device="cuda")[:T].int()
            s["k_pages"], s["v_pages"] = _pages(g, c, pages, dt)
        if c["mode"] == "train":
            s["grad_q"], s["grad_k"] = _randn(g, T, N, H, dtype=dt), _randn(g, T, NK, H, dtype=dt)
        return s
    s["lengths"], s["granted"], s["table"], s["pages"], s["free"], s["count"] = _requests(c, g, -1)
    B, total = c["requests"], sum(_spread(c["new_lo"], c["new_hi"], c["requests"]))
    n = c["new_hi"]
    if c["family"] == "keep":
        s["k_pages"], s["v_pages"] = _pages(g, c, s["pages"], dt, c["layers"])
        # the accepted path: every request keeps up to its drafts, fewer as they go on; some requests end
        keep = torch.rand(B, n, generator=g, device="cuda") < torch.linspace(0.95, 0.2, n, device="cuda")
        keep &= torch.arange(n, device="cuda") < s["granted"][:, None]
        order = torch.where(keep, torch.arange(n, device="cuda"), 2 * n).sort(1).values
        s["path"] = torch.where(order < n, order, 0).int()
        s["kept"] = torch.where(torch.rand(B, generator=g, device="cuda") < 0.1, -1, keep.sum(1)).int()
        return s
    # queries that look for some keys more than for others, as trained heads do
    rows = total + c["spare_rows"]
    s["q"] = _randn(g, rows, c["heads"], c["size"], dtype=dt, scale=1.5)
    s["k_pages"], s["v_pages"] = _pages(g, c, s["pages"], dt)
    s["scale"] = c["size"] ** -0.5
    s["row_start"] = torch.cat((s["granted"].new_zeros(1), s["granted"].cumsum(0).int())).int()
    s["out"] = torch.zeros_like(s["q"])
    s["mask"] = None
    if c["kind"] == "tree":
        # each draft hangs on an earlier one (or on the context) and sees the drafts above it, and itself
        parent = (torch.rand(B, n, generator=g, device="cuda") * torch.arange(n, device="cuda")).long()
        sees = torch.eye(n, dtype=torch.bool, device="cuda").expand(B, n, n).clone()
        for i in range(1, n):
            sees[:, i] |= sees[torch.arange(B, device="cuda"), parent[:, i]]
        words = (n + 31) // 32
        bits = torch.zeros(B, n, words * 32, dtype=torch.int64, device="cuda")
        bits[:, :, :n] = sees.long()
        packed = (bits.view(B, n, words, 32) << torch.arange(32, device="cuda")).sum(3)
        packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()
        s["mask"] = torch.zeros(rows, words, dtype=torch.int32, device="cuda")
        s["mask"][:total] = packed[torch.arange(n, device="cuda") < s["granted"][:, None]]
    return s


# ------------------------------------------------------------------------------------- one pass

def _package():
    import importlib
    return importlib.import_module("intel-extension-for-openxla_b200")


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["family"]](state, state["case"])


def _run_own(s):
    ixk, c = _package(), s["case"]
    if c["family"] == "extend":
        step = ixk.paged_extend(s["table"], s["lengths"], s["new"], s["free"], s["count"], rows=s["rows"], page_size=c["page"])
        return {"table": s["table"], "row_start": step.row_start, "granted": step.granted, "request": step.request,
                "position": step.position, "slot": step.slot, "free_count": step.free_count}
    if c["family"] == "qk":
        common = {"q_gain": s["q_gain"], "k_gain": s["k_gain"], "gain_offset": s["offset"], "eps": 1e-6, "cos": s["cos"], "sin": s["sin"],
                  "positions": s["positions"], "half_split": c["half"]}
        if c["mode"] == "cache":
            q, _ = ixk.qk_norm_rotary_forward(s["q"], s["k"], v=s["v"], slots=s["slots"], k_pages=s["k_pages"], v_pages=s["v_pages"], **common)
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        q, k = ixk.qk_norm_rotary_forward(s["q"], s["k"], **common)
        out = {"q": q, "k": k}
        if c["mode"] == "train":
            out["dq"], out["dk"], out["dq_gain"], out["dk_gain"] = ixk.qk_norm_rotary_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], **common)
        return out
    if c["family"] == "tree":
        out, lse = ixk.fmha_paged_forward(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["row_start"], s["granted"],
                                          scale=s["scale"], mask=s["mask"], out=s["out"], with_lse=c["lse"])
        return {"out": out, "lse": lse[:sum(_spread(c["new_lo"], c["new_hi"], c["requests"]))]} if c["lse"] else {"out": out}
    lengths, count = ixk.paged_keep(s["table"], s["lengths"], s["granted"], s["kept"], s["free"], s["count"], page_size=c["page"],
                                    path=s["path"], k_pages=s["k_pages"], v_pages=s["v_pages"])
    return {"lengths": lengths, "free_count": count, "free": s["free"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _pages_of(tokens, page):
    return (tokens + page - 1) // page


def _plain_extend(s, c):
    S, rows, columns = c["page"], s["rows"], s["table"].shape[1]
    lengths, new, free, count = s["lengths"].long(), s["new"].long(), s["free"], s["count"].long()
    end = new.cumsum(0)
    have, want = _pages_of(lengths, S), _pages_of(lengths + new, S)
    fits = (lengths >= 0) & (want <= columns) & (end <= rows)
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    first = upto - need
    taken = torch.where(served, need, 0).sum(0, keepdim=True)
    # the table's new places
    column = torch.arange(columns, device="cuda")
    fresh = served[:, None] & (column >= have[:, None]) & (column < want[:, None])
    at = count - 1 - (first[:, None] + column - have[:, None])
    s["table"].copy_(torch.where(fresh, free[torch.where(fresh, at, 0)], s["table"]))
    row_start = torch.cat((end.new_zeros(1), end)).clamp(max=rows)
    r = torch.arange(rows, device="cuda")
    of = torch.searchsorted(row_start[1:], r, right=True)
    inside = of < len(new)
    of = torch.where(inside, of, 0)
    valid = inside & served[of]
    position = torch.where(valid, lengths[of] + r - row_start[of], 0)
    slot = s["table"][of, position // S].long() * S + position % S
    none = torch.full_like(r, -1)
    return {"table": s["table"], "row_start": row_start.int(), "granted": torch.where(served, new, 0).int(),
            "request": torch.where(valid, of, none).int(), "position": torch.where(valid, position, none).int(),
            "slot": torch.where(valid, slot, none).int(), "free_count": (count - taken).int()}


def _turn(x, cos, sin, rotary, half, back=False):
    """Every head's first `rotary` elements, turned by the angles of its token (or back)."""
    c, s = cos[:, None, :], (-sin if back else sin)[:, None, :]
    x1, x2 = (x[..., :rotary // 2], x[..., rotary // 2:rotary]) if half else (x[..., 0:rotary:2], x[..., 1:rotary:2])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    turned = torch.cat((y1, y2), -1) if half else torch.stack((y1, y2), -1).flatten(-2)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_norm(x, gain, s, c, cos, sin):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (s["offset"] + gain.float())
    return _turn(y, cos, sin, c["rotary"], c["half"])


def _plain_norm_back(grad, x, gain, s, c, cos, sin):
    g, x = _turn(grad.float(), cos, sin, c["rotary"], c["half"], back=True), x.float()
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    xh = x * rstd
    h = g * (s["offset"] + gain.float())
    return (h - xh * (h * xh).mean(-1, keepdim=True)) * rstd, (g * xh).sum((0, 1))


def _plain_qk(s, c):
    dt = s["q"].dtype
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    q, k = (_plain_norm(s[x], s[x + "_gain"], s, c, cos, sin).to(dt) for x in ("q", "k"))
    if c["mode"] == "cache":
        slots = s["slots"].long()
        s["k_pages"].view(-1, c["kv_heads"], c["size"])[slots] = k
        s["v_pages"].view(-1, c["kv_heads"], c["size"])[slots] = s["v"]
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    out = {"q": q, "k": k}
    if c["mode"] == "train":
        pt = s["q_gain"].dtype
        dq, dq_gain = _plain_norm_back(s["grad_q"], s["q"], s["q_gain"], s, c, cos, sin)
        dk, dk_gain = _plain_norm_back(s["grad_k"], s["k"], s["k_gain"], s, c, cos, sin)
        out.update(dq=dq.to(dt), dk=dk.to(dt), dq_gain=dq_gain.to(pt), dk_gain=dk_gain.to(pt))
    return out


def _plain_tree(s, c):
    """The batch padded to its longest request, the keys gathered out of their pages."""
    B, S, N, NK, H, n = c["requests"], c["page"], c["heads"], c["kv_heads"], c["size"], c["new_hi"]
    keys = c["hi"] + n
    lengths, granted, start = s["lengths"].long(), s["granted"].long(), s["row_start"].long()
    t, j = torch.arange(keys, device="cuda"), torch.arange(n, device="cuda")
    slots = s["table"].long()[:, t // S] * S + t % S
    k = s["k_pages"].view(-1, NK, H)[slots].permute(0, 2, 3, 1).float()            # [B, NK, H, keys]
    v = s["v_pages"].view(-1, NK, H)[slots].permute(0, 2, 1, 3).float()            # [B, NK, keys, H]
    row = torch.where(j < granted[:, None], start[:-1, None] + j, 0)
    q = s["q"][row].float().view(B, n, NK, N // NK, H).permute(0, 2, 1, 3, 4).reshape(B, NK, n * (N // NK), H)
    draft = t - lengths[:, None]                                                   # [B, keys]
    if s["mask"] is None:
        sees = draft[:, None, :] <= j[None, :, None]
    else:
        d = draft.clamp(0, n - 1)[:, None, :]
        words = torch.gather(s["mask"][row].long(), 2, (d // 32).expand(B, n, keys))
        sees = (draft[:, None, :] < granted[:, None, None]) & ((draft[:, None, :] < 0) | ((words >> (d % 32) & 1) > 0))
    sees = (sees & (t < (lengths + granted)[:, None])[:, None, :]).repeat_interleave(N // NK, 1)[:, None]
    z = torch.where(sees, (q @ k) * s["scale"], -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    o = o.view(B, NK, n, N // NK, H).permute(0, 2, 1, 3, 4).reshape(B, n, N, H)
    there = j < granted[:, None]
    s["out"][:int(sum(_spread(c["new_lo"], c["new_hi"], B)))] = o[there].to(s["out"].dtype)
    out = {"out": s["out"]}
    if c["lse"]:
        lse = (top + total.log()).view(B, NK, n, N // NK).permute(0, 2, 1, 3).reshape(B, n, N)
        out["lse"] = lse[there]
    return out


def _plain_keep(s, c):
    S, n, pages = c["page"], s["path"].shape[1], s["pages"]
    lengths, granted, kept, path, count = s["lengths"].long(), s["granted"].long(), s["kept"].long(), s["path"].long(), s["count"].long()
    j = torch.arange(n, device="cuda")
    before = torch.cat((torch.full_like(path[:, :1], -1), path[:, :-1]), 1)
    fine = (j < kept[:, None]) & (path > before) & (path < granted[:, None])
    fine = fine.long().cumprod(1)
    moved = fine.sum(1)
    # what moves is gathered in whole before it is put down
    b, i = torch.nonzero(fine, as_tuple=True)
    source, target = lengths[b] + path[b, i], lengths[b] + i
    source, target = (s["table"][b, p // S].long() * S + p % S for p in (source, target))
    for cache in (s["k_pages"], s["v_pages"]):
        flat = cache.view(c["layers"], -1, c["kv_heads"], c["size"])
        flat[:, target] = flat[:, source]
    after = torch.where(kept < 0, 0, lengths + moved)
    low, high = _pages_of(after, S), _pages_of(lengths + granted, S)
    columns = torch.arange(s["table"].shape[1], device="cuda")
    loose = (columns >= low[:, None]) & (columns < high[:, None])
    back = s["table"][loose]
    place = count + torch.arange(len(back), device="cuda")
    s["free"][place.clamp(max=pages - 1)] = back
    return {"lengths": after.int(), "free_count": (count + len(back)).int(), "free": s["free"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


_PLAIN = {"extend": _plain_extend, "qk": _plain_qk, "tree": _plain_tree, "keep": _plain_keep}


# ------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions in 64 bits, a request or a head at a time; moved and whole values have none."""
    c, s, f64 = case, prepare(case, seed), torch.float64
    if c["family"] in ("extend", "keep"):
        return None
    if c["family"] == "qk":
        rot, H = c["rotary"], c["size"]
        phase = torch.complex(s["cos"].to(f64), s["sin"].to(f64))[s["positions"].long()]

        def pairs(x):           # a head's rotated elements as complex numbers
            x = x[..., :rot]
            x = torch.stack((x[..., :rot // 2], x[..., rot // 2:]), -1) if c["half"] else x.reshape(*x.shape[:-1], rot // 2, 2)
            return torch.view_as_complex(x.contiguous())

        def elements(z, rest):
            x = torch.view_as_real(z)
            x = x.transpose(-1, -2).flatten(-2) if c["half"] else x.flatten(-2)
            return torch.cat((x, rest[..., rot:]), -1)

        out = {}
        for name in ("q", "k"):
            x, w = s[name].to(f64), s[name + "_gain"].to(f64) + s["offset"]
            size = (x.square().sum(-1, keepdim=True) / H + 1e-6).sqrt()
            unit = x / size
            y = unit * w
            out[name] = elements(pairs(y) * phase[:, None], y)
            if c["mode"] == "train":
                g = s["grad_" + name].to(f64)
                g = elements(pairs(g) * phase[:, None].conj(), g)
                out["d" + name + "_gain"] = torch.einsum("tnh,tnh->h", g, unit)
                a = g * w
                # the part along the head's own direction does not count
                out["d" + name] = (a - unit * ((a * unit).sum(-1, keepdim=True) / H)) / size
        if c["mode"] == "cache":
            k_pages, v_pages = s["k_pages"].to(f64), s["v_pages"].to(f64)
            k_pages.view(-1, c["kv_heads"], H).index_copy_(0, s["slots"].long(), out.pop("k"))
            v_pages.view(-1, c["kv_heads"], H).index_copy_(0, s["slots"].long(), s["v"].to(f64))
            out.update(k_pages=k_pages, v_pages=v_pages)
        return out
    out, lse = torch.zeros_like(s["q"], dtype=f64), []
    lengths, granted, start = s["lengths"].tolist(), s["granted"].tolist(), s["row_start"].tolist()
    group = c["heads"] // c["kv_heads"]
    for b in range(c["requests"]):
        L, n, r0 = lengths[b], granted[b], start[b]
        used = s["table"][b, :(L + n + c["page"] - 1) // c["page"]].long()
        k = s["k_pages"][used].flatten(0, 1)[:L + n]
        v = s["v_pages"][used].flatten(0, 1)[:L + n]
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        if s["mask"] is not None:
            i = torch.arange(n, device="cuda")
            hidden = (s["mask"][r0:r0 + n].long()[:, i // 32] >> (i % 32)) % 2 == 0
        rows = []
        for h in range(c["heads"]):
            z = s["q"][r0:r0 + n, h].to(f64) @ k[:, h // group].to(f64).t() * s["scale"]
            z[:, L:].masked_fill_(hidden, -math.inf)
            out[r0:r0 + n, h] = torch.softmax(z, 1) @ v[:, h // group].to(f64)
            rows.append(torch.logsumexp(z, 1))
        lse.append(torch.stack(rows, 1))
    return {"out": out, "lse": torch.cat(lse)} if c["lse"] else {"out": out}


# ------------------------------------------------------------------------------------- what it takes

def work(case):
    """Each input once, each output once; the two products of attention over the keys that a row sees."""
    c = case
    B = c.get("requests", 0)
    if c["family"] == "extend":
        new = sum(_spread(c["new_lo"], c["new_hi"], B))
        # lengths and counts in, counts, row starts and the three maps out; a table word a request, taken pages in and out
        return {"bytes": 20.0 * B + 12.0 * (new + c["spare_rows"]) + 8.0 * new / c["page"], "flops": 0.0}
    e = 4.0 if c["dtype"] == "fp32" else 2.0
    if c["family"] == "qk":
        T, H = c["tokens"], c["size"]
        both = (c["heads"] + c["kv_heads"]) * T * H * e
        tables = T * (c["rotary"] * 4.0 + 4.0)
        if c["mode"] == "cache":
            return {"bytes": 2.0 * both + 2.0 * c["kv_heads"] * T * H * e + tables + 4.0 * T, "flops": 8.0 * both / e}
        return {"bytes": (5.0 if c["mode"] == "train" else 2.0) * both + tables, "flops": (24.0 if c["mode"] == "train" else 8.0) * both / e}
    new, lengths = _spread(c["new_lo"], c["new_hi"], B), _spread(c["lo"], c["hi"], B)
    token = 2.0 * c["kv_heads"] * c["size"] * e
    if c["family"] == "tree":
        keys, rows, mean = sum(lengths) + sum(new), sum(new), sum(new) / B
        visible = sum(lengths) * mean + rows * (mean + 1.0) / 2.0       # (the lengths are dealt apart from the new tokens)
        return {"bytes": keys * token + 2.0 * rows * c["heads"] * c["size"] * e + 4.0 * keys / c["page"],
                "flops": 4.0 * c["heads"] * c["size"] * visible}
    moved = 0.5 * sum(new)
    return {"bytes": 2.0 * moved * c["layers"] * token + 4.0 * sum(new) + 16.0 * B, "flops": 0.0}
