"""Operators of a layer that answers many requests at once, with their plain forms.

* ``PagedKV.share`` / ``attend(shared=)``: the last t tokens of every sequence against its 8-bit pages, where sequences have pages in
  common (forks of one prompt, a tree of them): what is shared is read once for all of them.  Value = e4m3 code * scale of the
  (page, head); the token at position p sees the positions <= p of its own sequence.
* ``Adapters.add``: out = y + s_a (x A_a^T) B_a^T for every token, with the low-rank adapter a of its request, or out = y
  where it has none; y is the shared projection of the same x.
* ``norm_rope_heads``: every head's norm (x / sqrt(mean x^2 + eps) * (1 + w)), then the rotation of its first 2F dims: frequency f turns
  the dims (f, f + F) by the angle p_a(f) * inv_freq[f], with the token's position p_a on that frequency's axis a (time, height,
  width).  The heads also go out unrotated where a memory path reads them.
"""
import heapq
import math

import torch

own = False

D = 256                  # head dim of the converted model
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _shared(name, common, docs, ways, tails, t=1, page=64, H=24, G=4, dtype="bf16"):
    return {"op": "shared", "name": name, "common": common, "docs": docs, "ways": ways, "tails": tails, "t": t, "page": page, "H": H, "G": G,
            "dtype": dtype}


def _adapter(name, tokens, ids, ranks, d_in=5120, d_out=12288, dtype="bf16"):
    return {"op": "adapter", "name": name, "tokens": tokens, "ids": ids, "ranks": ranks, "d_in": d_in, "d_out": d_out, "dtype": dtype}


def _rope(name, B, t, start, image, memory=True, gated=True, H=24, G=4, sections="11,11,10", dtype="bf16"):
    return {"op": "rope", "name": name, "B": B, "t": t, "start": start, "image": image, "memory": memory, "gated": gated, "H": H, "G": G,
            "sections": sections, "dtype": dtype}


def _text(xs):
    return ",".join(str(x) for x in xs)


def _ints(s):
    return [int(x) for x in s.split(",") if x]


def _spread(n, lo, hi, step=7919):
    """n lengths between lo and hi, evenly over their logarithm, in a mixed order, odd ones among them."""
    xs = [int(lo * (hi / lo) ** (i / max(n - 1, 1))) for i in range(n)]
    return [xs[(i * step) % n] for i in range(n)] if math.gcd(step, n) == 1 else xs


def listed():
    return [
        # one question answered two ways: latency
        _shared("shared_pair", 300, "0", "2", "5,9"),
        # 64 users behind one long instruction, each at its own length
        _shared("shared_instruction", 8000, "0", "64", _text(_spread(64, 1, 1500))),
        # an instruction under eight documents under eight questions each
        _shared("shared_tree", 1500, _text(_spread(8, 2000, 12000, 3)), "8,8,8,8,8,8,8,8", _text(_spread(64, 1, 300))),
        # a long document, sixteen questions about it
        _shared("shared_document", 131072, "0", "16", _text(_spread(16, 20, 500, 7))),
        # three drafted tokens checked at once, small pages, fp16, eight query heads to a KV head
        _shared("shared_drafts", 4001, "0,333", "20,11", _text(_spread(31, 3, 400)), t=3, page=16, H=16, G=2, dtype="fp16"),
        # one user, one adapter on the key projection: latency
        _adapter("adapter_one", "1", "0", "16", d_out=1024),
        # one decode step of 64 requests, each with its own adapter beside the query projection, or none
        _adapter("adapter_step", _text([1] * 64), _text([(i * 37) % 61 - (i % 16 == 5) * 99 for i in range(64)]), _text([16, 8, 32, 16] * 16)),
        # packed prompts: several requests to an adapter, odd lengths
        _adapter("adapter_prompts", "2048,1,777,3000,130,64,513,1659", "0,1,2,0,3,-1,1,4", "16,64,32,8,16"),
        # the output projection of four long prompts, rank 64, fp16
        _adapter("adapter_long", "8192,8191,4097,5000", "1,0,3,2", "64,64,64,64", d_in=6144, d_out=5120, dtype="fp16"),
        # one decode step of 64 conversations, far into them, some behind images
        _rope("rope_step", 64, 1, 120000, "24,32"),
        # a prompt with images among its text
        _rope("rope_prompt", 1, 8191, 0, "32,45"),
        # a batch of long prompts of a kept layer: no memory path, fp16
        _rope("rope_batch", 4, 16384, 1000, "40,40", memory=False, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "adapter", "adapter", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    G = rng.choice([1, 2, 4])
    R = rng.choice([1, 2, 4, 6, 8])
    if op == "shared":
        docs = [rng.choice([0, _log(rng, 1, 12000)]) for _ in range(rng.choice([1, 1, 2, 3, 7]))]
        ways = [_log(rng, 1, 64 // len(docs)) for _ in docs]
        t = rng.choice([1, 1, 1, 2, 3, 5])
        n = sum(ways)
        tails = [t - 1 + _log(rng, 1, 20000 // n) for _ in range(n)]
        return {"op": op, "common": _log(rng, 1, 60000 // n + 3000), "docs": _text(docs), "ways": _text(ways), "tails": _text(tails), "t": t,
                "page": rng.choice([16, 32, 64, 128]), "H": G * R, "G": G, "dtype": dtype}
    if op == "adapter":
        n = _log(rng, 1, 96)
        m = rng.randint(1, max(1, n))
        each = 1 if rng.random() < 0.4 else 16384 // n
        return {"op": op, "tokens": _text([_log(rng, 1, each) for _ in range(n)]), "ids": _text([rng.randint(-1, m - 1) for _ in range(n)]),
                "ranks": _text([rng.choice([4, 8, 16, 32, 64, 128]) if rng.random() < 0.3 else 16 for _ in range(m)]),
                "d_in": rng.choice([512, 1000, 2560, 5120]), "d_out": rng.choice([256, 1024, 5000, 6144]), "dtype": dtype}
    B = _log(rng, 1, 64)
    pairs = rng.choice([8, 16, 32, 64])
    h = rng.randint(0, pairs // 3)
    w = rng.randint(0, pairs // 3)
    return {"op": op, "B": B, "t": 1 if rng.random() < 0.3 else _log(rng, 1, 32768 // B), "start": _log(rng, 1, 250000),
            "image": f"{rng.randint(1, 48)},{rng.randint(1, 48)}", "memory": rng.random() < 0.5, "gated": rng.random() < 0.7, "H": G * R, "G": G,
            "sections": f"{pairs - h - w},{h},{w}", "dtype": dtype}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "shared":
        t, H, G, L = case["t"], case["H"], case["G"], case["page"]
        rows, lens, _ = _tree(case)
        filled = {}
        for r, n in zip(rows, lens):
            for j, p in enumerate(r):
                filled[p] = max(filled.get(p, 0), min(L, n - j * L))
        by = sum(filled.values()) * 2 * G * D + len(filled) * 8 * G + 4 * sum(map(len, rows)) + 4 * len(lens) * t * H * D
        return {"bytes": by, "flops": 4 * H * D * sum(t * n - t * (t - 1) // 2 for n in lens)}
    if op == "adapter":
        tokens, ids, ranks = _ints(case["tokens"]), _ints(case["ids"]), _ints(case["ranks"])
        i, o = case["d_in"], case["d_out"]
        by = 4 * o * sum(tokens) + sum(2 * i * n for n, a in zip(tokens, ids) if a >= 0) + sum(2 * ranks[a] * (i + o) for a in set(ids) if a >= 0)
        return {"bytes": by, "flops": sum(2 * n * ranks[a] * (i + o) for n, a in zip(tokens, ids) if a >= 0)}
    heads = case["B"] * case["t"] * (case["H"] + case["G"])
    return {"bytes": heads * D * 2 * (3 if case["memory"] else 2) + 24 * case["B"] * case["t"], "flops": heads * (4 * D + 6 * sum(_ints(case["sections"])))}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _rand(g, shape, dtype):
    """Normalised heads: components of order one, heads of somewhat different size."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    return x * (0.75 + 0.5 * torch.rand(shape[-2], 1, generator=g, device="cuda")).to(dtype)


def _steps(case):
    """How a server comes to the tree: the calls of its cache, in order, and the number of its slots."""
    docs, ways, tails = _ints(case["docs"]), _ints(case["ways"]), _ints(case["tails"])
    n, nd = len(tails), len(docs)
    root, mid, leaves = [n], list(range(n + 1, n + 1 + nd)), list(range(n))
    src = [m for m, w in zip(mid, ways) for _ in range(w)]
    calls = [("reserve", root, [case["common"]]), ("fork", root * nd, mid), ("free", root), ("reserve", mid, docs), ("fork", src, leaves),
             ("free", mid), ("reserve", leaves, tails)]
    return calls, n + 1 + nd


def _tree(case):
    """The sequences' pages and lengths, with pages given out lowest first: full pages shared by a fork, a partial one copied."""
    L = case["page"]
    calls, slots = _steps(case)
    rows, lens, refs, free, top = [[] for _ in range(slots)], [0] * slots, {}, [], 0

    def take():
        nonlocal top
        p = heapq.heappop(free) if free else top
        top = max(top, p + 1)
        refs[p] = 1
        return p

    for name, a, *b in calls:
        for i, s in enumerate(a):
            if name == "reserve":
                lens[s] += b[0][i]
                while len(rows[s]) * L < lens[s]:
                    rows[s].append(take())
            elif name == "fork":
                d, full = b[0][i], lens[s] // L
                rows[d], lens[d] = rows[s][:full], lens[s]
                for p in rows[d]:
                    refs[p] += 1
                if lens[s] % L:
                    rows[d].append(take())
            else:
                for p in rows[s]:
                    refs[p] -= 1
                    if not refs[p]:
                        heapq.heappush(free, p)
                rows[s], lens[s] = [], 0
    n = len(_ints(case["tails"]))
    return rows[:n], lens[:n], top


def _fill(g, pages, scale):
    """Codes and scales as they come from normalised heads of different sizes."""
    P = pages.shape[1]
    for p in range(0, P, 256):
        part = pages[0, p:p + 256]
        x = torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float32)
        e = torch.randint(-1, 3, part.shape[:2], generator=g, device="cuda")
        part.copy_((x * 64).clamp_(-448, 448).to(torch.float8_e4m3fn))
        scale[0, p:p + 256] = torch.ldexp(torch.ones((), device="cuda"), e - 6)


def _prepare_shared(case, g):
    page, G = case["page"], case["G"]
    rows, lens, top = _tree(case)
    P = top + 3
    width = max(map(len, rows)) + 1
    st = {"lens": lens}
    if own:
        from heimdall_b200 import PagedKV
        calls, slots = _steps(case)
        c = PagedKV(1, P, G, slots, page=page, dim=D, max_len=width * page)
        for name, *args in calls:
            getattr(c, name)(*args)
        st["pool"] = {"k": c.k_pages, "v": c.v_pages, "ks": c.k_scale, "vs": c.v_scale}
        st["c"], st["plan"] = c, c.share(range(len(lens)))
    else:
        code = lambda: torch.zeros(1, P, G, page, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        st["pool"] = {"k": code(), "v": code(), "ks": torch.zeros(1, P, G, device="cuda"), "vs": torch.zeros(1, P, G, device="cuda")}
    table = torch.zeros(len(lens), width, dtype=torch.int64)
    for b, r in enumerate(rows):
        table[b, :len(r)] = torch.tensor(r)
    st["table"], st["host_table"] = table.cuda(), rows
    st["n"] = torch.tensor(lens, device="cuda")
    _fill(g, st["pool"]["k"], st["pool"]["ks"])
    _fill(g, st["pool"]["v"], st["pool"]["vs"])
    st["q"] = _rand(g, (len(lens), case["t"], case["H"], D), _dtype(case))
    return st


def _prepare_adapter(case, g):
    dt, i, o = _dtype(case), case["d_in"], case["d_out"]
    tokens, ids, ranks = _ints(case["tokens"]), _ints(case["ids"]), _ints(case["ranks"])
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    a = [(rand(r, i) * i ** -0.5).to(dt) for r in ranks]
    b = [(rand(o, r) * 0.3 * r ** -0.5).to(dt) for r in ranks]
    s = [2.0 if k % 3 else 0.7 for k in range(len(ranks))]
    per = torch.tensor([max(k, -1) for k in ids], dtype=torch.int32).repeat_interleave(torch.tensor(tokens)).cuda()
    st = {"x": rand(sum(tokens), i).to(dt), "y": rand(sum(tokens), o).to(dt), "ids": per, "ranks": ranks, "a": a, "b": b, "s": s}
    if own:
        from heimdall_b200 import Adapters
        st["adapters"] = Adapters(a, b, s)
    else:
        st["a_all"], st["b_all"] = torch.cat(a), torch.cat([y.t() for y in b])
        st["of"] = torch.arange(len(ranks)).repeat_interleave(torch.tensor(ranks)).cuda()
        st["s_all"] = torch.tensor(s).repeat_interleave(torch.tensor(ranks)).cuda()
    return st


def _axes(sections):
    """The axis of each frequency: dealt in turn, an axis that has all of its own leaves the rest to the first."""
    n, F = len(sections), sum(sections)
    return [f % n if f < n * sections[f % n] else 0 for f in range(F)]


def _prepare_rope(case, g):
    B, t, H, G, dt = case["B"], case["t"], case["H"], case["G"], _dtype(case)
    rows, cols = _ints(case["image"])
    sections = _ints(case["sections"])
    F = sum(sections)
    # 100 tokens of text, then an image, and so on: in text all axes count on together, an image's patches lie on a grid that starts at
    # the next position, and the text behind it goes on after the largest
    each, size = 100 + rows * cols, 100 + max(rows, cols)
    i = torch.arange(t, device="cuda")
    k, j = i // each, i % each
    patch = (j - 100).clamp(min=0)
    text = j < 100
    base = k * size
    p = torch.stack([base + torch.where(text, j, 100), base + torch.where(text, j, 100 + patch // cols), base + torch.where(text, j, 100 + patch % cols)])
    start = torch.randint(max(1, case["start"] // 2), case["start"] + 2, (B,), generator=g, device="cuda")
    pos = p[:, None] + start[None, :, None]
    w = lambda: (torch.randn(D, generator=g, device="cuda") * 0.1)
    return {"qg": _rand(g, (B, t, H, D * (2 if case["gated"] else 1)), dt), "kl": _rand(g, (B, t, G, D), dt), "qw": w(), "kw": w(), "pos": pos,
            "inv_freq": (1e7 ** (-torch.arange(F, device="cuda", dtype=torch.float64) / F)).float(),
            "axes": _axes(sections), "memory": case["memory"], "gated": case["gated"]}


def prepare(case, seed):
    st = {"shared": _prepare_shared, "adapter": _prepare_adapter, "rope": _prepare_rope}[case["op"]](case, _gen(seed))
    st["op"] = case["op"]
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _shared_plain(st):
    q, pool, table, n = st["q"], st["pool"], st["table"], st["n"]
    B, t, H, _ = q.shape
    G, L = pool["k"].shape[2:4]
    there = torch.arange(table.shape[1] * L, device=q.device)
    values = lambda c, s: (c[0][table].float() * s[0][table][..., None, None]).transpose(1, 2).reshape(B, G, -1, D)
    qq = q.float().reshape(B, t, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, -1, D)
    s = torch.matmul(qq, values(pool["k"], pool["ks"]).transpose(2, 3)) * D ** -0.5
    last = (n[:, None] - t + torch.arange(t, device=q.device)).repeat_interleave(H // G, 1)
    s = s.masked_fill((there > last[..., None])[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, values(pool["v"], pool["vs"])) / p.sum(-1, keepdim=True)
    return o.reshape(B, G, t, H // G, D).transpose(1, 2).reshape(B, t, H, D).to(q.dtype)


def _adapter_plain(st):
    x, y = st["x"], st["y"]
    h = torch.matmul(x.float(), st["a_all"].float().t()) * st["s_all"]
    h = torch.where(st["ids"][:, None] == st["of"][None], h, torch.zeros_like(h))
    return (y.float() + torch.matmul(h, st["b_all"].float())).to(y.dtype)


def _norm(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w)


def _rope_plain(st):
    qg, kl, axes = st["qg"], st["kl"], torch.tensor(st["axes"], device="cuda")
    F = len(st["axes"])
    angle = st["pos"][axes].permute(1, 2, 0).double() * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def rotate(x):
        a, b = x[..., :F], x[..., F:2 * F]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * F:]], -1).transpose(1, 2).contiguous()

    q, k = _norm(qg[..., :D], st["qw"]), _norm(kl, st["kw"])
    out = [rotate(q).to(qg.dtype), rotate(k).to(qg.dtype)]
    return out + [q.to(qg.dtype), k.to(qg.dtype)] if st["memory"] else out


def run(state):
    op = state["op"]
    if op == "shared":
        return state["c"].attend(0, state["q"], shared=state["plan"])[0] if own else _shared_plain(state)
    if op == "adapter":
        return state["adapters"].add(state["y"], state["x"], state["ids"]) if own else _adapter_plain(state)
    if own:
        from heimdall_b200 import norm_rope_heads
        q, k, qr, kr = norm_rope_heads(state["qg"], state["kl"], state["qw"], state["kw"], state["pos"], state["inv_freq"], axes=state["axes"],
                                       eps=EPS, gated=state["gated"], memory=state["memory"])
        return [qr, kr, q, k] if state["memory"] else [qr, kr]
    return _rope_plain(state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "shared":
        pool, q, L = st["pool"], st["q"], case["page"]
        B, t, H, _ = q.shape
        R = H // case["G"]
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(st["lens"]):
            pages = torch.tensor(st["host_table"][b], device="cuda")
            for g in range(case["G"]):
                k = (pool["k"][0, pages, g].double() * pool["ks"][0, pages, g].double()[:, None, None]).reshape(-1, D)[:n]
                v = (pool["v"][0, pages, g].double() * pool["vs"][0, pages, g].double()[:, None, None]).reshape(-1, D)[:n]
                for i in range(t):
                    m = n - t + i + 1
                    a = q[b, i, g * R:g * R + R].double() @ k[:m].T / math.sqrt(D)
                    o[b, i, g * R:g * R + R] = torch.softmax(a, -1) @ v[:m]
        return o
    if case["op"] == "adapter":
        out = st["y"].double()
        for i in set(st["ids"].tolist()) - {-1}:
            rows = torch.nonzero(st["ids"] == i)[:, 0]
            out[rows] += st["s"][i] * ((st["x"][rows].double() @ st["a"][i].double().T) @ st["b"][i].double().T)
        return out
    F, f64 = len(st["axes"]), torch.float64
    turned, plain = [], []
    for x, w in ((st["qg"][..., :D], st["qw"]), (st["kl"], st["kw"])):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.double())
        z = x.transpose(1, 2).clone()
        for f, a in enumerate(st["axes"]):
            turn = torch.polar(torch.ones((), dtype=f64, device="cuda"), st["pos"][a].double() * st["inv_freq"][f].double())[:, None]
            c = torch.complex(z[..., f], z[..., f + F]) * turn
            z[..., f], z[..., f + F] = c.real, c.imag
        turned.append(z)
        plain.append(x)
    return turned + plain if case["memory"] else turned
