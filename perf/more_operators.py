"""The paged-cache operators of the pack, as measured: their cases, inputs, plain forms and exact values.

Operators of a stream whose keys and values live in pages:
  rope    rotary positions of q and k: interleaved or half layout, all or part of the head, one axis or
          several, frequencies scaled for long contexts, forward or its gradient (the inverse rotation)
  append  a chunk's q and k rotated, its k and v written to the pages behind what is cached
  attend  a chunk of new tokens a sequence over everything cached, the new tokens included
  fork    branches dropped, branched anew off their parents (full pages shared, a partly filled
          last page copied), and room made for their next tokens
  compact the pages in use moved to the front of the pool

A cache is k, v [layers, pages, page, heads, dim], a table [sequences, width] of page numbers (-1 for
none), the tokens each sequence holds, and how many sequences hold each page.  Free pages are given
out lowest first, in the order of sequences and of their pages.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of a stream, where latency counts
        {"name": "rope 1x12+12x128", "op": "rope", "T": 1, "Hq": 12, "Hk": 12, "D": 128, "rot": 128,
         "layout": "interleaved", "scaling": "none", "axes": 1, "dtype": "bf16", "inverse": False, "far": 33792},
        # q and k in the fused projection of a 1408x768 chunk, (frame, row, column) positions
        {"name": "rope 3d 8448x12+12x128", "op": "rope", "T": 8448, "Hq": 12, "Hk": 12, "D": 128, "rot": 128,
         "layout": "interleaved", "scaling": "none", "axes": 3, "dtype": "bf16", "inverse": False, "far": 1024},
        # gradients of a ragged batch: shared key heads, half of an odd-sized head, positions far past training
        {"name": "rope inverse 4099x24+4x80", "op": "rope", "T": 4099, "Hq": 24, "Hk": 4, "D": 80, "rot": 40,
         "layout": "half", "scaling": "yarn", "axes": 1, "dtype": "f32", "inverse": True, "far": 1000000},
        # 64 streams, one new token each
        {"name": "append 64x1 12+12x128", "op": "append", "B": 64, "new": 1, "cached": 4096, "Hq": 12, "Hk": 12,
         "D": 128, "page": 64, "rot": 128, "layout": "half", "scaling": "none", "dtype": "bf16"},
        # two streams' chunks of a 1408x768 step, windows of 128 tokens as pages
        {"name": "append 2x8448 12+12x128", "op": "append", "B": 2, "new": 8448, "cached": 8448, "Hq": 12, "Hk": 12,
         "D": 128, "page": 128, "rot": 128, "layout": "interleaved", "scaling": "linear", "dtype": "bf16"},
        # one stream's next token over a short cache: latency
        {"name": "attend 1x1 over 2000 12/12x128", "op": "attend", "B": 1, "new": 1, "cached": 2000, "Hq": 12,
         "Hk": 12, "D": 128, "page": 64, "causal": True, "dtype": "bf16"},
        # many streams of uneven length, one token each, shared key heads: the cache's bytes count
        {"name": "attend 48x1 over 16896 32/8x128", "op": "attend", "B": 48, "new": 1, "cached": 16896, "Hq": 32,
         "Hk": 8, "D": 128, "page": 64, "causal": True, "dtype": "bf16"},
        # uneven prompts behind uneven prefixes, narrow heads, small pages
        {"name": "attend 7x1537 over 1001 16/4x64", "op": "attend", "B": 7, "new": 1537, "cached": 1001, "Hq": 16,
         "Hk": 4, "D": 64, "page": 16, "causal": True, "dtype": "f16"},
        # a 1408x768 step's chunk over three cached chunks, every token seen: the largest
        {"name": "attend 1x8448 over 25344 12/12x128", "op": "attend", "B": 1, "new": 8448, "cached": 25344, "Hq": 12,
         "Hk": 12, "D": 128, "page": 128, "causal": False, "dtype": "bf16"},
        # a small search: three branches of one short stream
        {"name": "fork 3 of 1x1000", "op": "fork", "layers": 2, "B": 1, "n": 3, "tokens": 1000, "new": 1, "page": 16,
         "H": 12, "D": 128, "dtype": "bf16"},
        # two streams at an odd length, eight branches in six blocks
        {"name": "fork 8 of 2x8525", "op": "fork", "layers": 6, "B": 2, "n": 8, "tokens": 8525, "new": 200, "page": 128,
         "H": 12, "D": 128, "dtype": "bf16"},
        # a pool of windows with holes in it, four blocks
        {"name": "compact 100 of 220", "op": "compact", "layers": 4, "pages": 400, "used": 220, "moved": 100,
         "page": 128, "H": 12, "D": 128, "dtype": "bf16"},
    ]


def _between(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, round(v / step) * step))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend", "attend", "fork", "compact"))
    dt = rng.choice(("bf16", "f16"))
    layout = rng.choice(("interleaved", "half"))
    scaling = rng.choice(("none", "linear", "ntk", "yarn"))
    Hk = rng.choice((1, 2, 3, 4, 8, 12))
    group = rng.choice((1, 1, 2, 3, 4, 6, 8)) if Hk <= 8 else 1
    page = rng.choice((16, 32, 48, 64, 128, 256))
    if op == "rope":
        D = _between(rng, 16, 256, 2)
        return {"op": op, "T": _between(rng, 1, 8448), "Hq": Hk * group, "Hk": Hk, "D": D,
                "rot": min(D, 6 + _between(rng, 2, D, 2)), "layout": layout, "scaling": scaling,
                "axes": rng.choice((1, 1, 3)), "dtype": rng.choice(("bf16", "f16", "f32")),
                "inverse": rng.random() < 0.4, "far": _between(rng, 64, 4000000)}
    if op == "append":
        B = _between(rng, 1, 64)
        D = rng.choice((64, 128))
        return {"op": op, "B": B, "new": _between(rng, 1, 8448 // B), "cached": _between(rng, 1, 8448),
                "Hq": Hk * group, "Hk": Hk, "D": D, "page": page, "rot": D // rng.choice((1, 2)), "layout": layout,
                "scaling": scaling, "dtype": dt}
    if op == "attend":
        D = rng.choice((64, 128, 128))
        B = _between(rng, 1, 64)
        new = rng.choice((1, 1, _between(rng, 2, 16), _between(rng, 2, 4096)))
        new = max(1, min(new, 8448 // B))
        cached = _between(rng, 1, min(33792, 400000 // B))
        return {"op": op, "B": B, "new": new, "cached": cached, "Hq": Hk * group, "Hk": Hk, "D": D, "page": page,
                "causal": rng.random() < 0.7, "dtype": dt}
    if op == "fork":
        B = rng.randint(1, 8)
        return {"op": op, "layers": rng.randint(1, 6), "B": B, "n": rng.randint(1, 16), "tokens": _between(rng, 30, 4096),
                "new": _between(rng, 1, 400), "page": page, "H": Hk, "D": rng.choice((64, 128)), "dtype": dt}
    used = _between(rng, 4, 220)
    return {"op": op, "layers": rng.randint(1, 4), "pages": 2 * used + rng.randint(0, 30), "used": used,
            "moved": rng.randint(1, max(1, used // 2)), "page": page, "H": Hk, "D": rng.choice((64, 128)), "dtype": dt}


def _ragged(B, n):
    """B lengths up to n that differ as streams' lengths do, the same for a case each time; one is n."""
    r = random.Random(1000 * B + n)
    return [n] + [max(1, round(n * r.uniform(0.1, 1.0))) for _ in range(B - 1)]


def _lengths(case):
    """New and cached tokens of each sequence."""
    B = case["B"]
    return _ragged(B, case["new"]), _ragged(B, case["cached"])[::-1]


# ------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    e = {"f32": 4}.get(case["dtype"], 2)
    if op == "rope":  # q and k read and written; a position a token
        n = case["T"] * (case["Hq"] + case["Hk"])
        return {"bytes": 2 * e * n * case["D"] + 4 * case["T"] * case["axes"], "flops": 3 * n * case["rot"]}
    if op == "append":  # q, k and v read and written
        n, _ = _lengths(case)
        heads = case["Hq"] + 2 * case["Hk"]
        return {"bytes": 2 * e * sum(n) * heads * case["D"],
                "flops": 3 * sum(n) * (case["Hq"] + case["Hk"]) * case["rot"]}
    if op == "attend":  # q read, out written, each cached key and value read once
        new, cached = _lengths(case)
        pairs = 0
        for n, c in zip(new, cached):
            pairs += n * c + (n * (n + 1) // 2 if case["causal"] else n * n)
        b = 2 * e * sum(new) * case["Hq"] * case["D"] + 2 * e * (sum(new) + sum(cached)) * case["Hk"] * case["D"]
        return {"bytes": b, "flops": 4 * pairs * case["Hq"] * case["D"]}
    row = 2 * e * case["layers"] * case["H"] * case["D"]  # k and v of a token in every layer
    if op == "fork":  # the tokens in the last pages, read and written; a table row a branch
        t, p = case["tokens"], case["page"]
        return {"bytes": case["n"] * (2 * row * (t % p) + 16 * -(-(t + case["new"]) // p)),
                "flops": case["n"] * (t // p + 1)}
    return {"bytes": 2 * row * case["page"] * case["moved"] + 12 * case["pages"], "flops": case["pages"]}


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


THETA, ORIGINAL, FACTOR = 10000.0, 4096, 8.0


def _sections(rot, axes):
    """Rotated channels of each axis: two thirds rounded down to even for rows and columns, the rest for frames."""
    if axes == 1:
        return (rot,)
    third = rot // 6 * 2
    return (rot - 2 * third, third, third)


def _pool(g, dtype, layers, pages, page, H, D):
    k = torch.empty(layers, pages, page, H, D, device="cuda", dtype=dtype)
    v = torch.empty_like(k)
    for t in (k, v):
        for layer in t:
            layer.normal_(generator=g)
    return k, v


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(g, seed, case, lens, spare, width=None):
    """A pool whose pages lie in no order, with sequences of `lens` tokens, and their table."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = width or max(need)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    refs = [0] * pages
    for p in order[:at]:
        refs[p] = 1
    H = case["Hk"] if "Hk" in case else case["H"]
    k, v = _pool(g, DTYPES[case["dtype"]], case.get("layers", 1), pages, page, H, case["D"])
    return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs}


def _finish(s):
    """Table, lengths and reference counts as tensors, and the program's handle on them."""
    for name in ("table", "lens", "refs"):
        s[name] = _i32(s[name])
    if own:
        import flashvsr_sm89_ops_b200 as ops
        s["kv"] = ops.PagedKV(s["k"], s["v"], s["table"], s["lens"], s["refs"])


def _handle(case, axes=1):
    import flashvsr_sm89_ops_b200 as ops
    return ops.Rope(case["rot"], theta=THETA, layout=case["layout"],
                    scaling=None if case["scaling"] == "none" else case["scaling"], factor=FACTOR,
                    original_len=ORIGINAL, axes=None if axes == 1 else _sections(case["rot"], axes))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "rope":
        T, D = case["T"], case["D"]
        qkv = _randn(g, DTYPES[case["dtype"]], T, (case["Hq"] + 2 * case["Hk"]) * D)
        s["q"] = qkv[:, :case["Hq"] * D].unflatten(1, (case["Hq"], D))
        s["k"] = qkv[:, case["Hq"] * D:-case["Hk"] * D].unflatten(1, (case["Hk"], D))
        shape = (T,) if case["axes"] == 1 else (T, case["axes"])
        s["positions"] = torch.randint(0, case["far"], shape, device="cuda", generator=g, dtype=torch.int32)
        if own:
            s["rope"] = _handle(case, case["axes"])
    elif op == "append":
        new, cached = _lengths(case)
        s |= _cache(g, seed, case, [a + b for a, b in zip(new, cached)], 3)
        D = case["D"]
        qkv = _randn(g, DTYPES[case["dtype"]], sum(new), (case["Hq"] + 2 * case["Hk"]) * D)
        q, k, v = qkv.split((case["Hq"] * D, case["Hk"] * D, case["Hk"] * D), 1)
        s["nq"], s["nk"], s["nv"] = q.unflatten(1, (-1, D)), k.unflatten(1, (-1, D)), v.unflatten(1, (-1, D))
        s["cu"] = _i32([sum(new[:i]) for i in range(case["B"] + 1)])
        _finish(s)
        if own:
            s["rope"] = _handle(case)
    elif op == "attend":
        new, cached = _lengths(case)
        s |= _cache(g, seed, case, [a + b for a, b in zip(new, cached)], 3)
        s["q"] = 2 * _randn(g, DTYPES[case["dtype"]], sum(new), case["Hq"], case["D"])
        s["cu"] = _i32([sum(new[:i]) for i in range(case["B"] + 1)])
        _finish(s)
    elif op == "fork":
        # the branches of an earlier fork have their own tokens behind their parents' full pages by now
        B, n, page = case["B"], case["n"], case["page"]
        full, part = divmod(case["tokens"], page)
        width = -(-(case["tokens"] + case["new"]) // page) + 2
        own_pages = width - 1 - full
        s |= _cache(g, seed, case, [case["tokens"]] * B, n * own_pages + 5, width)
        free = [p for p, r in enumerate(s["refs"]) if r == 0]
        random.Random(seed + 1).shuffle(free)
        s["src"] = [i % B for i in range(n)]
        for i in range(n):
            mine = free[i * own_pages:(i + 1) * own_pages - 1]
            row = s["table"][i % B][:full] + mine
            for p in row:
                s["refs"][p] += 1
            s["table"].append(row + [-1] * (width - len(row)))
            s["lens"].append(case["tokens"] + 1)
        for i in range(n):  # a branch's table holds exactly the pages that its tokens need
            row, keep = s["table"][B + i], -(-s["lens"][B + i] // page)
            for j in range(keep, width):
                if row[j] >= 0:
                    s["refs"][row[j]] -= 1
                    row[j] = -1
        s["src"], s["dst"] = _i32(s["src"]), _i32([B + i for i in range(n)])
        s["more"] = _i32([0] * B + [case["new"]] * n)
        _finish(s)
    else:
        pages, used, moved, page = case["pages"], case["used"], case["moved"], case["page"]
        r = random.Random(seed)
        holes = set(r.sample(range(used), moved))
        held = [p for p in range(used) if p not in holes] + r.sample(range(used, pages), moved)
        r.shuffle(held)
        B = min(8, used)
        cuts = [round(i * used / B) for i in range(B + 1)]
        width = max(b - a for a, b in zip(cuts, cuts[1:])) + 1
        s["table"] = [held[a:b] + [-1] * (width - b + a) for a, b in zip(cuts, cuts[1:])]
        s["lens"] = [(b - a) * page - min(i, page - 1) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]
        taken = set(held)
        s["refs"] = [1 if p in taken else 0 for p in range(pages)]
        s["k"], s["v"] = _pool(g, DTYPES[case["dtype"]], case["layers"], pages, page, case["H"], case["D"])
        _finish(s)
        s["table0"], s["refs0"] = s["table"].clone(), s["refs"].clone()
    return s


# ------------------------------------------------------------------------------- plain forms
def _frequencies(case, axes):
    """Angle of one position for each pair of rotated channels (64 bits), the pair's axis, and the factor
    that the scaling puts on the rotated channels."""
    freq, axis = [], []
    for a, d in enumerate(_sections(case["rot"], axes)):
        i = torch.arange(0, d, 2, dtype=torch.float64)
        theta = THETA
        if case["scaling"] == "ntk" and d > 2:
            theta = THETA * FACTOR ** (d / (d - 2))
        f = theta ** (-i / d) if d else i
        if case["scaling"] == "linear":
            f = f / FACTOR
        if case["scaling"] == "yarn" and d:
            # pairs that turn more than 32 times over the original length stay, those below one turn
            # are stretched, a ramp between
            low = max(math.floor(d * math.log(ORIGINAL / (32 * 2 * math.pi)) / (2 * math.log(THETA))), 0)
            high = min(math.ceil(d * math.log(ORIGINAL / (1 * 2 * math.pi)) / (2 * math.log(THETA))), d // 2 - 1)
            ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
            f = f * (1 - ramp) + f / FACTOR * ramp
        freq.append(f)
        axis += [a] * (d // 2)
    scale = 0.1 * math.log(FACTOR) + 1 if case["scaling"] == "yarn" else 1.0
    return torch.cat(freq).cuda(), torch.tensor(axis).cuda(), scale


def _rotated(x, positions, case, axes=1, inverse=False):
    """x [T, H, D] with its first `rot` channels turned by the positions' angles."""
    freq, axis, scale = _frequencies(case, axes)
    p = positions.double()
    angle = (p[:, None] if axes == 1 else p)[:, axis] * freq
    c, s = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    if inverse:
        s = -s
    rot = case["rot"]
    y = x.float().clone()
    if case["layout"] == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        y = torch.cat((a * c - b * s, b * c + a * s, y[..., rot:]), -1)
    else:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2] = a * c - b * s
        y[..., 1:rot:2] = b * c + a * s
    return y.to(x.dtype)


def _places(s):
    """Sequence, position in it and slot of the pool of each new token."""
    cu, lens, page = s["cu"].long(), s["lens"].long(), s["case"]["page"]
    t = torch.arange(s["nq"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[seq] - (cu[seq + 1] - cu[seq]) + t - cu[seq]
    return pos, s["table"].long()[seq, pos // page] * page + pos % page


def _plain_append(s):
    pos, slot = _places(s)
    for pool, x in ((s["k"], _rotated(s["nk"], pos, s["case"])), (s["v"], s["nv"])):
        pool[0].view(-1, *pool.shape[3:])[slot] = x
    return _rotated(s["nq"], pos, s["case"]), s["k"], s["v"]


def _plain_attend(s):
    case = s["case"]
    new, cached = _lengths(case)
    page, Hq, Hk, D = case["page"], case["Hq"], case["Hk"], case["D"]
    g = Hq // Hk
    out = torch.empty_like(s["q"])
    at = 0
    for b, (n, c) in enumerate(zip(new, cached)):
        L = n + c
        pages = s["table"][b, :-(-L // page)].long()
        k = s["k"][0][pages].view(-1, Hk, D)[:L].float().permute(1, 2, 0)
        v = s["v"][0][pages].view(-1, Hk, D)[:L].float().transpose(0, 1)
        q = s["q"][at:at + n].float().view(n, Hk, g, D).permute(1, 2, 0, 3)
        seen = None
        if case["causal"] and n > 1:
            seen = torch.arange(L, device="cuda") <= torch.arange(c, L, device="cuda")[:, None]
        step = max(1, 2 ** 30 // (g * n * L))
        for h in range(0, Hk, step):
            x = torch.matmul(q[h:h + step], k[h:h + step, None]) / math.sqrt(D)
            if seen is not None:
                x = x.masked_fill(~seen, float("-inf"))
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(x, v[h:h + step, None]) / x.sum(-1, keepdim=True)
            out.view(-1, Hk, g, D)[at:at + n, h:h + step] = o.permute(2, 0, 1, 3).to(out.dtype)
        at += n
    return out


def _free_pages(refs, n):
    """The n lowest free pages."""
    return torch.argsort((refs > 0).int(), stable=True)[:n]


def _plain_fork(s):
    case = s["case"]
    page, n = case["page"], case["n"]
    table, lens, refs, src, dst = s["table"], s["lens"], s["refs"], s["src"].long(), s["dst"].long()
    W = table.shape[1]
    # drop the branches
    gone = table[dst]
    refs.index_add_(0, gone.clamp(min=0).view(-1).long(), -(gone >= 0).int().view(-1))
    table[dst] = -1
    lens[dst] = 0
    # branch anew: full pages shared, a partly filled one copied
    full, part = lens[src] // page, lens[src] % page
    j = torch.arange(W, device="cuda")
    rows = torch.where(j < full[:, None], table[src], -1)
    refs.index_add_(0, rows.clamp(min=0).view(-1).long(), (rows >= 0).int().view(-1))
    if case["tokens"] % page:
        fresh = _free_pages(refs, n)
        was = table[src].gather(1, full[:, None].long())[:, 0].long()
        rows.scatter_(1, full[:, None].long(), fresh[:, None].int())
        refs[fresh] = 1
        t = case["tokens"] % page
        for pool in (s["k"], s["v"]):
            pool[:, fresh, :t] = pool[:, was, :t]
    table[dst] = rows
    lens[dst] = lens[src]
    # room for the next tokens
    have, want = (lens + page - 1) // page, (lens + s["more"] + page - 1) // page
    new = (j >= have[:, None]) & (j < want[:, None])
    rank = torch.cumsum(new.view(-1), 0) - 1
    fresh = _free_pages(refs, min(refs.numel(), table.numel()))
    place = fresh[rank.clamp(0, fresh.numel() - 1)].view_as(new)
    table.copy_(torch.where(new, place, table))
    refs.index_add_(0, place.view(-1), new.int().view(-1))
    lens += s["more"]
    return table, lens, refs, s["k"], s["v"]


def _plain_compact(s):
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    table, refs = s["table"], s["refs"]
    held = refs > 0
    used = held.sum()
    p = torch.arange(refs.numel(), device="cuda")
    holes, movers = p[~held & (p < used)], p[held & (p >= used)]
    to = p.clone()
    to[movers] = holes
    for pool in (s["k"], s["v"]):
        pool[:, holes] = pool[:, movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    return table, s["lens"], refs, s["k"], s["v"]


def _plain(s):
    op = s["case"]["op"]
    if op == "rope":
        return tuple(_rotated(s[n], s["positions"], s["case"], s["case"]["axes"], s["case"]["inverse"])
                     for n in ("q", "k"))
    return {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact}[op](s)


# ------------------------------------------------------------------------------- the calls
def _calls(s):
    import flashvsr_sm89_ops_b200 as ops
    case = s["case"]
    op = case["op"]
    if op == "rope":
        return ops.fused_rope(s["q"], s["k"], s["positions"], s["rope"], inverse=case["inverse"])
    kv = s["kv"]
    if op == "append":
        return kv.append(0, s["nk"], s["nv"], s["cu"], q=s["nq"], rope=s["rope"]), kv.k, kv.v
    if op == "attend":
        return kv.attend(0, s["q"], s["cu"], causal=case["causal"], max_new=case["new"])
    if op == "fork":
        kv.release(s["dst"])
        kv.fork(s["src"], s["dst"])
        kv.reserve(s["more"])
    else:
        kv.table.copy_(s["table0"])
        kv.refs.copy_(s["refs0"])
        kv.compact()
    return kv.table, kv.lens, kv.refs, kv.k, kv.v


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------- exact values
def _turned_64(x, positions, case, axes=1, sign=1.0):
    """The rotation as a product of complex numbers in 64 bits."""
    T, H, D = x.shape
    x = x.double()
    rot, at, out = case["rot"], 0, []
    positions = positions.double().reshape(T, -1)
    half = case["layout"] == "half"
    z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) if half else \
        torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous())
    scale = 1 + 0.1 * math.log(FACTOR) if case["scaling"] == "yarn" else 1.0
    for a, d in enumerate(_sections(rot, axes)):
        turns = []
        for i in range(d // 2):
            base = THETA * (FACTOR ** (d / (d - 2)) if case["scaling"] == "ntk" and d > 2 else 1)
            w = math.exp(-2 * i / d * math.log(base))
            if case["scaling"] == "linear":
                w /= FACTOR
            if case["scaling"] == "yarn":
                at_turns = lambda n: d * math.log(ORIGINAL / (n * 2 * math.pi)) / (2 * math.log(THETA))
                lo, hi = max(math.floor(at_turns(32)), 0), min(math.ceil(at_turns(1)), d // 2 - 1)
                m = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
                w = w * (1 - m) + w / FACTOR * m
            turns.append(w)
        angle = sign * positions[:, a:a + 1] * torch.tensor(turns, dtype=torch.float64, device=x.device)
        out.append(z[..., at:at + d // 2] * torch.polar(torch.full_like(angle, scale), angle)[:, None])
        at += d // 2
    z = torch.cat(out, -1)
    flat = torch.cat((z.real, z.imag), -1) if half else torch.view_as_real(z).flatten(-2)
    return torch.cat((flat, x[..., rot:]), -1)


def _attend_64(s):
    case = s["case"]
    new, cached = _lengths(case)
    page, D, g = case["page"], case["D"], case["Hq"] // case["Hk"]
    out, at = [], 0
    for b, (n, c) in enumerate(zip(new, cached)):
        pos = torch.arange(n + c, device="cuda")
        slot = s["table"].long()[b, pos // page] * page + pos % page
        k, v = (p[0].flatten(0, 1)[slot] for p in (s["k"], s["v"]))
        heads = []
        for h in range(case["Hq"]):
            kd, vd = k[:, h // g].double(), v[:, h // g].double()
            rows = []
            for i in range(0, n, 2048):
                x = torch.mm(s["q"][at + i:min(at + i + 2048, at + n), h].double(), kd.T).mul_(D ** -0.5)
                if case["causal"]:
                    last = c + i + torch.arange(x.shape[0], device="cuda")[:, None]
                    x[pos[None] > last] = -math.inf
                x -= torch.logsumexp(x, 1, keepdim=True)
                rows.append(torch.mm(x.exp_(), vd))
            heads.append(torch.cat(rows))
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)


def _fork_by_hand(s):
    """The tables in plain Python, one page at a time."""
    page = s["case"]["page"]
    table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
    src, dst, more = s["src"].tolist(), s["dst"].tolist(), s["more"].tolist()
    for d in dst:
        for p in table[d]:
            if p >= 0:
                refs[p] -= 1
        table[d], lens[d] = [-1] * len(table[d]), 0
    copies = []
    for a, d in zip(src, dst):
        for j in range(lens[a] // page):
            table[d][j] = table[a][j]
            refs[table[a][j]] += 1
        lens[d] = lens[a]
    for a, d in zip(src, dst):
        if lens[a] % page:
            p = refs.index(0)
            refs[p] = 1
            table[d][lens[a] // page] = p
            copies.append((table[a][lens[a] // page], p, lens[a] % page))
    for b, n in enumerate(more):
        for j in range(-(-lens[b] // page), -(-(lens[b] + n) // page)):
            p = refs.index(0)
            refs[p] = 1
            table[b][j] = p
        lens[b] += n
    k, v = s["k"].clone(), s["v"].clone()
    for a, d, n in copies:
        k[:, d, :n].copy_(s["k"][:, a, :n])
        v[:, d, :n].copy_(s["v"][:, a, :n])
    return _i32(table), _i32(lens), _i32(refs), k, v


def _compact_by_hand(s):
    refs, table = s["refs0"].tolist(), s["table0"].tolist()
    used = sum(r > 0 for r in refs)
    k, v, to = s["k"].clone(), s["v"].clone(), {}
    hole = 0
    for p in range(used, len(refs)):
        if refs[p]:
            while refs[hole]:
                hole += 1
            to[p] = hole
            k[:, hole].copy_(s["k"][:, p])
            v[:, hole].copy_(s["v"][:, p])
            refs[hole], refs[p] = refs[p], 0
    return _i32([[to.get(p, p) for p in row] for row in table]), s["lens"], _i32(refs), k, v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        sign = -1.0 if case["inverse"] else 1.0
        return tuple(_turned_64(s[n], s["positions"], case, case["axes"], sign) for n in ("q", "k"))
    if op == "append":
        new, cached = _lengths(case)
        pos = torch.cat([torch.arange(c, c + n, device="cuda") for n, c in zip(new, cached)])
        k, v = s["k"].double(), s["v"].double()
        turned, t = _turned_64(s["nk"], pos, case), 0
        rows, at = s["table"].tolist(), pos.tolist()
        slots = []
        for b, n in enumerate(new):
            for i in range(n):
                slots.append(rows[b][at[t] // case["page"]] * case["page"] + at[t] % case["page"])
                t += 1
        slots = torch.tensor(slots, device="cuda")
        k[0].flatten(0, 1).index_copy_(0, slots, turned)
        v[0].flatten(0, 1).index_copy_(0, slots, s["nv"].double())
        return _turned_64(s["nq"], pos, case), k, v
    if op == "attend":
        return _attend_64(s)
    return _fork_by_hand(s) if op == "fork" else _compact_by_hand(s)
