"""Cases of the paged-cache operators: rotary positions, pages of a KV cache, and attention over a shared prefix.

Kinds of case (``case["op"]``):

* ``rotate``   rotary positions on q and k, forward or backward, out of place
* ``append``   rotary positions (and the model's q/k norm) on new tokens, with k and v written into the pages of a cache
* ``fork``     sequences copied into new slots that share their full pages, then room made for the next token
* ``compact``  finished sequences freed and the pages still in use moved to the front of the pool
* ``attend``   attention of new tokens over paged keys, groups of sequences sharing a prefix

``run`` computes the plain form (elementary torch operations in 32 bits) or, with ``own``, calls the framework.
Pages are (layers, pages, kv heads, rows of a page, head dim); a sequence's row of ``table`` lists its pages, -1 past
the last; ``lens`` counts its tokens, the new ones included; ``refs`` counts the table entries that name each page.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # One decode step of 32 chats: q and k of one layer, ten heads of 128 as in the d20 preset.
        dict(name="rotate step", op="rotate", rows=32, hq=10, hk=10, d=128, rot=128, layout="half", scale="none",
             factor=1.0, dtype="bf16", grad=False, positions=2048),
        # A training micro-batch of the d20 preset: 32 sequences of 2048 tokens.
        dict(name="rotate batch", op="rotate", rows=65536, hq=10, hk=10, d=128, rot=128, layout="half", scale="none",
             factor=1.0, dtype="bf16", grad=False, positions=2048),
        # The gradient for interleaved pairs, half of the head, long-context frequencies, shared kv heads, 32 bits.
        dict(name="rotate gradient", op="rotate", rows=40961, hq=16, hk=4, d=128, rot=64, layout="interleaved",
             scale="parts", factor=4.0, dtype="fp32", grad=True, positions=8192),
        # One decode step of 32 chats: a layer's new k and v into the cache, with the model's q/k norm.
        dict(name="append step", op="append", seqs=32, t=1, hq=10, hk=10, d=128, rot=128, layout="half", scale="none",
             factor=1.0, dtype="bf16", norm=True, page=64, width=32),
        # User turns of ragged lengths prefilled together, small pages, shared kv heads, part of the head.
        dict(name="append turns", op="append", seqs=48, t=300, hq=16, hk=4, d=64, rot=32, layout="interleaved",
             scale="linear", factor=2.0, dtype="fp16", norm=False, page=16, width=96),
        # Seven more samples of one prompt, the d12 preset's cache.
        dict(name="fork 7", op="fork", parents=1, children=7, tokens=1000, layers=12, hk=6, d=128, page=64, width=32,
             dtype="bf16"),
        # A sampling run: four prompts into 63 samples each, the d20 preset's cache.
        dict(name="fork 252", op="fork", parents=4, children=252, tokens=1997, layers=20, hk=10, d=128, page=64,
             width=32, dtype="bf16"),
        # Half of the sequences of a server are done: the d20 preset's cache, 512 pages of 64 tokens.
        dict(name="compact", op="compact", seqs=48, done=24, tokens=640, layers=20, hk=10, d=128, page=64, width=16,
             pages=512, dtype="bf16"),
        # A few chats behind one system prompt: latency counts.
        dict(name="attend chats", op="attend", groups=1, members=4, shared=512, tail=64, t=1, hq=10, hk=10, d=128,
             page=64, width=16, dtype="bf16", idle=False),
        # 64 samples of one prompt of 2000 tokens, ten heads of 128.
        dict(name="attend samples", op="attend", groups=1, members=64, shared=1984, tail=256, t=1, hq=10, hk=10, d=128,
             page=64, width=40, dtype="bf16", idle=True),
        # A long document behind 256 requests, shared kv heads.
        dict(name="attend document", op="attend", groups=1, members=256, shared=32768, tail=1000, t=1, hq=16, hk=4,
             d=128, page=128, width=272, dtype="bf16", idle=False),
        # User turns prefilled behind their system prompts: many new tokens a sequence, small pages and heads.
        dict(name="attend turns", op="attend", groups=3, members=11, shared=1456, tail=400, t=210, hq=12, hk=6, d=64,
             page=16, width=128, dtype="fp16", idle=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "fork", "compact", "attend", "attend"])
    d = rng.choice([64, 128])
    hk = rng.choice([1, 2, 3, 4, 6, 8, 10])
    hq = hk * rng.choice([1, 1, 2, 4])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    scale = rng.choice(["none", "linear", "ntk", "parts"])
    turn = dict(rot=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["half", "interleaved"]), scale=scale,
                factor=1.0 if scale == "none" else rng.choice([2.0, 4.0, 8.0]))
    page = rng.choice([16, 32, 64, 128])
    if op == "rotate":
        return dict(op=op, rows=_log(rng, 1, 40000), hq=hq, hk=hk, d=d, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    grad=rng.random() < 0.5, positions=_log(rng, 64, 65536), **turn)
    if op == "append":
        seqs, t = _log(rng, 1, 256), rng.choice([1, 1, _log(rng, 2, 200)])
        return dict(op=op, seqs=seqs, t=t, hq=hq, hk=hk, d=d, dtype=dtype, norm=rng.random() < 0.5, page=page,
                    width=(t + _log(rng, page, 2000)) // page + 1, **turn)
    if op == "fork":
        tokens = _log(rng, 1, 4000)
        return dict(op=op, parents=rng.randint(1, 5), children=_log(rng, 1, 200), tokens=tokens,
                    layers=_log(rng, 1, 20), hk=hk, d=d, page=page, width=tokens // page + 2, dtype=dtype)
    if op == "compact":
        seqs, tokens = _log(rng, 2, 100), _log(rng, 1, 1000)
        return dict(op=op, seqs=seqs, done=rng.randint(1, seqs), tokens=tokens, layers=_log(rng, 1, 12), hk=hk, d=d,
                    page=page, width=tokens // page + 1, pages=seqs * (tokens // page + 1) + rng.randint(0, 40),
                    dtype=dtype)
    groups, members = rng.choice([1, 1, 2, _log(rng, 2, 40)]), _log(rng, 1, 128)
    t = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 150)])
    shared = rng.choice([0, 1, 1]) * _log(rng, 1, 16384 // (groups if t == 1 else groups * t)) // page * page
    tail = t + _log(rng, 1, 600)
    if groups * members * t > 4096 or groups * members * tail > 100000:
        members = max(1, min(4096 // (groups * t), 100000 // (groups * tail)))
    return dict(op=op, groups=groups, members=members, shared=shared, tail=tail, t=t, hq=hq, hk=hk, d=d, page=page,
                width=(shared + tail) // page + 1, dtype=dtype, idle=t == 1 and rng.random() < 0.3)


# ---- inputs -------------------------------------------------------------------------------------


def _lengths(g, count, most):
    """Lengths of `count` sequences, from half of `most` to `most`."""
    return torch.randint(max(1, most // 2), most + 1, (count,), generator=g, device="cuda", dtype=torch.int32)


def _new_tokens(case, count):
    """New tokens of each sequence, from half of the case's `t` to `t`: ragged, and the same for every seed."""
    t = case["t"]
    return [t - (i * 40503 % 65536) * (t // 2 + 1) // 65536 for i in range(count)]


def _frequencies(case, base, real):
    """Radians a position of each pair, for the case's long-context rule, and the factor on cos and sin."""
    rot, f = case["rot"], case["factor"]
    if case["scale"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    w = base ** (-torch.arange(0, rot, 2, device="cuda", dtype=real) / rot)
    if case["scale"] == "linear":
        return w / f, 1.0
    if case["scale"] == "parts":
        # Pairs that turn often over the original length keep their frequency, those that turn less than once are
        # slowed down by the factor, those between are blended.
        keep = ((2048 * w / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return w * (keep + (1 - keep) / f), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _tables(case, positions):
    if own:
        from rs_nanogpt_b200.ops import rotary
        scaling = None if case["scale"] == "none" else rotary.Scaling(case["scale"], case["factor"], original_len=2048)
        return rotary.tables(case["rot"], positions, base=10000.0, scaling=scaling, device="cuda")
    w, mul = _frequencies(case, 10000.0, torch.float64)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * w
    return (angle.cos() * mul).float(), (angle.sin() * mul).float()


def _rows(counts):
    """(sequence, tokens of it that follow) of each row of sequences that lie one after another."""
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts)
    first = counts.cumsum(0) - counts
    back = (first + counts)[seq] - 1 - torch.arange(len(seq), device="cuda")
    return seq, back


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    s = dict(case=case)
    if case["op"] == "rotate":
        s["cos"], s["sin"] = _tables(case, case["positions"])
        s["q"], s["k"] = randn(case["rows"], case["hq"], case["d"]), randn(case["rows"], case["hk"], case["d"])
        first = torch.randint(0, case["positions"], (1,), generator=g, device="cuda")
        s["pos"] = ((torch.arange(case["rows"], device="cuda") + first) % case["positions"]).int()
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s

    if case["op"] in ("append", "attend"):
        hq, hk, d, page, width = (case[n] for n in ("hq", "hk", "d", "page", "width"))
        b = case["seqs"] if case["op"] == "append" else case["groups"] * case["members"]
        shared = 0 if case["op"] == "append" else case["shared"]
        counts = torch.tensor(_new_tokens(case, b), device="cuda", dtype=torch.int32)
        tail = (width * page if case["op"] == "append" else case["tail"]) - case["t"]
        lens = shared + counts + torch.randint(0, tail + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        # Every group's shared pages, then each sequence's own, anywhere in the pool.
        sp, groups = shared // page, case.get("groups", b)
        pages = groups * sp + b * (width - sp)
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        own_pages = ids[groups * sp:].view(b, width - sp)
        table = torch.cat([ids[:groups * sp].view(groups, sp).repeat_interleave(b // groups, 0), own_pages], 1)
        used = torch.arange(width, device="cuda") * page < lens[:, None]
        s["table"] = torch.where(used, table, -1).int()
        if case.get("idle"):
            lens[5::7] = 0  # slots whose request has ended
        s["lens"], s["counts"], s["scale"] = lens, counts, 1 / math.sqrt(d)
        n = int(counts.sum())
        s["seq"], s["back"] = _rows(counts)
        s["q"] = randn(n, hq, d)
        s["k_pages"], s["v_pages"] = randn(pages, hk, page, d), randn(pages, hk, page, d)
        s["q_out"] = torch.empty_like(s["q"])
        if case["op"] == "append":
            s["k"], s["v"] = randn(n, hk, d), randn(n, hk, d)
            s["cos"], s["sin"] = _tables(case, width * page)
        else:
            # Rows of each sequence side by side, for products over all sequences at once.
            at = torch.arange(case["t"], device="cuda")
            s["pad"] = (counts.cumsum(0) - counts)[:, None] + at.clamp(max=case["t"] - 1)
            s["pad"] = torch.where(at < counts[:, None], s["pad"], 0)
            s["unpad"] = s["seq"] * case["t"] + counts[s["seq"]] - 1 - s["back"]
            s["lse"] = torch.empty(n, hq, device="cuda", dtype=torch.float32)
        if own:
            from rs_nanogpt_b200.ops import paged
            s["plan"] = paged.PrefixPlan([(b // groups, shared)] * groups, counts.tolist(), n_head=hq, n_kv_head=hk,
                                         head_dim=d, page=page, table_width=width, device="cuda")
        return s

    # Page tables of sequences whose pages lie anywhere in the pool.
    page, width = case["page"], case["width"]
    seqs = case["parents"] + case["children"] if case["op"] == "fork" else case["seqs"]
    held = case["parents"] if case["op"] == "fork" else seqs
    pages = case.get("pages", held * width + 2 * case.get("children", 0))
    lens = torch.zeros(seqs, device="cuda", dtype=torch.int32)
    lens[:held] = _lengths(g, held, case["tokens"])
    used = torch.arange(width, device="cuda") * page < lens[:, None]
    table = torch.full((seqs, width), -1, device="cuda", dtype=torch.int32)
    table[used] = torch.randperm(pages, generator=g, device="cuda")[:int(used.sum())].int()
    refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
    refs[table[used].long()] = 1
    order = torch.randperm(seqs, generator=g, device="cuda")  # slots in use and free ones lie mixed
    s["table"], s["lens"], s["refs"] = table[order].contiguous(), lens[order].contiguous(), refs
    s["out"] = tuple(torch.empty_like(s[n]) for n in ("table", "lens", "refs"))
    shape = (case["layers"], pages, case["hk"], page, case["d"])
    s["k_pages"], s["v_pages"] = randn(*shape), randn(*shape)
    slot = torch.argsort(order)
    if case["op"] == "fork":
        s["children"] = slot[held:].int()
        s["parents"] = slot[torch.arange(case["children"], device="cuda") % held].int()
        s["add"] = torch.zeros(seqs, device="cuda", dtype=torch.int32)
        s["add"][slot[held:]] = 1
    else:
        s["done"] = slot[:case["done"]].int()
    return s


# ---- plain forms ----------------------------------------------------------------------------------


def _turned(x, cos, sin, layout, back):
    """x (rows, heads, d) in 32 bits with its first pairs turned: y1 = x1 cos + x2 sin, y2 = x2 cos - x1 sin."""
    half = cos.shape[1]
    c, sn = cos[:, None], (-sin if back else sin)[:, None]
    if layout == "half":
        x1, x2, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([x1 * c + x2 * sn, x2 * c - x1 * sn, rest], -1)
    x1, x2, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    return torch.cat([torch.stack([x1 * c + x2 * sn, x2 * c - x1 * sn], -1).flatten(-2), rest], -1)


def _plain_rotate(s):
    case, at = s["case"], s["pos"].long()
    c, sn = s["cos"][at], s["sin"][at]
    return [_turned(x.float(), c, sn, case["layout"], case["grad"]).to(x.dtype) for x in (s["q"], s["k"])]


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    at = s["lens"][s["seq"]].long() - 1 - s["back"]
    q, k = (_turned(x.float(), s["cos"][at], s["sin"][at], case["layout"], False) for x in (s["q"], s["k"]))
    if case["norm"]:
        q, k = (x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() for x in (q, k))
    where = s["table"][s["seq"], at // page].long()
    s["k_pages"][where, :, at % page] = k.to(s["k"].dtype)
    s["v_pages"][where, :, at % page] = s["v"]
    return {"q": q.to(s["q"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _free_pages_first(refs):
    return torch.argsort((refs > 0).int(), stable=True).int()


def _plain_fork(s):
    page, table, lens, refs = s["case"]["page"], s["table"].clone(), s["lens"].clone(), s["refs"].clone()
    entry = torch.arange(table.shape[1], device="cuda")
    parents, children = s["parents"].long(), s["children"].long()
    rows, n = table[parents], lens[parents]
    full, rest = n // page, n % page
    new = _free_pages_first(refs)[((rest > 0).long().cumsum(0) - 1).clamp(min=0)]
    rows = torch.where(entry < full[:, None], rows, -1)
    rows = torch.where((entry == full[:, None]) & (rest > 0)[:, None], new[:, None], rows)
    last = table[parents, full.clamp(max=table.shape[1] - 1).long()]
    src, dst = (x[rest > 0].long() for x in (last, new))
    copied = torch.arange(page, device="cuda") < rest[rest > 0][:, None]  # filled rows of the parent's last page
    for x in (s["k_pages"], s["v_pages"]):
        x[:, dst] = torch.where(copied[:, None, :, None], x[:, src], x[:, dst])
    table[children], lens[children] = rows, n
    refs.scatter_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).int().flatten())
    # Room for the next tokens: each sequence's missing pages, lowest free page first.
    have, want = (lens + page - 1) // page, (lens + s["add"] + page - 1) // page
    before = (want - have).cumsum(0) - (want - have)
    fresh = (entry >= have[:, None]) & (entry < want[:, None])
    rank = (before[:, None] + entry - have[:, None]).clamp(0, len(refs) - 1)
    table = torch.where(fresh, _free_pages_first(refs)[rank.long()], table)
    refs.scatter_add_(0, table.clamp(min=0).flatten().long(), fresh.int().flatten())
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "table": table, "lens": lens + s["add"], "refs": refs}


def _plain_compact(s):
    table, lens, refs, done = s["table"].clone(), s["lens"].clone(), s["refs"].clone(), s["done"].long()
    rows = table[done]
    refs.scatter_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).int().flatten())
    table[done], lens[done] = -1, 0
    live, at = refs > 0, torch.arange(len(refs), device="cuda")
    src = torch.nonzero(live & (at >= live.sum()))[:, 0]   # in use past the end of what is needed
    dst = torch.nonzero(~live & (at < live.sum()))[:, 0]   # as many holes before it
    for x in (s["k_pages"], s["v_pages"]):
        x[:, dst] = x[:, src]
    to = at.clone()
    to[src] = dst
    refs[dst], refs[src] = refs[src], 0
    table = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "table": table, "lens": lens, "refs": refs}


def _plain_attend(s):
    case = s["case"]
    hq, hk, d, page, t = (case[n] for n in ("hq", "hk", "d", "page", "t"))
    groups, m, b, sp = case["groups"], case["members"], len(s["lens"]), case["shared"] // page
    share = hq // hk

    def by_group(x):  # (sequences, kv heads, query heads of one, t, ..) to (groups, kv heads, all rows, ..)
        return x.reshape(groups, m, hk, share * t, -1 if x.numel() else 0).transpose(1, 2).flatten(2, 3)

    def by_sequence(x):  # and back
        return x.view(groups, hk, m, share * t, x.shape[-1]).transpose(1, 2).reshape(b, hk, share, t, x.shape[-1])

    # Keys and values of the shared pages once a group, of the others a sequence: (.., kv heads, tokens, d).
    first, rest = s["table"].view(groups, m, case["width"])[:, 0, :sp], s["table"][:, sp:]
    kp, vp, ks, vs = (x[pages.clamp(min=0).long()].float().transpose(1, 2).flatten(2, 3)
                      for pages in (first, rest) for x in (s["k_pages"], s["v_pages"]))
    q = s["q"].float()[s["pad"]].view(b, t, hk, share, d).permute(0, 2, 3, 1, 4)
    scores = torch.cat([by_sequence(by_group(q) @ kp.mT),
                        (q.flatten(2, 3) @ ks.mT).view(b, hk, share, t, -1)], -1) * s["scale"]
    # Token i of a sequence's new ones sees the keys up to its own.
    sees = (s["lens"] - s["counts"])[:, None] + 1 + torch.arange(t, device="cuda")
    hidden = torch.arange(scores.shape[-1], device="cuda") >= sees[:, None, None, :, None]
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    o = by_sequence(by_group(p[..., :sp * page]) @ vp)
    o = o + (p[..., sp * page:].flatten(2, 3) @ vs).view(b, hk, share, t, d)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(b * t, hq, d)[s["unpad"]]
    lse = torch.where(total > 0, top + total.log(), -math.inf).permute(0, 3, 1, 2, 4).reshape(b * t, hq)[s["unpad"]]
    return {"out": o.to(s["q"].dtype), "lse": lse}


# ---- the framework's operators ----------------------------------------------------------------------


def _own(s):
    from rs_nanogpt_b200.ops import paged, rotary
    case, op = s["case"], s["case"]["op"]
    if op == "rotate":
        turn = rotary.rotate_bwd if case["grad"] else rotary.rotate
        return list(turn(s["q"], s["k"], s["pos"], s["cos"], s["sin"], case["layout"], s["q_out"], s["k_out"]))
    if op == "append":
        q = paged.append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["plan"],
                         s["cos"], s["sin"], layout=case["layout"], qk_eps=EPS if case["norm"] else None,
                         q_out=s["q_out"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "attend":
        out = paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["plan"], out=s["q_out"],
                              lse=s["lse"], scale=s["scale"])
        return {"out": out, "lse": s["lse"]}
    if op == "fork":
        state = paged.fork_pages(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["refs"], s["parents"],
                                 s["children"], out=s["out"])
        state = paged.grow_pages(*state, s["add"], case["page"], out=s["out"])
    else:
        state = paged.free_pages(s["table"], s["lens"], s["refs"], s["done"], out=s["out"])
        state = paged.compact_pages(s["k_pages"], s["v_pages"], *state, out=s["out"])
    return dict(zip(("table", "lens", "refs"), state), k_pages=s["k_pages"], v_pages=s["v_pages"])


def run(state):
    if own:
        return _own(state)
    return {"rotate": _plain_rotate, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
            "attend": _plain_attend}[state["case"]["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    hk, d = case["hk"], case["d"]
    if case["op"] == "rotate":
        values = case["rows"] * (case["hq"] + hk) * d
        tables = 4 * case["rot"] * min(case["rows"], case["positions"])
        return {"bytes": 2 * size * values + 4 * case["rows"] + tables,
                "flops": 3 * case["rows"] * (case["hq"] + hk) * case["rot"]}
    if case["op"] == "append":
        rows = sum(_new_tokens(case, case["seqs"]))
        tables = 4 * case["rot"] * min(rows, case["width"] * case["page"])
        values = rows * (case["hq"] + hk) * d
        return {"bytes": 2 * size * (values + rows * hk * d) + 12 * rows + tables, "flops": 3 * values}
    if case["op"] == "attend":
        b = case["groups"] * case["members"]
        mean_t = sum(_new_tokens(case, b)) / b
        busy = 6 / 7 if case["idle"] and b > 5 else 1.0
        tail = (case["tail"] - case["t"]) / 2  # of a sequence, before its new tokens
        keys = case["groups"] * case["shared"] + busy * b * (tail + mean_t)
        seen = busy * b * mean_t * (case["shared"] + tail + (mean_t + 1) / 2)
        rows = b * mean_t * case["hq"]
        return {"bytes": size * (2 * keys * hk * d + 2 * rows * d) + 4 * rows, "flops": 4 * seen * case["hq"] * d}
    row = 2 * case["layers"] * hk * d * size  # bytes of one token's k and v over all layers
    meta = 8 * (case["width"] + 1)            # of a slot, read and written
    if case["op"] == "fork":
        rest = sum(n % case["page"] for n in range(max(1, case["tokens"] // 2), case["tokens"] + 1))
        rest /= case["tokens"] + 1 - max(1, case["tokens"] // 2)
        return {"bytes": (case["parents"] + case["children"]) * (rest * row + meta), "flops": 0}
    live = (case["seqs"] - case["done"]) * (0.75 * case["tokens"] / case["page"] + 0.5)
    moved = live * max(0.0, 1 - live / case["pages"])
    return {"bytes": 2 * moved * case["page"] * row + case["seqs"] * meta + 8 * case["pages"], "flops": 0}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------


def _exact_turn(case, x, positions, sign):
    w, mul = _frequencies(case, 10000.0, torch.float64)
    y = x.double().clone()
    angle = positions.double()[:, None, None] * w
    i = torch.arange(case["rot"] // 2, device="cuda")
    one, two = (i, i + case["rot"] // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(y[..., one], y[..., two]) * torch.polar(torch.full_like(angle, mul), -sign * angle)
    y[..., one], y[..., two] = z.real, z.imag
    return y


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # pages are moved and tables counted: no number is computed
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return [_exact_turn(case, x, s["pos"], -1 if case["grad"] else 1) for x in (s["q"], s["k"])]
    if case["op"] == "append":
        at = s["lens"].long()[s["seq"]] - s["back"] - 1
        q, k = _exact_turn(case, s["q"], at, 1), _exact_turn(case, s["k"], at, 1)
        if case["norm"]:
            q, k = (x * math.sqrt(case["d"]) / (x.norm(dim=-1, keepdim=True) ** 2 + case["d"] * EPS).sqrt()
                    for x in (q, k))
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        where = s["table"].gather(1, (torch.arange(case["width"] * case["page"], device="cuda") // case["page"])
                                  .expand(case["seqs"], -1))[s["seq"], at].long()
        kp[where, :, at - at // case["page"] * case["page"]] = k
        vp[where, :, at - at // case["page"] * case["page"]] = s["v"].double()
        return {"q": q, "k_pages": kp, "v_pages": vp}
    # Attention, a sequence at a time.
    out, lse, row = torch.zeros_like(s["q"], dtype=torch.float64), torch.full_like(s["lse"], -math.inf).double(), 0
    share = case["hq"] // case["hk"]
    for i, (n, count) in enumerate(zip(s["lens"].tolist(), s["counts"].tolist())):
        if n > 0:
            pages = s["table"][i, :(n + case["page"] - 1) // case["page"]].long()
            k, v = (x[pages].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (s["k_pages"], s["v_pages"]))
            q = s["q"][row:row + count].double().unflatten(1, (case["hk"], share)).permute(1, 2, 0, 3).flatten(1, 2)
            z = torch.baddbmm(torch.zeros((), device="cuda", dtype=torch.float64), q, k.mT, beta=0, alpha=s["scale"])
            hidden = torch.ones(count, n, device="cuda", dtype=torch.bool).triu(n - count + 1)
            z = z.unflatten(1, (share, count)).masked_fill(hidden, -math.inf)
            o = torch.softmax(z, -1).flatten(1, 2) @ v
            out[row:row + count] = o.unflatten(1, (share, count)).permute(2, 0, 1, 3).flatten(1, 2)
            lse[row:row + count] = torch.logsumexp(z, -1).permute(2, 0, 1).flatten(1)
        row += count
    return {"out": out, "lse": lse}
