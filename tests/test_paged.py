"""Paged cache operators: page bookkeeping against a model in Python lists, the append
and the attention against their definitions in 64 bits."""
import math
import random

import pytest
import torch

gpu = pytest.mark.gpu
checked = pytest.mark.usefixtures("kernel_ok")
DEV = "cuda"


# ---- page bookkeeping --------------------------------------------------------------------


class Model:
    """The rules of the page operators in plain Python; a page's content is a list of row tags."""

    def __init__(self, pages, page, width, slots):
        self.page, self.width = page, width
        self.refs = [0] * pages
        self.rows = [[0] * page for _ in range(pages)]
        self.table = [[] for _ in range(slots)]
        self.lens = [0] * slots

    def lowest(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        return free[:n] if len(free) >= n else None

    def grow(self, add):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        used = 0
        for s, a in enumerate(add):
            if a < 0 or self.lens[s] + a > self.width * self.page:
                continue
            need = -(-(self.lens[s] + a) // self.page) - len(self.table[s])
            if used + need <= len(free):
                for p in free[used:used + need]:
                    self.table[s].append(p)
                    self.refs[p] = 1
                self.lens[s] += a
            used += need

    def fork(self, parents, children):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        rank, made = 0, []
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < len(self.lens) and 0 <= c < len(self.lens)) or self.lens[c] or c in children[:i]:
                continue
            part = self.lens[p] % self.page
            new = None
            if part:
                rank += 1
                if rank > len(free):
                    continue
                new = free[rank - 1]
            made.append((p, c, part, new))
        before = {p: (list(self.table[p]), self.lens[p]) for p, *_ in made}
        for p, c, part, new in made:
            table, n = before[p]
            self.table[c] = table[:n // self.page]
            for q in self.table[c]:
                self.refs[q] += 1
            if part:
                self.rows[new][:part] = self.rows[table[-1]][:part]
                self.table[c].append(new)
                self.refs[new] = 1
            self.lens[c] = n

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lens):
                for q in self.table[s]:
                    self.refs[q] -= 1
                self.table[s], self.lens[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.rows[b] = list(self.rows[a])
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(q, q) for q in t] for t in self.table]


def _state(m):
    table = torch.full((len(m.lens), m.width), -1, dtype=torch.int32)
    for s, t in enumerate(m.table):
        table[s, :len(t)] = torch.tensor(t, dtype=torch.int32)
    return table, torch.tensor(m.lens, dtype=torch.int32), torch.tensor(m.refs, dtype=torch.int32)


def _pools(m, layers, heads, d, dtype, pad=0):
    """Pools whose rows carry the model's tags: value = tag + layer / 4, head in the second element."""
    p, r = len(m.refs), m.page
    tags = torch.tensor(m.rows, dtype=torch.float32)
    x = torch.zeros(layers, p + pad, heads, r, d)
    x[:, :p] = tags[None, :, None, :, None] + torch.arange(layers)[:, None, None, None, None] * 0.25
    x[..., 1] = torch.arange(heads)[None, None, :, None]
    return x.to(dtype).to(DEV)[:, :p]


def _check_state(m, got):
    for want, have, name in zip(_state(m), got, ("table", "lens", "refs")):
        assert torch.equal(want, have.cpu()), name


def _check_pools(m, k, v, layers, heads, d, dtype):
    want = _pools(m, layers, heads, d, dtype)
    assert torch.equal(k, want) and torch.equal(v, want)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@gpu
@checked
@pytest.mark.parametrize("seed,pages,page,width,slots,layers,heads,d,dtype,in_place", [
    (0, 40, 8, 6, 9, 2, 3, 64, torch.bfloat16, True), (1, 300, 16, 12, 40, 1, 1, 128, torch.float16, False),
    (2, 20000, 32, 4, 700, 1, 1, 16, torch.float32, True), (3, 64, 1, 20, 12, 2, 2, 8, torch.bfloat16, False),
    (4, 33, 7, 9, 6, 3, 2, 24, torch.float16, True)])
def test_random_histories(seed, pages, page, width, slots, layers, heads, d, dtype, in_place):
    from rs_nanogpt_b200.ops import paged
    rng = random.Random(seed)
    m = Model(pages, page, width, slots)
    for q in range(pages):
        m.rows[q] = [rng.randint(1, 100) for _ in range(page)]
    k, v = (_pools(m, layers, heads, d, dtype, pad=2) for _ in range(2))  # layers at a stride of their own
    state = tuple(t.to(DEV) for t in _state(m))
    for step in range(30):
        op = rng.choice(["grow", "grow", "fork", "fork", "free", "compact"])
        out = state if in_place else None
        if op == "grow":
            add = [rng.choice([0, 0, 1, 1, rng.randint(0, page * 2)]) if m.lens[s] or rng.random() < 0.3 else 0
                   for s in range(slots)]
            add = [min(a, width * page - m.lens[s]) for s, a in enumerate(add)]
            trial = [sum(-(-(m.lens[s] + a) // page) - len(m.table[s]) for s, a in enumerate(add))]
            if trial[0] > sum(r == 0 for r in m.refs):
                continue
            m.grow(add)
            state = paged.grow_pages(*state, _i32(add), page, out=out)
        elif op == "fork":
            empty = [s for s in range(slots) if m.lens[s] == 0]
            held = [s for s in range(slots) if m.lens[s]]
            if not empty or not held:
                continue
            children = rng.sample(empty, rng.randint(1, min(len(empty), sum(r == 0 for r in m.refs)) or 1))
            if len(children) > sum(r == 0 for r in m.refs):
                continue
            parents = [rng.choice(held) for _ in children]
            m.fork(parents, children)
            state = paged.fork_pages(k, v, *state, _i32(parents), _i32(children), out=out)
        elif op == "free":
            seqs = rng.sample(range(slots), rng.randint(0, slots // 2))
            m.free(seqs)
            state = paged.free_pages(*state, _i32(seqs), out=out)
        else:
            m.compact()
            state = paged.compact_pages(k, v, *state, out=out)
        _check_state(m, state)
    _check_pools(m, k, v, layers, heads, d, dtype)


@gpu
def test_what_cannot_be_done_is_skipped_and_reported():
    from rs_nanogpt_b200.ops import paged
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    m = Model(6, 4, 3, 6)
    m.grow([5, 4, 0, 0, 0, 0])
    k, v = (_pools(m, 1, 1, 8, torch.float32) for _ in range(2))
    state = tuple(t.to(DEV) for t in _state(m))
    # Pages run out in the middle of a list: the first two children have theirs.
    m.grow([0, 4, 0, 0, 0, 0])
    state = paged.grow_pages(*state, _i32([0, 4, 0, 0, 0, 0]), 4)
    assert kernel_status(True) == 0
    parents, children = [0, 0, 0, 1], [2, 3, 4, 5]
    m.fork(parents, children)
    state = paged.fork_pages(k, v, *state, _i32(parents), _i32(children))
    assert kernel_status(True) == 6 and m.lens == [5, 8, 5, 5, 0, 8]
    _check_state(m, state)
    # A slot that lacks a page keeps its length, one that has room grows.
    m.grow([3, 1, 0, 0, 0, 0])
    state = paged.grow_pages(*state, _i32([3, 1, 0, 0, 0, 0]), 4)
    assert kernel_status(True) == 6 and m.lens[:2] == [8, 8]
    _check_state(m, state)
    for call in (lambda: paged.fork_pages(k, v, *state, _i32([0, 0, 7, 0]), _i32([1, 9, 4, -1])),
                 lambda: paged.grow_pages(*state, _i32([0, 0, -1, 0, 0, 0]), 4),
                 lambda: paged.grow_pages(*state, _i32([5, 0, 0, 0, 0, 0]), 4),   # past the table's width
                 lambda: paged.free_pages(*state, _i32([6]))):
        after = call()
        assert kernel_status(True) == 5
        _check_state(m, after)
    m.free([1, 1, 5])  # named twice: freed once
    state = paged.free_pages(*state, _i32([1, 1, 5]))
    _check_state(m, state)
    m.fork([2, 3], [4, 4])  # named twice: the first mention counts
    state = paged.fork_pages(k, v, *state, _i32([2, 3]), _i32([4, 4]))
    _check_state(m, state)
    assert kernel_status(True) == 5
    paged.copy_pages(k, v, _i32([0, 6]), _i32([1, 2]))
    assert kernel_status(True) == 5


@gpu
@checked
def test_empty_calls_and_page_copies():
    from rs_nanogpt_b200.ops import paged
    k = torch.randn(2, 7, 3, 4, 16, device=DEV)
    v = torch.randn_like(k)
    k0, v0 = k.clone(), v.clone()
    paged.copy_pages(k, v, _i32([5, -1, 0]), _i32([1, 2, 6]))
    k0[:, 1], k0[:, 6], v0[:, 1], v0[:, 6] = k0[:, 5], k0[:, 0], v0[:, 5], v0[:, 0]
    assert torch.equal(k, k0) and torch.equal(v, v0)
    none = _i32([])
    paged.copy_pages(k, v, none, none)
    m = Model(7, 4, 3, 2)
    state = tuple(t.to(DEV) for t in _state(m))
    state = paged.fork_pages(k, v, *state, none, none)
    state = paged.free_pages(*state, none)
    state = paged.compact_pages(k, v, *state)
    _check_state(m, state)
    assert torch.equal(k, k0)


@gpu
def test_page_refusals():
    from rs_nanogpt_b200.ops import paged
    k = torch.zeros(1, 6, 2, 4, 8, device=DEV)
    m = Model(6, 4, 3, 4)
    table, lens, refs = (t.to(DEV) for t in _state(m))
    one = _i32([0])
    for call in (lambda: paged.fork_pages(k, k, table.long(), lens, refs, one, one),
                 lambda: paged.fork_pages(k, k, table, lens[:2], refs, one, one),
                 lambda: paged.fork_pages(k, k, table, lens, refs[:5], one, one),
                 lambda: paged.fork_pages(k, k, table, lens, refs, one, _i32([1, 2])),
                 lambda: paged.fork_pages(k, k[:, :5], table, lens, refs, one, one),
                 lambda: paged.fork_pages(k[..., :6], k[..., :6], table, lens, refs, one, one),
                 lambda: paged.fork_pages(k.transpose(2, 3), k.transpose(2, 3), table, lens, refs, one, one),
                 lambda: paged.grow_pages(table, lens, refs, one, 4),
                 lambda: paged.grow_pages(table, lens, refs, torch.zeros_like(lens), 4,
                                          out=(table, torch.empty_like(lens), refs)),
                 lambda: paged.free_pages(table, lens, refs, one.cpu()),
                 lambda: paged.compact_pages(k.cpu(), k.cpu(), table, lens, refs),
                 lambda: paged.copy_pages(k, k, one, _i32([1, 2]))):
        with pytest.raises(RuntimeError):
            call()


# ---- append and attention -------------------------------------------------------------------


class Batch:
    """Sequences in groups with shared prefixes over pages in random order; rows of pages that hold
    no token are NaN."""

    def __init__(self, groups, tails, q_lens, hq, hk, d, page, dtype, seed=0, spare=3, empty=(), slots=None, fill=True):
        from rs_nanogpt_b200.ops import paged
        g = torch.Generator().manual_seed(seed)
        n = sum(c for c, _ in groups)
        shared = [s for c, s in groups for _ in range(c)]
        self.lens = [s + t for s, t in zip(shared, tails)]
        for e in empty:
            self.lens[e] = 0
        self.q_lens = [q_lens] * n if isinstance(q_lens, int) else list(q_lens)
        width = max(-(-(s + t) // page) for s, t in zip(shared, tails)) + 2
        total = sum(s // page for _, s in groups) + sum(-(-t // page) for t in tails) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.table = torch.full((n, width), -1, dtype=torch.int32)
        i = 0
        for c, s in groups:
            pre = [order.pop() for _ in range(s // page)]
            for _ in range(c):
                ids = pre + [order.pop() for _ in range(-(-tails[i] // page))]
                if i not in empty:
                    self.table[i, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                i += 1
        self.k = torch.full((total, hk, page, d), float("nan"), dtype=dtype)
        self.v = self.k.clone()
        if fill:
            for s in range(n):
                for p in range(0, self.lens[s], page):
                    r = min(page, self.lens[s] - p)
                    q = int(self.table[s, p // page])
                    for x in (self.k, self.v):
                        x[q, :, :r] = torch.randn(hk, r, d, generator=g).to(dtype)
        self.page, self.d, self.hq, self.hk, self.n = page, d, hq, hk, n
        self.slots = list(range(n)) if slots is None else slots
        rows = max(self.slots) + 1
        table, lens = torch.full((rows, width), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
        table[self.slots], lens[self.slots] = self.table, torch.tensor(self.lens, dtype=torch.int32)
        self.dev_table, self.dev_lens = table.to(DEV), lens.to(DEV)
        self.q = torch.randn(sum(self.q_lens), hq, d, generator=g).to(dtype)
        self.plan = paged.PrefixPlan(groups, self.q_lens, n_head=hq, n_kv_head=hk, head_dim=d, page=page,
                                     table_width=width, slots=slots, device=DEV)

    def reference(self, scale):
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64)
        row = 0
        for s in range(self.n):
            n, t = self.lens[s], self.q_lens[s]
            ids = self.table[s, :-(-n // self.page)].long()
            k, v = (x[ids].transpose(0, 1).reshape(self.hk, -1, self.d)[:, :n].double() for x in (self.k, self.v))
            for i in range(t):
                see = n - t + 1 + i
                if see > 0:
                    for h in range(self.hq):
                        z = k[h * self.hk // self.hq, :see] @ self.q[row + i, h].double() * scale
                        lse[row + i, h] = torch.logsumexp(z, 0)
                        out[row + i, h] = torch.softmax(z, 0) @ v[h * self.hk // self.hq, :see]
            row += t
        return out, lse

    def run(self, scale=None, **kw):
        from rs_nanogpt_b200.ops import paged
        return paged.attention(self.q.to(DEV), self.k.to(DEV), self.v.to(DEV), self.dev_table, self.dev_lens, self.plan,
                               scale=scale, **kw)


def _check_attention(b, out, lse, scale):
    """Rounding P to the values' type moves the output by at most half a unit of max |v|, rounding the
    output by half a unit of it again; scores of |q| |k| up to ~20 in fp32 are off by less than
    head_dim 2^-24 |q| |k| scale < 2e-4, and move output and LSE by as much (twice for the output)."""
    ref, ref_lse = b.reference(scale)
    unit = 2.0 ** -8 if b.q.dtype == torch.bfloat16 else 2.0 ** -11
    vmax = b.v[torch.isfinite(b.v)].abs().max().item() if torch.isfinite(b.v).any() else 1.0
    err = (out.cpu().double() - ref).abs().max().item()
    assert err <= (2 * unit + 4e-4) * vmax, err
    seen = torch.isfinite(ref_lse)
    got = lse.cpu().double()
    assert torch.equal(torch.isfinite(got), seen)
    assert not seen.any() or (got - ref_lse)[seen].abs().max().item() <= 2e-4


CASES = {
    # groups (sequences, shared tokens), tails, new tokens, hq, hk, d, page
    "one token": ([(1, 0)], [1], 1, 1, 1, 128, 64),
    "plain paged": ([(1, 0)] * 5, [1, 63, 64, 65, 500], 1, 3, 3, 128, 64),
    "samples": ([(9, 192)], [1, 5, 64, 65, 30, 1, 200, 128, 63], 1, 4, 4, 128, 64),
    "one key past a tile": ([(3, 64)], [1, 1, 1], 1, 2, 1, 64, 16),
    "ragged groups": ([(1, 32), (4, 96), (2, 0), (5, 16)], [7, 1, 33, 15, 16, 17, 90, 2, 3, 200, 1, 31], 1, 6, 3, 64,
                      16),
    "many heads of one": ([(6, 128)], [9, 40, 3, 77, 1, 64], 1, 24, 2, 128, 32),
    "small pages": ([(3, 40)], [1, 9, 70], 1, 4, 2, 64, 8),
    "large pages": ([(20, 512)], list(range(1, 21)), 1, 2, 2, 128, 256),
    "many sequences": ([(150, 64)], [1 + 7 * i % 90 for i in range(150)], 1, 2, 1, 64, 32),
    "two tokens": ([(4, 64)], [2, 10, 64, 66], 2, 4, 2, 128, 64),
    "turns": ([(3, 128), (2, 64)], [50, 100, 65, 64, 129], [50, 97, 64, 1, 30], 4, 2, 64, 64),
    "a turn alone": ([(1, 0)], [300], [300], 2, 1, 128, 128),
    "long shares": ([(1, 0), (3, 20480)], [15000, 40, 7, 130], 1, 4, 2, 64, 64),
    "long shares of many rows": ([(2, 10240)], [70, 40], [33, 40], 10, 5, 64, 128),
    "many rows of one prefix": ([(30, 256)], [1 + 11 * i % 140 for i in range(30)], 1, 8, 1, 128, 64),
    "many rows, small heads and pages": ([(4, 40), (2, 1000)], [90, 200, 33, 129, 31, 64], [90, 150, 33, 128, 5, 64],
                                         6, 2, 64, 8),
    "a part of a tile": ([(1, 0), (1, 0)], [130, 257], [130, 129], 3, 1, 128, 256),
    "no new tokens for one": ([(3, 32)], [5, 20, 9], [1, 0, 2], 2, 2, 64, 32),
}


@gpu
@checked
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CASES)
def test_attention(name, dtype):
    b = Batch(*CASES[name], dtype)
    lse = torch.empty(b.q.shape[:2], device=DEV)
    scale = 1 / math.sqrt(b.d)
    _check_attention(b, b.run(lse=lse), lse, scale)


@gpu
@checked
def test_empty_slots_rows_without_keys_and_slot_order():
    groups, tails = [(4, 64), (3, 0), (2, 32)], [5, 6, 70, 8, 3, 1, 200, 2, 2]
    for empty in ((0,), (0, 1, 2, 3), (2, 4, 8), tuple(range(9))):
        b = Batch(groups, tails, 1, 4, 2, 64, 32, torch.bfloat16, empty=empty, slots=[3, 0, 11, 7, 2, 1, 9, 8, 4])
        lse = torch.empty(9, 4, device=DEV)
        out = b.run(lse=lse)
        _check_attention(b, out, lse, 1 / 8)
        assert all(out[e].abs().max() == 0 for e in empty)


@gpu
@checked
def test_sequences_shorter_than_the_prefix():
    """A member that holds fewer tokens than its group shares sees only its own."""
    b = Batch([(3, 192)], [9, 30, 1], 1, 4, 4, 128, 64, torch.bfloat16)
    for lens in ([70, 222, 193], [5, 64, 1], [201, 0, 100]):
        b.lens = lens
        b.dev_lens = _i32(lens)
        lse = torch.empty(3, 4, device=DEV)
        _check_attention(b, b.run(lse=lse), lse, 1 / math.sqrt(128))


@gpu
@checked
def test_strides_scale_and_pool_views():
    from rs_nanogpt_b200.ops import paged
    b = Batch([(5, 64)], [5, 6, 70, 8, 3], 1, 4, 2, 64, 32, torch.bfloat16)
    fused = torch.full((5, 3, 4 * 64 + 2), 7.0, device=DEV, dtype=torch.bfloat16)
    fused[:, 1, :256] = b.q.view(5, 256).to(DEV)
    q = fused[:, 1, :256].view(5, 4, 64)
    pool = torch.full((b.k.shape[0], 3, *b.k.shape[1:]), float("nan"), device=DEV, dtype=torch.bfloat16)
    pool[:, 0], pool[:, 2] = b.k.to(DEV), b.v.to(DEV)  # k and v of a page side by side
    out = torch.full((4, 5, 64), 3.0, device=DEV, dtype=torch.bfloat16).transpose(0, 1)
    lse = torch.empty(5, 4, device=DEV)
    paged.attention(q, pool[:, 0], pool[:, 2], b.dev_table, b.dev_lens, b.plan, out=out, lse=lse, scale=0.3)
    _check_attention(b, out, lse, 0.3)


@gpu
@checked
def test_infinite_and_nan_values_stay_with_the_rows_that_see_them():
    b = Batch([(3, 64)], [10, 20, 30], 1, 2, 2, 64, 32, torch.bfloat16)
    b.v[int(b.table[1, 2]), 0, 3, 5] = float("nan")   # a key that only sequence 1 sees, kv head 0
    b.k[int(b.table[2, 2]), 1, 0] = float("inf")      # sequence 2, kv head 1
    out = b.run().float().cpu()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, 1]).all() and torch.isfinite(out[2, 0]).all()
    assert torch.isnan(out[1, 0, 5]) and not torch.isfinite(out[2, 1]).any()
    assert torch.isfinite(out[1, 0, :5]).all()


@gpu
@checked
def test_large_scores_do_not_overflow():
    b = Batch([(4, 128)], [3, 70, 64, 1], 1, 2, 1, 128, 64, torch.bfloat16)
    b.q = b.q * 30
    lse = torch.empty(4, 2, device=DEV)
    out = b.run(lse=lse)
    ref, ref_lse = b.reference(1 / math.sqrt(128))
    # Scores up to ~400: fp32 errors of 128 2^-24 |q||k| scale, about 0.005, move the output by twice that.
    assert (out.double().cpu() - ref).abs().max() <= (2 ** -7 + 0.02) * b.v[torch.isfinite(b.v)].abs().max()
    assert (lse.double().cpu() - ref_lse).abs().max() <= 0.01


@gpu
@checked
def test_other_stream_repeats_and_graph():
    """The same answer on another stream, every time, and from a captured graph that follows the lengths."""
    from rs_nanogpt_b200.ops import paged
    b = Batch([(40, 256)], [1 + 5 * i % 77 for i in range(40)], 1, 4, 2, 128, 64, torch.bfloat16)
    first = b.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = b.run()
    s.synchronize()
    assert torch.equal(first, other)
    q, k, v = b.q.to(DEV), b.k.to(DEV), b.v.to(DEV)
    out = torch.empty_like(q)
    lens = b.dev_lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, b.dev_table, lens, b.plan, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    lens[:20] -= lens[:20] // 3
    graph.replay()
    want = paged.attention(q, k, v, b.dev_table, lens, b.plan)
    assert torch.equal(out, want) and not torch.equal(out, first)


@gpu
@checked
def test_offsets_past_32_bits():
    """Pages beyond 2^31 elements of the pool, written by the append and read by the attention."""
    from rs_nanogpt_b200.ops import paged
    pages, hk, page, d = 140000, 2, 64, 128
    assert pages * hk * page * d > 2 ** 31
    k = torch.empty(pages, hk, page, d, device=DEV, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    ids = [139999, 3, 135000, 131072, 139000]
    table, lens = _i32([ids]), _i32([300])
    plan = paged.PrefixPlan([(1, 0)], [300], n_head=2, n_kv_head=2, head_dim=d, page=page, table_width=5)
    torch.manual_seed(0)
    x = torch.randn(3, 300, hk, d, device=DEV).bfloat16()
    paged.append(x[0], x[1], x[2], k, v, table, lens, plan)
    at = torch.arange(300, device=DEV)
    assert torch.equal(k[_i32(ids).long()[at // page], :, at % page], x[1])
    out = paged.attention(x[0], k, v, table, lens, plan)
    z = torch.einsum("qhd,khd->hqk", x[0].double(), x[1].double()) / math.sqrt(d)
    z.masked_fill_(torch.ones(300, 300, device=DEV, dtype=torch.bool).triu(1), -math.inf)
    ref = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), x[2].double())
    assert (out.double() - ref).abs().max() <= (2 * 2 ** -8 + 4e-4) * x[2].abs().max()


@gpu
@checked
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout,rot,norm", [("half", 128, True), ("interleaved", 32, False), ("half", 20, True),
                                             ("interleaved", 6, True), ("half", 0, True), ("half", 0, False)])
def test_append(layout, rot, norm, dtype):
    """A value is off by half a unit of its type and by fp32 rounding (2^-19 of its head's norm)."""
    from rs_nanogpt_b200.ops import paged, rotary
    d, hq, hk, page, eps = 128, 6, 2, 16, 1e-6
    b = Batch([(2, 32), (1, 0), (2, 16)], [5, 40, 17, 1, 16], [5, 33, 17, 1, 2], hq, hk, d, page, dtype, seed=4,
              slots=[4, 0, 2, 1, 3])
    n = b.q.shape[0]
    fused = torch.randn(n, (hq + 2 * hk) * d, device=DEV).to(dtype)
    q, k, v = (x.view(n, -1, d) for x in fused.split([hq * d, hk * d, hk * d], 1))
    cos, sin = rotary.tables(rot, 4096) if rot else (None, None)
    kp, vp = b.k.to(DEV), b.v.to(DEV)
    want_k, want_v = kp.cpu().double(), vp.cpu().double()
    pos = torch.cat([torch.arange(m - t, m) for m, t in zip(b.lens, b.q_lens)])
    seq = torch.repeat_interleave(torch.arange(5), torch.tensor(b.q_lens))
    i = torch.arange(rot // 2)
    one, two = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)

    def turned(x):
        x = x.double().cpu()
        y = x.clone()
        if rot:
            a = pos.double()[:, None] * torch.pow(10000.0, -2.0 * i.double() / rot)
            c, s = a.cos()[:, None], a.sin()[:, None]
            y[..., one], y[..., two] = x[..., one] * c + x[..., two] * s, x[..., two] * c - x[..., one] * s
        return y / (y.square().mean(-1, keepdim=True) + eps).sqrt() if norm else y

    want_q, new_k = turned(q), turned(k)
    where = b.table[seq, pos // page].long()
    want_k[where, :, pos % page], want_v[where, :, pos % page] = new_k, v.double().cpu()
    got_q = paged.append(q, k, v, kp, vp, b.dev_table, b.dev_lens, b.plan, cos, sin, layout=layout,
                         qk_eps=eps if norm else None, q_out=q)  # in place in the fused rows
    assert got_q.data_ptr() == fused.data_ptr()
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    for got, want in ((got_q, want_q), (kp, want_k)):
        want = want.nan_to_num(0.0)
        got = got.double().cpu().nan_to_num(0.0)
        tol = want.abs() * unit * 1.001 + want.norm(dim=-1, keepdim=True) * 2.0 ** -19 + 2.0 ** -25
        assert ((got - want).abs() <= tol).all()
    assert torch.equal(vp.double().cpu().nan_to_num(0.0), want_v.nan_to_num(0.0))


@gpu
def test_append_reports_what_it_cannot_place():
    from rs_nanogpt_b200.ops import paged, rotary
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    k = torch.zeros(4, 1, 8, 64, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    plan = paged.PrefixPlan([(1, 0)] * 3, 1, n_head=1, n_kv_head=1, head_dim=64, page=8, table_width=2)
    x = torch.ones(3, 1, 64, device=DEV, dtype=torch.bfloat16)
    table = _i32([[0, -1], [1, 9], [2, -1]])
    paged.append(x, x, x, k, v, table, _i32([3, 0, 8]), plan)
    assert kernel_status(True) == 0  # an empty slot has nothing to place
    assert k[0, 0, 2].sum() == 64 and k[2, 0, 7].sum() == 64 and k.sum() == 128
    for lens in ([9, 0, 0], [0, 10, 0], [17, 0, 0]):
        paged.append(x, x, x, k, v, table, _i32(lens), plan)
        assert kernel_status(True) == 5
    cos, sin = rotary.tables(64, 4)
    paged.append(x, x, x, k, v, table, _i32([5, 0, 0]), plan, cos, sin)
    assert kernel_status(True) == 5
    assert k.sum() == 128
    paged.attention(x, k, v, _i32([[0, -1], [1, 9], [2, -1]]), _i32([0, 9, 0]), plan)
    assert kernel_status(True) == 5


@gpu
def test_append_and_attention_refusals():
    from rs_nanogpt_b200.ops import paged
    b = Batch([(2, 32)], [5, 6], 1, 4, 2, 64, 32, torch.bfloat16)
    q, k, v, t, n, plan = b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), b.dev_table, b.dev_lens, b.plan
    kv = torch.zeros(2, 2, 64, device=DEV, dtype=torch.bfloat16)

    def call(q=q, k=k, v=v, t=t, n=n, plan=plan, **kw):
        return paged.attention(q, k, v, t, n, plan, **kw)

    other = paged.PrefixPlan([(2, 32)], 1, n_head=2, n_kv_head=2, head_dim=64, page=32, table_width=t.shape[1])
    bad = [lambda: call(q=q.float()), lambda: call(q=q.half()), lambda: call(q=q[:1]), lambda: call(q=q[:, :3]),
           lambda: call(q=q[..., :32]), lambda: call(k=k[:, :, :24], v=v[:, :, :24]), lambda: call(k=k[:, :1]),
           lambda: call(k=k.transpose(1, 2), v=v.transpose(1, 2)), lambda: call(t=t.long()), lambda: call(n=n[:1]),
           lambda: call(t=t[:1], n=n[:1]), lambda: call(plan=other), lambda: call(lse=torch.empty(2, 4)),
           lambda: call(out=torch.empty_like(q).float()), lambda: call(q=q.cpu()), lambda: call(scale=0.0),
           lambda: paged.append(q, kv[..., :32], kv, k, v, t, n, plan),
           lambda: paged.append(q, kv, kv[:, :1], k, v, t, n, plan),
           lambda: paged.append(q, kv, kv, k[..., :32], v, t, n, plan),
           lambda: paged.append(q[:1], kv[:1], kv[:1], k, v, t, n, plan),
           lambda: paged.append(q, kv, kv, k, v, t, n, plan, cos=torch.zeros(9, 64, device=DEV))]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("kw", [dict(groups=[(2, 5)]), dict(groups=[(2, 1024)]), dict(q_lens=[1]), dict(q_lens=[1, -1]),
                                dict(slots=[0]), dict(slots=[0, -1]), dict(n_kv_head=3)])
def test_plan_refusals_cpu(kw):
    from rs_nanogpt_b200.ops import paged
    args = dict(groups=[(2, 32)], q_lens=1, n_head=4, n_kv_head=2, head_dim=64, page=32, table_width=4, device="cpu")
    paged.PrefixPlan(**args)
    with pytest.raises(ValueError):
        paged.PrefixPlan(**{**args, **kw})


@pytest.mark.parametrize("groups,q_lens,split", [
    ([(1, 64), (3, 32), (2, 0)], [3, 40, 1, 0, 2, 5], [0, 0, 0, 0, 0, 0]),        # too short a prefix to be worth a run
    ([(1, 6400), (30, 3200), (2, 0)], [3] + [5] * 29 + [0, 2, 5], [0] + [1] * 30 + [0, 0]),
    ([(2, 3200), (9, 3200)], [300, 200] + [1] * 9, [0, 0] + [1] * 9),             # long prompts fill their tiles alone
])
def test_plan_items_cpu(groups, q_lens, split):
    """Every (row, head) pair is in one item of its own keys, and in one of the shared keys where its group is
    split; own keys begin where the shared run ends, or at 0."""
    from rs_nanogpt_b200.ops import paged
    plan = paged.PrefixPlan(groups, q_lens, n_head=6, n_kv_head=2, head_dim=64, page=32, table_width=256, device="cpu")
    shared_of = [s for n, s in groups for _ in range(n)]
    seq = [i for i, t in enumerate(q_lens) for _ in range(3 * t)]
    seen = {0: [0] * len(seq), 1: [0] * len(seq)}
    for list_, most, mark in ((plan.items, 16, 0), (plan.big_items, 256, paged.BIG)):
        for i, (shared, first, count, row0, rows, key0, keys, alone) in enumerate(list_.tolist()):
            assert 0 < rows <= most
            for p in range(row0, row0 + rows):
                seen[shared][p] += 1
                assert (plan.shared_item if shared else plan.own_item)[p] == i + mark
                if shared:
                    assert (key0, keys) == (0, shared_of[seq[p]])
                else:
                    assert key0 == split[seq[p]] * shared_of[seq[p]] and alone == (key0 == 0)
    assert seen[0] == [1] * len(seq)
    assert seen[1] == [split[i] for i in seq]
