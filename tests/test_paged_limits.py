"""Paged cache operators at their limits: pages that run out, plans and tensors that do not fit,
operands that lie over one another, values that a row may not see, states without entries."""
import math
import random

import pytest
import torch

from test_paged import CASES, DEV, Batch, Model, _check_state, _i32, _pools, _state

gpu = pytest.mark.gpu
checked = pytest.mark.usefixtures("kernel_ok")


# ---- pages that run out ------------------------------------------------------------------


@gpu
def test_refused_slots_keep_their_tokens():
    """The append writes new tokens only: a slot whose growth was refused loses none of what it holds,
    nor do those that share its pages."""
    from rs_nanogpt_b200.ops import paged
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    page, d = 8, 64
    k = torch.zeros(3, 1, page, d, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    table, lens, refs = torch.full((4, 3), -1, device=DEV, dtype=torch.int32), _i32([0] * 4), _i32([0] * 3)
    state, room = (table, lens, refs), _i32([0] * 4)

    def new(slots, t, fill):
        plan = paged.PrefixPlan([(len(slots), 0)], t, n_head=1, n_kv_head=1, head_dim=d, page=page, table_width=3,
                                slots=slots)
        x = torch.full((len(slots) * t, 1, d), float(fill), device=DEV, dtype=torch.bfloat16)
        paged.append(x, x, x, k, v, table, lens, plan, room=room)
        room[slots] = 0

    paged.grow_pages(*state, _i32([8, 0, 5, 0]), page, out=state, room=room)
    assert room.tolist() == [8, 0, 5, 0]
    new([0], 8, 1)
    new([2], 5, 2)
    kk, vv = k.view(1, *k.shape), v.view(1, *v.shape)
    paged.fork_pages(kk, vv, *state, _i32([0]), _i32([1]), out=state)  # a full page, shared
    paged.grow_pages(*state, _i32([0, 0, 0, 8]), page, out=state, room=room)
    new([3], 8, 3)
    assert kernel_status(True) == 0
    before = k.clone(), v.clone(), [x.clone() for x in state]
    # No page is free: slots 0 and 1 are refused, slot 2 has room in its own page.
    paged.grow_pages(*state, _i32([1, 2, 0, 0]), page, out=state, room=room)
    assert kernel_status(True) == 6
    paged.grow_pages(*state, _i32([0, 0, 1, 0]), page, out=state, room=room)
    assert kernel_status(True) == 0 and lens.tolist() == [8, 8, 6, 8] and room.tolist() == [0, 0, 1, 0]
    new([0, 2], 1, 9)
    assert kernel_status(True) == 6
    new([1], 2, 9)
    assert kernel_status(True) == 6
    own = int(table[2, 0])
    assert (k[own, 0, 5] == 9).all()
    for x, was in ((k, before[0]), (v, before[1])):
        x[own, 0, 5] = 0
        assert torch.equal(x, was)
    # More rows than were granted: those that were not are left out.
    paged.grow_pages(*state, _i32([0, 0, 1, 0]), page, out=state, room=room)
    new([2], 3, 7)
    assert kernel_status(True) == 6
    assert (k[own, 0, 6] == 7).all() and (k[own, 0, 4] == 2).all()
    # A slot that is freed has no room either.
    paged.free_pages(*state, _i32([3]), out=state, room=room)
    paged.grow_pages(*state, _i32([1, 0, 0, 0]), page, out=state, room=room)
    paged.free_pages(*state, _i32([0]), out=state, room=room)
    assert room.tolist() == [0] * 4 and kernel_status(True) == 0


@gpu
def test_a_refused_slot_refuses_no_other():
    """Slots are served in order; one that cannot be served takes nothing from those after it."""
    from rs_nanogpt_b200.ops import paged
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    m = Model(2, 4, 3, 2)
    m.grow([4, 1])
    state = paged.grow_pages(*(x.to(DEV) for x in _state(m)), _i32([1, 1]), 4)  # slot 1 needs no page
    assert kernel_status(True) == 6 and state[1].tolist() == [4, 2]
    m = Model(3, 4, 8, 4)
    m.grow([4, 0, 0, 0])
    state = paged.grow_pages(*(x.to(DEV) for x in _state(m)), _i32([9, 2, 0, 4]), 4)
    assert kernel_status(True) == 6
    assert state[1].tolist() == [4, 2, 0, 4] and state[2].tolist() == [1, 1, 1]
    assert state[0][:, 0].tolist() == [0, 1, -1, 2]


def _grow_in_order(m, add):
    """Model.grow where a refused slot takes nothing."""
    free = [p for p, r in enumerate(m.refs) if r == 0]
    refused = False
    for s, a in enumerate(add):
        if a < 0 or m.lens[s] + a > m.width * m.page:
            continue
        need = -(-(m.lens[s] + a) // m.page) - len(m.table[s])
        if need > len(free):
            refused = True
            continue
        for _ in range(need):
            p = free.pop(0)
            m.table[s].append(p)
            m.refs[p] = 1
        m.lens[s] += a
    return refused


@gpu
@pytest.mark.parametrize("seed,pages,page,width,slots", [(0, 11, 4, 5, 7), (1, 90, 3, 6, 61), (2, 400, 2, 9, 1500),
                                                         (3, 20000, 1, 40, 1100), (4, 5, 16, 3, 40)])
def test_growing_past_the_pool(seed, pages, page, width, slots):
    from rs_nanogpt_b200.ops import paged
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    rng = random.Random(seed)
    m = Model(pages, page, width, slots)
    state = tuple(x.to(DEV) for x in _state(m))
    room, held = _i32([0] * slots), [0] * slots
    refusals = 0
    for _ in range(12):
        most = max(1, 2 * pages * page // slots)
        add = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(slots)]
        add = [min(a, width * page - m.lens[s]) for s, a in enumerate(add)]
        before = list(m.lens)
        refused = _grow_in_order(m, add)
        held = [h + n - b for h, n, b in zip(held, m.lens, before)]
        state = paged.grow_pages(*state, _i32(add), page, out=state if rng.random() < 0.5 else None, room=room)
        assert kernel_status(True) == (6 if refused else 0)
        refusals += refused
        _check_state(m, state)
        assert room.tolist() == held
        gone = rng.sample(range(slots), slots // 4)
        m.free(gone)
        held = [0 if s in set(gone) else h for s, h in enumerate(held)]
        state = paged.free_pages(*state, _i32(gone), out=state if rng.random() < 0.5 else None, room=room)
        assert room.tolist() == held
    assert refusals


# ---- plans and operands that do not fit ------------------------------------------------------


@gpu
@checked
def test_a_plan_for_other_pages_is_refused():
    from rs_nanogpt_b200.ops import paged
    b = Batch([(30, 64)], [5] * 30, 1, 4, 2, 64, 32, torch.bfloat16)
    b.run()
    for page in (8, 16, 64):
        b.plan = paged.PrefixPlan([(30, 64)], 1, n_head=4, n_kv_head=2, head_dim=64, page=page,
                                  table_width=b.table.shape[1] * 32 // page)
        with pytest.raises(RuntimeError, match="page"):
            b.run()


@gpu
@checked
def test_more_tiles_than_are_counted_are_refused():
    """The limit counts the keys of the plan's shared runs, not only those that the table at hand can name."""
    from rs_nanogpt_b200.ops import paged
    b = Batch([(30, 64)], [5] * 30, 1, 4, 2, 64, 32, torch.bfloat16)
    b.plan = paged.PrefixPlan([(30, 1 << 30)], 1, n_head=4, n_kv_head=2, head_dim=64, page=32, table_width=1 << 25)
    assert len(b.plan.items) + len(b.plan.big_items) > 30  # the shared run is one of its own
    with pytest.raises(RuntimeError, match="32-bit"):
        b.run()


@gpu
@checked
def test_outputs_over_other_operands_are_refused():
    from rs_nanogpt_b200.ops import paged, rotary
    n, h, d = 6, 2, 64
    cos, sin = rotary.tables(32, 64)
    pos = torch.arange(n, device=DEV, dtype=torch.int32)
    buf = torch.randn(8 * n * h * d, device=DEV).bfloat16()

    def block(at, heads=h):
        return buf[at * d:at * d + n * heads * d].view(n, heads, d)

    q, k, far, far2 = block(0), block(n * h), block(2 * n * h), block(3 * n * h)
    wide = buf[:n * d].view(n, 1, d).expand(n, h, d)
    for args in [dict(q_out=k, k_out=far), dict(q_out=far, k_out=q), dict(q_out=far, k_out=far),
                 dict(q_out=block(n * h + 1), k_out=far), dict(q_out=far, k_out=block(2 * n * h + h)),
                 dict(q_out=wide, k_out=far), dict(q_out=k, k_out=k), dict(q_out=far, k_out=wide)]:
        before = buf.clone()
        with pytest.raises(RuntimeError):
            rotary.rotate(q, k, pos, cos, sin, **args)
        assert torch.equal(buf, before)
    with pytest.raises(RuntimeError):
        rotary.rotate(q, q, pos, cos, sin, q_out=q, k_out=q)
    # What shares a buffer without lying over one another is served: column blocks of a row, heads in turn,
    # heads before rows, one after another.
    fused = torch.randn(n, 3, h, d, device=DEV).bfloat16()
    turns = torch.randn(n, h, 3, d, device=DEV).bfloat16()
    first = torch.randn(3, h, n, d, device=DEV).bfloat16().permute(2, 0, 1, 3)
    ragged = torch.randn(n, 7 * d, device=DEV).bfloat16()
    for a, b in [(fused[:, 0], fused[:, 1]), (fused[:, 2], fused[:, 0]), (turns[:, :, 0], turns[:, :, 2]),
                 (first[:, 0], first[:, 1]), (ragged[:, 2 * d:].view(n, 5, d), ragged[:, :2 * d].view(n, 2, d)),
                 (ragged[:1, d:2 * d].view(1, 1, d), ragged[:1, 2 * d:4 * d].view(1, 2, d)), (q, k), (q, q)]:
        want = rotary.rotate(a.clone(), b.clone(), pos[:len(a)], cos, sin)
        got = rotary.rotate(a, b, pos[:len(a)], cos, sin, q_out=far, k_out=far2) if a is b else rotary.rotate(
            a, b, pos[:len(a)], cos, sin, q_out=a, k_out=b)
        for x, y in zip(want, got):  # up to a step of the type, where another alignment orders the products otherwise
            assert ((x.float() - y.float()).abs() <= x.float().abs() * 2.0 ** -7).all()
    # The append and the attention.
    c = Batch([(1, 0)], [n], n, h, h, d, 32, torch.bfloat16)
    kp, vp, t, lens = c.k.to(DEV), c.v.to(DEV), c.dev_table, c.dev_lens
    for args in [(q, k, far, k), (q, k, far, far), (q, k, far, block(n * h + 1)), (q, k, far, wide)]:
        with pytest.raises(RuntimeError):
            paged.append(*args[:3], kp, vp, t, lens, c.plan, q_out=args[3])
    paged.append(fused[:, 0], fused[:, 1], fused[:, 2], kp, vp, t, lens, c.plan, q_out=fused[:, 0])
    with pytest.raises(RuntimeError):
        paged.attention(q, kp, vp, t, lens, c.plan, out=block(1))
    with pytest.raises(RuntimeError):
        paged.attention(q, kp, vp, t, lens, c.plan, out=wide)
    want = paged.attention(q, kp, vp, t, lens, c.plan)
    assert torch.equal(paged.attention(q, kp, vp, t, lens, c.plan, out=q), want)


# ---- what a row may not see ------------------------------------------------------------------


HIDDEN = {
    # groups, tails, new tokens, hq, hk, d, page; (sequence, token, element, value) of the values' first kv head
    "a short turn": ([(1, 0)], [40], [40], 1, 1, 64, 16, [(0, 20, 3, math.nan), (0, 33, 9, math.inf)]),
    "heads of one": ([(1, 0), (1, 0)], [30, 9], [5, 1], 4, 2, 128, 32, [(0, 27, 0, -math.inf), (1, 8, 127, math.nan)]),
    "a long turn": ([(1, 0)], [300], [300], 2, 1, 128, 64, [(0, 150, 5, math.nan), (0, 299, 90, math.inf)]),
    "turns behind a prefix": ([(3, 128)], [70, 200, 33], [70, 150, 33], 4, 2, 64, 16,
                              [(0, 190, 1, math.nan), (1, 300, 2, math.inf), (2, 140, 63, math.nan)]),
    "a turn in parts": ([(1, 0)], [12000], [60], 2, 1, 64, 64, [(0, 11970, 5, math.nan), (0, 11999, 6, -math.inf)]),
    "a few tokens in parts": ([(1, 0)], [6000], [8], 2, 1, 64, 64, [(0, 5994, 31, math.nan), (0, 5999, 2, math.inf)]),
    "a long turn in parts": ([(1, 0)], [9000], [200], 4, 4, 128, 128, [(0, 8900, 100, math.nan)]),
    "many samples": ([(40, 512)], [1 + i for i in range(40)], 1, 8, 1, 128, 64,
                     [(3, 515, 17, math.nan), (0, 7, 20, math.inf)]),
}


@gpu
@checked
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", HIDDEN)
def test_values_that_a_row_does_not_see_do_not_reach_it(name, dtype):
    """A NaN or infinite value reaches the rows that see its key and no other, of the same tile and before it."""
    groups, tails, q_lens, hq, hk, d, page, bad = HIDDEN[name]
    b = Batch(groups, tails, q_lens, hq, hk, d, page, dtype)
    for s, at, e, x in bad:
        b.v[int(b.table[s, at // page]), 0, at % page, e] = x
    lse = torch.empty(b.q.shape[:2], device=DEV)
    scale = 1 / math.sqrt(d)
    out = b.run(lse=lse).double().cpu()
    ref, ref_lse = b.reference(scale)
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isinf(), ref.isinf())
    assert ref.isnan().any() or ref.isinf().any()
    ok = ref.isfinite()
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    vmax = b.v[torch.isfinite(b.v)].abs().max().item()
    # As for finite values: P and the output are rounded to the type, scores are off by less than 2e-4.
    assert (out - ref)[ok].abs().max() <= (2 * unit + 4e-4) * vmax
    assert (lse.double().cpu() - ref_lse).abs().max() <= 2e-4
    from rs_nanogpt_b200.ops import paged
    q = b.q.to(DEV)
    paged.attention(q, b.k.to(DEV), b.v.to(DEV), b.dev_table, b.dev_lens, b.plan, out=q)
    assert torch.equal(q.double().cpu().nan_to_num(7.0), out.nan_to_num(7.0))


@gpu
@checked
def test_members_shorter_than_the_prefix_do_not_see_its_end():
    b = Batch([(4, 192)], [9, 30, 1, 5], 1, 4, 4, 128, 64, torch.bfloat16)
    b.v[int(b.table[0, 1]), 0, 40, 11] = math.nan  # token 104 of the shared pages
    b.v[int(b.table[0, 2]), 1, 3, 12] = math.inf   # token 131
    for lens in ([70, 222, 193, 104], [104, 105, 131, 132]):
        b.lens = lens
        b.dev_lens = _i32(lens)
        out = b.run().double().cpu()
        ref, _ = b.reference(1 / math.sqrt(128))
        assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isinf(), ref.isinf())
        ok = ref.isfinite()
        vmax = b.v[torch.isfinite(b.v)].abs().max().item()
        assert (out - ref)[ok].abs().max() <= (2 * 2.0 ** -8 + 4e-4) * vmax


# ---- states without entries, rows without a place --------------------------------------------


@gpu
@checked
@pytest.mark.parametrize("pages,width,slots", [(5, 3, 0), (5, 0, 4), (0, 3, 4), (0, 0, 0)])
def test_states_without_entries(pages, width, slots):
    """Fresh outputs are written whole, also where the table has no entries."""
    from rs_nanogpt_b200.ops import paged
    table = torch.full((slots, width), -1, device=DEV, dtype=torch.int32)
    lens, refs = _i32([0] * slots), _i32([0] * pages)
    none, k = _i32([]), torch.zeros(1, pages, 1, 4, 8, device=DEV)
    for call in (lambda out: paged.grow_pages(table, lens, refs, _i32([0] * slots), 4, out=out),
                 lambda out: paged.free_pages(table, lens, refs, none, out=out),
                 lambda out: paged.fork_pages(k, k.clone(), table, lens, refs, none, none, out=out),
                 lambda out: paged.compact_pages(k, k.clone(), table, lens, refs, out=out)):
        out = tuple(torch.full_like(x, 77) for x in (table, lens, refs))
        call(out)
        for x, want in zip(out, (table, lens, refs)):
            assert torch.equal(x, want)
        assert all(torch.equal(x, want) for x, want in zip(call((table, lens, refs)), (table, lens, refs)))


@gpu
@checked
def test_rows_without_a_place_are_zero():
    """The rows of q of a slot that holds no tokens, or fewer than its rows, are 0, not what memory held."""
    from rs_nanogpt_b200.ops import paged
    b = Batch([(3, 0)], [5, 6, 9], [2, 6, 4], 4, 2, 64, 32, torch.bfloat16)
    b.dev_lens = _i32([0, 4, 9])
    k, v = (torch.randn(12, 2, 64, device=DEV).bfloat16() for _ in range(2))
    out = torch.full(b.q.shape, 7.0, device=DEV, dtype=torch.bfloat16)
    q = b.q.to(DEV)
    paged.append(q, k, v, b.k.to(DEV), b.v.to(DEV), b.dev_table, b.dev_lens, b.plan, q_out=out)
    assert (out[:4] == 0).all() and torch.equal(out[4:], q[4:])


# ---- how near the attention comes ------------------------------------------------------------


@gpu
@checked
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CASES)
def test_attention_error_scales_with_the_probabilities(name, dtype):
    """Rounding each p_j to the type (relative error up to u) moves an output by a sum of terms u p_j v_j of
    either sign: by more than 7 u sqrt(sum (p_j v_j)^2) in one element of 2e10 (Hoeffding). fp16 loses up to
    2^-25 of the largest p on small ones. The output is rounded once, by u |o|. Scores, exponentials and sums
    in fp32: scores are off by less than 2e-4, which counts twice, and sums by less than 1e-4, both times
    sum p_j |v_j|. An output of zeros is far outside of this, also behind a prefix of 20000 tokens."""
    b = Batch(*CASES[name], dtype)
    out = b.run().double()
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    row = 0
    for s in range(b.n):
        n, t = b.lens[s], b.q_lens[s]
        ids = b.table[s, :-(-n // b.page)].long()
        k, v = (x[ids].transpose(0, 1).flatten(1, 2)[:, :n].to(DEV).double().repeat_interleave(b.hq // b.hk, 0)
                for x in (b.k, b.v))
        z = torch.einsum("thd,hnd->htn", b.q[row:row + t].to(DEV).double(), k) / math.sqrt(b.d)
        z.masked_fill_(torch.ones(t, n, device=DEV, dtype=torch.bool).triu(n - t + 1), -math.inf)
        p = torch.softmax(z, -1)
        ref, mass = p @ v, p @ v.abs()
        tol = 7 * unit * (p.square() @ v.square()).sqrt() + unit * ref.abs() + 5e-4 * mass
        if dtype == torch.float16:
            tol += 2.0 ** -25 * p.amax(-1, keepdim=True) * v.abs().sum(1, keepdim=True)
        got = out[row:row + t].transpose(0, 1)
        assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).max().item()
        assert (ref.abs() > tol).any(-1).all()
        row += t
