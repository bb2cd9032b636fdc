"""The decoder over the paged cache: what it refuses, what a refusal leaves behind, and its numbers with
output projections that let the attention through."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
checked = pytest.mark.usefixtures("kernel_ok")


def _store(seq=512, vocab=1000, depth=2):
    """Random weights; the output projections, too, are drawn, so that the logits depend on the attention."""
    from rs_nanogpt_b200.config import d_model
    from rs_nanogpt_b200.models.params import ParamStore, init_params
    cfg = d_model(depth, vocab_size=vocab, sequence_len=seq)
    store = ParamStore(cfg, "cuda")
    init_params(store, seed=5, mode="bench")
    g = torch.Generator(device="cuda").manual_seed(6)
    for name in store.names():
        if name.endswith("c_proj.weight"):
            store.param(name).normal_(0.0, 0.05, generator=g)
    store.refresh_work()
    return cfg, store


def _tokens(cfg, n, seed=0):
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _state(dec):
    c = dec.cache
    return [x.clone() for x in (c.table, c.lens, c.refs, c.k, c.v)]


def _unchanged(dec, was):
    return all(torch.equal(a, b) for a, b in zip(_state(dec), was))


def _close(got, ref):
    # bf16 activations through two blocks against fp32: the tolerance of the contiguous cache's test.
    assert (got.float() - ref).abs().max().item() <= 5e-2 * max(1.0, ref.abs().max().item())


@gpu
@checked
def test_logits_that_depend_on_the_attention():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    from rs_nanogpt_b200.models.reference import ReferenceGpt
    cfg, store = _store()
    ref = ReferenceGpt(store, torch.float32)
    dec = PagedDecoder(store, pages=40, max_seqs=8, max_len=400, page=32)

    def expect(seqs):
        return torch.stack([ref.forward(torch.tensor([s], device="cuda"))[0, -1] for s in seqs])

    system = [_tokens(cfg, 130), _tokens(cfg, 70, 1)]
    _close(dec.feed(system, [0, 4]), expect(system))
    # They do depend on it: without the first half of a prompt they are others.
    a, b = expect([system[0]]), expect([system[0][65:]])
    assert (a - b).abs().max() > 0.3 * max(1.0, a.abs().max().item())
    dec.cache.fork([0, 0, 4], [1, 2, 5])
    slots, groups = [0, 1, 2, 4, 5], [(3, 128), (2, 64)]
    seqs = [system[0] for _ in range(3)] + [system[1] for _ in range(2)]
    for i, lens in enumerate(([5, 40, 1, 33, 7], [1] * 5, [2, 3, 4, 5, 6], [1] * 5)):
        new = [_tokens(cfg, n, 10 * i + j + 2) for j, n in enumerate(lens)]
        seqs = [s + t for s, t in zip(seqs, new)]
        _close(dec.feed(new, slots, groups), expect(seqs))
    dec.cache.check()


@gpu
@pytest.mark.usefixtures("kernel_ok")
@pytest.mark.parametrize("slots", [[0, 8], [8], [0, -1], [-1], [1 << 40, 0]])
def test_slots_outside_the_cache_are_refused(slots):
    from rs_nanogpt_b200.models.paged import PagedDecoder
    cfg, store = _store()
    dec = PagedDecoder(store, pages=20, max_seqs=8, max_len=200, page=32)
    dec.feed([_tokens(cfg, 40)], [7])
    was = _state(dec)
    with pytest.raises(ValueError):
        dec.feed([[1]] * len(slots), slots)
    assert _unchanged(dec, was)


@gpu
@checked
def test_refused_arguments_leave_the_cache_as_it_was():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    cfg, store = _store()
    dec = PagedDecoder(store, pages=20, max_seqs=4, max_len=200, page=32)
    dec.feed([_tokens(cfg, 64), _tokens(cfg, 40, 1)], [0, 1])
    was = _state(dec)
    for groups in ([(2, 33)], [(3, 0)], [(1, 0)], [(2, 32 * 100)], [(-1, 0), (3, 0)]):
        with pytest.raises(ValueError):
            dec.feed([[1], [2]], [0, 1], groups)
        assert _unchanged(dec, was)


@gpu
@checked
def test_tokens_outside_the_vocabulary_are_refused():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    cfg, store = _store()
    dec = PagedDecoder(store, pages=20, max_seqs=4, max_len=200, page=32)
    dec.feed([_tokens(cfg, 64), _tokens(cfg, 40, 1)], [0, 1])
    was = _state(dec)
    for ids in ([cfg.vocab_size], [-1], [1 << 40]):
        with pytest.raises(ValueError):
            dec.feed([[3], ids], [0, 1])
        assert _unchanged(dec, was)


@gpu
def test_appends_to_a_full_pool_change_nothing():
    """A refused grow, used all the same: no page is written, of the slot or of those that share it."""
    from rs_nanogpt_b200.models.paged import PagedDecoder
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    cfg, store = _store()
    dec = PagedDecoder(store, pages=5, max_seqs=4, max_len=200, page=32)
    dec.feed([_tokens(cfg, 64)], [0])
    dec.cache.fork([0], [1])
    dec.feed([_tokens(cfg, 96, 1)], [2])
    was = _state(dec)
    assert kernel_status(True) == 0
    dec.cache.grow([0, 1, 0, 0])
    assert kernel_status(True) == 6
    dec.forward(torch.tensor([5], device="cuda"), dec.plan([(1, 0)], [1], [1]))
    assert kernel_status(True) == 6 and _unchanged(dec, was)
    # Reserved in two steps, written in one.
    dec.cache.free([2])
    dec.cache.grow([0, 1, 0, 0])
    dec.cache.grow([0, 2, 0, 0])
    new = _tokens(cfg, 3, 2)
    dec.forward(torch.tensor(new, device="cuda"), dec.plan([(1, 0)], [3], [1]))
    assert kernel_status(True) == 0
    from rs_nanogpt_b200.models.reference import ReferenceGpt
    ref = ReferenceGpt(store, torch.float32).forward(torch.tensor([_tokens(cfg, 64) + new + [9]], device="cuda"))[:, -1]
    _close(dec.feed([[9]], [1]), ref)


@gpu
@checked
def test_feeds_that_do_not_fit_raise_and_change_nothing():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    cfg, store = _store()
    dec = PagedDecoder(store, pages=5, max_seqs=4, max_len=150, page=32)
    dec.feed([_tokens(cfg, 64)], [0])
    dec.cache.fork([0], [1])
    dec.feed([_tokens(cfg, 70, 1)], [2])
    was = _state(dec)
    with pytest.raises(RuntimeError, match="out of pages"):
        dec.feed([[1], [2] * 27], [1, 2])
    with pytest.raises(RuntimeError, match="out of pages"):
        dec.feed([[1]], [1])
    assert _unchanged(dec, was)
    with pytest.raises(ValueError, match="max_len"):
        dec.feed([[1] * 81], [2])
    assert _unchanged(dec, was)
    dec.feed([[2] * 26], [2])  # what fits is served
    dec.cache.free([2])
    dec.feed([[1] * 86], [1])  # up to max_len
    assert dec.cache.lens.tolist() == [64, 150, 0, 0]
    with pytest.raises(ValueError, match="max_len"):
        dec.feed([[1]], [1])


@gpu
@checked
def test_samples_need_empty_slots():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    cfg, store = _store()
    dec = PagedDecoder(store, pages=30, max_seqs=4, max_len=200, page=32)
    alone = dec.sample_many(_tokens(cfg, 50), 2, 6, 1.0, 50, seed=1)
    for used in (0, 1):
        dec.feed([_tokens(cfg, 40, 3)], [used])
        was = _state(dec)
        with pytest.raises(ValueError, match="slot"):
            dec.sample_many(_tokens(cfg, 50), 2, 6, 1.0, 50, seed=1)
        assert _unchanged(dec, was)
        dec.cache.free([used])
    dec.feed([_tokens(cfg, 40, 3)], [3])  # another slot may be in use
    assert dec.sample_many(_tokens(cfg, 50), 2, 6, 1.0, 50, seed=1) == alone
    assert dec.cache.lens.tolist() == [0, 0, 0, 40]


@gpu
@checked
@pytest.mark.parametrize("kind", ["parts", "linear"])
def test_scaling_sharpens_behind_the_norm(kind, monkeypatch):
    """Frequencies scaled by parts multiply the scores by (0.1 ln(factor) + 1)^2, although the norm of q and k
    divides a common factor of theirs away."""
    from rs_nanogpt_b200.models.paged import PagedDecoder
    from rs_nanogpt_b200.ops import paged, rotary
    cfg, store = _store(seq=128)
    f = 16.0
    dec = PagedDecoder(store, 20, 2, 300, page=32, scaling=rotary.Scaling(kind, f, original_len=128))
    calls, attention = [], paged.attention

    def spy(q, k, v, *args, **kw):
        q = q.clone()
        out = attention(q, k, v, *args, **kw)
        calls.append((q, k.clone(), v.clone(), out.clone()))
        return out

    monkeypatch.setattr(paged, "attention", spy)
    x = _tokens(cfg, 250)
    dec.feed([x], [0])
    table, mul = dec.cache.table[0].long(), 0.1 * math.log(f) + 1 if kind == "parts" else 1.0
    for q, k, v, out in calls:
        # Unit root mean square: nothing of the factor is left in q and k.
        assert (q.double().square().mean(-1) - 1).abs().max() < 0.02
        k, v = (y[table[:8]].transpose(0, 1).flatten(1, 2)[:, :250].double() for y in (k, v))
        z = torch.einsum("qhd,hkd->hqk", q.double(), k) * (mul * mul / math.sqrt(cfg.head_dim))
        z.masked_fill_(torch.ones(250, 250, device="cuda", dtype=torch.bool).triu(1), -math.inf)
        ref = torch.einsum("hqk,hkd->qhd", torch.softmax(z, -1), v)
        assert (out.double() - ref).abs().max() <= (2 * 2.0 ** -8 + 4e-4) * v.abs().max()


@gpu
def test_check_waits_for_the_stream_it_is_called_on():
    from rs_nanogpt_b200.models.paged import PagedCache
    from rs_nanogpt_b200.ops._ext import kernel_status
    kernel_status(True)
    cache = PagedCache(1, 1, 64, 2, 32, 2, 128)
    add = torch.tensor([64, 32], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second or more
        cache.grow(add)
        with pytest.raises(RuntimeError, match="out of pages"):
            cache.check()
    torch.cuda.synchronize()
    assert kernel_status(True) == 0
