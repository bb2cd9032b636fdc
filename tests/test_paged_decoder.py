"""Generation over the paged cache against the fp32 PyTorch model and the contiguous cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _store(seq=512, vocab=1000, depth=2):
    from rs_nanogpt_b200.config import d_model
    from rs_nanogpt_b200.models.params import ParamStore, init_params
    cfg = d_model(depth, vocab_size=vocab, sequence_len=seq)
    store = ParamStore(cfg, "cuda")
    init_params(store, seed=5, mode="bench")
    store.refresh_work()
    return cfg, store


def _close(got, ref):
    # bf16 activations through two blocks against fp32: the tolerance of the contiguous cache's test.
    scale = max(1.0, ref.abs().max().item())
    assert (got.float() - ref).abs().max().item() <= 5e-2 * scale


@pytest.mark.usefixtures("kernel_ok")
def test_feeds_forks_and_frees_match_the_model():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    from rs_nanogpt_b200.models.reference import ReferenceGpt
    cfg, store = _store()
    ref = ReferenceGpt(store, torch.float32)
    dec = PagedDecoder(store, pages=40, max_seqs=8, max_len=400, page=32)
    g = torch.Generator().manual_seed(0)

    def tokens(n):
        return torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()

    def expect(seqs):
        return torch.stack([ref.forward(torch.tensor([s], device="cuda"))[0, -1] for s in seqs])

    # Two system prompts, three and two chats behind them, turns of ragged lengths, then single tokens.
    system = [tokens(130), tokens(70)]
    _close(dec.feed(system, [0, 4]), expect(system))
    dec.cache.fork([0, 0, 4], [1, 2, 5])
    slots, groups = [0, 1, 2, 4, 5], [(3, 128), (2, 64)]
    seqs = [system[0] for _ in range(3)] + [system[1] for _ in range(2)]
    for lens in ([5, 40, 1, 33, 7], [1] * 5, [1] * 5, [2, 3, 4, 5, 6]):
        new = [tokens(n) for n in lens]
        seqs = [s + t for s, t in zip(seqs, new)]
        _close(dec.feed(new, slots, groups), expect(seqs))
    # One chat ends; the pool is compacted and its pages serve another.
    dec.cache.free([1])
    dec.cache.compact()
    fresh = tokens(60)
    new = [tokens(1) for _ in range(4)] + [fresh]
    seqs = [s + t for s, t in zip([seqs[0], seqs[2], seqs[3], seqs[4]], new)] + [fresh]
    _close(dec.feed(new, [0, 2, 4, 5, 7], [(2, 128), (2, 64), (1, 0)]), expect(seqs))
    dec.cache.check()
    used = int((dec.cache.refs > 0).sum())
    assert (dec.cache.refs[:used] > 0).sum() >= used - 3  # the fresh sequence took the lowest free pages
    dec.cache.free([0, 2, 4, 5, 7])
    assert int(dec.cache.refs.abs().sum()) == 0


@pytest.mark.usefixtures("kernel_ok")
def test_sample_many_greedy_and_graph():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    _, store = _store()
    prompt = [(7 * i + 3) % 1000 for i in range(150)]
    dec = PagedDecoder(store, pages=60, max_seqs=6, max_len=256, page=32)
    outs = dec.sample_many(prompt, 6, 9, temperature=0.0)
    assert all(o == outs[0] for o in outs)  # greedy: every sample the same
    seq = list(prompt)
    dec2 = PagedDecoder(store, pages=60, max_seqs=1, max_len=256, page=64)
    logits = dec2.feed([seq], [0])
    for tok in outs[0]:
        # The chosen token is the largest logit up to bf16 ties between the two page sizes' roundings.
        assert logits[0, tok] >= logits[0].max() - 0.05 * logits[0].abs().max()
        logits = dec2.feed([[tok]], [0])
    a = dec.sample_many(prompt, 5, 12, 1.0, 50, seed=3, use_graph=True)
    b = dec.sample_many(prompt, 5, 12, 1.0, 50, seed=3, use_graph=False)
    assert a == b and len({tuple(o) for o in a}) > 1
    assert int(dec.cache.refs.sum()) == 0


def test_out_of_pages_and_refusals():
    from rs_nanogpt_b200.models.paged import PagedDecoder
    from rs_nanogpt_b200.ops import rotary
    from rs_nanogpt_b200.ops._ext import kernel_status
    _, store = _store()
    with pytest.raises(ValueError):
        PagedDecoder(store, 8, 2, 1024)
    dec = PagedDecoder(store, 4, 4, 600, page=32, scaling=rotary.Scaling("parts", 2.0, original_len=512))
    for bad in (lambda: dec.feed([[1], []], [0, 1]), lambda: dec.feed([[1], [2]], [0, 0]), lambda: dec.feed([], []),
                lambda: dec.sample_many([1], 5, 1), lambda: dec.sample_many([], 1, 1),
                lambda: dec.sample_many([1] * 600, 1, 2)):
        with pytest.raises(ValueError):
            bad()
    kernel_status(True)
    with pytest.raises(RuntimeError, match="out of pages"):
        dec.sample_many([1] * 100, 4, 4)
    assert kernel_status(True) == 0
