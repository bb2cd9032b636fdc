"""Paged KV cache operators (kernels: ``csrc/kernels/pages.cu``,
``csrc/kernels/rotary.cu``, ``csrc/kernels/paged_attn.cu``).

A cache is a pool of pages, ``k`` and ``v`` of shape (layers, pages, kv heads,
rows of a page, head_dim), and three int32 tensors on the device:

* ``table`` (slots, width)  the pages of each slot's sequence in order, -1 past the last
* ``lens``  (slots)         its tokens; 0 means the slot is empty
* ``refs``  (pages)         how many table entries name the page; 0 means it is free

Sequences that were forked from one another share their full pages; a partly
filled page belongs to one sequence, so appending never needs a copy. The state
operators return ``(table, lens, refs)``; ``out`` takes three tensors for the
result, which may be the inputs themselves (in place) and are fresh ones by
default. No operator waits for the device: pages that run out or an index out
of range are reported by ``kernel_status`` and the entry concerned is skipped.

A fourth tensor, ``room`` (slots) int32, zero at first, keeps apart the tokens
that ``grow_pages`` granted and those that are written: growing adds to it,
``append`` writes no more of a slot's tokens than it says, and whoever has
written a slot's tokens (into all layers) sets its entry to 0. It is optional;
without it, an append after a growth that was refused writes over the last
tokens that the cache holds, in pages that others may share, so the caller has
to look at ``kernel_status`` in between.
"""
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import rotary
from ._ext import count_launches, ext

State = Tuple[torch.Tensor, torch.Tensor, torch.Tensor]


def _out(table, lens, refs, out) -> State:
    return (torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)) if out is None else out


def fork_pages(k, v, table, lens, refs, parents, children, out: Optional[State] = None) -> State:
    """Make slot ``children[i]`` (empty; int32) a copy of slot ``parents[i]``.
    Full pages are shared; the filled rows of a partly filled last page go to
    the lowest free page, in the list's order. A child that is not empty, named
    twice (its first mention counts), out of range or without a page to be had
    is skipped and reported."""
    out = _out(table, lens, refs, out)
    ext().pages_fork(k, v, table, lens, refs, parents, children, *out)
    return out


def grow_pages(table, lens, refs, add, page: int, out: Optional[State] = None,
               room: Optional[torch.Tensor] = None) -> State:
    """Make room for ``add[s]`` (int32, one a slot) more tokens in every slot:
    ``lens`` grows by it and missing pages are the lowest free ones, in the
    order of the slots. A slot that lacks more pages than are left when its turn
    comes keeps its length, is reported and takes nothing from those after it.
    What is granted is added to ``room``."""
    out = _out(table, lens, refs, out)
    ext().pages_grow(table, lens, refs, add, page, *out, room)
    return out


def free_pages(table, lens, refs, seqs, out: Optional[State] = None, room: Optional[torch.Tensor] = None) -> State:
    """Empty the slots ``seqs`` (int32); pages that nobody else holds are free.
    The slots' entries of ``room`` become 0."""
    out = _out(table, lens, refs, out)
    ext().pages_free(table, lens, refs, seqs, *out, room)
    return out


def compact_pages(k, v, table, lens, refs, out: Optional[State] = None) -> State:
    """Move pages so that the L ones in use are the first L of the pool: the
    i-th page in use past L (ascending) takes the i-th free number below L."""
    out = _out(table, lens, refs, out)
    ext().pages_compact(k, v, table, lens, refs, *out)
    return out


def copy_pages(k, v, src, dst) -> None:
    """Copy pages ``src[i]`` to ``dst[i]`` (int32) in every layer of k and v.
    Pairs with a negative source are skipped; no page may be both a source and
    a target, nor a target twice."""
    ext().pages_copy(k, v, src, dst)


# (row, query head) pairs of an item, as in csrc/kernels/paged_attn.cuh: up to
# SMALL_ROWS on mma.sync, up to BIG_ROWS (two tiles of 128) on tcgen05. Runs of more
# than BIG_FROM pairs go to tcgen05: 64 rows of one prefix of 1984 tokens take 30.6 us
# as four items on mma.sync and 40.7 us there, 128 rows of 8192 tokens 87.7 and 65.2 us.
SMALL_ROWS, BIG_ROWS, BIG_FROM, BIG = 16, 256, 64, 1 << 30


def _cost(pairs, keys, over: int):
    """Time of a run of ``keys`` keys for ``pairs`` pairs, in tiles of the tcgen05
    kernel (2.3 us of an SM); a tile of a warp on mma.sync takes 0.036 of one, and
    an item as long as ``over`` tiles before its first."""
    big = -(-pairs // BIG_ROWS) * (over + -(-keys // 128))
    small = -(-pairs // SMALL_ROWS) * (over + -(-keys // 32)) * 0.036
    return np.where(pairs > BIG_FROM, big, small)


class PrefixPlan:
    """Which rows belong to which sequence and which sequences share a prefix.

    ``groups`` lists (sequences, shared tokens): so many sequences, one after
    another, whose first ``shared`` tokens (whole pages) lie in the same pages.
    ``q_lens`` is the number of new tokens of each sequence (one number for
    all, or a list); the rows of q, k and v hold them one sequence after another.
    ``slots`` names each sequence's row of the cache's table (0, 1, 2, ... by
    default). A plan depends on nothing that changes from step to step, so one
    plan serves every layer and every step of a batch, and a captured graph.
    Making one takes the host 0.3 ms for a few sequences to 0.8 ms for 256 (lists
    in Python, eight copies to the device), more than the attention of one layer:
    it is meant to be kept."""

    def __init__(self, groups: Sequence[Tuple[int, int]], q_lens: Union[int, Sequence[int]] = 1, *, n_head: int,
                 n_kv_head: int, head_dim: int, page: int, table_width: int, slots: Optional[Sequence[int]] = None,
                 device="cuda"):
        n_seq = sum(n for n, _ in groups)
        if n_kv_head <= 0 or n_head % n_kv_head:
            raise ValueError(f"{n_head} query heads cannot share {n_kv_head} kv heads")
        if any(n < 0 or s < 0 or s % page or s > table_width * page for n, s in groups):
            raise ValueError(f"groups must be (sequences, shared tokens), shared a multiple of the page ({page}) "
                             f"within the table ({table_width} pages): {list(groups)}")
        t = np.full(n_seq, q_lens, np.int64) if isinstance(q_lens, int) else np.asarray(list(q_lens), np.int64)
        if len(t) != n_seq or (t < 0).any():
            raise ValueError(f"q_lens must be one length for each of the {n_seq} sequences")
        slot = np.arange(n_seq) if slots is None else np.asarray(list(slots), np.int64)
        if len(slot) != n_seq or (slot < 0).any():
            raise ValueError(f"slots must be one table row for each of the {n_seq} sequences")
        share = n_head // n_kv_head
        self.rows, self.share, self.max_slot = int(t.sum()), share, int(slot.max(initial=-1))
        self.max_shared = max((s for _, s in groups), default=0)
        self.n_head, self.n_kv_head, self.head_dim, self.page, self.table_width = (n_head, n_kv_head, head_dim, page,
                                                                                   table_width)
        start = np.concatenate([[0], np.cumsum(t)])
        seq = np.repeat(np.arange(n_seq), t)
        back = start[seq + 1] - 1 - np.arange(self.rows)
        lists, of_pair = ([], []), np.full((2, self.rows * share), -1, np.int64)

        def add(shared, first, count, row0, row1, key0, keys, alone=0):
            pairs = (row1 - row0) * share
            big = int(pairs > BIG_FROM)
            items, most = lists[big], (SMALL_ROWS, BIG_ROWS)[big]
            for r in range(0, pairs, most):
                n = min(most, pairs - r)
                p0 = row0 * share + r
                of_pair[shared, p0:p0 + n] = len(items) + BIG * big
                after = keys if shared else back[(p0 + n - 1) // share]
                items.append((shared, first, count, p0, n, key0, after, alone))

        at = 0
        own_from = np.zeros(n_seq, np.int64)
        for n, shared in groups:
            # The shared keys as a run of their own, for the rows of all: its tiles are
            # fuller, but it is an item more and every pair has two runs to join (0.018
            # of a tile's time for 100 values). Prompts of many tokens fill their tiles
            # alone, and short prefixes are soon read again.
            pairs = t[at:at + n] * share
            apart = _cost(pairs, shared, 0).sum()
            together = _cost(pairs.sum(), shared, 3) + pairs.sum() * head_dim * 1.8e-4
            if n > 1 and shared > 0 and apart > together:
                add(1, at, n, start[at], start[at + n], 0, shared)
                own_from[at:at + n] = shared
            at += n
        for s in range(n_seq):
            add(0, slot[s], 1, start[s], start[s + 1], own_from[s], 0, int(own_from[s] == 0))

        def dev(x):
            return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).to(device)

        kinds = sum(1 for x in lists if x)
        self.launches = kinds + (kinds > 0)  # of an attention call: a kernel for either kind of items, and the join
        self.items, self.big_items = (dev(np.asarray(x, np.int64).reshape(-1, 8)) for x in lists)
        self.shared_item, self.own_item = dev(of_pair[1]), dev(of_pair[0])
        self.slot_of_seq, self.row_slot, self.row_back = dev(slot), dev(slot[seq]), dev(back)


def append(q, k, v, k_pages, v_pages, table, lens, plan: PrefixPlan, cos=None, sin=None, layout: str = "half",
           qk_eps: Optional[float] = None, q_out: Optional[torch.Tensor] = None,
           room: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Write the new tokens' keys and values into one layer's pages (pages, kv
    heads, rows of a page, head_dim), turned by their positions (``cos``,
    ``sin`` of ``rotary.tables``; none: not turned) and, with ``qk_eps``, each
    head of q and k divided by its root mean square as the model does after
    RoPE (rs-nanogpt src/model/attention.rs:68-116), which takes a factor common
    to ``cos`` and ``sin`` out again (see ``rotary.Scaling``). ``lens`` counts the new
    tokens already (``grow_pages`` comes first); with ``room``, tokens that it
    did not grant are left out and reported. Returns q, turned and normed alike,
    in ``q_out`` (which may be q); rows without a place in the cache, those
    of an empty slot among them, are 0 there."""
    if q_out is None:
        q_out = torch.empty_like(q)
    ext().paged_append(q, k, v, k_pages, v_pages, table, lens, plan.row_slot, plan.row_back, cos, sin,
                       rotary.interleaved(layout), 0.0 if qk_eps is None else qk_eps, qk_eps is not None, q_out,
                       room)
    return q_out


def attention(q, k_pages, v_pages, table, lens, plan: PrefixPlan, out: Optional[torch.Tensor] = None,
              lse: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of the new tokens ``q`` (rows, heads, head_dim) over one
    layer's pages, the keys that a group shares read once for all its rows.
    ``lens`` counts the new tokens; the last of them sees all of its sequence. A
    row without keys (an empty slot) gives 0. A NaN or infinite value reaches
    the rows that see its key and no others. The probabilities are rounded to
    the values' type before they meet them, their sum is not. ``out`` may be q. ``lse`` (rows, heads) fp32 takes
    the log of each row's softmax sum (-inf without keys). ``scale`` is
    1 / sqrt(head_dim) by default."""
    if out is None:
        out = torch.empty_like(q)
    ext().paged_attention(q, k_pages, v_pages, table, lens, plan.items, plan.big_items, plan.slot_of_seq, plan.row_slot,
                          plan.row_back, plan.shared_item, plan.own_item, plan.max_slot, plan.page,
                          plan.max_shared, q.shape[-1] ** -0.5 if scale is None else scale, out, lse)
    count_launches(plan.launches)
    return out
