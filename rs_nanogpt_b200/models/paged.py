"""Generation over a paged KV cache whose sequences share prefixes.

``PagedCache`` owns the pages of all layers, the page tables, lengths and
reference counts (``rs_nanogpt_b200.ops.paged``). ``PagedDecoder`` runs the GPT
over it: ``feed`` appends any number of new tokens to any of its sequences and
returns the logits of each one's last token; ``fork`` copies sequences without
copying what they share; ``sample_many`` draws many completions of one prompt,
which is prefilled, stored and, in every decode step, read once for all of them.

The decoder's positions may go past the trained ``sequence_len`` with a
``rotary.Scaling``. Its sums are the cached forward's of ``models/decode.py``
(rs-nanogpt src/model/gpt.rs:80-131) except that the divisor of the q/k norm is
kept in fp32 instead of being rounded to bf16 first, and that the softmax's
probabilities are rounded to bf16 before they meet the values, as in the
training forward; the decode step there keeps them in fp32.
"""
from typing import List, Optional, Sequence, Tuple

import torch

from ..ops import gemm, paged, rotary
from ..ops import layers as L
from ..ops._ext import kernel_status
from .decode import draw_uniforms
from .params import ParamStore


class PagedCache:
    """Pages (layers, pages, kv heads, page, head_dim) for up to ``max_seqs``
    sequences of up to ``max_len`` tokens. All changes are made on the device
    and in place; ``check`` (which waits for the current stream) raises when
    pages ran out."""

    def __init__(self, n_layer: int, n_kv_head: int, head_dim: int, pages: int, page: int, max_seqs: int, max_len: int,
                 dtype=torch.bfloat16, device="cuda"):
        if min(pages, page, max_seqs, max_len) <= 0:
            raise ValueError("paged cache: pages, page, max_seqs and max_len must be positive")
        self.page, self.width = page, -(-max_len // page)
        shape = (n_layer, pages, n_kv_head, page, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.table = torch.full((max_seqs, self.width), -1, **ints)
        self.lens = torch.zeros(max_seqs, **ints)
        self.refs = torch.zeros(pages, **ints)
        self.room = torch.zeros(max_seqs, **ints)  # tokens granted and not yet written

    @property
    def state(self) -> paged.State:
        return self.table, self.lens, self.refs

    def _list(self, x) -> torch.Tensor:
        return torch.as_tensor(x, dtype=torch.int32, device=self.table.device)

    def grow(self, add) -> None:
        """Room for ``add[s]`` more tokens in every slot ``s``."""
        paged.grow_pages(*self.state, self._list(add), self.page, out=self.state, room=self.room)

    def fork(self, parents, children) -> None:
        paged.fork_pages(self.k, self.v, *self.state, self._list(parents), self._list(children), out=self.state)

    def free(self, seqs) -> None:
        paged.free_pages(*self.state, self._list(seqs), out=self.state, room=self.room)

    def compact(self) -> None:
        paged.compact_pages(self.k, self.v, *self.state, out=self.state)

    def check(self) -> None:
        torch.cuda.current_stream(self.table.device).synchronize()  # the status is read on the default stream
        status = kernel_status()
        if status == 6:
            raise RuntimeError("paged cache: out of pages")
        if status:
            raise RuntimeError(f"paged cache: kernel status {status}")


class PagedDecoder:
    def __init__(self, store: ParamStore, pages: int, max_seqs: int, max_len: int, page: int = 64,
                 scaling: Optional[rotary.Scaling] = None):
        cfg = store.cfg
        if store.device.type != "cuda" or store.work is None:
            raise ValueError("PagedDecoder needs a CUDA parameter store with its bf16 working copy")
        if cfg.head_dim not in (64, 128):
            raise ValueError(f"PagedDecoder supports head_dim 64 and 128, got {cfg.head_dim}")
        if scaling is None and max_len > cfg.sequence_len:
            raise ValueError(f"max_len ({max_len}) exceeds sequence_len ({cfg.sequence_len}) without rotary scaling")
        self.store, self.cfg, self.max_len = store, cfg, max_len
        self.cache = PagedCache(cfg.n_layer, cfg.n_head, cfg.head_dim, pages, page, max_seqs, max_len,
                                device=store.device)
        # q and k are normed after the turn, so the scaling's factor on them goes into the scores.
        self.cos, self.sin = rotary.tables(cfg.head_dim, self.cache.width * page, cfg.rope_base, scaling, store.device,
                                           sharpen=False)
        self.scale = cfg.head_dim ** -0.5 * (scaling.sharpening ** 2 if scaling else 1.0)

    def plan(self, groups: Sequence[Tuple[int, int]], q_lens,
             slots: Optional[Sequence[int]] = None) -> paged.PrefixPlan:
        """Sequences ``slots`` in ``groups`` of (count, shared tokens), as ``PrefixPlan``."""
        cfg = self.cfg
        return paged.PrefixPlan(groups, q_lens, n_head=cfg.n_head, n_kv_head=cfg.n_head, head_dim=cfg.head_dim,
                                page=self.cache.page, table_width=self.cache.width, slots=slots,
                                device=self.store.device)

    @torch.no_grad()
    def forward(self, ids: torch.Tensor, plan: paged.PrefixPlan) -> torch.Tensor:
        """``ids`` (rows,) int64 on the device: the new tokens of the plan's
        sequences, one sequence after another; the cache has grown by them.
        Rows of a slot that could not grow are written nowhere (and reported).
        Returns the final normed hidden states (rows, C)."""
        cfg, st, cache = self.cfg, self.store, self.cache
        n, c, h, eps = ids.shape[0], cfg.n_embd, cfg.n_head, cfg.norm_eps
        x = L.embedding(ids, st.work_of("wte.weight"))
        y = torch.empty_like(x)
        for i in range(cfg.n_layer):
            p = f"blocks.{i}."
            qkv = gemm.linear(L.rmsnorm(x, eps), st.qkv_work(i))
            q, k, v = qkv.view(n, 3, h, cfg.head_dim).unbind(1)
            paged.append(q, k, v, cache.k[i], cache.v[i], cache.table, cache.lens, plan, self.cos, self.sin, qk_eps=eps,
                         q_out=q, room=cache.room)
            paged.attention(q, cache.k[i], cache.v[i], cache.table, cache.lens, plan, out=y.view(n, h, cfg.head_dim),
                            scale=self.scale)
            x = gemm.linear_residual(y, st.work_of(p + "attn.c_proj.weight"), x)
            a = gemm.linear_relu2_act(L.rmsnorm(x, eps), st.work_of(p + "mlp.c_fc.weight"))
            x = gemm.linear_residual(a, st.work_of(p + "mlp.c_proj.weight"), x)
        cache.room.index_fill_(0, plan.row_slot.long(), 0)
        return L.rmsnorm(x, eps)

    def _check_fits(self, slots: Sequence[int], new: Sequence[int]) -> None:
        """Reads the cache's lengths and free pages: the growth that follows is granted whole."""
        cache = self.cache
        *held, free = torch.cat([cache.lens, (cache.refs <= 0).sum(dtype=torch.int32).view(1)]).tolist()
        need = 0
        for s, n in zip(slots, new):
            if held[s] + n > self.max_len:
                raise ValueError(f"feed: {held[s]} tokens in slot {s} and {n} new ones exceed max_len ({self.max_len})")
            need += -(-(held[s] + n) // cache.page) - -(-held[s] // cache.page)
        if need > free:
            raise RuntimeError(f"paged cache: out of pages ({need} needed, {free} free)")

    @torch.no_grad()
    def feed(self, tokens: Sequence[Sequence[int]], slots: Sequence[int],
             groups: Optional[Sequence[Tuple[int, int]]] = None) -> torch.Tensor:
        """Append ``tokens[i]`` to the sequence in slot ``slots[i]``; ``groups``
        as in ``plan`` (none: nothing shared). Returns the (sequences, vocab)
        bf16 logits of their last tokens. Raises, and leaves the cache as it
        was, where a sequence would pass ``max_len`` or the pages run out."""
        lens = [len(t) for t in tokens]
        if not lens or min(lens) == 0 or len(slots) != len(tokens) or len(set(slots)) != len(slots):
            raise ValueError("feed: one slot of its own and at least one token for each sequence")
        if min(slots) < 0 or max(slots) >= self.cache.lens.shape[0]:
            raise ValueError(f"feed: slots must be below {self.cache.lens.shape[0]}, got {list(slots)}")
        ids = [t for s in tokens for t in s]
        if min(ids) < 0 or max(ids) >= self.cfg.vocab_size:
            raise ValueError(f"feed: token ids must be below the vocabulary's size, {self.cfg.vocab_size}")
        dev = self.store.device
        plan = self.plan(groups or [(len(tokens), 0)], lens, slots)
        self._check_fits(slots, lens)
        add = torch.zeros_like(self.cache.lens)
        add[torch.tensor(list(slots), device=dev)] = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.cache.grow(add)  # after all checks: a refused call leaves the cache as it was
        hidden = self.forward(torch.tensor(ids, dtype=torch.int64, device=dev), plan)
        last = torch.tensor(lens, device=dev).cumsum(0) - 1
        return gemm.linear(hidden[last], self.store.work_of("lm_head.weight"))

    @torch.no_grad()
    def sample_many(self, prompt: Sequence[int], n: int, max_new: int, temperature: float = 1.0, top_k: int = 50,
                    seed: int = 0, use_graph: bool = True) -> List[List[int]]:
        """``n`` completions of ``max_new`` tokens of one prompt, in slots 0..n-1,
        which have to be empty (and are emptied again at the end). The prompt is prefilled
        once and forked; a decode step is one graph replay."""
        cache, dev, v = self.cache, self.store.device, self.cfg.vocab_size
        if not 0 < n <= cache.lens.shape[0] or max_new <= 0 or not prompt:
            raise ValueError("sample_many: a prompt, up to max_seqs samples and at least one new token")
        if len(prompt) + max_new - 1 > self.max_len:
            raise ValueError(f"sample_many: prompt ({len(prompt)}) + {max_new} new tokens exceed max_len "
                             f"({self.max_len})")
        if cache.lens[:n].any():
            raise ValueError(f"sample_many: slots 0 to {n - 1} have to be empty")
        logits = self.feed([prompt], [0]).expand(n, v).contiguous()
        cache.fork([0] * (n - 1), list(range(1, n)))
        shared = len(prompt) // cache.page * cache.page
        plan = self.plan([(n, shared)], 1)
        out = torch.zeros(n, max_new, device=dev, dtype=torch.int32)
        uniforms = draw_uniforms(seed, max_new, n).to(dev)
        count, unused = (torch.zeros(n, device=dev, dtype=torch.int32) for _ in range(2))
        ids = torch.zeros(n, device=dev, dtype=torch.int64)
        one = torch.zeros_like(cache.lens)
        one[:n] = 1

        def sample():
            L.sample_tokens(logits, temperature, top_k, uniforms, count, out, ids, unused, False)

        def step():
            cache.grow(one)
            logits.copy_(gemm.linear(self.forward(ids, plan), self.store.work_of("lm_head.weight")))
            sample()

        sample()
        steps = max_new - 1
        if use_graph and steps > 2:
            step()  # also sets the kernels' attributes, which a capture may not
            side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
            for _ in range(steps - 1):
                graph.replay()
        else:
            for _ in range(steps):
                step()
        cache.free(list(range(n)))
        cache.check()
        return out.tolist()
