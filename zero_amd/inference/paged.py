"""Decoding over a paged KV cache: sequences of different lengths in one batch, prompt chunks on a filled cache, trees of
drafted tokens, sampling.

The contiguous cache of inference.decode gives every sequence of a batch one shared length and takes one token a step.
Here a sequence owns pages (``PagedKVCache``), a step carries any number of new tokens per sequence as packed rows
(``Step``), and each layer runs ops.kv_append_paged and ops.attn_paged on them (``forward_paged``).  ``generate_paged`` is
what inference.decode.generate calls for prompts of different lengths and for drafting: a smaller decoder (the surrogate a
target was grafted through shares its tokens) proposes a tree of tokens, the target scores all nodes in one step, and the
path that the target itself would have taken is kept: greedy tokens are those of decoding without a draft and sampled ones
are drawn from the same distributions, up to the rounding of products with other row counts (which can change the places
of near-equal logits, and with them the token that a given number draws)."""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from .. import ops
from ..distributed.tensor_parallel import TPContext
from .decode import BF16, check_drawn, draw_tokens, eos_ids, mlp_infer, qkv_infer


def ancestors(parents: Sequence[int]) -> List[int]:
    """For every node of a tree (parents[i] < i, -1 = the root) the nodes on its path from the root, itself included, as
    an integer of bits."""
    seen: List[int] = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"tree: parent {p} of node {i} does not come before it")
        seen.append((1 << i) | (seen[p] if p >= 0 else 0))
    return seen


def depths(parents: Sequence[int]) -> List[int]:
    out: List[int] = []
    for p in parents:
        out.append(out[p] + 1 if p >= 0 else 0)
    return out


def tree_mask(trees: Sequence[Sequence[int]], device) -> torch.Tensor:
    """ops.attn_paged's mask of a batch of trees, given as the parents of their nodes: int64 [all nodes, words]."""
    words = max(1, -(-max((len(t) for t in trees), default=1) // 64))
    rows = [[(bits >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for t in trees for bits in ancestors(t)]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).reshape(-1, words).view(np.int64)).to(device)


class Step:
    """What one forward over new tokens needs on the device: their positions and cache rows, the lengths with them, and
    which rows of the packed tokens are whose."""

    def __init__(self, positions, slots, ctx, cu, page_table, mask):
        dev = page_table.device
        T, B = len(positions), len(ctx)
        host = torch.tensor(list(positions) + list(slots) + list(ctx) + list(cu), dtype=torch.int32)
        at = host.to(dev)                                            # one copy for all four
        self.positions, self.slots, self.ctx_lens, self.cu_q = at[:T], at[T:2 * T], at[2 * T:2 * T + B], at[2 * T + B:]
        self.tokens, self.cu = T, list(cu)
        self.max_q = max(max(b - a for a, b in zip(cu, cu[1:])), 1)
        self.max_ctx = max(max(ctx), 1)
        self.page_table, self.mask = page_table, mask


class PagedKVCache:
    """Keys (after rotation) and values of ``max_seqs`` sequences in pages of ``page_size`` tokens that are handed out as
    the sequences grow: one tensor [layers, 2, pages, page_size, local kv heads * hd] bf16, so that rows move for all
    layers at once.  ``n_pages`` may be less than max_seqs * max_len needs."""

    def __init__(self, n_layers: int, max_seqs: int, max_len: int, kv_width: int, device, page_size: int = 64,
                 n_pages: Optional[int] = None):
        if min(n_layers, max_seqs, max_len, kv_width, page_size) <= 0:
            raise ValueError("PagedKVCache: sizes must be positive")
        cols = -(-max_len // page_size)
        self.n_pages = max_seqs * cols if n_pages is None else int(n_pages)
        self.page_size, self.max_len, self.max_seqs = page_size, max_len, max_seqs
        self.kv = torch.empty((n_layers, 2, self.n_pages, page_size, kv_width), dtype=BF16, device=device)
        self.lengths = [0] * max_seqs
        self.pages: List[List[int]] = [[] for _ in range(max_seqs)]
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._host_table = torch.full((max_seqs, cols), -1, dtype=torch.int32)
        self._table: Optional[torch.Tensor] = None

    @classmethod
    def for_decoder(cls, decoder, max_seqs: int, max_len: int, device, page_size: int = 64, n_pages=None):
        layers = decoder.model.layers[: decoder.config.num_hidden_layers]
        return cls(len(layers), max_seqs, max_len, layers[0].self_attn.k_proj.weight.shape[0], device, page_size, n_pages)

    @property
    def page_table(self) -> torch.Tensor:
        if self._table is None:
            self._table = self._host_table.to(self.kv.device)
        return self._table

    def grow(self, b: int, rows: int):
        """Pages for ``rows`` rows of sequence b."""
        self._grow_all([(b, rows)])

    def _grow_all(self, wanted):
        """Pages for (sequence, rows) pairs: for all of them, or, refused, for none."""
        need = []
        for b, rows in wanted:
            if rows > self.max_len:
                raise ValueError(f"KV cache too small: {rows} > {self.max_len}")
            need.append(max(-(-rows // self.page_size) - len(self.pages[b]), 0))
        if sum(need) > len(self._free):
            raise RuntimeError(f"KV cache out of pages: {sum(need)} needed (of sequences "
                               f"{[b for (b, _), n in zip(wanted, need) if n]}), {len(self._free)} are free")
        for (b, _), n in zip(wanted, need):
            for _ in range(n):
                pg = self._free.pop()
                self._host_table[b, len(self.pages[b])] = pg
                self.pages[b].append(pg)
                self._table = None

    def truncate(self, b: int, rows: int):
        """Sequence b ends at ``rows``; pages past it go back."""
        self.lengths[b] = min(self.lengths[b], rows)
        while len(self.pages[b]) > -(-rows // self.page_size):
            self._free.append(self.pages[b].pop())
            self._host_table[b, len(self.pages[b])] = -1
            self._table = None

    def release(self, b: int):
        self.truncate(b, 0)

    def row(self, b: int, r: int) -> int:
        """Flat cache row of row r of sequence b."""
        return self.pages[b][r // self.page_size] * self.page_size + r % self.page_size

    def step(self, counts: Sequence[int], trees: Optional[Sequence[Sequence[int]]] = None) -> Step:
        """The next ``counts[b]`` tokens of every sequence (0 allowed), behind its length, as a chain, or as the trees
        ``trees[b]`` of parents (counts[b] nodes).  The lengths move with ``advance``, so that a step may be repeated."""
        if len(counts) != self.max_seqs or sum(counts) <= 0 or min(counts) < 0:
            raise ValueError("step: a count for each sequence, and some token")
        if trees is not None and [len(t) for t in trees] != list(counts):
            raise ValueError("step: trees and counts differ")
        mask = None if trees is None else tree_mask(trees, self.kv.device)       # (refuses what is no tree, before pages go)
        self._grow_all([(b, self.lengths[b] + n) for b, n in enumerate(counts)])
        positions, slots, ctx, cu = [], [], [], [0]
        for b, n in enumerate(counts):
            base = self.lengths[b]
            positions += [base + d for d in (range(n) if trees is None else depths(trees[b]))]
            slots += [self.row(b, base + i) for i in range(n)]
            ctx.append(base + n)
            cu.append(cu[-1] + n)
        return Step(positions, slots, ctx, cu, self.page_table, mask)

    def advance(self, counts: Sequence[int]):
        for b, n in enumerate(counts):
            self.lengths[b] += n

    def keep(self, paths: Sequence[Sequence[int]]):
        """After a step of trees: the nodes ``paths[b]`` (a path from the root, in order) become the next rows of sequence
        b, the others are dropped."""
        src, dst = [], []
        for b, path in enumerate(paths):
            base = self.lengths[b]
            for d, node in enumerate(path):
                if node != d:
                    src.append(self.row(b, base + node))
                    dst.append(self.row(b, base + d))
        if src:
            rows = self.kv.view(-1, self.n_pages * self.page_size, self.kv.shape[-1])
            at = torch.tensor([src, dst], dtype=torch.int64).to(rows.device)
            rows.index_copy_(1, at[1], rows.index_select(1, at[0]))      # all read before the first is written
        for b, path in enumerate(paths):
            self.lengths[b] += len(path)
            self.truncate(b, self.lengths[b])


@torch.no_grad()
def forward_paged(decoder, x: torch.Tensor, cache: PagedKVCache, step: Step, rows: Optional[torch.Tensor] = None,
                  tp: Optional[TPContext] = None) -> torch.Tensor:
    """x [T, d]: embeddings of the step's packed tokens.  Appends their keys and values and returns the logits [T, V] (or
    of the rows listed in ``rows``, int64) in bf16.  The cache's lengths stay: see ``advance`` / ``keep``."""
    tp = tp or TPContext()
    model = decoder.model
    if x.shape[0] != step.tokens:
        raise ValueError(f"forward_paged: {x.shape[0]} rows for a step of {step.tokens} tokens")
    cos_t, sin_t = model.rotary_emb.tables(cache.max_len, x.device)
    h = x.to(BF16).contiguous()
    for li, layer in enumerate(model.layers[: decoder.config.num_hidden_layers]):
        a, (_, _, hd, _) = layer.self_attn, layer.cfg_dims
        nh, nkv = a.q_proj.weight.shape[0] // hd, a.k_proj.weight.shape[0] // hd      # local (sharded) head counts
        k, v = cache.kv[li, 0], cache.kv[li, 1]
        q = ops.kv_append_paged(qkv_infer(layer, h), cos_t, sin_t, k, v, step.positions, step.slots, nh, nkv, hd)
        ao = ops.attn_paged(q, k, v, step.page_table, step.ctx_lens, step.cu_q, step.max_q, step.max_ctx, nh, nkv, hd,
                            hd ** -0.5, tree_mask=step.mask)
        # row-parallel projections: every rank holds a slice of the contraction; ONE rank adds the residual
        xa = tp.reduce(ops.gemm(ao, a.o_proj.weight.detach(), residual=h if tp.lead else None))
        h = mlp_infer(layer, xa, tp)
    if rows is not None:
        h = h.index_select(0, rows)
    hn, _ = ops.rmsnorm_fwd(h, model.norm.weight, model.norm.variance_epsilon, save_stats=False)
    return ops.gemm(hn, decoder.lm_head.weight.detach())


def _embed(decoder, tokens: Sequence[int], device) -> torch.Tensor:
    return decoder.model.get_input_embeddings()(torch.tensor(list(tokens), dtype=torch.int64).to(device))


def draft_tree(width: int, depth: int) -> List[int]:
    """Parents of ``width`` chains of ``depth`` nodes under a common root, level by level."""
    return [-1] + [0 if level == 0 else 1 + (level - 1) * width + c for level in range(depth) for c in range(width)]


def accepted_path(parents: Sequence[int], tokens: Sequence[int], drawn: Sequence[int]) -> List[int]:
    """The nodes from the root on that a decoder which drew ``drawn[i]`` after node i would have taken: a child is taken if
    its token is the one drawn after its parent (the first of equal ones)."""
    path = [0]
    while True:
        nxt = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == drawn[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


def _assistant_tp(assistant, tp: TPContext) -> TPContext:
    """How the assistant runs beside a decoder of the group ``tp``: split over the same ranks, or whole on each of them (all
    draft alike: equal weights, equal tokens, kernels that repeat themselves bit for bit)."""
    layer = assistant.model.layers[0]
    nh, _, hd, _ = layer.cfg_dims
    parts = nh * hd // layer.self_attn.q_proj.weight.shape[0]
    if parts != tp.world and parts != 1:
        raise ValueError(f"generate: the assistant is split over {parts} ranks, the decoder's group has {tp.world}")
    return tp if parts == tp.world else TPContext()


def _draft(assistant, cache: PagedKVCache, roots: Sequence[Optional[int]], width: int, depth: int, tp) -> List[List[int]]:
    """Tokens of the tree draft_tree(width, depth) under each root (None: a finished sequence, no nodes): the ``width``
    likeliest after the root, then the likeliest after each.  Each level runs the nodes so far again, as the tree of one
    step: an earlier step's rows would be seen by all branches."""
    device = cache.kv.device
    tokens = [[] if r is None else [r] for r in roots]
    live = [b for b, r in enumerate(roots) if r is not None]
    for level in range(depth):
        trees = [draft_tree(width, level) if t else [] for t in tokens]
        step = cache.step([len(t) for t in trees], trees)
        last = [step.cu[b + 1] - 1 - i for b in live for i in reversed(range(width if level else 1))]
        logits = forward_paged(assistant, _embed(assistant, [t for ts in tokens for t in ts], device), cache, step,
                               torch.tensor(last).to(device), tp)
        top = logits.float().topk(width, -1).indices if level == 0 else logits.float().argmax(-1).view(-1, width)
        for b, new in zip(live, top.tolist()):
            tokens[b] += new
    return tokens


@torch.no_grad()
def generate_paged(decoder, prompts: Sequence[torch.Tensor], max_new_tokens: int, eos_token_id=None, pad_token_id=None,
                   sampling: Optional[dict] = None, generator=None, assistant=None, draft_width: int = 2,
                   draft_depth: int = 4, page_size: int = 64, tp: Optional[TPContext] = None,
                   assistant_prompts: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """New token ids [B, <= max_new_tokens] (int64) for prompts [S_b, d] of any lengths; sequences that ended are filled
    with ``pad_token_id``.  ``sampling``: ops.sample's settings (None: the largest logit).  ``assistant``: a decoder of the
    same vocabulary that drafts draft_width chains of draft_depth tokens a step (its prompts default to the decoder's); under
    tensor parallelism split over the same ranks as the decoder, or whole on every rank."""
    tp = tp or TPContext()
    if not prompts:
        raise ValueError("generate: no prompts")
    if assistant_prompts is not None and len(assistant_prompts) != len(prompts):
        raise ValueError(f"generate: {len(assistant_prompts)} prompts for the assistant, {len(prompts)} for the decoder")
    B, device = len(prompts), prompts[0].device
    eos, pad = eos_ids(decoder, eos_token_id, pad_token_id)
    pad = 0 if pad is None else pad
    if max_new_tokens <= 0:
        return torch.empty((B, 0), dtype=torch.int64, device=device)
    nodes = 1 + draft_width * draft_depth if assistant is not None else 1
    if assistant is not None and (draft_width < 1 or draft_depth < 1):
        raise ValueError("generate: draft_width and draft_depth must be positive")
    if assistant is not None and assistant.lm_head.weight.shape[0] != decoder.lm_head.weight.shape[0]:
        raise ValueError(f"generate: vocabularies differ: {assistant.lm_head.weight.shape[0]} tokens of the assistant, "
                         f"{decoder.lm_head.weight.shape[0]} of the decoder")
    helper_tp = None if assistant is None else _assistant_tp(assistant, tp)
    u = None
    if sampling is not None:                             # the numbers that decode.generate draws; drafts past the end: any
        u = torch.rand((max_new_tokens, B), generator=generator, device=device)
        u = torch.cat([u, torch.zeros((nodes, B), device=device)])

    def fill(dec, rows, tp):
        lens = [int(p.shape[0]) for p in rows]
        if min(lens) == 0:
            raise ValueError("generate: an empty prompt")
        d = dec.config.hidden_size
        if any(p.dim() != 2 or p.shape[1] != d for p in rows):
            raise ValueError(f"generate: prompts must be [tokens, {d}] (an assistant of another width needs its own)")
        c = PagedKVCache.for_decoder(dec, B, max(lens) + max_new_tokens + nodes, device, page_size)
        st = c.step(lens)
        ends = torch.tensor([e - 1 for e in st.cu[1:]]).to(device)
        logits = forward_paged(dec, torch.cat([p.to(BF16) for p in rows]), c, st, ends, tp)
        c.advance(lens)
        return c, logits

    def draw(logits, where):                             # where: (sequence, index of the token) of every row
        if sampling is None:
            return draw_tokens(logits, None, None).tolist()
        us = u[torch.tensor([i for _, i in where]).to(device), torch.tensor([b for b, _ in where]).to(device)]
        return draw_tokens(logits, us, sampling).tolist()

    cache, logits = fill(decoder, prompts, tp)
    helper = None
    if assistant is not None:
        helper, _ = fill(assistant, prompts if assistant_prompts is None else assistant_prompts, helper_tp)
    out: List[List[int]] = [[] for _ in range(B)]
    done = [False] * B

    def emit(b, token):                                  # (a row that is not taken may have nothing to draw from)
        if not done[b]:
            out[b].append(check_drawn([token])[0])
            done[b] = token in eos or len(out[b]) >= max_new_tokens

    for b, t in enumerate(draw(logits, [(b, 0) for b in range(B)])):
        emit(b, t)
    while not all(done):
        roots = [None if done[b] else out[b][-1] for b in range(B)]
        if helper is None:
            tokens = [[] if r is None else [r] for r in roots]
            trees = [[-1] * len(t) for t in tokens]
        else:
            tokens = _draft(assistant, helper, roots, draft_width, draft_depth, helper_tp)
            trees = [draft_tree(draft_width, draft_depth) if t else [] for t in tokens]
            # the assistant's rows of the last level: its step stopped one level short of them
            st = helper.step([len(t) for t in trees], trees)
            forward_paged(assistant, _embed(assistant, [t for ts in tokens for t in ts], device), helper, st,
                          torch.zeros(1, dtype=torch.int64, device=device), helper_tp)
        step = cache.step([len(t) for t in trees], trees if helper is not None else None)
        logits = forward_paged(decoder, _embed(decoder, [t for ts in tokens for t in ts], device), cache, step, None, tp)
        where = [(b, len(out[b]) + d) for b in range(B) for d in depths(trees[b])]
        drawn = draw(logits, where)
        paths, at = [], 0
        for b in range(B):
            n = len(tokens[b])
            mine = drawn[at:at + n]
            path = accepted_path(trees[b], tokens[b], mine) if n else []
            at += n
            paths.append(path)
            for node in path:
                emit(b, mine[node])
        cache.keep(paths)
        if helper is not None:
            helper.keep(paths)
    length = max(len(o) for o in out)
    return torch.tensor([o + [pad] * (length - len(o)) for o in out], dtype=torch.int64, device=device)
