"""generate_paged's bookkeeping on the CPU: the decoders are stand-ins whose next token is a function of the tokens that a
row sees, read back from the cache rows, page table, lengths and masks that the attention kernel would be given.  What a
draft has to see, which drafts are accepted and what stays in both caches is then exact."""
from types import SimpleNamespace

import pytest
import torch

from zero_amd.distributed.tensor_parallel import TPContext
from zero_amd.inference import paged

V, D = 50, 4


class Model:
    """rule(tokens) -> next token.  ``seen``: (tokens, next) of every row of every step; ``steps``: rows and tp of each."""

    def __init__(self, rule, vocab=V, world=1):
        w = lambda *s: SimpleNamespace(weight=torch.zeros(*s))  # noqa: E731
        layer = SimpleNamespace(self_attn=SimpleNamespace(q_proj=w(8 // world, D), k_proj=w(4 // world, D)),
                                cfg_dims=(4, 2, 2, 1e-5))
        self.rule, self.vocab = rule, vocab
        self.config = SimpleNamespace(hidden_size=D, num_hidden_layers=1, vocab_size=vocab)
        self.generation_config = None
        self.lm_head = w(vocab, D)
        self.model = SimpleNamespace(layers=[layer], get_input_embeddings=lambda: self.embed)
        self.seen, self.steps = [], []

    def embed(self, ids):
        assert int(ids.max()) < self.vocab and int(ids.min()) >= 0          # (the real gather reads what is there)
        return torch.nn.functional.pad(ids[:, None].to(torch.bfloat16), (0, D - 1))


def fake_forward(decoder, x, cache, step, rows=None, tp=None):
    assert x.shape == (step.tokens, D)
    decoder.steps.append((step.tokens, tp))
    flat = cache.kv[0, 0].view(-1, cache.kv.shape[-1])
    flat[step.slots.long(), 0] = x[:, 0].to(torch.bfloat16)
    cu, ctx = step.cu_q.tolist(), step.ctx_lens.tolist()
    out = torch.full((step.tokens, decoder.vocab), -1.0)
    for b, L in enumerate(ctx):
        at = [int(step.page_table[b, r // cache.page_size]) * cache.page_size + r % cache.page_size for r in range(L)]
        n = cu[b + 1] - cu[b]
        for i in range(n):
            t = cu[b] + i
            new = [j for j in range(n) if (j <= i if step.mask is None else (int(step.mask[t, j // 64]) >> (j % 64)) & 1)]
            tokens = [int(flat[at[r], 0]) for r in list(range(L - n)) + [L - n + j for j in new]]
            assert int(step.positions[t]) == len(tokens) - 1
            nxt = decoder.rule(tokens)
            decoder.seen.append((tokens, nxt))
            # the second and third likeliest: two other tokens, the same everywhere
            out[t, (nxt + 7) % decoder.vocab], out[t, (nxt + 3) % decoder.vocab], out[t, nxt] = 0.5, 1.0, 2.0
    return (out if rows is None else out.index_select(0, rows)).to(torch.bfloat16)


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    monkeypatch.setattr(paged, "forward_paged", fake_forward)
    kept = []
    real = paged.PagedKVCache.keep
    monkeypatch.setattr(paged.PagedKVCache, "keep", lambda self, paths: kept.append([list(p) for p in paths]) or real(self, paths))
    return kept


def prompt(*ids):
    return torch.nn.functional.pad(torch.tensor(ids, dtype=torch.bfloat16)[:, None], (0, D - 1))


def mixed(tokens):
    x = 7
    for t in tokens:
        x = (x * 31 + t + 1) % 1009
    return x % V


def text(rule, ids, n):
    out = list(ids)
    for _ in range(n):
        out.append(rule(out))
    return out[len(ids):]


PROMPTS = [(3, 1, 4), (1,), (5, 9, 2, 6, 5, 3, 5)]


def check_seen(model, texts):
    """Every row saw the tokens of its own sequence so far and then a drafted path, nothing else."""
    for tokens, _ in model.seen:
        fits = [sum(a == b for a, b in zip(tokens, t)) for t in texts]
        assert any(tokens == t[:len(tokens)] or f >= len(p) for t, f, p in zip(texts, fits, PROMPTS))


@pytest.mark.parametrize("width,depth", [(1, 1), (1, 4), (2, 3), (3, 2)])
@pytest.mark.parametrize("page", [1, 3, 64])
def test_a_decoder_that_drafts_for_itself_accepts_every_draft(stand_ins, width, depth, page):
    m, helper, n = Model(mixed), Model(mixed), 13
    got = paged.generate_paged(m, [prompt(*p) for p in PROMPTS], n, assistant=helper, draft_width=width, draft_depth=depth,
                               page_size=page)
    assert got.tolist() == [text(mixed, p, n) for p in PROMPTS]
    rounds = -(-(n - 1) // (depth + 1))                      # the first token comes from the prompts
    assert len(m.steps) == 1 + rounds
    assert stand_ins == [[list(accepted(width, depth))] * 3] * (2 * rounds)
    full = [list(p) + text(mixed, p, n + depth + 1) for p in PROMPTS]
    check_seen(m, full)
    check_seen(helper, full)
    # the assistant ran depth levels and the last level's rows a round, and saw true prefixes with the chains it likes behind
    assert len(helper.steps) == 1 + rounds * (depth + 1)
    own = {tuple(t) for t, _ in helper.seen}
    for f, p in zip(full, PROMPTS):
        for k in range(len(p), len(p) + n - 1):
            assert tuple(f[:k]) in own


def accepted(width, depth):
    return [0] + [1 + level * width for level in range(depth)]


def test_the_second_chain_is_taken_where_the_first_is_wrong(stand_ins):
    """An assistant whose likeliest token after a root is another one, with the right one second and all later ones right."""
    def shy(tokens):
        return (mixed(tokens) - 3) % V if len(tokens) in roots else mixed(tokens)       # + 3 is its second choice
    ids, n = PROMPTS[0], 13
    roots = {len(ids) + 1 + 3 * k for k in range(9)}          # the lengths at which a round of two drafted tokens starts
    m = Model(mixed)
    got = paged.generate_paged(m, [prompt(*ids)], n, assistant=Model(shy), draft_width=2, draft_depth=2)
    assert got.tolist() == [text(mixed, ids, n)]
    assert stand_ins == [[[0, 2, 4]]] * 8 and len(m.steps) == 1 + 4


def test_an_assistant_that_is_always_wrong_changes_nothing(stand_ins):
    m = Model(mixed)
    got = paged.generate_paged(m, [prompt(*p) for p in PROMPTS], 6, assistant=Model(lambda t: (mixed(t) + 1) % V), draft_width=2,
                               draft_depth=3)
    assert got.tolist() == [text(mixed, p, 6) for p in PROMPTS] and len(m.steps) == 1 + 5
    assert stand_ins == [[[0]] * 3] * 10


def test_an_end_token_inside_a_drafted_path_ends_the_sequence(stand_ins):
    want = [text(mixed, p, 20) for p in PROMPTS]
    eos = want[0][3]
    got = paged.generate_paged(Model(mixed), [prompt(*p) for p in PROMPTS], 20, eos_token_id=eos, pad_token_id=49,
                               assistant=Model(mixed), draft_width=2, draft_depth=4).tolist()
    for g, w in zip(got, want):
        end = w.index(eos) + 1 if eos in w else len(w)
        assert g[:end] == w[:end] and all(t == 49 for t in g[end:])
    assert got[0][3] == eos


def test_generation_without_an_assistant(stand_ins):
    m = Model(mixed)
    got = paged.generate_paged(m, [prompt(*p) for p in PROMPTS], 5, page_size=2)
    assert got.tolist() == [text(mixed, p, 5) for p in PROMPTS] and len(m.steps) == 5


@pytest.mark.parametrize("vocab", [V - 1, V + 1])
def test_an_assistant_of_another_vocabulary_is_refused(stand_ins, vocab):
    """Its drafts are looked up in the decoder's embedding table and the decoder's tokens in its own."""
    m, helper = Model(mixed), Model(mixed, vocab=vocab)
    with pytest.raises(ValueError, match="vocabular"):
        paged.generate_paged(m, [prompt(*p) for p in PROMPTS], 6, assistant=helper)
    assert not m.steps and not helper.steps


def test_an_assistant_that_is_whole_on_every_rank_runs_whole(stand_ins):
    """Under tensor parallelism a whole assistant's products are not summed over the ranks, those of a split one are; one
    that is split over another number of ranks is refused."""
    group = TPContext(1, 2, reduce_fn=lambda part: part)
    for world in (1, 2):
        m, helper = Model(mixed, world=2), Model(mixed, world=world)
        got = paged.generate_paged(m, [prompt(*PROMPTS[0])], 6, assistant=helper, tp=group)
        assert got.tolist() == [text(mixed, PROMPTS[0], 6)] and m.steps and helper.steps
        assert all(tp is group for _, tp in m.steps)
        for _, tp in helper.steps:
            assert tp is group if world == 2 else tp.world == 1 and tp.lead and tp.reduce("x") == "x"
    for tp, world in ((group, 4), (None, 2)):
        with pytest.raises(ValueError, match="ranks"):
            paged.generate_paged(Model(mixed, world=tp.world if tp else 1), [prompt(*PROMPTS[0])], 6, tp=tp,
                                 assistant=Model(mixed, world=world))


def drawing(undrawable):
    """draw_tokens for sampled rows: the likeliest, or -1 (what ops.sample gives for a row it cannot draw from) where the
    likeliest token is one of ``undrawable``."""
    def draw(logits, u, sampling):
        top = logits.float().argmax(-1)
        return torch.tensor([-1 if int(t) in undrawable else int(t) for t in top])
    return draw


def test_a_row_without_a_drawable_token_counts_only_where_it_is_taken(stand_ins, monkeypatch):
    """Rows of drafts that are not accepted, and of what follows the end of a sequence, may hold NaN."""
    ids, n = PROMPTS[0], 7
    want = text(mixed, ids, n)

    def wild(tokens):                                        # what follows drafts that are never in the text: 41
        return 41 if any(t in (30, 33) for t in tokens[len(ids):]) else mixed(tokens)
    assert not {30, 33, 41} & set(want)
    monkeypatch.setattr(paged, "draw_tokens", drawing({41}))
    got = paged.generate_paged(Model(wild), [prompt(*ids)], n, assistant=Model(lambda t: 30), draft_width=2, draft_depth=1,
                               sampling=dict(temperature=1.0))
    assert got.tolist() == [want]
    eos = want[2]                                            # a full draft goes on behind the end token
    monkeypatch.setattr(paged, "draw_tokens", drawing({want[3]}))
    got = paged.generate_paged(Model(mixed), [prompt(*ids)], n, assistant=Model(mixed), draft_width=1, draft_depth=4,
                               sampling=dict(temperature=1.0), eos_token_id=eos)
    assert got.tolist() == [want[:3]]
    for helper in (None, Model(mixed)):                      # and is refused in the text itself, the first token among it
        for bad in (want[0], want[3]):
            monkeypatch.setattr(paged, "draw_tokens", drawing({bad}))
            with pytest.raises(FloatingPointError):
                paged.generate_paged(Model(mixed), [prompt(*ids)], n, assistant=helper, sampling=dict(temperature=1.0))
