"""Decoding over the paged cache on the GPU: chunks, ragged batches and trees against the causal forward over whole
sequences, and generate() with masks, sampling and drafts against decoding each sequence alone."""
import pytest
import torch

from oracle import zero_oracle as zo
from tests.golden.configs import GOLDEN_CONFIGS
from tests.test_graft_gpu import _model, maxrel

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def graft():
    spec = GOLDEN_CONFIGS["graft"]
    params, cfg, model = _model(spec)
    return spec["dec"], params, model.decoder


def full_logits(decoder, x):
    with torch.no_grad():
        return decoder(inputs_embeds=x[None], use_cache=False)["logits"][0]


@pytest.mark.parametrize("page", [5, 64])
def test_chunks_and_single_tokens_match_the_causal_forward(graft, page):
    """Prompts of different lengths in chunks, then single tokens, one sequence pausing: 1e-2 as for the contiguous cache."""
    from zero_amd.inference.paged import PagedKVCache, forward_paged
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(1)
    lens, B = [61, 9, 140], 3
    xs = [torch.randn(n, dec.hidden, generator=g).to(torch.bfloat16).to(DEV) for n in lens]
    want = [full_logits(decoder, x) for x in xs]
    cache = PagedKVCache.for_decoder(decoder, B, 150, DEV, page_size=page)
    for counts in ([40, 5, 3], [0, 1, 100], [19, 0, 30], [1, 1, 1], [1, 1, 6], [0, 1, 0]):
        at = list(cache.lengths)
        step = cache.step(counts)
        got = forward_paged(decoder, torch.cat([x[a:a + n] for x, a, n in zip(xs, at, counts)]), cache, step)
        cache.advance(counts)
        for b, n in enumerate(counts):
            if n:
                assert maxrel(got[step.cu[b]:step.cu[b + 1]], want[b][at[b]:at[b] + n]) <= 1e-2, (counts, b)
    assert cache.lengths == lens


def test_every_node_of_a_tree_matches_its_path(graft):
    """Trees over different prefixes; then a path is kept and decoding goes on from it."""
    from zero_amd.inference.paged import PagedKVCache, forward_paged
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(2)
    lens, trees = [23, 70], [[-1, 0, 0, 1, 1, 2, 4, 5], [-1, 0, 1, 1, 1, 4]]
    xs = [torch.randn(n, dec.hidden, generator=g).to(torch.bfloat16).to(DEV) for n in lens]
    nodes = [torch.randn(len(t), dec.hidden, generator=g).to(torch.bfloat16).to(DEV) for t in trees]
    cache = PagedKVCache.for_decoder(decoder, 2, 100, DEV, page_size=16)
    forward_paged(decoder, torch.cat(xs), cache, cache.step(lens))
    cache.advance(lens)
    step = cache.step([len(t) for t in trees], trees)
    got = forward_paged(decoder, torch.cat(nodes), cache, step)
    paths = []
    for b, t in enumerate(trees):
        for i in range(len(t)):
            path = [i]
            while t[path[0]] >= 0:
                path.insert(0, t[path[0]])
            want = full_logits(decoder, torch.cat([xs[b], nodes[b][path]]))[-1]
            assert maxrel(got[step.cu[b] + i], want) <= 1e-2, (b, i)
        paths.append(path)
    cache.keep(paths)
    assert cache.lengths == [n + len(p) for n, p in zip(lens, paths)]
    more = torch.randn(2, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    nxt = forward_paged(decoder, more, cache, cache.step([1, 1]))
    for b in range(2):
        assert maxrel(nxt[b], full_logits(decoder, torch.cat([xs[b], nodes[b][paths[b]], more[b:b + 1]]))[-1]) <= 1e-2


def same_tokens(got, want, decoder, prompt, params, dec, greedy=True):
    """Equal tokens; where greedy ones part, the oracle's fp32 logits of the two must be as near as its own distance from
    the bf16 decoder (2e-2 of the largest logit) allows, and what follows is another text."""
    got, want = got.tolist(), want.tolist()
    for i, (a, b) in enumerate(zip(got, want)):
        if a != b:
            assert greedy
            x = prompt
            if i:
                wte = decoder.model.get_input_embeddings()
                x = torch.cat([prompt, wte(torch.tensor(want[:i], device=DEV))])
            lg = zo.llama_forward(params, x[None].float().cpu(), dec)[0, -1]
            assert abs(float(lg[a] - lg[b])) <= 2 * 2e-2 * float(lg.abs().max()), (i, a, b)
            return
    assert len(got) == len(want)


def prompts_of(dec, seed, lens):
    g = torch.Generator().manual_seed(seed)
    S = max(lens)
    x = torch.randn(len(lens), S, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    mask = torch.zeros(len(lens), S, dtype=torch.int64, device=DEV)
    for b, n in enumerate(lens):                               # right- and left-padded ones, a hole in the last
        if b % 2:
            mask[b, S - n:] = 1
        else:
            mask[b, :n] = 1
    return x, mask


def test_generate_with_a_mask_decodes_each_prompt_as_alone(graft):
    dec, params, decoder = graft
    x, mask = prompts_of(dec, 3, [30, 12, 1, 25])
    mask[3, 5:9] = 0
    got = decoder.generate(inputs_embeds=x, attention_mask=mask, max_new_tokens=7)
    assert tuple(got.shape) == (4, 7)
    for b in range(4):
        alone = x[b][mask[b] != 0]
        same_tokens(got[b], decoder.generate(inputs_embeds=alone[None], max_new_tokens=7)[0], decoder, alone, params, dec)


@pytest.mark.parametrize("width,depth", [(1, 1), (2, 3), (3, 2)])
def test_generate_with_an_assistant_gives_the_same_tokens(graft, width, depth):
    """The decoder as its own draft (everything is accepted), and a shorter one."""
    import copy
    dec, params, decoder = graft
    short = copy.copy(decoder)
    short._modules = dict(decoder._modules)
    short.model = copy.copy(decoder.model)
    short.model._modules = dict(decoder.model._modules)
    short.model.layers = torch.nn.ModuleList(list(decoder.model.layers)[:1])
    x, _ = prompts_of(dec, 4, [18, 18])
    want = decoder.generate(inputs_embeds=x, max_new_tokens=9)
    for helper in (decoder, short):
        got = decoder.generate(inputs_embeds=x, max_new_tokens=9, assistant=helper, draft_width=width, draft_depth=depth)
        for b in range(2):
            same_tokens(got[b], want[b], decoder, x[b], params, dec)
    eos = int(want[0, 2])
    ended = decoder.generate(inputs_embeds=x[:1], max_new_tokens=9, eos_token_id=eos, pad_token_id=3, assistant=short,
                             draft_width=width, draft_depth=depth)[0].tolist()
    first = want[0].tolist().index(eos)
    if ended[:first + 1] == want[0].tolist()[:first + 1]:
        assert len(ended) == first + 1


def test_generate_samples(graft):
    """top_k = 1 is greedy; equal generators give equal tokens; settings move the tokens; an assistant leaves them among the
    kept ones; bad settings and rows that cannot be drawn from are refused."""
    dec, params, decoder = graft
    x, _ = prompts_of(dec, 5, [16, 16, 16])
    gen = lambda: torch.Generator(device=DEV).manual_seed(8)  # noqa: E731
    greedy = decoder.generate(inputs_embeds=x, max_new_tokens=6)
    assert torch.equal(decoder.generate(inputs_embeds=x, max_new_tokens=6, do_sample=True, top_k=1), greedy)
    assert torch.equal(decoder.generate(inputs_embeds=x, max_new_tokens=6, do_sample=True, temperature=0.0), greedy)
    kw = dict(inputs_embeds=x, max_new_tokens=6, do_sample=True, temperature=1.5, top_k=40, top_p=0.95)
    a, b = decoder.generate(generator=gen(), **kw), decoder.generate(generator=gen(), **kw)
    assert torch.equal(a, b) and not torch.equal(a, greedy)
    # With a draft the logits come from products of other row counts, and near-equal ones change places in the falling order
    # that a draw goes by: the tokens may part, but each is one of the 40 likeliest after its own prefix, up to twice the
    # distance that a bf16 logit keeps from the oracle's (2e-2 of the largest).
    drafted = decoder.generate(generator=gen(), assistant=decoder, draft_width=2, draft_depth=2, **kw)
    assert torch.equal(drafted, decoder.generate(generator=gen(), assistant=decoder, draft_width=2, draft_depth=2, **kw))
    wte = decoder.model.get_input_embeddings()
    for b in range(3):
        lg = zo.llama_forward(params, torch.cat([x[b], wte(drafted[b, :-1])])[None].float().cpu(), dec)[0, 15:]
        for i, t in enumerate(drafted[b].tolist()):
            assert float(lg[i, t]) >= float(lg[i].topk(40).values[-1]) - 2 * 2e-2 * float(lg[i].abs().max()), (b, i)
    assert torch.equal(decoder.generate(inputs_embeds=x, max_new_tokens=6, do_sample=True, top_k=1, assistant=decoder),
                       decoder.generate(inputs_embeds=x, max_new_tokens=6, assistant=decoder))
    with pytest.raises(ValueError):
        decoder.generate(inputs_embeds=x, max_new_tokens=2, do_sample=True, top_p=1.5)
    w = decoder.model.norm.weight
    keep = w.detach().clone()
    with torch.no_grad():
        w[3] = float("nan")
    try:
        with pytest.raises(FloatingPointError):
            decoder.generate(inputs_embeds=x, max_new_tokens=2, do_sample=True)
    finally:
        with torch.no_grad():
            w.copy_(keep)


def test_paged_tensor_parallel_two_rank_threads(graft):
    """forward_paged through sharded layers (W = 2 rank threads) against the unsharded decoder: chunk, tree, single token."""
    import threading
    from zero_amd.distributed.tensor_parallel import ThreadSimGroup, shard_llama_
    from zero_amd.inference.paged import PagedKVCache, forward_paged
    dec, params, decoder = graft
    spec = GOLDEN_CONFIGS["graft"]
    g = torch.Generator().manual_seed(6)
    xs = torch.randn(40, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    tree = [-1, 0, 0, 2]

    def steps(d, tp=None):
        c = PagedKVCache.for_decoder(d, 1, 64, DEV, page_size=16)
        out = [forward_paged(d, xs[:30], c, c.step([30]), tp=tp)]
        c.advance([30])
        out.append(forward_paged(d, xs[30:34], c, c.step([4], [tree]), tp=tp))
        c.keep([[0, 2, 3]])
        out.append(forward_paged(d, xs[34:35], c, c.step([1]), tp=tp))
        return out

    want = steps(decoder)
    W = 2
    group, results, errors = ThreadSimGroup(W), [None] * 2, []
    shards = []
    for r in range(W):
        m = _model(spec)[2]
        shard_llama_(m.decoder, r, W)
        shards.append(m.decoder)

    def run(r):
        try:
            torch.cuda.set_device(0)
            results[r] = steps(shards[r], group.context(r))
        except Exception as e:      # a dead rank must not leave the other one waiting at the rendezvous
            errors.append(e)
            group._bar.abort()

    threads = [threading.Thread(target=run, args=(r,)) for r in range(W)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    for r in range(W):
        for a, b in zip(results[r], want):
            assert maxrel(a, b) <= 1.5e-2
