"""The serving path's state on the GPU: rotary tables under several caches, sequences beside others, launches without shares,
what a draft proposes and what of it is accepted."""
import gc
import threading

import pytest
import torch

from oracle import zero_oracle as zo
from tests.golden.configs import GOLDEN_CONFIGS
from tests.test_graft_gpu import _model, maxrel
from tests.test_paged_gpu import agree, call, make

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


def test_a_contiguous_cache_goes_on_after_a_paged_call_of_another_length(graft):
    """The plan of native steps reads the rotary tables by address; other lengths are asked for in between, and memory is
    handed out anew."""
    from zero_amd.inference.decode import KVCache, forward_cached
    from zero_amd.inference.paged import PagedKVCache, forward_paged
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(11)
    xs = torch.randn(1, 24, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)

    def steps(between):
        cache = KVCache(len(decoder.model.layers), 1, 40, decoder.model.layers[0].self_attn.k_proj.weight.shape[0], DEV)
        out = [forward_cached(decoder, xs[:, :20], cache)]
        for t in range(20, 24):
            out.append(forward_cached(decoder, xs[:, t:t + 1], cache))
            between(t)
        return out

    def disturb(t):
        for n in (1500 * (t - 18), 17):
            c = PagedKVCache.for_decoder(decoder, 1, n, DEV, page_size=16)
            forward_paged(decoder, xs[0, :5], c, c.step([5]))
        gc.collect()
        junk.extend(torch.full((40, n), 3.0, device=DEV) for n in (16, 32, 64, 128))

    junk = []
    want = steps(lambda t: None)
    for a, b in zip(steps(disturb), want):
        assert torch.equal(a, b)
    assert all(bool((j == 3).all()) for j in junk)


def test_a_captured_step_goes_on_after_other_lengths(graft):
    """forward_paged in a graph, replayed after longer and shorter caches were used on the same decoder."""
    from zero_amd.inference.paged import PagedKVCache, forward_paged
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(12)
    xs = torch.randn(30, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    cache = PagedKVCache.for_decoder(decoder, 1, 64, DEV, page_size=16)
    forward_paged(decoder, xs[:29], cache, cache.step([29]))
    cache.advance([29])
    step, x = cache.step([1]), xs[29:30].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = forward_paged(decoder, x, cache, step)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = forward_paged(decoder, x, cache, step)
    for n in (3000, 17, 9000):
        c = PagedKVCache.for_decoder(decoder, 1, n, DEV, page_size=16)
        forward_paged(decoder, xs[:5], c, c.step([5]))
        junk = [torch.full((64, w), 3.0, device=DEV) for w in (16, 32, 64, 128)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and all(bool((j == 3).all()) for j in junk)


@pytest.mark.parametrize("Hq,Hkv,hd,page", [(8, 2, 128, 16), (12, 4, 64, 64)])
@pytest.mark.parametrize("tree", [False, True])
def test_attn_paged_sequences_among_different_neighbours(Hq, Hkv, hd, page, tree):
    """The same sequences alone, in other orders and beside others that send the call to another kernel and other shares: the
    cuts of the keys, and so the last bits, go by the whole batch, the answer within the tolerance does not."""
    c = make([(1, 900), (30, 200), (2, 5), (3, 700), (90, 1500)], Hq, Hkv, hd, page, tree=tree, seed=14)
    for some in ([0], [0, 2], [3, 0], [1, 0], [4, 3, 2, 1, 0], [0, 4], [2, 1], [1]):
        rows = [t for b in some for t in range(c["cu"][b], c["cu"][b + 1])]
        cu = [0]
        for b in some:
            cu.append(cu[-1] + c["cu"][b + 1] - c["cu"][b])
        part = dict(c, q=c["q"][rows], table=c["table"][some], ctx=[c["ctx"][b] for b in some], cu=cu,
                    mask=None if c["mask"] is None else c["mask"][rows].contiguous())
        agree(call(part), part)


@pytest.mark.parametrize("seqs,hd,page", [([(200, 900), (60, 300), (1, 70)], 128, 64), ([(200, 900), (60, 300), (1, 70)], 128, 24),
                                          ([(300, 900), (90, 200)], 64, 64), ([(300, 900), (90, 200)], 64, 100)])
@pytest.mark.parametrize("tree", [False, True])
def test_attn_paged_more_work_than_two_rounds_is_not_shared_out(seqs, hd, page, tree):
    """T * Hq of 131072 rows and more (196608 of width 64): every row tile goes over all its keys, without shares and merge."""
    from zero_amd import ops
    c = make(seqs, 512, 4, hd, page, tree=tree, seed=15)
    T = c["cu"][-1]
    assert ops.attn_paged_ws_floats(len(seqs), T, seqs[0][0], seqs[0][1], 512, 4, hd) == 0
    agree(call(c), c)


@pytest.fixture
def kept(monkeypatch):
    from zero_amd.inference import paged
    paths = []
    real = paged.PagedKVCache.keep
    monkeypatch.setattr(paged.PagedKVCache, "keep", lambda self, p: paths.append([list(x) for x in p]) or real(self, p))
    return paths


@pytest.mark.parametrize("width,depth", [(1, 4), (2, 3), (3, 2)])
def test_a_decoder_that_drafts_for_itself_is_believed(graft, kept, width, depth):
    """Drafts of the decoder's own are accepted whole, but where two logits are so near that other row counts of the
    products change their order: in three of four rounds at the least (of random drafts from this vocabulary next to none
    would be)."""
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(16)
    x = torch.randn(3, 21, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    decoder.generate(inputs_embeds=x, max_new_tokens=16, assistant=decoder, draft_width=width, draft_depth=depth)
    rounds = [p for step in kept for p in step if p]
    whole = sum(len(p) == depth + 1 for p in rounds)
    assert len(rounds) >= 6 and 4 * whole >= 3 * len(rounds), rounds


def test_what_a_draft_proposes_is_what_its_decoder_finds_likeliest(graft):
    """paged._draft's tokens against the causal forward of the same tokens (1e-2 of the largest logit apart, as in the other
    tests of it: a token is the likeliest, or within twice that) and, after a path is kept, the next logits against the fp32
    oracle.  Two bf16 forwards may be as far from each other as the sum of their distances from the oracle: at most 2e-2 each
    in the tests of cached decoding.  Tokens' embeddings are 50 times smaller than random ones, so every layer's roundings
    reach the last logits here: the training path itself was 0.0077 and 0.0097 from the oracle, this path 0.0085 and 0.0109,
    the two 0.0072 and 0.0122 apart."""
    from zero_amd.inference import paged
    dec, params, decoder = graft
    g = torch.Generator().manual_seed(17)
    lens, width, depth = [19, 44], 3, 3
    xs = [torch.randn(n, dec.hidden, generator=g).to(torch.bfloat16).to(DEV) for n in lens]
    cache = paged.PagedKVCache.for_decoder(decoder, 3, 100, DEV, page_size=16)
    paged.forward_paged(decoder, torch.cat(xs), cache, cache.step(lens[:1] + [0] + lens[1:]))
    cache.advance([lens[0], 0, lens[1]])
    roots = [5, None, 9]
    tokens = paged._draft(decoder, cache, roots, width, depth, None)
    assert [len(t) for t in tokens] == [1 + width * depth, 0, 1 + width * depth]
    wte = decoder.model.get_input_embeddings()
    parents = paged.draft_tree(width, depth)
    for x, t in ((xs[0], tokens[0]), (xs[1], tokens[2])):
        assert len(set(t[1:1 + width])) == width
        for i in range(1, len(parents)):
            path, j = [], parents[i]
            while j >= 0:
                path.insert(0, t[j])
                j = parents[j]
            lg = full_logits(decoder, torch.cat([x, wte(torch.tensor(path, device=DEV))]))[-1].float()
            least = lg.topk(width).values[(i - 1) % width] if parents[i] == 0 else lg.max()
            assert float(lg[t[i]]) >= float(least) - 2e-2 * float(lg.abs().max()), i
    st = cache.step([len(t) for t in tokens], [parents, [], parents])
    paged.forward_paged(decoder, wte(torch.tensor([t for ts in tokens for t in ts], device=DEV)), cache, st)
    path = [0, 2, 5, 8]                                       # the second chain
    cache.keep([path, [], path])
    nxt = paged.forward_paged(decoder, wte(torch.tensor([7, 7], device=DEV)), cache, cache.step([1, 0, 1]))
    for row, x, t in ((0, xs[0], tokens[0]), (1, xs[1], tokens[2])):
        ids = torch.tensor([t[j] for j in path] + [7], device=DEV)
        seq = torch.cat([x, wte(ids)])
        assert maxrel(nxt[row], zo.llama_forward(params, seq[None].float().cpu(), dec)[0, -1]) <= 2e-2
        assert maxrel(nxt[row], full_logits(decoder, seq)[-1]) <= 2e-2 + 2e-2


def test_a_whole_assistant_beside_a_split_decoder(graft, kept):
    """Two rank threads: the decoder is split, the assistant (the same decoder, whole) runs on each rank by itself.  Both
    ranks give the same tokens, each the likeliest after its own prefix up to twice the distance that a bf16 logit keeps from
    the oracle's (2e-2 of the largest), and drafts are accepted."""
    from zero_amd.distributed.tensor_parallel import ThreadSimGroup, shard_llama_
    from zero_amd.inference.decode import generate
    dec, params, decoder = graft
    spec = GOLDEN_CONFIGS["graft"]
    g = torch.Generator().manual_seed(18)
    x = torch.randn(2, 17, dec.hidden, generator=g).to(torch.bfloat16).to(DEV)
    W = 2
    group, results, errors = ThreadSimGroup(W), [None] * W, []
    split = [shard_llama_(_model(spec)[2].decoder, r, W) for r in range(W)]
    whole = [_model(spec)[2].decoder for _ in range(W)]

    def run(r):
        try:
            torch.cuda.set_device(0)
            results[r] = generate(split[r], x, max_new_tokens=11, assistant=whole[r], draft_width=2, draft_depth=2,
                                  tp=group.context(r))
        except Exception as e:      # a dead rank must not leave the other one waiting at the rendezvous
            errors.append(e)
            group._bar.abort()

    threads = [threading.Thread(target=run, args=(r,)) for r in range(W)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    assert torch.equal(results[0], results[1])
    wte = decoder.model.get_input_embeddings()
    for b in range(2):
        lg = zo.llama_forward(params, torch.cat([x[b], wte(results[0][b, :-1])])[None].float().cpu(), dec)[0, 16:]
        for i, t in enumerate(results[0][b].tolist()):
            assert float(lg[i, t]) >= float(lg[i].max()) - 2 * 2e-2 * float(lg[i].abs().max()), (b, i)
    rounds = [p for step in kept for p in step if p]
    assert 2 * sum(len(p) > 1 for p in rounds) >= len(rounds), rounds
