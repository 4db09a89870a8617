"""The rotary tables' lifetime and values: kernels, captured graphs and DecodePlan read them by address."""
import gc
import weakref

import pytest
import torch

from zero_amd.models import llama


def config(**kw):
    return llama.LlamaConfig(vocab_size=40, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                             num_key_value_heads=1, head_dim=64, **kw)


@pytest.mark.parametrize("S", [1, 2, 63, 64, 1000, 1024, 1025, 5003])
def test_rows_do_not_depend_on_the_length_asked_for(S):
    """Every length gives the rows of the formula, bit for bit, after shorter and after longer ones."""
    cfg = config()
    rot = llama.LlamaRotaryEmbedding(cfg)
    f = (llama.llama3_inv_freq(cfg)[:, None] @ torch.arange(S, dtype=torch.float32)[None, :]).t()
    for first in (S, 1, 9000):
        rot.tables(first, "cpu")
        cos, sin = rot.tables(S, "cpu")
        assert cos.shape == sin.shape == (S, 32) and cos.is_contiguous() and sin.is_contiguous()
        assert torch.equal(cos, f.cos().bfloat16().float()) and torch.equal(sin, f.sin().bfloat16().float())


def test_lengths_in_turn_share_one_table(monkeypatch):
    """Two caches of different lengths, used in turn, do not make the tables again at every step."""
    made = []
    real = llama.llama3_inv_freq
    monkeypatch.setattr(llama, "llama3_inv_freq", lambda cfg: made.append(1) or real(cfg))
    rot = llama.LlamaRotaryEmbedding(config())
    for _ in range(5):
        for S in (700, 90, 331):
            rot.tables(S, "cpu")
    assert len(made) == 1
    for S in range(1, 20000, 37):
        rot.tables(S, "cpu")
    assert len(made) <= 6                                    # a longer one is at least twice as long


def test_tables_stay_where_they_were_handed_out():
    """Whoever keeps only the address (a captured graph, a plan of native calls) reads the same rows after longer and
    shorter lengths were asked for: as long as the module lives, no table's memory is given back."""
    rot = llama.LlamaRotaryEmbedding(config())
    tables = [rot.tables(S, "cpu") for S in (70, 3000, 8, 20000)]
    kept = [t.clone() for pair in tables for t in pair]
    where = [(t.data_ptr(), t.numel()) for pair in tables for t in pair]
    del tables
    gc.collect()
    junk = [torch.full((n,), 7.0) for _ in range(8) for _, n in where]
    held = [t for tables in rot._cache.values() for t in tables]
    for (ptr, n), want in zip(where, kept):
        home = [t for pair in held for t in pair if t.data_ptr() == ptr and t.numel() >= n]
        assert home and torch.equal(home[0][:want.shape[0]], want)
    assert all(j[0] == 7 for j in junk)


def test_tables_made_in_inference_mode_serve_training():
    rot = llama.LlamaRotaryEmbedding(config())
    with torch.inference_mode():
        rot.tables(90, "cpu")
    cos, _ = rot.tables(33, "cpu")
    x = torch.ones(33, 32, requires_grad=True)
    (x * cos).sum().backward()                               # (cos is saved for the gradient)
    assert torch.equal(x.grad, cos)


def test_decode_plan_holds_the_tables_it_points_into():
    """The plan's structs hold addresses; the tables they name must live as long as the plan."""
    from zero_amd.inference.decode import DecodePlan, KVCache
    dec = llama.LlamaForCausalLM(config())
    cache = KVCache(1, 1, 16, 64, "cpu")
    cos, sin = torch.zeros(16, 32), torch.zeros(16, 32)
    plan = DecodePlan(dec, cache, cos, sin)
    assert plan.structs[0].cos_t == cos.data_ptr() and plan.structs[0].sin_t == sin.data_ptr()
    alive = [weakref.ref(cos), weakref.ref(sin)]
    del cos, sin
    gc.collect()
    assert all(r() is not None for r in alive)
