"""Refusals of the paged-cache operators and of sampling: at the C boundary (every check comes before any launch, so
these run without a GPU) and in the tensor wrappers."""
import ctypes

import pytest
import torch

OK, EINVAL = 0, -22
BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 63) // 64 * 64            # an aligned address; nothing reads it


def append(**kw):
    from zero_amd._lib import lib
    a = dict(qkv=PTR, cos=PTR, sin=PTR, q=PTR, k=PTR, v=PTR, pos=PTR, slots=PTR, T=0, Hq=8, Hkv=2, hd=128, rot=128, P=16,
             ldqkv=12 * 128, ldq=8 * 128, rows=64, inter=0)
    a.update(kw)
    return lib.zk_kv_append_paged(*a.values(), None)


def attn(**kw):
    from zero_amd._lib import lib
    a = dict(q=PTR, k=PTR, v=PTR, out=PTR, table=PTR, ctx=PTR, cu=PTR, mask=None, ws=PTR, wsf=1 << 40, T=0, B=3, max_q=4,
             max_ctx=100, Hq=8, Hkv=2, hd=128, page=16, pages=20, cols=7, ldt=7, words=0, ldq=1024, ldo=1024, scale=0.1)
    a.update(kw)
    return lib.zk_attn_paged(*a.values(), None)


def sample(**kw):
    from zero_amd._lib import lib
    a = dict(logits=PTR, u=PTR, tr=None, kr=None, pr=None, mr=None, t=1.0, k=0, p=1.0, mp=0.0, tok=PTR, lp=PTR, rows=0,
             V=100, ld=100)
    a.update(kw)
    return lib.zk_sample(*a.values(), None)


def test_calls_without_rows_are_fine():
    assert append() == OK and attn() == OK and sample() == OK


@pytest.mark.parametrize("bad", [dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(Hq=7), dict(hd=96), dict(rot=0), dict(rot=24),
                                 dict(rot=144), dict(P=0), dict(ldqkv=1535), dict(ldqkv=1528), dict(ldq=1020), dict(ldq=512),
                                 dict(rows=0), dict(rows=1 << 31), dict(qkv=None), dict(cos=None), dict(sin=None), dict(q=None),
                                 dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(qkv=PTR + 2),
                                 dict(k=PTR + 8), dict(q=PTR + 4), dict(cos=PTR + 4)], ids=str)
def test_append_refusals(bad):
    assert append(**bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(T=-1), dict(B=0), dict(max_q=0), dict(max_ctx=0), dict(Hq=9), dict(hd=80), dict(page=0),
                                 dict(pages=0), dict(cols=0), dict(ldt=6), dict(page=1 << 20, pages=1 << 12), dict(ldq=1000),
                                 dict(ldo=1023), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(table=None),
                                 dict(ctx=None), dict(cu=None), dict(mask=PTR, words=0), dict(q=PTR + 2), dict(k=PTR + 2),
                                 dict(out=PTR + 8), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(B=1 << 30), dict(B=1 << 28, Hkv=2), dict(T=1 << 30),
                                 dict(max_q=1 << 31), dict(max_ctx=1 << 31), dict(Hq=1 << 18, Hkv=1 << 18)], ids=str)
def test_attention_refusals(bad):
    assert attn(**bad) == EINVAL


def test_attention_workspace_is_checked():
    from zero_amd import ops
    need = ops.attn_paged_ws_floats(2, 2, 1, 100000, 8, 2, 128)
    if need:
        long = dict(B=2, T=2, max_q=1, max_ctx=100000, pages=10000, cols=7000, ldt=7000)
        assert attn(ws=None, **long) == EINVAL and attn(wsf=need - 1, **long) == EINVAL and attn(ws=PTR + 4, **long) == EINVAL


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(V=0), dict(ld=99), dict(logits=None), dict(u=None), dict(tok=None),
                                 dict(lp=None), dict(logits=PTR + 1), dict(t=-0.5), dict(t=float("nan")), dict(t=2.0 ** 21),
                                 dict(k=-1), dict(p=0.0), dict(p=1.5), dict(p=float("nan")), dict(mp=-0.1), dict(mp=1.1),
                                 dict(mp=float("nan"))], ids=str)
def test_sample_refusals(bad):
    assert sample(**bad) == EINVAL


@pytest.mark.parametrize("call,good,bad", [
    (append, dict(T=0), dict(T=1 << 24)),                                             # a token a workgroup of 256 threads
    (sample, dict(rows=0), dict(rows=1 << 22)),                                       # a row a workgroup of 1024
    (attn, dict(T=0), dict(T=4096, B=4096, max_q=1, max_ctx=1 << 18, Hq=32, Hkv=8, ldq=4096, ldo=4096)),     # shares
    (attn, dict(T=0), dict(T=65536, B=65536, max_q=1, max_ctx=8200, Hq=64, Hkv=4, ldq=8192, ldo=8192)),      # merge
    (attn, dict(T=0), dict(T=1 << 22, B=1 << 22, max_q=1, max_ctx=1536, Hq=16, Hkv=1, ldq=2048, ldo=2048)),  # of few shares
    (attn, dict(T=0), dict(T=1 << 23, B=4, max_q=1 << 22, max_ctx=1 << 22, Hq=128, Hkv=1, ldq=16384, ldo=16384)),
], ids=["append", "sample", "attention-shares", "attention-merge", "attention-merge-few", "attention-tiles"])
def test_calls_of_more_threads_than_a_launch_has_are_refused_before_it(call, good, bad):
    """2^32 threads and more are no launch."""
    assert call(**good) == OK and call(**bad) == EINVAL


def test_attention_workspace_of_a_call_that_cannot_be_launched():
    from zero_amd import ops
    from zero_amd._lib import ZeroHipError
    with pytest.raises(ZeroHipError):
        ops.attn_paged_ws_floats(4096, 4096, 1, 1 << 18, 32, 8, 128)
    assert ops.attn_paged_ws_floats(4096, 4096, 1, 1 << 17, 32, 8, 128) > 0


def test_wrappers_refuse_host_tensors():
    from zero_amd import ops
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="device"):
        ops.sample(b(2, 8), torch.zeros(2))
    with pytest.raises(ValueError, match="device"):
        ops.kv_append_paged(b(2, 512), torch.zeros(4, 32), torch.zeros(4, 32), b(2, 4, 128), b(2, 4, 128), i(2), i(2), 4, 2, 64)
    with pytest.raises(ValueError, match="device"):
        ops.attn_paged(b(2, 256), b(2, 4, 128), b(2, 4, 128), i(2).view(1, 2), i(1), i(2), 2, 8, 4, 2, 64, 0.1)


# ---- the host side of the paged cache -------------------------------------------------------------------------------
def cache_of(**kw):
    from zero_amd.inference.paged import PagedKVCache
    a = dict(n_layers=2, max_seqs=3, max_len=20, kv_width=8, device="cpu", page_size=4)
    a.update(kw)
    return PagedKVCache(**a)


def test_cache_hands_out_pages_and_takes_them_back():
    c = cache_of(n_pages=6)
    st = c.step([5, 0, 9])                                    # 2 + 0 + 3 pages
    assert [len(p) for p in c.pages] == [2, 0, 3] and len({p for ps in c.pages for p in ps}) == 5
    assert st.cu == [0, 5, 5, 14] and st.max_q == 9 and st.max_ctx == 9 and st.mask is None
    assert st.positions.tolist() == list(range(5)) + list(range(9)) and st.ctx_lens.tolist() == [5, 0, 9]
    assert st.slots.tolist() == [c.row(0, r) for r in range(5)] + [c.row(2, r) for r in range(9)]
    assert len(set(st.slots.tolist())) == 14
    for b, ps in enumerate(c.pages):
        assert c.page_table[b].tolist() == ps + [-1] * (5 - len(ps))
    assert c.lengths == [0, 0, 0]
    c.advance([5, 0, 9])
    nxt = c.step([1, 1, 1])                                   # 5 -> 6 and 9 -> 10 fit their pages; sequence 1 takes the last
    assert nxt.positions.tolist() == [5, 0, 9] and len(c._free) == 0
    with pytest.raises(RuntimeError, match="out of pages"):
        c.step([4, 0, 0])                                     # 9 rows: a third page
    c.advance([1, 1, 1])
    c.truncate(2, 4)
    assert c.lengths == [6, 1, 4] and len(c._free) == 2 and c.page_table[2].tolist() == c.pages[2] + [-1] * 4
    c.release(0)
    assert c.lengths[0] == 0 and len(c._free) == 4
    with pytest.raises(ValueError, match="too small"):
        c.step([21, 0, 0])
    for bad in ([0, 0, 0], [1, 1]):
        with pytest.raises(ValueError):
            c.step(bad)
    with pytest.raises(ValueError):
        c.step([2, 0, 0], [[-1], [], []])
    free = list(c._free)
    for bad in ([[-1, 1], [], []], [[-1, -2], [], []], [[0, 0], [], []]):
        with pytest.raises(ValueError, match="parent"):
            c.step([2, 0, 0], bad)
    with pytest.raises(ValueError):
        c.step([-1, 2, 0])
    assert c._free == free                                    # nothing was handed out for them
    with pytest.raises(ValueError):
        cache_of(page_size=0)


@pytest.mark.parametrize("counts,error", [([8, 4, 8], RuntimeError), ([4, 21, 0], ValueError), ([0, 1, 21], ValueError)],
                         ids=str)
def test_a_refused_step_hands_out_nothing(counts, error):
    """A step that does not fit leaves the pages as they were, those of the sequences before the one that did not fit too."""
    c = cache_of(n_pages=4)
    c.step([3, 0, 0])
    before = (list(c._free), [list(p) for p in c.pages], c.page_table.clone(), list(c.lengths))
    with pytest.raises(error):
        c.step(counts)
    assert (c._free, c.pages, c.lengths) == (before[0], before[1], before[3]) and torch.equal(c.page_table, before[2])
    c.release(0)
    c.step([0, 0, 16])                                        # all four pages


def test_cache_keeps_a_path_of_a_tree():
    """Rows of the path move to the front, over pages, for all layers; sources that are destinations of others first read."""
    c = cache_of(max_seqs=2, page_size=3)
    c.kv.fill_(0.5)                                           # (fresh memory may hold NaN, which equals nothing)
    c.step([4, 2]); c.advance([4, 2])
    trees = [[-1, 0, 0, 1, 2, 3, 4], [-1]]
    st = c.step([7, 1], trees)
    assert st.positions.tolist() == [4, 5, 5, 6, 6, 7, 7, 2]
    rows = c.kv.view(2, 2, -1, 8)
    for i, s in enumerate(st.slots.tolist()):
        rows[:, :, s] = float(i + 1)
    before = rows[:, :, [c.row(0, r) for r in range(4)]].clone()
    c.keep([[0, 2, 4, 6], [0]])
    assert c.lengths == [8, 3] and len(c.pages[0]) == 3
    got = [rows[:, :, c.row(0, 4 + d)].unique().tolist() for d in range(4)]
    assert got == [[1.0], [3.0], [5.0], [7.0]]
    assert torch.equal(rows[:, :, [c.row(0, r) for r in range(4)]], before)
    c.keep([[], [0]])                                          # a finished sequence keeps nothing
    assert c.lengths == [8, 4]


def test_tree_masks_and_paths():
    from zero_amd.inference.paged import accepted_path, ancestors, depths, draft_tree, tree_mask
    assert draft_tree(2, 3) == [-1, 0, 0, 1, 2, 3, 4] and draft_tree(3, 0) == [-1]
    assert depths(draft_tree(2, 3)) == [0, 1, 1, 2, 2, 3, 3]
    assert ancestors([-1, 0, 0, 1]) == [0b1, 0b11, 0b101, 0b1011]
    with pytest.raises(ValueError):
        ancestors([-1, 1])
    m = tree_mask([[-1, 0], list(range(-1, 129))], "cpu")     # a pair, and a chain of 130: three words
    assert tuple(m.shape) == (132, 3) and m[1].tolist() == [3, 0, 0]
    assert m[2 + 129].tolist() == [-1, -1, 3] and m[2 + 63].tolist() == [-1, 0, 0]
    t = draft_tree(2, 2)                                      # root, a b, a' b'
    tok = [9, 4, 5, 6, 7]
    assert accepted_path(t, tok, [5, 0, 7, 0, 1]) == [0, 2, 4]
    assert accepted_path(t, tok, [4, 7, 7, 0, 1]) == [0, 1]
    assert accepted_path(t, tok, [3, 6, 7, 0, 1]) == [0]
    assert accepted_path([-1, 0, 0], [1, 2, 2], [2, 0, 0]) == [0, 1]


def test_generate_refuses_prompts_that_do_not_fit():
    from types import SimpleNamespace
    from zero_amd.inference.paged import generate_paged
    dec = SimpleNamespace(config=SimpleNamespace(hidden_size=16), generation_config=None)
    for prompts, more in (([], {}), ([torch.zeros(0, 16)], {}), ([torch.zeros(3, 8)], {}), ([torch.zeros(2, 3, 16)], {}),
                          ([torch.zeros(3, 16)], dict(assistant=dec, draft_depth=0)),
                          ([torch.zeros(3, 16)], dict(assistant=dec, assistant_prompts=[]))):
        with pytest.raises(ValueError):
            generate_paged(dec, prompts, 4, **more)
