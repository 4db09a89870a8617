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
                                 dict(out=PTR + 8)], ids=str)
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
