"""Paged-cache operators on the GPU against 64-bit plain forms (tests/paged_ref.py)."""
import math
import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
HALF_STEP = 2.0 ** -8            # a bf16 rounding, relative


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF16)


def make(seqs, Hq, Hkv, hd, page, tree=False, seed=0, spare=3, words=None, poison=True):
    """seqs: (new, cached) per sequence.  Unused pages and the rows past a sequence's end hold NaN."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    need = [-(-c // page) for _, c in seqs]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g)
    k, v = _normal(g, n_pages, page, Hkv * hd), _normal(g, n_pages, page, Hkv * hd)
    cols = max(max(need), 1) + 1
    table = torch.full((len(seqs), cols), -7, dtype=torch.int32)
    at = 0
    used = torch.zeros(n_pages, page, dtype=torch.bool)
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m].to(torch.int32)
        at += m
        for r in range(seqs[b][1]):
            used[int(table[b, r // page]), r % page] = True
    if poison:
        k[~used], v[~used] = math.nan, math.nan
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    mask = None
    if tree:
        W = words or -(-max(n for n, _ in seqs) // 64)
        mask = torch.zeros((cu[-1], W), dtype=torch.int64)
        for b, (n, _) in enumerate(seqs):
            seen = []
            for i in range(n):
                bits = (1 << i) | (seen[rng.randint(max(0, i - 5), i - 1)] if i else 0)
                seen.append(bits)
                for w in range(W):
                    x = (bits >> (64 * w)) & (2 ** 64 - 1)
                    mask[cu[b] + i, w] = x - 2 ** 64 if x >= 2 ** 63 else x
    q = _normal(g, cu[-1], Hq * hd, scale=1.5)
    return dict(q=q, k=k, v=v, table=table, ctx=[c for _, c in seqs], cu=cu, mask=mask, Hq=Hq, Hkv=Hkv, hd=hd)


def call(c, **kw):
    from zero_amd import ops
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return ops.attn_paged(d(c["q"]), d(c["k"]), d(c["v"]), d(c["table"]), d(torch.tensor(c["ctx"], dtype=torch.int32)),
                          d(torch.tensor(c["cu"], dtype=torch.int32)), max(max(b - a for a, b in zip(c["cu"], c["cu"][1:])), 1),
                          max(max(c["ctx"]), 1), c["Hq"], c["Hkv"], c["hd"], c["hd"] ** -0.5, tree_mask=d(c["mask"]), **kw)


def agree(out, c):
    """|out - o| <= a rounding of o + a rounding of every p (moves o by that share of sum p |v|) + 2^-11 of the same
    for the fp32 work: scores of 128 products (128 * 2^-24 * sum |q k| * scale < 2^-12 here), exponential, sums."""
    want, mag = ref.attention(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["cu"], c["Hq"], c["Hkv"], c["hd"],
                              c["hd"] ** -0.5, c["mask"])
    own = ~want.isnan().all(1)
    got = out.double().cpu()[own]
    want, mag = want[own], mag[own]
    assert torch.isfinite(got).all()
    tol = HALF_STEP * want.abs() + (HALF_STEP + 2.0 ** -11) * mag + 1e-30
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


SEQS = {
    "one": [(1, 1)],
    "one-long": [(1, 1025)],
    "singles": [(1, 1), (1, 63), (1, 64), (1, 65), (1, 200), (1, 31), (1, 97)],
    "some-empty": [(0, 5), (1, 17), (0, 0), (3, 3), (0, 64)],
    "chunks": [(17, 17), (33, 100), (1, 300), (64, 64), (70, 129)],
    "long-chunk": [(150, 331)],
}


@pytest.mark.parametrize("seqs", SEQS.values(), ids=SEQS.keys())
@pytest.mark.parametrize("Hq,Hkv,hd,page", [(8, 2, 128, 16), (3, 1, 128, 1), (4, 4, 64, 7), (20, 2, 64, 64),
                                            (17, 1, 128, 100), (6, 2, 128, 1024)])
def test_attn_paged_chain(seqs, Hq, Hkv, hd, page):
    c = make(seqs, Hq, Hkv, hd, page, seed=len(seqs))
    agree(call(c), c)


@pytest.mark.parametrize("seqs", [[(2, 2)], [(7, 30), (16, 16), (1, 65)], [(64, 200), (13, 13)], [(65, 130), (3, 70)],
                                  [(130, 391)]], ids=str)
@pytest.mark.parametrize("Hq,Hkv,hd,page", [(8, 2, 128, 16), (5, 1, 64, 24), (4, 4, 128, 5), (12, 4, 64, 64)])
def test_attn_paged_tree(seqs, Hq, Hkv, hd, page):
    c = make(seqs, Hq, Hkv, hd, page, tree=True, seed=7)
    agree(call(c), c)


def test_attn_paged_rows_that_see_nothing():
    """A clear mask over an empty prefix: zeros; over a prefix: the prefix alone, whatever the hidden rows hold."""
    c = make([(4, 4), (5, 40)], 8, 2, 128, 8, tree=True, seed=3)
    c["mask"][1] = 0
    c["mask"][4:] = 0
    for j in range(35, 40):                                          # the new rows of sequence 1 are seen by nobody
        c["k"][int(c["table"][1, j // 8]), j % 8] = math.nan
        c["v"][int(c["table"][1, j // 8]), j % 8] = math.inf
    out = call(c)
    assert (out[1] == 0).all()
    agree(out, c)


def test_attn_paged_large_scores():
    """Scores of several thousand, of both signs: the running maximum is subtracted before every exponential."""
    c = make([(1, 130), (40, 150)], 8, 2, 128, 16, seed=5)
    c["k"] *= 64
    c["q"] *= 16
    want, mag = ref.attention(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["cu"], 8, 2, 128, 128 ** -0.5)
    got = call(c).double().cpu()
    # a score of up to 128 * 96 * 256 * scale ~ 3e5 / 2^24-steps of its partial sums: p off by up to 2^-3 in the worst
    # case where two keys are that near; the bound is on the value's magnitude, and nothing overflows
    assert torch.isfinite(got).all() and ((got - want).abs() <= 0.25 * mag + HALF_STEP * want.abs()).all()


def test_attn_paged_bad_pages_are_not_seen():
    """Page numbers out of range (never read: the kernel compares each with the page count) hide their rows."""
    c = make([(1, 100), (20, 90)], 4, 2, 64, 16, seed=9)
    c["table"][0, 2], c["table"][1, 0], c["table"][1, 3] = c["k"].shape[0], -1, 2 ** 31 - 1
    agree(call(c), c)


def test_attn_paged_strided_rows_behind_the_last_sequence_and_out():
    """q and out as column slices of wider rows; rows of out past cu_q[B] and the columns beside stay as they were."""
    from zero_amd import ops
    c = make([(3, 20), (18, 60)], 4, 2, 64, 16, seed=11)
    T, w = c["cu"][-1], 4 * 64
    wide_q = torch.full((T + 5, w + 16), math.nan, dtype=BF16)
    wide_q[:T, 8:8 + w] = c["q"]
    wide_o = torch.full((T + 5, w + 24), 7.0, dtype=BF16, device=DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    got = ops.attn_paged(wide_q.to(DEV)[:, 8:8 + w], c["k"].to(DEV), c["v"].to(DEV), c["table"].to(DEV), i32(c["ctx"]),
                         i32(c["cu"]), 18, 60, 4, 2, 64, 64 ** -0.5, out=wide_o[:, 16:16 + w])
    agree(got[:T], c)
    assert (wide_o[T:] == 7).all() and (wide_o[:, :16] == 7).all() and (wide_o[:, 16 + w:] == 7).all()


def test_attn_paged_is_bitwise_reproducible_and_independent_of_its_neighbours():
    c = make([(1, 900), (30, 200), (1, 5)], 8, 2, 128, 16, seed=13)
    a, b = call(c), call(c)
    assert torch.equal(a, b)


def test_attn_paged_far_page_offsets():
    """Cache rows whose byte offset passes 2^32 (a cache of 4.5 GiB an array)."""
    Hkv, hd, page = 8, 128, 64
    pages = (9 << 29) // (page * Hkv * hd * 2) + 1
    from zero_amd import ops
    k = torch.empty((pages, page, Hkv * hd), dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(1)
    far = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    kk, vv, q = _normal(g, 3, page, Hkv * hd), _normal(g, 3, page, Hkv * hd), _normal(g, 1, 2 * Hkv * hd)
    for i in range(3):
        k[int(far[0, i])], v[int(far[0, i])] = kk[i].to(DEV), vv[i].to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = ops.attn_paged(q.to(DEV), k, v, far.to(DEV), i32([150]), i32([0, 1]), 1, 150, 16, 8, 128, 128 ** -0.5)
    c = dict(q=q, k=kk, v=vv, table=torch.tensor([[0, 1, 2]]), ctx=[150], cu=[0, 1], mask=None, Hq=16, Hkv=8, hd=128)
    agree(out, c)
    # and the append reaches them
    T = 2
    qkv = _normal(g, T, (16 + 2 * Hkv) * hd)
    cos, sin = torch.ones(4, hd // 2), torch.zeros(4, hd // 2)
    slots = [(pages - 1) * page + 5, 3]
    ops.kv_append_paged(qkv.to(DEV), cos.to(DEV), sin.to(DEV), k, v, i32([0, 1]), i32(slots), 16, 8, hd)
    for t, s in enumerate(slots):
        assert torch.equal(k.view(-1, Hkv * hd)[s].cpu(), qkv[t, 16 * hd:24 * hd])
        assert torch.equal(v.view(-1, Hkv * hd)[s].cpu(), qkv[t, 24 * hd:])


@pytest.mark.parametrize("Hq,Hkv,hd,rot", [(8, 2, 128, 128), (8, 2, 128, 64), (3, 1, 64, 64), (4, 4, 64, 16), (17, 1, 128, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,page", [(1, 16), (37, 5), (130, 64)])
def test_kv_append_paged(Hq, Hkv, hd, rot, interleaved, T, page):
    """q, k: one rounding of the turned pair (two products and a sum in fp32: 3 * 2^-24 of |x| + |y| beside it);
    v: exact; every other cache row untouched; padding tokens and slots out of range append nothing."""
    from zero_amd import ops
    g = torch.Generator().manual_seed(T + rot)
    pages, P, W = -(-T // page) + 2, 300, (Hq + 2 * Hkv) * hd
    qkv = _normal(g, T, W + 8)[:, :W]
    ang = torch.rand(P, rot // 2, generator=g) * 6.28
    cos, sin = ang.cos(), ang.sin()
    k, v = _normal(g, pages, page, Hkv * hd), _normal(g, pages, page, Hkv * hd)
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32)
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    if T > 30:
        slots[3], slots[4], pos[5], pos[6] = -1, pages * page, -1, P
    kd, vd, qd = k.to(DEV), v.to(DEV), qkv.to(DEV)
    got = ops.kv_append_paged(qd, cos.to(DEV), sin.to(DEV), kd, vd, pos.to(DEV), slots.to(DEV), Hq, Hkv, hd,
                              interleaved=interleaved)
    assert torch.equal(qd.cpu(), qkv)
    want_k, want_v = k.double().view(-1, Hkv, hd), v.clone().view(-1, Hkv * hd)
    near_k = torch.zeros_like(want_k)
    for t in range(T):
        x = qkv[t].double().view(Hq + 2 * Hkv, hd)
        if not 0 <= int(pos[t]) < P:
            assert (got[t] == 0).all()
            continue
        c, s = cos[int(pos[t])].double(), sin[int(pos[t])].double()
        turned = ref.rotate(x[:Hq + Hkv], c, s, interleaved)
        size = ref.rotate(x[:Hq + Hkv].abs(), c.abs(), -s.abs(), interleaved).abs() + x[:Hq + Hkv].abs()
        tol = HALF_STEP * turned.abs() + 2.0 ** -21 * size
        assert ((got[t].double().cpu().view(Hq, hd) - turned[:Hq]).abs() <= tol[:Hq]).all(), t
        if 0 <= int(slots[t]) < pages * page:
            want_k[int(slots[t])], near_k[int(slots[t])] = turned[Hq:], tol[Hq:]
            want_v[int(slots[t])] = qkv[t, (Hq + Hkv) * hd:]
    assert ((kd.double().cpu().view(-1, Hkv, hd) - want_k).abs() <= near_k).all()
    assert torch.equal(vd.cpu().view(-1, Hkv * hd), want_v)


def test_kv_append_paged_turns_like_rope():
    """Half layout over the whole head: bit for bit zk_rope's rows."""
    from zero_amd import ops
    g = torch.Generator().manual_seed(2)
    T, Hq, Hkv, hd = 9, 6, 2, 128
    qkv = _normal(g, T, (Hq + 2 * Hkv) * hd).to(DEV)
    ang = torch.rand(T, hd // 2, generator=g) * 6.28
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    k = torch.zeros((2, 8, Hkv * hd), dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    at = torch.arange(T, dtype=torch.int32, device=DEV)
    q = ops.kv_append_paged(qkv, cos, sin, k, v, at, at, Hq, Hkv, hd)
    turned = ops.rope_(qkv.clone(), cos, sin, T, Hq + Hkv, hd)
    assert torch.equal(q, turned[:, :Hq * hd])
    assert torch.equal(k.view(-1, Hkv * hd)[:T], turned[:, Hq * hd:(Hq + Hkv) * hd])


def test_decode_step_of_the_three_operators_in_a_captured_graph():
    """append -> attention -> (a product as the model's head) -> sample, captured once and replayed over growing caches
    with eager work between the replays; every replay equals the eager run of the same step."""
    from zero_amd import ops
    g = torch.Generator().manual_seed(4)
    B, Hq, Hkv, hd, page, V = 3, 8, 2, 64, 16, 501
    cols, P = 8, 200
    kv = torch.zeros((2, B * cols, page, Hkv * hd), dtype=BF16, device=DEV)
    table = torch.arange(B * cols, dtype=torch.int32, device=DEV).view(B, cols)
    ang = torch.rand(P, hd // 2, generator=g) * 6.28
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    head = _normal(g, 504, Hq * hd).to(DEV)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    pos, slots, ctx = (torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(3))
    qkv = torch.zeros((B, (Hq + 2 * Hkv) * hd), dtype=BF16, device=DEV)
    u = torch.zeros(B, device=DEV)
    ws = torch.empty(max(1, ops.attn_paged_ws_floats(B, B, 1, cols * page, Hq, Hkv, hd)), device=DEV)

    def step(kv):
        q = ops.kv_append_paged(qkv, cos, sin, kv[0], kv[1], pos, slots, Hq, Hkv, hd)
        o = ops.attn_paged(q, kv[0], kv[1], table, ctx, cu, 1, cols * page, Hq, Hkv, hd, hd ** -0.5, ws=ws)
        logits = ops.gemm(o, head)[:, :V]
        return (o, logits) + ops.sample(logits, u, temperature=0.8, top_k=40, top_p=0.9)

    def feed(i):
        at = [3 + i * 7, i, 40 + i * 13]
        qkv.copy_(_normal(g, *qkv.shape).to(DEV))
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        slots.copy_(torch.tensor([b * cols * page + a for b, a in enumerate(at)], dtype=torch.int32))
        ctx.copy_(torch.tensor([a + 1 for a in at], dtype=torch.int32))
        u.copy_(torch.rand(B, generator=g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        feed(0)
        step(kv)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(kv)
    for i in range(5):
        feed(i)
        other = kv.clone()
        want = step(other)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kv, other)
        for a, b in zip(held, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("Hq,Hkv,hd,page", [(8, 2, 128, 64), (16, 2, 64, 128), (6, 1, 128, 48)])
@pytest.mark.parametrize("tree", [False, True])
def test_attn_paged_shares_of_long_ragged_sequences(Hq, Hkv, hd, page, tree):
    """Many-row tiles whose keys are dealt out over workgroups by the sequences' own lengths, and merged."""
    c = make([(37, 3001), (70, 700), (9, 20), (0, 90), (41, 41), (33, 1999)], Hq, Hkv, hd, page, tree=tree, seed=21)
    agree(call(c), c)


@pytest.mark.parametrize("Hq,Hkv,hd,tree", [(20, 2, 64, False), (17, 1, 128, False), (20, 4, 128, True)])
def test_attn_paged_shares_of_many_rows(Hq, Hkv, hd, tree):
    """More rows than waves fit the GPU at once, some of their sequences shared out; heads that no group of eight ends with."""
    c = make([(300, 1900), (250, 700), (1, 900)], Hq, Hkv, hd, 32, tree=tree, seed=24)
    agree(call(c), c)


@pytest.mark.parametrize("ctx", [5000, 40001])
@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 1, 128), (4, 2, 64), (40, 2, 128)])
def test_attn_paged_single_tokens_far_into_the_cache(ctx, Hq, Hkv, hd):
    c = make([(1, ctx), (1, 300)], Hq, Hkv, hd, 64, seed=22, poison=False)
    agree(call(c), c)


@pytest.mark.parametrize("B,ctx,Hq,Hkv,hd", [(3, 270, 4, 4, 128), (30, 700, 8, 8, 128), (6, 1023, 32, 32, 64),
                                            (40, 300, 32, 8, 128), (70, 1000, 16, 16, 64)])
@pytest.mark.parametrize("tree", [False, True])
def test_attn_paged_batches_of_short_sequences(B, ctx, Hq, Hkv, hd, tree):
    """Lengths where eight waves take a whole sequence: up to 4 new tokens, ragged."""
    rng = random.Random(B)
    seqs = [(1 + b % (16 // (Hq // Hkv)) % 4, ctx) if b == 0 else (n, max(n, rng.randrange(1, ctx)))
            for b, n in ((b, rng.choice([0, 1, 1, 2, 4])) for b in range(B))]
    c = make(seqs, Hq, Hkv, hd, 48, tree=tree, seed=B, words=1 if tree else None)
    agree(call(c), c)


def test_attn_paged_whole_sequences_infinities_and_nan():
    """The same form with infinities and NaN in new rows that only some tokens see."""
    Hq = Hkv = 16
    c = make([(4, 500), (2, 130), (1, 33), (3, 257), (0, 9), (4, 4), (4, 400), (2, 511)], Hq, Hkv, 64, 16, tree=True, seed=5)
    for b, n in ((0, 4), (1, 2), (3, 3), (5, 4), (6, 4)):
        for j, val in ((1, math.inf), (n - 1, math.nan)):
            r = c["ctx"][b] - n + j
            c["v"][int(c["table"][b, r // 16]), r % 16, 5 + j::17] = val
    want, mag = ref.attention(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["cu"], Hq, Hkv, 64, 0.125, c["mask"])
    differ_like(call(c), want, torch.nan_to_num(mag, nan=0.0, posinf=0.0))


def test_attn_paged_more_sequences_than_lanes():
    """150 sequences, some without new tokens: the layout of shares is found over several rounds of 64."""
    rng = random.Random(1)
    seqs = [(rng.choice([0, 1, 3, 20, 34]), 0) for _ in range(150)]
    seqs = [(n, n + rng.randrange(0, 330)) for n, _ in seqs]
    c = make(seqs, 4, 2, 64, 16, seed=23)
    agree(call(c), c)


def differ_like(got, want, mag):
    """Where the formula is finite: as ``agree``; where it is infinite or NaN: the same."""
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    tol = HALF_STEP * want.abs() + (HALF_STEP + 2.0 ** -11) * mag + 1e-30
    assert ((got - want).abs()[fin] <= tol[fin]).all()


@pytest.mark.parametrize("seqs", [[(1, 40), (3, 9)], [(8, 50), (5, 5)], [(40, 130), (70, 70)], [(1, 1100), (2, 650)],
                                  [(40, 900), (9, 300)]], ids=["few", "some", "many", "few-shared", "many-shared"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("tree", [False, True])
def test_attn_paged_infinities_and_nan_reach_those_that_see_them_only(seqs, page, tree):
    """New rows whose values hold infinities or NaN, seen by later tokens (or a branch) and hidden from the others."""
    Hq, Hkv, hd = 8, 2, 128
    c = make(seqs, Hq, Hkv, hd, page, tree=tree, seed=31)
    for b, (n, ctx) in enumerate(seqs):
        for j, val in ((n // 3, math.inf), (n // 2, math.nan), (n - 1, -math.inf)):
            r = ctx - n + j
            c["v"][int(c["table"][b, r // page]), r % page, 5 + j % 3::17] = val
    want, mag = ref.attention(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["cu"], Hq, Hkv, hd, hd ** -0.5, c["mask"])
    differ_like(call(c), want, torch.nan_to_num(mag, nan=0.0, posinf=0.0))


def test_attn_paged_nan_keys_reach_those_that_see_them_only():
    c = make([(40, 100), (1, 7)], 8, 2, 128, 64, seed=32)
    c["k"][int(c["table"][0, 80 // 64]), 80 % 64, 3] = math.nan        # key 80 = new token 20, head 0
    want, mag = ref.attention(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["cu"], 8, 2, 128, 128 ** -0.5)
    assert want[:20].isfinite().all() and want[20:40, :4 * 128].isnan().all()
    differ_like(call(c), want, torch.nan_to_num(mag))


def test_attn_paged_bounds_from_the_host_only_shape_the_launch():
    """max_q and max_ctx larger than needed (a captured graph's bounds) give the same answer within the tolerance, max_ctx
    smaller than a length too; tokens past max_q are left as they are."""
    from zero_amd import ops
    c = make([(2, 500), (1, 33)], 8, 2, 128, 16, seed=33)
    d = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in c.items()}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731

    def run(max_q, max_ctx, out=None):
        return ops.attn_paged(d["q"], d["k"], d["v"], d["table"], i32(c["ctx"]), i32(c["cu"]), max_q, max_ctx, 8, 2, 128,
                              128 ** -0.5, out=out)
    for max_q, max_ctx in ((2, 500), (2, 40), (7, 3000), (30, 100000), (30, 300)):
        agree(run(max_q, max_ctx), c)
    out = torch.full_like(d["q"], 9.0)
    run(1, 500, out)
    assert (out[1] == 9).all() and not (out[0] == 9).all() and not (out[2] == 9).all()


def test_operators_on_a_side_stream_and_two_at_once():
    """Inputs made on one stream and used on another that waited for it; two streams at the same time, a workspace each."""
    from zero_amd import ops
    cs = [make([(1, 3000), (20, 900)], 8, 2, 128, 64, seed=s) for s in (41, 42)]
    want = [call(c) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got.clear()
        for c, st in zip(cs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(call(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(5, 70000, device=DEV).to(BF16)
    u = torch.rand(5, device=DEV)
    a = ops.sample(x, u)
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        b = ops.sample(x, u)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_captured_graphs_with_a_workspace_each():
    """Two graphs of shared-out attention, replayed in turn and overlapping on two streams."""
    from zero_amd import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    graphs, outs, want, alive = [], [], [], []                  # a graph reads its inputs where they lay at capture
    for s in (51, 52):
        c = make([(20, 1500), (1, 700)], 8, 2, 128, 64, seed=s)
        d = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in c.items()}
        ws = torch.empty(max(1, ops.attn_paged_ws_floats(2, 21, 20, 1500, 8, 2, 128)), device=DEV)
        ctx, cu = i32(c["ctx"]), i32(c["cu"])
        f = lambda d=d, ws=ws, ctx=ctx, cu=cu: ops.attn_paged(d["q"], d["k"], d["v"], d["table"], ctx, cu, 20, 1500, 8, 2,  # noqa: E731
                                                              128, 128 ** -0.5, ws=ws)
        alive.append((d, ws, ctx, cu))
        want.append(f().clone())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()
        torch.cuda.synchronize()


def test_wrapper_refusals_on_the_device():
    from zero_amd import ops
    c = make([(2, 20)], 4, 2, 64, 16)
    d = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in c.items()}
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    ok = dict(q=d["q"], k_cache=d["k"], v_cache=d["v"], page_table=d["table"], ctx_lens=i32([20]), cu_q=i32([0, 2]), max_q=2,
              max_ctx=20, Hq=4, Hkv=2, hd=64, scale=0.1)
    ops.attn_paged(**ok)
    for bad in (dict(q=d["q"].float()), dict(q=d["q"][:, :128]), dict(Hkv=3), dict(k_cache=d["k"][:, ::2]),
                dict(v_cache=d["v"][:2]), dict(page_table=d["table"].long()), dict(ctx_lens=i32([20, 3])), dict(cu_q=i32([0])),
                dict(ctx_lens=d["q"][:1, 0]), dict(tree_mask=torch.zeros(3, 1, dtype=torch.int64, device=DEV)),
                dict(tree_mask=torch.zeros(2, 1, dtype=torch.int32, device=DEV)), dict(out=torch.empty(2, 64, device=DEV)),
                dict(ctx_lens=torch.tensor([20], dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.attn_paged(**{**ok, **bad})
    from zero_amd._lib import ZeroHipError
    with pytest.raises((ValueError, ZeroHipError)):
        ops.attn_paged(**{**ok, "max_q": 0})
    qkv = torch.zeros((2, 8 * 64), dtype=BF16, device=DEV)
    cos = torch.ones((4, 32), device=DEV)
    ok = dict(qkv=qkv, cos_t=cos, sin_t=cos, k_cache=d["k"], v_cache=d["v"], positions=i32([0, 1]), slots=i32([-1, -1]), Hq=4,
              Hkv=2, hd=64)
    ops.kv_append_paged(**ok)
    for bad in (dict(qkv=qkv[:, :256]), dict(cos_t=cos.double()), dict(sin_t=cos[:2]), dict(positions=i32([0])),
                dict(slots=i32([0, 1]).long()), dict(k_cache=d["k"].view(-1, 128)), dict(q_out=qkv)):
        with pytest.raises(ValueError):
            ops.kv_append_paged(**{**ok, **bad})
    for half in (4, 48):                                       # 8 values are no whole unit, 96 more than the head
        t = torch.ones((4, half), device=DEV)
        with pytest.raises(ZeroHipError):
            ops.kv_append_paged(**{**ok, "cos_t": t, "sin_t": t})
    x, u = torch.zeros((2, 9), dtype=BF16, device=DEV), torch.zeros(2, device=DEV)
    ops.sample(x, u)
    for bad in (dict(logits=x.float()), dict(logits=x.t()), dict(u=u[:1]), dict(u=u.double()), dict(temperature=-1.0),
                dict(temperature=math.nan), dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=2.0),
                dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]), dict(u=u.cpu())):
        with pytest.raises(ValueError):
            ops.sample(**{**dict(logits=x, u=u), **bad})
