"""ops.sample against a sort in 64-bit Python floats (tests/paged_ref.py), token for token."""
import math
import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def check_rows(x, u, T, k, p, mp, per_row=True, logits=None):
    from zero_amd import ops
    rows = x.shape[0]
    if per_row:
        par = dict(temperature=torch.tensor(T, device=DEV), top_k=torch.tensor(k, dtype=torch.int32, device=DEV),
                   top_p=torch.tensor(p, device=DEV), min_p=torch.tensor(mp, device=DEV))
    else:
        par = dict(temperature=T[0], top_k=k[0], top_p=p[0], min_p=mp[0])
    tok, logp = ops.sample(x.to(DEV) if logits is None else logits, torch.tensor(u, device=DEV), **par)
    for r in range(rows):
        i = r if per_row else 0
        t, lp = ref.sample_row(x[r].double().tolist(), f32(u[r]), f32(T[i]), k[i], f32(p[i]), f32(mp[i]))
        assert int(tok[r]) == t, (r, int(tok[r]), t, T[i], k[i], p[i], mp[i], u[r])
        got = float(logp[r])
        # a logarithm of 64-bit sums, rounded once to fp32
        assert got == lp or (math.isnan(got) and math.isnan(lp)) or abs(got - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (got, lp)


def settings(rng, rows):
    return ([rng.choice([0.0, 0.2, 0.7, 1.0, 3.0]) for _ in range(rows)], [rng.choice([0, 0, 1, 2, 17, 5000]) for _ in range(rows)],
            [rng.choice([1.0, 0.05, 0.5, 0.9, 0.999]) for _ in range(rows)], [rng.choice([0.0, 0.0, 0.01, 0.3, 1.0]) for _ in range(rows)])


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 1000, 1025, 9001, 32003])
@pytest.mark.parametrize("per_row", [True, False])
def test_sample_matches_the_sorted_row(V, per_row):
    g, rng = torch.Generator().manual_seed(V), random.Random(V)
    rows = 24 if V <= 9001 else 8
    x = (torch.randn(rows, V, generator=g) * 3).to(BF16)
    x[rows // 2:, : V // 3] = -math.inf if V > 2 else x[0, 0]
    u = [0.0, 1 - 2.0 ** -24] + [rng.random() * (1 - 2.0 ** -23) for _ in range(rows - 2)]
    check_rows(x, u, *settings(rng, rows), per_row=per_row)


def test_sample_a_vocabulary_of_several_parts():
    """More tokens than a workgroup holds at once (131 072)."""
    g, rng = torch.Generator().manual_seed(1), random.Random(1)
    rows, V = 6, 300007
    x = (torch.randn(rows, V, generator=g) * 2).to(BF16)
    x[3, :200000] = -math.inf
    x[4] = 1.5                                                   # one value: the rank is the token
    check_rows(x, [0.1, 0.5, 0.999, 0.3, 0.77, 0.0], [1.0, 0.5, 1.0, 2.0, 1.0, 0.0], [0, 0, 1000, 0, 0, 0],
               [1.0, 0.9, 1.0, 0.99, 1.0, 1.0], [0.0] * 5 + [0.1])


@pytest.mark.parametrize("V", [8192, 32768, 32769, 131072, 131073])
def test_sample_sizes_where_the_held_row_changes(V):
    g, rng = torch.Generator().manual_seed(V), random.Random(V)
    x = (torch.randn(5, V, generator=g) * 3).to(BF16)
    x[2, -1] = 30.0                                              # the last token is the only likely one
    x[3, -9:] = torch.tensor([9.0, 8.5, 9.0, 9.5, 8.0, 9.5, 9.0, 9.5, 9.0], dtype=BF16)
    check_rows(x, [0.3, 0.999, 0.5, 0.7, 0.0], [1.0, 0.8, 1.0, 0.3, 0.0], [0, 50, 0, 0, 0], [0.9, 1.0, 1.0, 1.0, 1.0],
               [0.0, 0.0, 0.0, 0.02, 0.0])


@pytest.mark.parametrize("V", [8201, 20011, 50021, 140003])
def test_sample_largest_logits_far_behind_the_first_ones(V):
    """The largest logit is not among the first 8192 tokens: 511, 512 and 513 values above those, or far beyond them."""
    g, rows = torch.Generator().manual_seed(V), 12
    x = (torch.randn(rows, V, generator=g)).to(BF16)
    late = 8192
    for r, key in enumerate((0x4000 + 511, 0x4000 + 512, 0x4000 + 513)):        # 0x4000: 2.0
        x[r, :late] = x[r, :late].clamp_max(2.0)
        x[r, 17] = 2.0
        x[r, late + 3 + r] = torch.tensor([key], dtype=torch.int16).view(BF16)[0]
        x[r, V - 1] = torch.tensor([key - 9], dtype=torch.int16).view(BF16)[0]
    x[3, :late] = -math.inf                                                      # nothing but what follows
    x[4, :late] = -1e30
    x[5, :late] = -(2.0 ** -100)                                                 # below zero, the largest is above
    x[5, late:] = x[5, late:] * 1e-30
    x[6, :late] = 1e-30
    x[7, late + 1] = math.inf
    x[8, V - 1] = math.nan
    x[9, :] = -math.inf
    x[9, V - 2] = -5.0
    x[10, :late] = x[10, :late] - 40.0
    x[11, V - 2] = 1e20
    T = [1.0, 30.0, 60.0, 1.0, 0.7, 1.0, 2.0, 1.0, 1.0, 1.0, 1.0, 2.0 ** 20]
    u = [0.2, 0.99, 0.999, 0.5, 0.3, 0.6, 0.9, 0.4, 0.4, 0.4, 0.8, 0.7]
    check_rows(x, u, T, [0, 0, 40, 0, 0, 0, 500, 0, 0, 0, 0, 0], [1.0, 1.0, 1.0, 0.9, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.5, 1.0],
               [0.0] * 8 + [0.0, 0.0, 0.05, 0.0])


@pytest.mark.parametrize("V", [8, 300, 4681, 32768])
def test_sample_many_rows_as_few(V):
    """More rows than CUs are counted in 16 bits, two rows a CU: the same tokens as in small batches, and the sorted rows'."""
    from zero_amd import ops
    g, rng, rows = torch.Generator().manual_seed(V), random.Random(V), 300
    x = (torch.randn(rows, V, generator=g) * 3).to(BF16)
    x[5] = 1.5                                                   # one value: a count of V
    x[6, ::2], x[6, 1::2] = 2.0, torch.tensor([0x4001], dtype=torch.int16).view(BF16)[0]    # two neighbouring values
    x[7] = -math.inf
    x[8, V - 1] = math.nan
    x[9, : V // 2] = -math.inf
    u = torch.tensor([rng.random() * (1 - 2.0 ** -23) for _ in range(rows)])
    T, k, p, mp = settings(rng, rows)
    T[5], k[5], p[5], mp[5], T[6], k[6], p[6], mp[6] = 1.0, 0, 1.0, 0.0, 1.0, 0, 1.0, 0.0
    par = [torch.tensor(T, device=DEV), torch.tensor(k, dtype=torch.int32, device=DEV), torch.tensor(p, device=DEV),
           torch.tensor(mp, device=DEV)]
    xd, ud = x.to(DEV), u.to(DEV)
    tok, logp = ops.sample(xd, ud, *par)
    halves = [ops.sample(xd[s], ud[s], *[v[s] for v in par]) for s in (slice(0, 150), slice(150, rows))]
    assert torch.equal(tok, torch.cat([h[0] for h in halves]))
    assert torch.equal(logp.nan_to_num(7.0), torch.cat([h[1] for h in halves]).nan_to_num(7.0))
    for r in list(range(4, 11)) + [200, 299]:
        t, lp = ref.sample_row(x[r].double().tolist(), float(u[r]), f32(T[r]), k[r], f32(p[r]), f32(mp[r]))
        got = float(logp[r])
        assert int(tok[r]) == t, (r, int(tok[r]), t)
        assert got == lp or (math.isnan(got) and math.isnan(lp)) or abs(got - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (r, got, lp)


def test_sample_ties_go_to_the_lowest_index():
    x = torch.tensor([[1.0, 3.0, -0.0, 3.0, 0.0, 3.0, -0.0, 1.0]] * 8).to(BF16)
    u = [0.0, 0.3, 0.4, 0.7, 0.0, 0.999, 0.5, 0.9]
    check_rows(x, u, [0.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 50.0], [0, 1, 2, 3, 4, 8, 0, 0], [1.0] * 6 + [0.34, 1.0], [0.0] * 8)
    y = torch.zeros(4, 70000).to(BF16)                            # more equal tokens than 16 bits count
    y[1, ::2] = -0.0
    y[2, 5] = 1e-30
    check_rows(y, [0.0, 0.9999, 0.5, 0.25], [1.0] * 4, [0, 0, 0, 33], [1.0, 1.0, 0.5, 1.0], [0.0] * 4)


def test_sample_extreme_rows():
    """Rows without a token, with NaN, infinities, the type's lowest value as a mask, values of far magnitudes."""
    low, big = torch.finfo(BF16).min, torch.finfo(BF16).max
    base = (torch.randn(12, 64, generator=torch.Generator().manual_seed(3)) * 2)
    base[0] = -math.inf
    base[1, 5] = math.nan
    base[2, 9] = -math.nan
    base[3, 7], base[3, 9] = math.inf, math.inf
    base[4, 8:] = low
    base[5] = low
    base[6, 1], base[6, 2] = big, low
    base[7] = torch.tensor([(-1.0) ** i * 2.0 ** (i - 60) for i in range(64)])
    base[8] = -torch.tensor([2.0 ** (i - 30) for i in range(64)])
    base[9, 1:] = -math.inf
    base[10] = math.inf
    x = base.to(BF16)
    for u in (0.0, 0.31, 0.97):
        check_rows(x, [u] * 12, [1.0] * 12, [0] * 12, [1.0] * 12, [0.0] * 12)
        check_rows(x, [u] * 12, [1e9] * 12, [0, 3] * 6, [0.8] * 12, [0.0] * 12)
        check_rows(x, [u] * 12, [0.0] * 12, [0] * 12, [1.0] * 12, [0.0] * 12)


def test_sample_settings_out_of_their_ranges_per_row():
    x = (torch.randn(10, 200, generator=torch.Generator().manual_seed(5)) * 2).to(BF16)
    nan = math.nan
    check_rows(x, [0.6] * 8 + [-1.0, 2.0], [-1.0, nan, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0],
               [0, 0, -3, 0, 0, 0, 0, 0, 0, 0], [1.0, 1.0, 1.0, -0.5, 0.0, 7.0, nan, 1.0, 1.0, 1.0],
               [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 5.0, nan, -1.0])


def test_sample_strided_rows_and_every_alignment():
    g = torch.Generator().manual_seed(6)
    wide = (torch.randn(9, 1200, generator=g) * 2).to(BF16)
    dev = wide.to(DEV)
    for start, V in ((0, 1000), (1, 999), (3, 513), (8, 800), (5, 1)):
        check_rows(wide[:, start:start + V], [0.05 + 0.1 * i for i in range(9)], [1.0] * 9, [0] * 9, [0.95] * 9, [0.0] * 9,
                   logits=dev[:, start:start + V])


def test_sample_follows_the_distribution():
    """A row's tokens over many u: shares within 5 standard deviations of their probability."""
    from zero_amd import ops
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], dtype=BF16)
    n = 40000
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n          # evenly spread: every share is exact to a step
    tok, logp = ops.sample(x.expand(n, 5).contiguous().to(DEV), u.float().to(DEV), temperature=0.7)
    p = torch.softmax(x.double() / f32(0.7), 0)
    share = torch.bincount(tok.cpu(), minlength=5).double() / n
    assert ((share - p).abs() <= 2.0 / n).all()
    assert torch.allclose(logp.cpu().double(), p.log()[tok.cpu()], rtol=1e-6, atol=1e-7)
