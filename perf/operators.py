"""Workloads of the serving operators: appending to a paged key / value cache, attention of new tokens
(single tokens, prompt chunks, trees of drafted tokens) over it, and drawing the next token from logits.

``run`` computes a case through ``zero_amd.ops`` where ``own`` is true and in plain 32- or 64-bit torch
operations where it is not; ``exact`` is the same result from the definitions in 64 bits.

Definitions
  append     q' = rot(q), cache[slot[t]] = (rot(k[t]), v[t]) for the packed rows q|k|v of T new tokens; rot turns
             the first 2 * cos.shape[1] values of a head by the angle row of the token's position, either pairing
             value i with value i + rot/2 (half layout) or 2i with 2i + 1 (interleaved layout).
  attention  new token i of sequence b sits in cache row ctx[b] - n[b] + i of the sequence, sees all rows before
             the new ones and, of the new ones, those up to its own (chain) or those its mask bits name (tree);
             query head h reads key / value head h // (Hq / Hkv).
  sample     tokens in falling order of their logit, ties by the lower index; w = exp((l - max) / T); top-k keeps
             the first k, top-p the shortest prefix that reaches p of their sum, min-p those with w >= min_p; the
             token drawn is the first whose running sum exceeds u times the kept sum.  T <= 0 takes the first.
"""
import math
import random

import numpy as np
import torch

own = False


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def listed():
    return [
        # one token of one conversation goes into the cache: pure latency
        dict(name="append-1", op="append", T=1, Hq=32, Hkv=8, hd=128, rot=128, interleaved=False, page=64),
        # a verification step of a batch (a few drafted tokens each), heads of the largest configuration, half of
        # the head rotated, interleaved pairs
        dict(name="append-batch", op="append", T=211, Hq=64, Hkv=8, hd=128, rot=64, interleaved=True, page=16),
        # a long prompt at once
        dict(name="append-prompt", op="append", T=8191, Hq=32, Hkv=8, hd=128, rot=128, interleaved=False, page=64),
        # single token of one conversation after an image prompt (577 + text)
        dict(name="decode-1", op="attention", B=1, Hq=32, Hkv=8, hd=128, page=64, new_lo=1, new_hi=1, ctx_lo=771,
             ctx_hi=771, tree=False, shape=1),
        # single tokens of a full batch of conversations of very different lengths
        dict(name="decode-batch", op="attention", B=48, Hq=32, Hkv=8, hd=128, page=64, new_lo=1, new_hi=1, ctx_lo=700,
             ctx_hi=8192, tree=False, shape=2),
        # single token at the end of the longest context, the heads one of eight ranks holds, odd pages
        dict(name="decode-long", op="attention", B=1, Hq=8, Hkv=1, hd=128, page=100, new_lo=1, new_hi=1, ctx_lo=131071,
             ctx_hi=131071, tree=False, shape=3),
        # trees of drafted tokens are verified for a small batch
        dict(name="tree-batch", op="attention", B=7, Hq=32, Hkv=8, hd=128, page=32, new_lo=17, new_hi=61, ctx_lo=1500,
             ctx_hi=5000, tree=True, shape=4),
        # a few heads of width 64, ragged chunks of three prompts
        dict(name="chunk-ragged", op="attention", B=3, Hq=16, Hkv=16, hd=64, page=24, new_lo=129, new_hi=517,
             ctx_lo=900, ctx_hi=4099, tree=False, shape=5),
        # a chunk of a long prompt over what is cached of it
        dict(name="chunk-long", op="attention", B=1, Hq=32, Hkv=8, hd=128, page=64, new_lo=2048, new_hi=2048,
             ctx_lo=32768, ctx_hi=32768, tree=False, shape=6),
        # the next token of one conversation
        dict(name="sample-1", op="sample", rows=1, V=128256, mode="nucleus", per_row=False),
        # a batch in which every conversation has settings of its own, some tokens forbidden, odd vocabulary
        dict(name="sample-batch", op="sample", rows=61, V=32003, mode="mixed", per_row=True),
        # every node of a large batch of drafted trees
        dict(name="sample-many", op="sample", rows=512, V=128256, mode="mixed", per_row=True),
    ]


_HEADS = [(32, 8, 128), (8, 1, 128), (64, 8, 128), (16, 4, 128), (6, 2, 128), (16, 16, 64), (32, 4, 64), (12, 4, 64)]
_PAGES = [1, 16, 24, 32, 64, 100, 256]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "tree", "chunk", "sample"])
    Hq, Hkv, hd = rng.choice(_HEADS)
    page = rng.choice(_PAGES)
    if op == "append":
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        return dict(op="append", T=_log_int(rng, 1, 8191), Hq=Hq, Hkv=Hkv, hd=hd, rot=rot,
                    interleaved=rng.random() < 0.3, page=page)
    if op == "sample":
        return dict(op="sample", rows=_log_int(rng, 1, 512), V=_log_int(rng, 257, 128256),
                    mode=rng.choice(["greedy", "plain", "topk", "nucleus", "minp", "mixed"]), per_row=rng.random() < 0.5)
    if op == "decode":
        B = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, min(131072, 262144 // B))
        return dict(op="attention", B=B, Hq=Hq, Hkv=Hkv, hd=hd, page=page, new_lo=1, new_hi=1,
                    ctx_lo=max(1, int(hi * rng.uniform(0.1, 1.0))), ctx_hi=hi, tree=False, shape=rng.randrange(1 << 20))
    if op == "tree":
        B, n = _log_int(rng, 1, 16), _log_int(rng, 2, 100)
        hi = max(n, _log_int(rng, 128, 16384 // max(1, B // 4)))
        return dict(op="attention", B=B, Hq=Hq, Hkv=Hkv, hd=hd, page=page, new_lo=max(1, n // 3), new_hi=n,
                    ctx_lo=max(n, hi // 3), ctx_hi=hi, tree=True, shape=rng.randrange(1 << 20))
    B, n = _log_int(rng, 1, 4), _log_int(rng, 65, 2048)
    hi = max(n, _log_int(rng, 512, 32768 // (2 * B if Hq > 32 else B)))
    return dict(op="attention", B=B, Hq=Hq, Hkv=Hkv, hd=hd, page=page, new_lo=max(1, n // 3), new_hi=n,
                ctx_lo=max(n, hi // 2), ctx_hi=hi, tree=False, shape=rng.randrange(1 << 20))


def _lengths(case):
    """New tokens and cached rows (the new ones among them) of every sequence, and the trees' parents."""
    rng = random.Random(case["shape"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    ctx = [max(n, _log_int(rng, case["ctx_lo"], case["ctx_hi"])) for n in new]
    new[0], ctx[0] = case["new_hi"], max(case["new_hi"], case["ctx_hi"])
    parents = None
    if case["tree"]:
        parents = [[-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)] for n in new]
    return new, ctx, parents


def _ancestors(parents):
    """For each node the nodes on its path from the root, itself included, as an integer of bits."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((1 << i) | (seen[p] if p >= 0 else 0))
    return seen


def work(case):
    if case["op"] == "append":
        width, kv = (case["Hq"] + 2 * case["Hkv"]) * case["hd"], case["Hkv"] * case["hd"]
        T = case["T"]
        return {"bytes": T * (2 * width * 2 + case["rot"] * 4 + 8),
                "flops": T * 3 * (case["Hq"] + case["Hkv"]) * case["rot"]}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["V"] * 2 + 4 + 4 + 8 + (16 if case["per_row"] else 0)),
                "flops": case["rows"] * case["V"] * 4}
    new, ctx, parents = _lengths(case)
    pairs = sum(n * (c - n) for n, c in zip(new, ctx))
    pairs += (sum(bin(a).count("1") for p in parents for a in _ancestors(p)) if parents
              else sum(n * (n + 1) // 2 for n in new))
    kv = sum(ctx) * case["Hkv"] * case["hd"] * 2 * 2
    q = sum(new) * case["Hq"] * case["hd"] * 2
    mask = sum(new) * ((max(new) + 63) // 64) * 8 if parents else 0
    return {"bytes": kv + 2 * q + mask + sum((c + case["page"] - 1) // case["page"] for c in ctx) * 4,
            "flops": 4 * pairs * case["Hq"] * case["hd"]}


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.float32) * scale).to(torch.bfloat16)

    if case["op"] == "append":
        T, Hq, Hkv, hd, page = case["T"], case["Hq"], case["Hkv"], case["hd"], case["page"]
        n_pages = (T + page - 1) // page + 5
        far = 131072 - T                                        # the tokens stand anywhere in a long context
        pos0 = rng.randrange(far)
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        ang = torch.arange(pos0, pos0 + T, dtype=torch.float64)[:, None] * inv[None, :]
        return dict(op="append", Hq=Hq, Hkv=Hkv, hd=hd, interleaved=case["interleaved"],
                    qkv=normal(T, (Hq + 2 * Hkv) * hd),
                    cos=ang.cos().to(torch.bfloat16).float().to(dev), sin=ang.sin().to(torch.bfloat16).float().to(dev),
                    k_cache=normal(n_pages, page, Hkv * hd), v_cache=normal(n_pages, page, Hkv * hd),
                    positions=torch.randperm(T, generator=g, device=dev).to(torch.int32),
                    slots=torch.randperm(n_pages * page, generator=g, device=dev)[:T].to(torch.int32))
    if case["op"] == "sample":
        rows, V = case["rows"], case["V"]
        x = torch.randn((rows, V), generator=g, device=dev) * 2.2
        likely = torch.randint(0, V, (rows, 24), generator=g, device=dev)   # a few words that fit
        x.scatter_add_(1, likely, torch.rand((rows, 24), generator=g, device=dev) * 9.0 + 2.0)
        if case["mode"] == "mixed":                                         # a grammar forbids words to some rows
            ban = torch.randint(0, V, (rows, V // 3), generator=g, device=dev)
            ban[::3] = ban[::3, :1]
            x.scatter_(1, ban, -math.inf)
        m = case["mode"]
        spec = {"greedy": (0.0, 0, 1.0, 0.0), "plain": (1.0, 0, 1.0, 0.0), "topk": (0.8, 50, 1.0, 0.0),
                "nucleus": (0.9, 0, 0.95, 0.0), "minp": (1.2, 0, 1.0, 0.05)}
        each = [spec[m]] * rows if m != "mixed" else [
            (rng.choice([0.0, 0.3, 0.7, 1.0, 1.6]), rng.choice([0, 0, 1, 20, 1000]), rng.choice([1.0, 0.5, 0.9, 0.99]),
             rng.choice([0.0, 0.0, 0.02, 0.1])) for _ in range(rows)]
        if case["per_row"]:
            f32 = lambda i: torch.tensor([e[i] for e in each], dtype=torch.float32, device=dev)  # noqa: E731
            par = dict(temperature=f32(0), top_k=torch.tensor([e[1] for e in each], dtype=torch.int32, device=dev),
                       top_p=f32(2), min_p=f32(3))
        else:
            t, k, p, mp = each[0]
            par = dict(temperature=t, top_k=k, top_p=p, min_p=mp)
        return dict(op="sample", logits=x.to(torch.bfloat16), u=torch.rand(rows, generator=g, device=dev), **par)
    B, Hq, Hkv, hd, page = case["B"], case["Hq"], case["Hkv"], case["hd"], case["page"]
    new, ctx, parents = _lengths(case)
    need = [(c + page - 1) // page for c in ctx]
    n_pages = sum(need) + sum(need) // 8 + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)     # pages were handed out in any order
    start = np.concatenate([[0], np.cumsum(need)])[:-1]
    col = torch.arange(max(need), device=dev)[None, :]
    table = order[(torch.tensor(start, device=dev)[:, None] + col).clamp_max(n_pages - 1)]
    table = torch.where(col < torch.tensor(need, device=dev)[:, None], table, torch.zeros_like(table)).contiguous()
    mask = None
    if parents:
        words = (max(new) + 63) // 64
        bits = [a for p in parents for a in _ancestors(p)]
        mask = torch.from_numpy(np.array([[(a >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for a in bits],
                                         dtype=np.uint64).view(np.int64)).to(dev)
    return dict(op="attention", Hq=Hq, Hkv=Hkv, hd=hd, scale=hd ** -0.5, q=normal(sum(new), Hq * hd, scale=1.5),
                k_cache=normal(n_pages, page, Hkv * hd), v_cache=normal(n_pages, page, Hkv * hd), page_table=table,
                ctx_lens=torch.tensor(ctx, dtype=torch.int32, device=dev),
                cu_q=torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=dev),
                max_q=max(new), max_ctx=max(ctx), tree_mask=mask)


def run(state):
    s = state
    if own:
        from zero_amd import ops
        if s["op"] == "append":
            q = ops.kv_append_paged(s["qkv"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["positions"], s["slots"],
                                    s["Hq"], s["Hkv"], s["hd"], interleaved=s["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        if s["op"] == "attention":
            return ops.attn_paged(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["ctx_lens"], s["cu_q"], s["max_q"],
                                  s["max_ctx"], s["Hq"], s["Hkv"], s["hd"], s["scale"], tree_mask=s["tree_mask"])
        return ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[s["op"]](s)


def _rotate(x, cos, sin, interleaved):
    """x [T, heads, hd] in 32 or 64 bits; cos / sin [T, rot / 2]."""
    half = cos.shape[1]
    c, n = cos[:, None, :], sin[:, None, :]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * n, b * c + a * n), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * c - b * n, b * c + a * n), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_append(s):
    Hq, Hkv, hd = s["Hq"], s["Hkv"], s["hd"]
    T, at = s["qkv"].shape[0], s["positions"].long()
    x = s["qkv"][:, :(Hq + Hkv) * hd].float().view(T, Hq + Hkv, hd)
    x = _rotate(x, s["cos"][at], s["sin"][at], s["interleaved"]).to(torch.bfloat16)
    slots = s["slots"].long()
    s["k_cache"].view(-1, Hkv * hd)[slots] = x[:, Hq:].reshape(T, Hkv * hd)
    s["v_cache"].view(-1, Hkv * hd)[slots] = s["qkv"][:, (Hq + Hkv) * hd:]
    return x[:, :Hq].reshape(T, Hq * hd), s["k_cache"], s["v_cache"]


def _plain_attention(s):
    Hq, Hkv, hd, dev = s["Hq"], s["Hkv"], s["hd"], s["q"].device
    G, n, L = Hq // Hkv, s["max_q"], s["max_ctx"]
    cu, ctx, T = s["cu_q"].long(), s["ctx_lens"].long(), s["q"].shape[0]
    B = ctx.numel()
    count = cu[1:] - cu[:-1]
    first = ctx - count                                                            # rows before the new ones
    row = (cu[:-1, None] + torch.arange(n, device=dev)).clamp_max(T - 1)           # [B, n] rows of q, padded
    q = s["q"].float()[row].view(B, n, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, hd)
    gather = lambda c: (c[s["page_table"].long()].reshape(B, -1, Hkv, hd)[:, :L].float()       # noqa: E731
                        .permute(0, 2, 1, 3))                                       # [B, Hkv, L, hd]
    sc = torch.matmul(q, gather(s["k_cache"]).transpose(2, 3).contiguous()) * s["scale"]
    key = torch.arange(L, device=dev)
    j = key[None, :] - first[:, None]                                              # [B, L]: which new token a row is
    if s["tree_mask"] is None:
        seen = j[:, None, :] <= torch.arange(n, device=dev)[None, :, None]
    else:
        words, jj = s["tree_mask"][row], j.clamp(0, n - 1)                          # [B, n, W]
        word = torch.gather(words, 2, (jj // 64)[:, None, :].expand(B, n, L))
        seen = (j[:, None, :] < 0) | (((word >> (jj % 64)[:, None, :]) & 1) != 0)
    seen = seen & (key < ctx[:, None])[:, None, :]
    sc = sc.view(B, Hkv, G, n, L).masked_fill_(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    sc = sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(B, Hkv, G * n, L), gather(s["v_cache"]).contiguous()).view(B, Hkv, G, n, hd)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq * hd)
    owner = torch.repeat_interleave(torch.arange(B, device=dev), count, output_size=T)
    return o[owner, torch.arange(T, device=dev) - cu[owner]].to(torch.bfloat16)


def _as_rows(v, rows, dtype, dev):
    """A setting as a column of one value a row, held in the type that the operator takes it in."""
    v = v if torch.is_tensor(v) else torch.full((rows,), v, dtype=dtype, device=dev)
    return v[:, None]


def _plain_sample(s):
    x, dev = s["logits"].double(), s["logits"].device
    rows, V = x.shape
    T = _as_rows(s["temperature"], rows, torch.float32, dev).double()
    k = _as_rows(s["top_k"], rows, torch.int32, dev).long()
    p = _as_rows(s["top_p"], rows, torch.float32, dev).double()
    mp = _as_rows(s["min_p"], rows, torch.float32, dev).double()
    greedy = T <= 0
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((val - val[:, :1]) / torch.where(greedy, torch.ones_like(T), T))
    rank = torch.arange(V, device=dev)[None, :]
    w = torch.where(rank < torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, torch.full_like(k, V))), w, 0.0)
    cum = torch.cumsum(w, 1)
    keep = (torch.nn.functional.pad(cum, (1, 0))[:, :-1] < p * cum[:, -1:]) | (p >= 1)
    keep = (keep & (w >= mp)) | (rank == 0)
    kept = torch.gather(cum, 1, keep.sum(1, keepdim=True) - 1)
    at = ((cum <= s["u"].double()[:, None] * kept) & keep).sum(1, keepdim=True).clamp_max(V - 1)
    return torch.gather(idx, 1, at)[:, 0], (torch.gather(w, 1, at).log() - kept.log())[:, 0].float()


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[s["op"]](s)


def _exact_append(s):
    Hq, Hkv, hd = s["Hq"], s["Hkv"], s["hd"]
    T, half = s["qkv"].shape[0], s["cos"].shape[1]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None, :]   # cos + i sin
    x = s["qkv"].double().view(T, Hq + 2 * Hkv, hd)
    pair = torch.arange(half, device=x.device)
    i, j = (2 * pair, 2 * pair + 1) if s["interleaved"] else (pair, pair + half)
    z = torch.complex(x[:, :Hq + Hkv, i], x[:, :Hq + Hkv, j]) * turn
    y = x.clone()
    y[:, :Hq + Hkv, i], y[:, :Hq + Hkv, j] = z.real, z.imag
    k, v = s["k_cache"].double(), s["v_cache"].double()
    page = k.shape[1]
    where = (s["slots"].long() // page, s["slots"].long() % page)
    k[where], v[where] = y[:, Hq:Hq + Hkv].flatten(1), y[:, Hq + Hkv:].flatten(1)
    return y[:, :Hq].flatten(1), k, v


def _exact_attention(s):
    Hq, Hkv, hd = s["Hq"], s["Hkv"], s["hd"]
    page, dev = s["k_cache"].shape[1], s["q"].device
    out = torch.zeros((s["q"].shape[0], Hq, hd), dtype=torch.float64, device=dev)
    k_rows, v_rows = s["k_cache"].view(-1, Hkv, hd), s["v_cache"].view(-1, Hkv, hd)
    cu, ctx = s["cu_q"].tolist(), s["ctx_lens"].tolist()
    for b, L in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        n = hi - lo
        t = torch.arange(L, device=dev)
        rows = s["page_table"][b].long()[t // page] * page + t % page
        if s["tree_mask"] is None:
            blind = t[None, :] > torch.arange(L - n, L, device=dev)[:, None]
        else:
            one = torch.ones((), dtype=torch.int64, device=dev)
            part = torch.stack([(s["tree_mask"][lo:hi, i // 64] & (one << (i % 64))) == 0 for i in range(n)], 1)
            blind = torch.cat((torch.zeros((n, L - n), dtype=torch.bool, device=dev), part), 1)
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            q = s["q"][lo:hi, h * hd:(h + 1) * hd].double()
            sc = (q @ k_rows[rows, kv].double().t()) * s["scale"]
            sc = sc.masked_fill(blind, -math.inf)
            out[lo:hi, h] = torch.exp(sc - torch.logsumexp(sc, 1, keepdim=True)) @ v_rows[rows, kv].double()
    return out.flatten(1)


def _exact_sample(s):
    """Equal logits are one step of the falling order: a step of c tokens of weight w adds c * w to the running sum."""
    x, (rows, V) = s["logits"], s["logits"].shape
    dev, ids, logp = x.device, [], []
    settings = [_as_rows(s[n], rows, d, dev)[:, 0].tolist() for n, d in (
        ("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))]
    u = s["u"].tolist()
    for r in range(rows):
        T, k, p, mp = (v[r] for v in settings)
        val, many = torch.unique(x[r].double(), return_counts=True)
        val, many = val.flip(0).cpu().numpy(), many.flip(0).cpu().numpy().astype(np.float64)
        w = np.exp((val - val[0]) / T) if T > 0 else (val == val[0]).astype(np.float64)
        before = np.cumsum(many) - many
        limit = 1 if T <= 0 else k if k > 0 else V
        many = np.clip(limit - before, 0, many)                                  # top-k
        if p < 1:                                                               # top-p
            goal = p * float((many * w).sum())
            run_ = np.concatenate([[0.0], np.cumsum(many * w)[:-1]])
            with np.errstate(divide="ignore", invalid="ignore"):
                part = np.ceil((goal - run_) / w)
            many = np.where(w > 0, np.clip(part, 0, many), 0.0)
            many[0] = max(many[0], 1.0)
        many = np.where(w >= mp, many, 0.0)                                     # min-p
        many[0] = max(many[0], 1.0)
        upto = np.cumsum(many * w)
        total = upto[-1]
        step = int(np.argmax(upto > u[r] * total))
        inside = int((u[r] * total - (upto[step] - many[step] * w[step])) / w[step])
        inside = min(max(inside, 0), int(many[step]) - 1)
        ids.append(int(torch.nonzero(x[r].double() == val[step])[inside, 0]))
        logp.append(math.log(w[step]) - math.log(total))
    return torch.tensor(ids, device=dev), torch.tensor(logp, dtype=torch.float64, device=dev)
