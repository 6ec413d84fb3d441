"""Speculative decoding with trees of drafted tokens, measured: what a step of it asks of this package, through the
public entry points.

Five kinds of case, over the head layouts that the tests and the benchmark use:
  mask     ops.tree_mask: the drafted trees' parents become the bits of who sees whom, and depths;
  attend   ops.attn_tree, ops.attn_tree_paged: the drafted tokens attend over the cache and their own branches;
  verify   ops.verify_drafts: drafted tokens against the target's logits, greedily or from given random numbers, with
           or without the drafter's probabilities;
  compact  ops.kv_compact, ops.kv_compact_paged: the accepted tokens' keys and values close up, in every layer;
  copy     ops.copy_pages: pages of the paged cache are copied in every layer (a row forks, or writes to a shared page).
"""

import math
import random

import torch

own = False   # False: the operators' plain forms in torch; True: the package's kernels

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_KEYS = dict(dtype="", B=0, T=0, shape="", H=0, K=0, D=0, past=0, page=0, ragged=False, short=False, window=0, sinks=0,
             vocab=0, temperature=0.0, probs=False, layers=0, pages=0)


def _case(name, kind, heads=(0, 0, 0), **kw):
    c = dict(_KEYS, name=name, kind=kind, H=heads[0], K=heads[1], D=heads[2])
    assert not set(kw) - set(c)
    c.update(kw)
    return c


def listed():
    return [
        # one conversation's drafted tree of a dozen tokens: the smallest call of all
        _case("mask_b1", "mask", B=1, T=12, shape="tree"),
        # a serving batch, a tree of its own for each row, the widest that a step drafts
        _case("mask_batch", "mask", B=64, T=256, shape="tree"),
        # the verify step of one short conversation over the contiguous cache: latency
        _case("attend_b1", "attend", (16, 8, 128), dtype="bf16", B=1, T=12, shape="tree", past=400),
        # sliding-window layers, one KV head of 256, first tokens kept, rows of their own lengths
        _case("attend_window", "attend", (8, 1, 256), dtype="fp16", B=8, T=26, shape="tree", past=8192, ragged=True,
              window=1024, sinks=4),
        # a large serving batch over the paged cache, trees of 64, some rows with smaller ones: the most work
        _case("attend_paged", "attend", (16, 8, 128), dtype="bf16", B=32, T=64, shape="tree", past=16383, page=64,
              ragged=True, short=True),
        # a chain of guesses verified greedily for one conversation
        _case("verify_greedy", "verify", dtype="bf16", B=1, T=5, shape="chain", vocab=32768),
        # a sampling batch: chains drawn by a drafter whose probabilities are known
        _case("verify_chain", "verify", dtype="bf16", B=32, T=6, shape="chain", vocab=131072, temperature=0.8, probs=True),
        # trees of a drafter's likeliest tokens in full precision, a vocabulary whose rows no vector load divides
        _case("verify_tree", "verify", dtype="fp32", B=8, T=40, shape="tree", vocab=100003, temperature=1.0, short=True),
        # one conversation's accepted branch, 28 layers of the contiguous cache
        _case("compact_b1", "compact", (16, 8, 128), dtype="bf16", B=1, T=12, shape="tree", past=200, layers=28),
        # a serving batch's, over pages
        _case("compact_paged", "compact", (16, 8, 128), dtype="bf16", B=64, T=26, shape="tree", past=60, page=16,
              layers=28, ragged=True),
        # a row writes to a page that it shares: one copy of it, 28 layers
        _case("copy_one", "copy", (12, 4, 64), dtype="bf16", page=16, layers=28, pages=1),
        # a prompt's last page for each of 64 continuations
        _case("copy_fork", "copy", (16, 8, 128), dtype="bf16", page=64, layers=28, pages=64),
    ]


# ---------------------------------------------------------------- more cases of the same ranges
_HEADS = [(16, 8, 128), (16, 8, 128), (12, 4, 64), (32, 8, 128), (8, 1, 256), (8, 4, 256), (16, 16, 64),
          (28, 4, 128), (8, 4, 32), (16, 1, 512)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["mask", "attend", "attend", "attend", "attend", "verify", "verify", "verify", "compact", "copy"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    heads = rng.choice(_HEADS)
    if heads[2] == 512 and dtype == "fp32":
        dtype = "bf16"
    shape = rng.choice(["chain", "tree", "tree", "tree", "star"])
    if kind == "mask":
        return _case("", kind, B=_log(rng, 1, 64), T=_log(rng, 1, 256), shape=shape, short=rng.random() < 0.3)
    if kind == "attend":
        window = rng.choice([0, 0, 0, 256, 1024, _log(rng, 4, 4096)])
        B = _log(rng, 1, 64)
        return _case("", kind, heads, dtype=dtype, B=B, T=rng.choice([1, _log(rng, 2, 16), _log(rng, 8, 64), _log(rng, 8, 128)]),
                     shape=shape, past=rng.choice([0, _log(rng, 16, 30000), _log(rng, 16, 30000)]),
                     page=rng.choice([0, 16, 32, 64, 128]), ragged=B > 1 and rng.random() < 0.6,
                     short=B > 1 and rng.random() < 0.4, window=window,
                     sinks=rng.choice([0, 1, 4, 16, _log(rng, 1, 128)]) if window else 0)
    if kind == "verify":
        T = rng.choice([1, _log(rng, 2, 10), _log(rng, 2, 10), _log(rng, 8, 64)])
        temperature = rng.choice([0.0, 1.0, 0.7, rng.uniform(0.2, 2.0)])
        return _case("", kind, dtype=dtype, B=_log(rng, 1, 64), T=T, shape=shape, vocab=_log(rng, 1000, 160000),
                     temperature=temperature, probs=temperature > 0 and rng.random() < 0.5,
                     short=rng.random() < 0.3)
    if kind == "compact":
        return _case("", kind, heads, dtype=dtype, B=_log(rng, 1, 64), T=_log(rng, 2, 64), shape=shape,
                     past=rng.choice([0, _log(rng, 1, 200)]), page=rng.choice([0, 16, 16, 32, 64]), layers=rng.randint(1, 32),
                     ragged=rng.random() < 0.5)
    return _case("", kind, heads, dtype=dtype, page=rng.choice([16, 32, 64, 128]), layers=rng.randint(1, 32),
                 pages=_log(rng, 1, 100))


def draw(rng):
    while True:
        c = _draw_once(rng)
        del c["name"]
        if c["kind"] == "attend":
            if c["T"] * c["H"] * c["B"] * (c["past"] + c["T"]) > 5e8 or c["B"] * c["K"] * c["D"] * c["past"] > 5e8:
                continue   # no more than the largest listed one's scores and keys
            if c["dtype"] == "fp32" and c["T"] * c["H"] * c["B"] * (c["past"] + c["T"]) > 5e7:
                continue
        if c["kind"] == "verify" and c["B"] * c["T"] * c["vocab"] > 3.2e7:
            continue
        if c["kind"] in ("compact", "copy") and 2 * c["layers"] * _pool(c) * _bits(c) / 8 > 1.0e9:
            continue
        return c


def _bits(c):
    return torch.finfo(DTYPES[c["dtype"]]).bits


# ---------------------------------------------------------------- inputs
def _rng(case):
    """One for each case, whatever the seed: seeds change the data, not the work."""
    return random.Random("%s %d %d" % (case["kind"], case["B"], case["T"]))


def _tree(rng, T, shape):
    """Parents of a drafted tree in level order: node 0 is the last token that was accepted for good."""
    if shape == "chain":
        return [t - 1 for t in range(T)]
    if shape == "star":
        return [-1] + [0] * (T - 1)
    parents = [-1]
    level = [0]
    while len(parents) < T:   # a level of about four times as many candidates as the last one, at most 16, unevenly spread
        n = min(T - len(parents), rng.randint(2, 4 * min(len(level), 4)))
        weights = [2.0 ** -i for i in range(len(level))]
        chosen = sorted(rng.choices(level, weights, k=n))
        level = list(range(len(parents), len(parents) + n))
        parents += chosen
    return parents


def _trees(case):
    """(parents [B][T], real nodes [B])"""
    rng, B, T = _rng(case), case["B"], case["T"]
    news = [rng.randint(0, T) if case["short"] and b else T for b in range(B)]
    return [_tree(rng, T, case["shape"]) for _ in range(B)], news


def _paths(case):
    """An accepted path [B][..] of each row's tree, from node 0 downwards."""
    rng = random.Random(7 + case["B"])
    out = []
    for parents in _trees(case)[0]:
        path = [0]
        while True:
            children = [t for t, p in enumerate(parents) if p == path[-1]]
            if not children or rng.random() < 0.2:
                break
            path.append(rng.choice(children))
        out.append(path)
    return out


def _pasts(case):
    rng, past = random.Random(99 + case["B"]), case["past"]
    return [rng.randint(past // 32, past) if case["ragged"] else past for _ in range(case["B"])]


def _pool(case):
    """Elements of a layer's K, all rows or pages."""
    if case["kind"] == "copy":
        return (2 * case["pages"] + 3) * case["K"] * case["page"] * case["D"]
    per = case["past"] + case["T"] + 16
    return case["B"] * case["K"] * case["D"] * (-(-per // case["page"]) * case["page"] if case["page"] else per)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    """Normal values of the dtype, made in slices of the first axis (no fp32 copy of a whole cache)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.chunk(max(1, out.numel() >> 26)):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return out


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(rows, page, seed):
    """Page table of rows that hold `rows` tokens, the pages anywhere in the pool; -1 behind a row's last page."""
    need = [-(-n // page) for n in rows]
    ids = list(range(sum(need) + 3))
    random.Random(seed).shuffle(ids)
    table = torch.full((len(rows), max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), sum(need) + 3


@torch.no_grad()
def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    B, T, H, K, D, P = (case[n] for n in ("B", "T", "H", "K", "D", "page"))
    dt = DTYPES.get(case["dtype"])
    s = {"case": case}
    if kind == "copy":
        n = case["pages"]
        shape = (2 * n + 3, K, P, D)
        ids = list(range(2 * n + 3))
        random.Random(seed).shuffle(ids)
        s["src"], s["dst"] = _i32(ids[:n]), _i32(ids[n:2 * n])
        s["k"] = [_randn(g, shape, dt) for _ in range(case["layers"])]
        s["v"] = [_randn(g, shape, dt) for _ in range(case["layers"])]
        return s
    parents, news = _trees(case)
    s["parents"] = _i32(parents)
    s["new_lens"] = _i32(news) if case["short"] else None
    if kind == "mask":   # (other trees with another seed: the parents moved by a permutation of the rows, one node hung elsewhere)
        rng = random.Random(seed)
        rng.shuffle(parents)
        for p in parents:
            t = rng.randrange(len(p))
            p[t] = rng.randint(-1, t - 1)
        s["parents"] = _i32(parents)
        return s
    if kind == "verify":
        return _prepare_verify(s, g, parents, seed)
    pasts = _pasts(case)
    s["pasts"], s["row_pos"] = pasts, _i32(pasts)
    longest = max(p + n for p, n in zip(pasts, news))
    s["longest"] = max(1, longest)
    if P:
        s["table"], pool = _table([p + n for p, n in zip(pasts, news)], P, seed)
        shape = (pool, K, P, D)
    else:
        shape = (B, K, s["longest"] + 16, D)
    if kind == "attend":
        s["mask"], s["depth"] = _mask_plain(s["parents"], None)
        # normalised, rotated keys and queries: gains near 1.3, so that scores have a standard deviation above 1
        s["k"], s["v"] = _randn(g, shape, dt, 1.3), _randn(g, shape, dt)
        s["q"] = _randn(g, (B, T, H, D), dt, 1.3).transpose(1, 2)
        return s
    paths = _paths(case)
    s["path"] = _i32([p + [-1] * (T - len(p)) for p in paths])
    s["count"] = _i32([len(p) for p in paths])
    s["k"] = [_randn(g, shape, dt) for _ in range(case["layers"])]
    s["v"] = [_randn(g, shape, dt) for _ in range(case["layers"])]
    return s


def _prepare_verify(s, g, parents, seed):
    """Target logits near the drafter's; a node's children are drawn from the drafter's probabilities, or are its
    likeliest tokens where those are not used."""
    case = s["case"]
    B, T, V = case["B"], case["T"], case["vocab"]
    dt = DTYPES[case["dtype"]]
    heat = case["temperature"] or 1.0
    s["logits"] = torch.empty(B, T, V, dtype=dt, device="cuda")
    s["probs"] = torch.empty(B, T, V, dtype=torch.float32, device="cuda") if case["probs"] else None
    tokens = torch.randint(V, (B, T), generator=g, device="cuda")
    for b in range(B):
        drafter = 3.0 * torch.randn(T, V, generator=g, device="cuda")
        drafter[:, torch.randint(V, (8,), generator=g, device="cuda")] += 9.0   # (a few likely tokens)
        s["logits"][b] = drafter + 0.4 * torch.randn(T, V, generator=g, device="cuda")
        most = max([1] + [sum(q == p for q in parents[b]) for p in set(parents[b]) if p >= 0])
        if case["probs"]:
            s["probs"][b] = (drafter / heat).softmax(-1)
            offers = torch.multinomial(s["probs"][b], most, replacement=True, generator=g)
        else:
            offers = drafter.topk(min(most, V), -1).indices
        seen = [0] * T
        where = []
        for t, p in enumerate(parents[b]):
            where.append(p * offers.shape[1] + seen[p] % offers.shape[1] if p >= 0 else 0)
            if p >= 0:
                seen[p] += 1
        tokens[b, 1:] = offers.flatten()[torch.tensor(where, device="cuda")][1:]
    s["tokens"] = tokens
    s["uniform"] = torch.rand(B, T, generator=g, device="cuda") if case["temperature"] else None
    return s


# ---------------------------------------------------------------- one pass, in plain torch
def _mask_plain(parents, new_lens):
    """vis(t) = {t} and vis(parent of t), by doubling the distance that is looked upwards."""
    B, T = parents.shape
    t = torch.arange(T, device=parents.device)
    up = torch.where((parents >= 0) & (parents < t), parents, -1).long()
    vis = torch.eye(T, dtype=torch.bool, device=parents.device).repeat(B, 1, 1)
    for _ in range(max(1, (T - 1).bit_length())):
        more = vis.gather(1, up.clamp(min=0)[..., None].expand(B, T, T))
        vis = vis | (more & (up >= 0)[..., None])
        up = torch.where(up >= 0, up.gather(1, up.clamp(min=0)), -1)
    if new_lens is not None:
        vis = vis & (t < new_lens[:, None])[..., None]
    depth = (vis.sum(-1) - 1).clamp(min=0).to(torch.int32)
    words = -(-T // 64)
    bits = torch.zeros(B, T, words * 64, dtype=torch.int64, device=parents.device)
    bits[..., :T] = vis.long()
    shift = torch.arange(64, device=parents.device)
    return (bits.view(B, T, words, 64) << shift).sum(-1), depth


def _unpack(mask, T):
    shift = torch.arange(64, device=mask.device)
    return ((mask[..., None] >> shift) & 1).flatten(-2)[..., :T].bool()


def _plain_attend(s):
    case = s["case"]
    B, T, H, K, D, P = (case[n] for n in ("B", "T", "H", "K", "D", "page"))
    S, k, v = s["longest"], s["k"], s["v"]
    if P:
        at = s["table"].long().clamp(min=0)
        k, v = (x[at].transpose(1, 2).reshape(B, K, -1, D) for x in (k, v))
    k, v = k[:, :, :S].float(), v[:, :, :S].float()
    t, keys, base = torch.arange(T, device="cuda"), torch.arange(S, device="cuda"), s["row_pos"].long()[:, None]
    depth = s["depth"].long()
    new = keys - base                                                   # [B, S]: which new token a slot holds
    slot = new.clamp(0, T - 1)
    there = (new >= 0) & (new < (s["new_lens"].long()[:, None] if case["short"] else T))
    pos = torch.where(new >= 0, base + depth.gather(1, slot), keys)     # the slots' positions
    see = _unpack(s["mask"], T).gather(2, slot[:, None].expand(B, T, S)) & there[:, None] | (new < 0)[:, None]
    if case["window"]:
        at = base + depth                                               # [B, T]: the queries' positions
        see &= (pos[:, None] > at[..., None] - case["window"]) | (pos < case["sinks"])[:, None]
    if case["short"]:
        see = see & (t < s["new_lens"][:, None])[..., None]
    w = s["q"].float().reshape(B, K, -1, D) @ k.transpose(-1, -2)
    w = w.view(B, K, -1, T, S).mul_(D ** -0.5).masked_fill_(~see[:, None, None], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = w.sum(-1, keepdim=True)
    y = w.view(B, K, -1, S) @ v
    y = y.view(B, K, -1, T, D) / total.clamp(min=1e-30)
    return y.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(s["q"].dtype)


def _plain_verify(s):
    """The nodes in order: a node whose parent is where the walk stands is accepted, or its token's share is taken out of
    what is left there. All rows at once."""
    case = s["case"]
    B, T, V, probs = case["B"], case["T"], case["vocab"], s["probs"]
    dev, heat = "cuda", case["temperature"]
    news = s["new_lens"].long() if case["short"] else torch.full((B,), T, device=dev)
    rows = torch.arange(B, device=dev)
    if heat:
        x = s["logits"].double() / heat
        mass = (x - x.amax(-1, keepdim=True)).exp_()
        del x
        u = s["uniform"].double()
        left, total, taken = mass[:, 0].clone(), mass[:, 0].sum(-1), torch.zeros(B, dtype=torch.float64, device=dev)
    else:
        best = s["logits"].float().argmax(-1)
    at = torch.zeros(B, dtype=torch.int64, device=dev)
    count = (news > 0).long()
    path = torch.full((B, T), -1, dtype=torch.int64, device=dev)
    path[:, 0] = torch.where(count > 0, 0, -1)
    out = torch.full((B, T + 1), -1, dtype=torch.int64, device=dev)
    for t in range(1, T):
        x = s["tokens"][:, t]
        child = (s["parents"][:, t] == at) & (t < news)
        if heat:
            q = probs[rows, at].double() if probs is not None else torch.zeros(B, V, dtype=torch.float64, device=dev).scatter_(1, x[:, None], 1.0)
            yes = child & (u[:, t] * q[rows, x] * total < left[rows, x])
            no = child & ~yes
            if probs is not None:
                taken = torch.where(no, taken + total, taken)
                rest = (mass[rows, at] - taken[:, None] * q).clamp(min=0)
            else:
                rest = left.masked_fill(q > 0, 0.0)
            left = torch.where(yes[:, None], mass[:, t], torch.where(no[:, None], rest, left))
            total = torch.where(child, left.sum(-1), total)
            taken = torch.where(yes, 0.0, taken)
        else:
            yes = child & (best[rows, at] == x)
        at = torch.where(yes, t, at)
        out[rows, torch.where(yes, count - 1, T)] = x
        path[rows, torch.where(yes, count, 0)] = torch.where(yes, t, path[:, 0])
        count = count + yes.long()
    if heat:
        none = left.sum(-1) <= 0
        upto = left.cumsum(-1)
        last = torch.searchsorted(upto, (u[:, :1] * left.sum(-1, keepdim=True)), right=True)[:, 0].clamp(max=V - 1)
        last = torch.where(none, s["logits"].float()[rows, at].argmax(-1), last)
    else:
        last = best[rows, at]
    out[rows, torch.where(count > 0, count - 1, T)] = last
    return out[:, :T], path.to(torch.int32), count.to(torch.int32)


def _plain_compact(s):
    case = s["case"]
    T, P = case["T"], case["page"]
    i = torch.arange(T, device="cuda")
    b, i = (i < s["count"][:, None]).nonzero(as_tuple=True)
    src = s["row_pos"].long()[b] + s["path"].long()[b, i]
    dst = s["row_pos"].long()[b] + i
    for x in (*s["k"], *s["v"]):
        if P:
            table = s["table"].long()
            x[table[b, dst // P], :, dst % P] = x[table[b, src // P], :, src % P]
        else:
            x[b, :, dst] = x[b, :, src]
    return {"k": s["k"], "v": s["v"]}


@torch.no_grad()
def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from sleuth_amd import ops

        if kind == "mask":
            return ops.tree_mask(s["parents"], s["new_lens"])
        if kind == "attend":
            seen = dict(scale=case["D"] ** -0.5, depth=s["depth"], new_lens=s["new_lens"], window=case["window"],
                        sinks=case["sinks"], max_kv_len=s["longest"])
            if case["page"]:
                return ops.attn_tree_paged(s["q"], s["k"], s["v"], s["table"], s["row_pos"], s["mask"], **seen)
            return ops.attn_tree(s["q"], s["k"], s["v"], s["mask"], row_pos=s["row_pos"], **seen)
        if kind == "verify":
            return ops.verify_drafts(s["logits"], s["tokens"], parents=s["parents"], uniform=s["uniform"],
                                     temperature=case["temperature"], draft_probs=s["probs"], new_lens=s["new_lens"])
        if kind == "compact":
            if case["page"]:
                ops.kv_compact_paged(s["k"], s["v"], s["table"], s["row_pos"], s["path"], s["count"])
            else:
                ops.kv_compact(s["k"], s["v"], s["path"], s["count"], row_pos=s["row_pos"])
        else:
            ops.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if kind == "mask":
        return _mask_plain(s["parents"], s["new_lens"])
    if kind == "attend":
        return _plain_attend(s)
    if kind == "verify":
        return _plain_verify(s)
    if kind == "compact":
        return _plain_compact(s)
    src, dst = s["src"].long(), s["dst"].long()
    for x in (*s["k"], *s["v"]):
        x[dst] = x[src]
    return {"k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- what a pass cannot do without
def _ancestors(parents, t):
    """t and what it hangs on, t first."""
    out = [t]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def work(case):
    kind = case["kind"]
    B, T, H, K, D = (case[n] for n in ("B", "T", "H", "K", "D"))
    if kind == "mask":   # parents in, bits and depths out; a bit is set for each ancestor
        return {"bytes": B * T * (4 + 4 + 8 * -(-T // 64)) + 4 * B * case["short"], "flops": B * T}
    e = _bits(case) // 8
    if kind == "copy":
        return {"bytes": 2 * 2 * case["layers"] * case["pages"] * K * case["page"] * D * e + 8 * case["pages"], "flops": 0}
    if kind == "compact":   # keys and values that change their place, in and out; the paths
        moved = sum(i != t for p in _paths(case) for i, t in enumerate(p))
        return {"bytes": 2 * 2 * case["layers"] * moved * K * D * e + 4 * B * (T + 2), "flops": 0}
    parents, news = _trees(case)
    if kind == "verify":   # the logits of the real nodes (and the drafter's probabilities), tokens and paths
        q = 4 if case["probs"] else 0
        return {"bytes": sum(news) * case["vocab"] * (e + q) + B * T * (8 + 4 + 4 + 8 + 4),
                "flops": sum(news) * case["vocab"] * (4 if case["temperature"] else 1)}
    pairs = keys = 0
    for p, past, n in zip(parents, _pasts(case), news):
        lowest = past
        for t in range(n):
            chain = _ancestors(p, t)
            at = past + len(chain) - 1
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            first = min(case["sinks"], low)   # (the first tokens outside the window)
            pairs += first + max(0, past - low) + sum(past + i >= low for i in range(len(chain)))
            lowest = min(lowest, low)
        if n:
            keys += past - lowest + min(case["sinks"], lowest) + n
    # K and V of the visible keys; the queries and bits in; the whole output, padding included, out
    return {"bytes": e * D * (2 * K * keys + H * (sum(news) + B * T)) + B * T * (4 + 8 * -(-T // 64)), "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------- the same in 64 bits
def _exact_attend(s, parents, news):
    case = s["case"]
    B, T, H, K, D, P = (case[n] for n in ("B", "T", "H", "K", "D", "page"))
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    for b, (past, n) in enumerate(zip(s["pasts"], news)):
        if not n:
            continue
        chains = [_ancestors(parents[b], t) for t in range(n)]
        hide = torch.ones(n, past + n, dtype=torch.bool)
        for t, chain in enumerate(chains):
            at = past + len(chain) - 1
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            hide[t, low:past] = False
            hide[t, :min(past, case["sinks"])] = False
            for j in chain:
                where = past + len(chains[j]) - 1
                if where >= low or where < case["sinks"]:
                    hide[t, past + j] = False
        hide = hide.cuda()
        if P:
            ids = s["table"][b, :-(-(past + n) // P)].long()
            k, v = (x[ids].transpose(0, 1).reshape(K, -1, D)[:, :past + n] for x in (s["k"], s["v"]))
        else:
            k, v = s["k"][b, :, :past + n], s["v"][b, :, :past + n]
        for h in range(H):
            a = (s["q"][b, h, :n].double() @ k[h * K // H].double().T.contiguous()) / math.sqrt(D)
            out[b, :n, h] = a.masked_fill(hide, -math.inf).softmax(-1) @ v[h * K // H].double()
    return out


def _exact_verify(s, parents, news):
    """Row by row, node by node, with normalised probabilities."""
    case = s["case"]
    B, T, V, heat = case["B"], case["T"], case["vocab"], case["temperature"]
    tokens, u = s["tokens"].tolist(), s["uniform"].tolist() if heat else None
    out = [[-1] * T for _ in range(B)]
    paths = [[-1] * T for _ in range(B)]
    counts = [0] * B
    for b in range(B):
        if not news[b]:
            continue
        path, at = [0], 0
        while True:
            children = [t for t in range(at + 1, news[b]) if parents[b][t] == at]
            logits = s["logits"][b, at].double()
            if not heat:
                best = int((logits == logits.max()).nonzero()[0])
                hit = [t for t in children if tokens[b][t] == best]
                last = best
            else:
                p = torch.softmax(logits / heat, -1)
                hit = []
                for t in children:
                    x = tokens[b][t]
                    if s["probs"] is not None:
                        q = s["probs"][b, at].double()
                        ok = u[b][t] * float(q[x]) < float(p[x])
                        if not ok:
                            rest = (p - q).clamp(min=0)
                    else:
                        ok = u[b][t] < float(p[x])
                        if not ok:
                            rest = p.clone()
                            rest[x] = 0
                    if ok:
                        hit = [t]
                        break
                    p = rest / rest.sum()
                last = None
            if not hit:
                break
            at = hit[0]
            path.append(at)
        if last is None:
            last = int((p.cumsum(-1) > u[b][0]).nonzero()[0])
        counts[b] = len(path)
        paths[b][:len(path)] = path
        out[b][:len(path)] = [tokens[b][t] for t in path[1:]] + [last]
    return (torch.tensor(out, device="cuda"), _i32(paths), _i32(counts))


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "mask":
        T = case["T"]
        news = s["new_lens"].tolist() if case["short"] else [T] * case["B"]
        words = -(-T // 64)
        mask = [[[0] * words for _ in range(T)] for _ in news]
        depth = [[0] * T for _ in news]
        for b, (p, n) in enumerate(zip(s["parents"].tolist(), news)):
            for t in range(n):
                chain = _ancestors(p, t)
                depth[b][t] = len(chain) - 1
                for j in chain:
                    mask[b][t][j // 64] |= 1 << j % 64
        signed = [[[x - (1 << 64) if x >> 63 else x for x in t] for t in b] for b in mask]
        return torch.tensor(signed, dtype=torch.int64, device="cuda"), _i32(depth)
    if kind == "copy":
        ids = list(zip(s["src"].tolist(), s["dst"].tolist()))
        res = {n: [x.double() for x in s[n]] for n in ("k", "v")}
        for n in ("k", "v"):
            for x, y in zip(s[n], res[n]):
                for a, b in ids:
                    y[b] = x[a].double()
        return res
    if kind == "compact":
        P = case["page"]
        res = {n: [x.double() for x in s[n]] for n in ("k", "v")}
        table = s["table"].tolist() if P else None
        for b, (past, path) in enumerate(zip(s["pasts"], _paths(case))):
            for i, t in enumerate(path):
                to, of = past + i, past + t
                for n in ("k", "v"):
                    for x, y in zip(s[n], res[n]):
                        if P:
                            y[table[b][to // P], :, to % P] = x[table[b][of // P], :, of % P].double()
                        else:
                            y[b, :, to] = x[b, :, of].double()
        return res
    parents, news = _trees(case)
    return _exact_attend(s, parents, news) if kind == "attend" else _exact_verify(s, parents, news)
