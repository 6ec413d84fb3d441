"""The paged cache and the attention sinks, measured: what a program that serves batches of long contexts with this
package has them do, through the public entry points.

Three kinds of case, over the head layouts that the tests and the benchmark use:
  append  ops.kv_append_paged: the new keys (RMSNorm, RoPE) and values of a step or of a chunk of prompts go into
          the pages that the table gives each row;
  paged   ops.attn_paged: the new tokens of each row (one in a decode step, a few in a verify step, a chunk of a
          prompt, a different number for each row of a padded batch) attend over its pages, with or without a sliding
          window whose first tokens stay visible;
  sinks   ops.attn_sinks: a sliding window and the first tokens over the contiguous cache: steps, whole prompts.
"""

import math

import torch

own = False   # False: the operators' plain forms in torch; True: the package's kernels

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
THETA = 1e6


def _case(name, kind, dtype, B, T, heads, past, page=0, ragged=False, short=False, window=0, sinks=0):
    H, K, D = heads
    return dict(name=name, kind=kind, dtype=dtype, B=B, T=T, H=H, K=K, D=D, past=past, page=page, ragged=ragged,
                short=short, window=window, sinks=sinks)


def listed():
    return [
        # the cache write of one decode step of a serving batch: 64 rows, each at a length of its own
        _case("append_step", "append", "bf16", 64, 1, (16, 8, 128), 4095, page=16, ragged=True),
        # the cache write of a chunk of four prompts of different lengths, padded to the longest
        _case("append_chunk", "append", "fp16", 4, 2048, (8, 4, 256), 6000, page=64, ragged=True, short=True),
        # the smallest attention call: one token of one short conversation
        _case("paged_decode_b1", "paged", "bf16", 1, 1, (16, 8, 128), 211, page=16),
        # a large serving batch of ragged lengths: the largest decode step
        _case("paged_decode_ragged", "paged", "bf16", 64, 1, (16, 8, 128), 32767, page=64, ragged=True),
        # speculative verify of 4 guesses for eight rows, two query heads per KV head
        _case("paged_verify", "paged", "fp16", 8, 5, (16, 8, 128), 6000, page=32, ragged=True),
        # one 512-token chunk of a long prompt, its prefix already in pages
        _case("paged_chunk", "paged", "bf16", 1, 512, (16, 8, 128), 15360, page=64),
        # a padded batch of prompt chunks, each row with its own past and its own number of new tokens: the most work
        _case("paged_chunk_batch", "paged", "bf16", 4, 2048, (8, 4, 256), 8191, page=128, ragged=True, short=True),
        # full precision: a prompt in the small 8 q / 4 KV head layout, head dim 32
        _case("paged_fp32", "paged", "fp32", 2, 333, (8, 4, 32), 700, page=16, ragged=True),
        # a decode step of sliding-window layers whose first four tokens stay visible
        _case("sinks_decode", "sinks", "bf16", 16, 1, (16, 8, 128), 8191, window=1024, sinks=4),
        # the same for a verify step of 3 guesses and one KV head of 256, rows of their own lengths
        _case("sinks_verify", "sinks", "bf16", 8, 4, (8, 1, 256), 8192, ragged=True, window=1024, sinks=4),
        # whole prompts on a sliding-window layer, the 12 q / 4 KV, head dim 64 layout
        _case("sinks_prompt", "sinks", "fp16", 2, 4093, (12, 4, 64), 0, window=1024, sinks=4),
        # a long prompt with a wide window
        _case("sinks_prompt_long", "sinks", "bf16", 1, 8192, (16, 8, 128), 0, window=2048, sinks=64),
    ]


# ---------------------------------------------------------------- more cases of the same ranges
_HEADS = [(16, 8, 128), (16, 8, 128), (12, 4, 64), (32, 8, 128), (8, 1, 256), (8, 4, 256), (16, 16, 64),
          (28, 4, 128), (8, 4, 32), (16, 1, 512)]
_MAX_BYTES, _MAX_FLOPS, _MAX_FLOPS_FP32 = 4.0e9, 2.6e11, 2e10


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["append", "append", "paged", "paged", "paged", "paged", "sinks", "sinks", "sinks"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
    heads = rng.choice(_HEADS)
    if heads[2] == 512 and dtype == "fp32":
        dtype = "bf16"
    page = 0 if kind == "sinks" else rng.choice([16, 16, 32, 64, 64, 128, 256])
    T = rng.choice([1, 1, rng.choice([2, 3, 4, 5, 8, 16]), _log(rng, 17, 4096), _log(rng, 17, 4096)])
    past = rng.choice([0, _log(rng, 16, 32000), _log(rng, 16, 32000)]) if T > 1 else _log(rng, 1, 32000)
    B = _log(rng, 1, 64) if T <= 16 else _log(rng, 1, 8)
    window = rng.choice([0, 0, 256, 1024, _log(rng, 64, 4096)]) if kind == "paged" else \
        rng.choice([256, 512, 1024, 2048, _log(rng, 64, 4096)]) if kind == "sinks" else 0
    return _case("", kind, dtype, B, T, heads, past, page=page, ragged=past > 0 and B > 1 and rng.random() < 0.6,
                 short=kind != "sinks" and T > 1 and B > 1 and rng.random() < 0.5, window=window,
                 sinks=rng.choice([1, 4, 4, 16, _log(rng, 1, 128)]) if window else 0)


def draw(rng):
    while True:
        c = _draw_once(rng)
        del c["name"]
        w = work(c)
        longest = max(p + n for p, n in _rows(c))
        if c["kind"] != "append" and (c["B"] * c["H"] * c["T"] * longest > 1.2e9 or
                                      c["B"] * c["K"] * c["D"] * longest > 2.6e9):
            continue   # the plain form's scores, or its 32-bit keys, would take more than the listed cases'
        if c["kind"] == "append" and w["bytes"] > 2e8:
            continue
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= (_MAX_FLOPS_FP32 if c["dtype"] == "fp32" else _MAX_FLOPS):
            return c


# ---------------------------------------------------------------- inputs
def _rows(case):
    """(tokens stored before the call, new tokens) of each row. One set per case: seeds change the data, not the work."""
    g = torch.Generator().manual_seed(1234)
    B, T, past = case["B"], case["T"], case["past"]
    pasts = torch.randint(past // 32, past + 1, (B,), generator=g).tolist() if case["ragged"] else [past] * B
    news = torch.randint(0, T + 1, (B,), generator=g).tolist() if case["short"] else [T] * B
    if case["short"]:
        news[0] = T   # the batch is padded to its longest row
    return list(zip(pasts, news))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    """Normal values of the dtype, made in slices of the first axis (no fp32 copy of a whole cache)."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.chunk(max(1, out.numel() >> 26)):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return out


def _rope_rows(pos, D):
    """fp32 cos/sin rows [..., D] of these positions, the two halves alike (sleuth_amd.rope's tables)."""
    inv = 1.0 / THETA ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    a = pos[..., None].double() * inv
    a = torch.cat([a, a], -1)
    return a.cos().float(), a.sin().float()


@torch.no_grad()
def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    kind, B, T, H, K, D, P = (case[n] for n in ("kind", "B", "T", "H", "K", "D", "page"))
    rows = _rows(case)
    s = {"case": case, "longest": max(p + n for p, n in rows),
         "row_pos": torch.tensor([p for p, _ in rows], dtype=torch.int32, device="cuda"),
         "new_lens": torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda") if case["short"] else None}
    if P:
        # The rows' pages lie anywhere in the pool, which holds a few more than are in use. A page that no query of
        # the call can see any more (behind the window, past the first tokens) was given back: -1, as is what lies
        # behind a row's last page.
        def kept(p, n, j):
            return not case["window"] or j * P < case["sinks"] or (j + 1) * P - 1 > p - case["window"]

        held = [[j for j in range(-(-(p + n) // P)) if kept(p, n, j)] for p, n in rows]
        pool = sum(map(len, held)) + 3
        ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((B, -(-(s["longest"]) // P) + 2), -1, dtype=torch.int32)
        for b, pages in enumerate(held):
            if pages:
                table[b, pages] = torch.tensor([ids.pop() for _ in pages], dtype=torch.int32)
        s["table"] = table.cuda()
        shape = (pool, K, P, D)
    else:
        cap = s["longest"] + 64
        shape = (B, K, cap, D)
    if kind == "append":
        s["k_cache"], s["v_cache"] = _randn(g, shape, dt), _randn(g, shape, dt)
        # k and v as the fused projection leaves them: views of its rows [B, T, 2 K D]
        y = _randn(g, (B, T, 2 * K * D), dt)
        s["k"], s["v"] = (x.view(B, T, K, D).transpose(1, 2) for x in y.split(K * D, -1))
        s["gain"] = 1.3 + 0.15 * torch.randn(D, generator=g, device="cuda")
        s["cos"], s["sin"] = _rope_rows(s["row_pos"].long()[:, None] + torch.arange(T, device="cuda"), D)
    else:
        # normalised, rotated keys and queries: gains near 1.3, so that scores have a standard deviation above 1
        s["k_cache"], s["v_cache"] = _randn(g, shape, dt, 1.3), _randn(g, shape, dt)
        s["q"] = _randn(g, (B, T, H, D), dt, 1.3).transpose(1, 2)
    return s


# ---------------------------------------------------------------- one pass
def _plain_append(s):
    case = s["case"]
    T, D, P = case["T"], case["D"], case["page"]
    k, v, half = s["k"].float(), s["v"], case["D"] // 2
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["gain"]
    a, z = k[..., :half], k[..., half:]
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    k = torch.cat([a * cos[..., :half] - z * sin[..., :half], z * cos[..., half:] + a * sin[..., half:]], -1)
    t = torch.arange(T, device="cuda")
    pos = s["row_pos"].long()[:, None] + t
    pages = s["table"].long().gather(1, (pos // P).clamp(max=s["table"].shape[1] - 1))
    real = (t < s["new_lens"][:, None]) if s["new_lens"] is not None else torch.ones_like(pos, dtype=torch.bool)
    b, t = real.nonzero(as_tuple=True)
    s["k_cache"][pages[b, t], :, pos[b, t] % P] = k[b, :, t].to(s["k_cache"].dtype)
    s["v_cache"][pages[b, t], :, pos[b, t] % P] = v[b, :, t]


def _plain_attend(s):
    case = s["case"]
    B, T, H, K, D, P = (case[n] for n in ("B", "T", "H", "K", "D", "page"))
    S = s["longest"]
    k, v = s["k_cache"], s["v_cache"]
    if P:
        at = s["table"].long().clamp(min=0)
        k, v = (x[at].transpose(1, 2).reshape(B, K, -1, D) for x in (k, v))
    k, v = k[:, :, :S].float(), v[:, :, :S].float()
    t, keys = torch.arange(T, device="cuda"), torch.arange(S, device="cuda")
    pos = s["row_pos"].long()[:, None] + t
    see = keys <= pos[..., None]                                       # [B, T, S]
    if case["window"]:
        see = see & ((keys > pos[..., None] - case["window"]) | (keys < case["sinks"]))
    if s["new_lens"] is not None:
        see = see & (t < s["new_lens"][:, None])[..., None]
    w = s["q"].float().reshape(B, K, -1, D) @ k.transpose(-1, -2)
    w = w.view(B, K, -1, T, S).mul_(D ** -0.5).masked_fill_(~see[:, None, None], -math.inf)
    w = w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = w.sum(-1, keepdim=True)
    y = w.view(B, K, -1, S) @ v
    y = y.view(B, K, -1, T, D) / total.clamp(min=1e-30)
    return y.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(s["q"].dtype)


@torch.no_grad()
def run(s):
    case = s["case"]
    if own:
        from sleuth_amd import ops

        if case["kind"] == "append":
            ops.kv_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["row_pos"],
                                new_lens=s["new_lens"], k_weight=s["gain"], eps=EPS, norm_k=True, cos=s["cos"],
                                sin=s["sin"])
            return {"k": s["k_cache"], "v": s["v_cache"]}
        seen = dict(scale=case["D"] ** -0.5, window=case["window"], sinks=case["sinks"], max_kv_len=s["longest"])
        if case["kind"] == "paged":
            return ops.attn_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["row_pos"],
                                  new_lens=s["new_lens"], **seen)
        where = dict(row_pos=s["row_pos"]) if case["ragged"] else dict(pos=case["past"])
        return ops.attn_sinks(s["q"], s["k_cache"], s["v_cache"], **where, **seen)
    if case["kind"] == "append":
        _plain_append(s)
        return {"k": s["k_cache"], "v": s["v_cache"]}
    return _plain_attend(s)


# ---------------------------------------------------------------- what a pass cannot do without
def _seen(past, new, window, sinks):
    """(query, key) pairs of a row's new queries, and the keys that any of them sees."""
    def one(p):   # keys that the query at p sees
        return p + 1 if not window or p + 1 <= window else window + min(sinks, p + 1 - window)

    if not new:
        return 0, 0
    low = max(0, past - window + 1) if window else 0   # the first query's first key
    return sum(one(p) for p in range(past, past + new)), past + new - low + min(sinks, low)


def work(case):
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    H, K, D, rows = case["H"], case["K"], case["D"], _rows(case)
    new = sum(n for _, n in rows)
    if case["kind"] == "append":   # k and v in and out, the gain, one cos and one sin row for each token
        return {"bytes": new * (4 * K * D * e + 2 * D * 4) + 4 * D, "flops": new * K * D * 8}
    seen = [_seen(p, n, case["window"], case["sinks"]) for p, n in rows]
    pairs, keys = sum(x[0] for x in seen), sum(x[1] for x in seen)
    # K and V of the visible keys; the queries in; the whole output, padding included, out
    return {"bytes": e * D * (2 * K * keys + H * (new + case["B"] * case["T"])), "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------- the same in 64 bits
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    rows, P, D = _rows(case), case["page"], case["D"]
    dev = s["k_cache"].device
    table = s["table"].tolist() if P else None
    if case["kind"] == "append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b, (past, new) in enumerate(rows):
            if not new:
                continue
            x, cos, sin = s["k"][b, :, :new].double(), s["cos"][b, :new].double(), s["sin"][b, :new].double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * s["gain"].double()
            x = x * cos + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * sin
            for j in range(past // P, (past + new - 1) // P + 1):   # page by page
                lo, hi = max(past, j * P), min(past + new, (j + 1) * P)
                kc[table[b][j], :, lo - j * P:hi - j * P] = x[:, lo - past:hi - past]
                vc[table[b][j], :, lo - j * P:hi - j * P] = s["v"][b, :, lo - past:hi - past].double()
        return {"k": kc, "v": vc}
    H, K, T = case["H"], case["K"], case["T"]
    out = torch.zeros(case["B"], T, H, D, dtype=torch.float64, device=dev)
    for b, (past, new) in enumerate(rows):
        if not new:
            continue
        n = past + new
        low = max(0, past - case["window"] + 1) if case["window"] else 0
        cut = max(0, min(case["sinks"], low))
        where = torch.tensor([*range(cut), *range(low, n)], device=dev)   # the keys that any query of the row sees
        if P:
            ids = torch.tensor(table[b], device=dev)[where // P]
            k, v = (c[ids, :, where % P].transpose(0, 1) for c in (s["k_cache"], s["v_cache"]))
        else:
            k, v = (c[b][:, where] for c in (s["k_cache"], s["v_cache"]))
        qpos = torch.arange(past, n, device=dev)[:, None]
        hide = where > qpos
        if case["window"]:
            hide |= (qpos - where >= case["window"]) & (where >= case["sinks"])
        for h in range(H):
            kk, vv = k[h * K // H].double(), v[h * K // H].double()
            a = (s["q"][b, h, :new].double() @ kk.T.contiguous()) / math.sqrt(D)
            out[b, :new, h] = a.masked_fill(hide, -math.inf).softmax(-1) @ vv
    return out
