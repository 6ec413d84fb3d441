"""The paged cache and attention with sinks (ops.kv_append_paged, attn_paged, attn_sinks) against 64-bit forms."""

from __future__ import annotations

import math

import pytest
import torch

from paged_oracle import Paged, assert_close, attend64, norm_rope64, visible
from sleuth_amd import _lib, ops
from sleuth_amd.rope import rope_tables

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def i32(xs, dev="cuda"):
    return torch.tensor(xs, dtype=torch.int32, device=dev)


# (dtype, H, K, D, page, pasts, T, news or None, window, sinks)
CASES = [
    # one token: lengths of one, page ends, tile ends, several tiles and parts
    (BF, 16, 8, 128, 16, [0, 1, 15, 16, 31, 32, 127, 128, 211], 1, None, 0, 0),
    (HF, 12, 4, 64, 32, [0, 63, 64, 200, 1500], 1, None, 0, 0),
    (SF, 8, 4, 32, 16, [0, 5, 31, 300], 1, None, 0, 0),
    (SF, 16, 8, 128, 64, [900, 3], 1, None, 0, 0),
    (SF, 8, 1, 256, 16, [130, 700], 1, None, 0, 0),
    (BF, 8, 4, 32, 16, [77, 1030], 1, None, 0, 0),
    (BF, 8, 1, 256, 128, [400, 1], 1, None, 0, 0),
    (BF, 16, 1, 512, 16, [0, 17, 333], 1, None, 0, 0),
    (HF, 16, 1, 512, 64, [1000], 2, None, 0, 0),
    (HF, 28, 4, 128, 16, [2500, 9], 1, None, 0, 0),
    # a few tokens
    (BF, 16, 8, 128, 16, [0, 1, 30, 500], 5, None, 0, 0),
    (HF, 32, 8, 128, 32, [100, 2000], 8, None, 0, 0),
    (BF, 8, 1, 256, 16, [61, 5], 4, None, 0, 0),
    (SF, 12, 4, 64, 16, [12, 400], 7, None, 0, 0),
    # chunks: more rows than a block, odd sizes, a past that ends inside a page
    (BF, 16, 8, 128, 16, [0, 37], 70, None, 0, 0),
    (BF, 16, 8, 128, 64, [300], 129, None, 0, 0),
    (HF, 12, 4, 64, 16, [0, 500], 65, None, 0, 0),
    (BF, 16, 16, 64, 32, [10], 200, None, 0, 0),
    (BF, 8, 4, 256, 16, [100, 0], 67, None, 0, 0),
    (HF, 8, 1, 256, 64, [9], 40, None, 0, 0),
    (SF, 8, 4, 32, 16, [0, 90], 101, None, 0, 0),
    (SF, 16, 8, 128, 16, [33], 50, None, 0, 0),
    (SF, 16, 16, 64, 32, [7], 150, None, 0, 0),
    (SF, 8, 4, 256, 16, [20], 33, None, 0, 0),
    (BF, 16, 1, 512, 32, [40], 37, None, 0, 0),
    (HF, 8, 4, 32, 16, [0], 300, None, 0, 0),
    (BF, 28, 4, 128, 32, [64], 45, None, 0, 0),
    (BF, 6, 2, 128, 16, [64, 3], 45, None, 0, 0),
    # fp32 chunks of more than 64 rows: two and three row blocks, tiles that the row's end cuts
    (SF, 16, 8, 128, 32, [70, 0], 130, None, 0, 0),
    (SF, 12, 4, 64, 16, [333], 100, None, 0, 0),
    (SF, 8, 1, 256, 16, [37], 21, None, 0, 0),
    (SF, 16, 8, 128, 16, [500, 20], 60, [60, 7], 100, 9),
    (SF, 8, 4, 256, 64, [90], 130, None, 33, 40),
    # padded batches: no new token, one, some, all
    (BF, 16, 8, 128, 16, [100, 50, 0, 700], 9, [9, 0, 1, 4], 0, 0),
    (HF, 12, 4, 64, 16, [30, 8, 0], 90, [90, 1, 0], 0, 0),
    (BF, 8, 4, 256, 32, [30, 8], 70, [2, 70], 0, 0),
    (SF, 8, 4, 64, 16, [30, 8], 40, [0, 33], 0, 0),
    # windows, with and without first tokens
    (BF, 16, 8, 128, 16, [0, 10, 64, 700, 2000], 1, None, 64, 4),
    (BF, 16, 8, 128, 16, [700], 1, None, 1, 0),
    (BF, 16, 8, 128, 16, [700], 1, None, 1, 1),
    (HF, 8, 1, 256, 32, [300, 31], 4, None, 100, 33),
    (SF, 8, 4, 64, 16, [300, 31], 3, None, 50, 5),
    (BF, 12, 4, 64, 16, [0, 250], 150, None, 40, 7),
    (BF, 16, 8, 128, 64, [1000], 140, None, 300, 64),
    (HF, 16, 8, 128, 16, [200, 90], 80, [80, 3], 16, 20),
    (SF, 8, 4, 32, 16, [200], 80, None, 33, 2),
    (BF, 16, 1, 512, 16, [150], 20, None, 48, 3),
    (BF, 8, 4, 256, 16, [400], 66, None, 64, 16),
    # head dim 512, chunks: part of a row block, several, a padded batch, a window, one KV head and two
    (BF, 8, 4, 512, 16, [100, 0], 45, [45, 7], 0, 0),
    (HF, 16, 2, 512, 16, [2, 300, 1000], 4, None, 0, 0),
    (BF, 16, 1, 512, 64, [500, 30], 9, None, 100, 9),
    (HF, 16, 1, 512, 128, [700, 3, 90], 33, [1, 33, 0], 20, 64),
    (BF, 4, 2, 512, 32, [15, 16, 31], 140, None, 0, 0),
    (BF, 8, 4, 32, 32, [40, 7], 90, [90, 33], 0, 0),
    (HF, 8, 4, 32, 16, [300], 150, None, 60, 5),
]


def _run_paged(dtype, H, K, D, page, pasts, T, news, window, sinks, seed=0, free=True):
    g = gen(seed)
    B = len(pasts)
    real = news if news is not None else [T] * B

    def freed(b, j):   # pages that no query of the call sees are given back
        p = pasts[b]
        return free and bool(window) and j * page >= sinks and (j + 1) * page - 1 <= p - window

    cache = Paged(g, [p + n for p, n in zip(pasts, real)], K, D, page, dtype, freed=freed)
    q = 1.3 * torch.randn(B, T, H, D, generator=g)
    q = q.to(dtype)
    for b, n in enumerate(real):
        q[b, n:] = math.nan   # what stands behind a row's last new token
    q = q.transpose(1, 2)
    scale = D ** -0.5
    got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts), scale=scale,
                         new_lens=i32(news) if news is not None else None, window=window, sinks=sinks)
    return got, *cache.want(q, pasts, real, window, sinks, scale)


def _id(c):
    return "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_attn_paged(case):
    got, want, bound = _run_paged(*case)
    assert_close(got, want, bound)


# ---------------------------------------------------------------- sinks over the contiguous cache
SINKS = [
    # (dtype, H, K, D, lens before, T, window, sinks, how the position is given)
    (BF, 16, 8, 128, [700], 1, 64, 4, "pos"),
    (BF, 16, 8, 128, [700, 3, 2000], 1, 300, 4, "rows"),
    (HF, 8, 1, 256, [333], 4, 100, 33, "dev"),
    (BF, 8, 1, 256, [333, 61], 4, 32, 0, "rows"),
    (SF, 8, 4, 32, [90], 1, 16, 1, "pos"),
    (SF, 16, 8, 128, [200, 7], 3, 50, 70, "rows"),
    (BF, 16, 1, 512, [130], 1, 48, 5, "pos"),
    (HF, 12, 4, 64, [0], 333, 64, 4, "pos"),
    (BF, 16, 8, 128, [0], 300, 100, 64, "pos"),
    (BF, 16, 8, 128, [500], 130, 1, 1, "dev"),
    (BF, 8, 4, 256, [40], 150, 70, 9, "pos"),
    (SF, 8, 4, 64, [0], 90, 20, 3, "pos"),
    (HF, 8, 4, 32, [10], 200, 33, 2, "pos"),
    (BF, 16, 1, 512, [0], 40, 16, 3, "pos"),
    (BF, 16, 16, 64, [100, 900], 70, 5000, 10, "rows"),   # a window no row fills
]


def _sinks_inputs(dtype, H, K, D, lens, T, window, sinks, how, seed=0, spare=70):
    g = gen(seed)
    B, cap = len(lens), max(lens) + T + spare
    kc = (1.3 * torch.randn(B, K, cap, D, generator=g)).to(dtype)
    vc = torch.randn(B, K, cap, D, generator=g).to(dtype)
    for b, n in enumerate(lens):   # behind a row's keys: NaN
        kc[b, :, n + T:], vc[b, :, n + T:] = math.nan, math.nan
    q = (1.3 * torch.randn(B, T, H, D, generator=g)).to(dtype).transpose(1, 2)
    return q, kc, vc


def _where(how, lens):
    if how == "rows":
        return dict(row_pos=i32(lens))
    return dict(pos=lens[0]) if how == "pos" else dict(pos_dev=torch.tensor([lens[0]], device="cuda"))


def _sinks_want(q, kc, vc, lens, window, sinks, scale):
    T = q.shape[2]
    out = [attend64(q[b], kc[b, :, :n + T], vc[b, :, :n + T], visible(torch.arange(n, n + T), torch.arange(n + T), window, sinks),
                    scale) for b, n in enumerate(lens)]
    return torch.stack([o for o, _ in out]), torch.stack([e for _, e in out])


@pytest.mark.gpu
@pytest.mark.parametrize("case", SINKS, ids=_id)
def test_attn_sinks(case):
    dtype, H, K, D, lens, T, window, sinks, how = case
    q, kc, vc = _sinks_inputs(*case)
    got = ops.attn_sinks(q.cuda(), kc.cuda(), vc.cuda(), scale=D ** -0.5, window=window, sinks=sinks, **_where(how, lens))
    assert_close(got, *_sinks_want(q, kc, vc, lens, window, sinks, D ** -0.5))


@pytest.mark.gpu
def test_sinks_of_a_wide_window_equal_the_plain_causal_attention():
    """A window that covers every row and any number of first tokens: ops.attn_decode's keys."""
    q, kc, vc = _sinks_inputs(BF, 16, 8, 128, [200], 3, 0, 0, "pos")
    q, kc, vc = q.cuda(), kc.cuda().nan_to_num(0.0), vc.cuda().nan_to_num(0.0)
    a = ops.attn_sinks(q, kc, vc, scale=0.1, window=4096, sinks=7, pos=200)
    b = ops.attn_decode(q, kc, vc, scale=0.1, pos=200)
    want, bound = _sinks_want(q.cpu(), kc.cpu(), vc.cpu(), [200], 0, 0, 0.1)
    assert_close(a, want, bound)
    assert_close(b, want, bound)


# ---------------------------------------------------------------- the cache write
APPENDS = [
    # (dtype, K, D, page, pasts, T, news, norm_k, rope, norm_v)
    (BF, 8, 128, 16, [0, 15, 16, 100], 1, None, True, True, False),
    (HF, 4, 256, 64, [10, 60], 70, [70, 3], True, True, False),
    (SF, 4, 32, 16, [0, 5, 31], 40, [0, 40, 1], True, True, True),
    (BF, 1, 512, 32, [7], 5, None, False, True, True),
    (HF, 3, 64, 128, [120, 0], 9, None, True, False, False),
    (SF, 2, 256, 16, [3], 17, None, False, False, False),
    (BF, 4, 32, 16, [33], 20, None, True, True, False),
    (SF, 16, 128, 16, [1, 2], 3, None, True, True, False),
]


def _append_inputs(dtype, K, D, page, pasts, T, news, norm_k, rope, norm_v):
    g = gen(5)
    B = len(pasts)
    real = news if news is not None else [T] * B
    cache = Paged(g, [p + n for p, n in zip(pasts, real)], K, D, page, dtype)
    cache.kp = torch.randn(cache.kp.shape, generator=g).to(dtype)
    cache.vp = torch.randn(cache.vp.shape, generator=g).to(dtype)
    y = torch.randn(B, T, 2 * K * D, generator=g).to(dtype)
    k, v = (x.view(B, T, K, D).transpose(1, 2) for x in y.split(K * D, -1))
    w = 1.3 + 0.15 * torch.randn(D, generator=g) if norm_k else None
    cos = sin = None
    if rope:
        tabs = rope_tables(D, max(pasts) + T, 1e4)
        at = torch.tensor(pasts)[:, None] + torch.arange(T)
        cos, sin = tabs[0][at], tabs[1][at]
    return cache, real, k, v, w, cos, sin


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPENDS, ids=_id)
def test_kv_append_paged(case):
    dtype, K, D, page, pasts, T, news, norm_k, rope, norm_v = case
    cache, real, k, v, w, cos, sin = _append_inputs(*case)
    kp, vp = cache.kp.cuda(), cache.vp.cuda()
    up = lambda t: None if t is None else t.cuda()   # noqa: E731
    y = torch.cat([k.transpose(1, 2).flatten(2), v.transpose(1, 2).flatten(2)], -1).cuda()   # the projection's rows
    kd, vd = (x.view(len(pasts), T, K, D).transpose(1, 2) for x in y.split(K * D, -1))
    ops.kv_append_paged(kd, vd, kp, vp, cache.table.cuda(), i32(pasts), new_lens=i32(news) if news is not None else None,
                        k_weight=up(w), eps=1e-6, norm_k=norm_k, norm_v=norm_v, cos=up(cos), sin=up(sin))
    eps = torch.finfo(dtype).eps / 2
    u = 2.0 ** -24
    touched = torch.zeros(cache.kp.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(real):
        rows = (None, None) if cos is None else (cos[b, :n], sin[b, :n])
        wk = norm_rope64(k[b, :, :n], w, 1e-6 if norm_k else None, *rows)
        wv = norm_rope64(v[b, :, :n], None, 1e-6 if norm_v else None, None, None)
        # what the two terms of a rotated channel may be off by: the sum of D squares, a root, a few products
        ak = norm_rope64(k[b, :, :n], w, 1e-6 if norm_k else None, None, None).abs()
        slack = (D + 24) * u * (ak + ak.roll(D // 2, -1))
        slack_v = (D + 24) * u * wv.abs()
        for i in range(n):
            pos = pasts[b] + i
            at = (int(cache.table[b, pos // page]), pos % page)
            touched[at] = True
            for got, want, s, plain in ((kp, wk, slack, not (norm_k or rope)), (vp, wv, slack_v, not norm_v)):
                x = got[at[0], :, at[1]].cpu().double()
                lim = torch.zeros(()) if plain else s[:, i] + eps * (1 + 1e-3) * want[:, i].abs()
                assert ((x - want[:, i]).abs() <= lim + (0 if plain else 1e-40)).all(), (b, i)
    # every other slot is as it was, bit for bit
    for got, was in ((kp.cpu(), cache.kp), (vp.cpu(), cache.vp)):
        keep = ~touched[:, None, :, None].expand_as(was)
        assert torch.equal(got[keep], was[keep])


@pytest.mark.gpu
def test_append_equals_the_contiguous_append_bit_for_bit():
    case = (BF, 8, 128, 16, [40, 40], 9, None, True, True, False)
    cache, real, k, v, w, cos, sin = _append_inputs(*case)
    kp, vp = cache.kp.cuda(), cache.vp.cuda()
    args = dict(k_weight=w.cuda(), eps=1e-6, norm_k=True, cos=cos[0].cuda(), sin=sin[0].cuda())
    ops.kv_append_paged(k.cuda(), v.cuda(), kp, vp, cache.table.cuda(), i32([40, 40]), **args)
    kc, vc = (torch.zeros(2, 8, 64, 128, dtype=BF, device="cuda") for _ in range(2))
    ops.kv_append(k.cuda(), v.cuda(), kc, vc, pos=40, **args)
    for b in range(2):
        for pos in range(40, 49):
            page = int(cache.table[b, pos // 16])
            assert torch.equal(kp[page, :, pos % 16], kc[b, :, pos]) and torch.equal(vp[page, :, pos % 16], vc[b, :, pos])


# ---------------------------------------------------------------- norm and RoPE of q inside the call
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H,K,D,T", [(BF, 16, 8, 128, 1), (BF, 16, 8, 128, 80), (HF, 8, 4, 32, 3), (SF, 8, 4, 64, 20),
                                           (HF, 8, 4, 256, 40), (BF, 16, 1, 512, 2), (SF, 8, 1, 256, 2), (BF, 12, 4, 64, 70)])
@pytest.mark.parametrize("what", ["norm", "rope", "both"])
def test_fused_q(dtype, H, K, D, T, what):
    """Raw q with norm and RoPE in the call: its rows are those of the 64-bit formula, rounded to the type, give or take
    one step of the type where the fp32 value lies next to a rounding border (which moves a score by at most
    eps * scale * sum |q k|)."""
    g = gen(3)
    pasts = [50, 9]
    cache = Paged(g, [p + T for p in pasts], K, D, 16, dtype)
    q = torch.randn(2, T, H, D, generator=g).to(dtype).transpose(1, 2)
    w = (1.2 + 0.1 * torch.randn(D, generator=g)) if what != "rope" else None
    tabs = rope_tables(D, 200, 1e4)
    at = torch.tensor(pasts)[:, None] + torch.arange(T)
    cos, sin = (tabs[0][at], tabs[1][at]) if what != "norm" else (None, None)
    up = lambda t: None if t is None else t.cuda()   # noqa: E731
    got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts), scale=D ** -0.5,
                         q_weight=up(w), eps=1e-6, norm_q=what != "rope", cos=up(cos), sin=up(sin))
    q64 = norm_rope64(q, w, 1e-6 if what != "rope" else None, None if cos is None else cos[:, None],
                      None if sin is None else sin[:, None])
    want, bound = cache.want(q64.to(dtype), pasts, [T, T], 0, 0, D ** -0.5)
    step = torch.finfo(dtype).eps
    for b in range(2):   # the step that a q value may be off by, on the scores: 2 e on the weights' quotient, as in attend64
        kk = cache.k[b].double().repeat_interleave(H // K, 0)
        a = (q64[b].abs() @ kk.abs().transpose(1, 2)).amax(-1) * D ** -0.5        # [H, T]
        vmax = cache.v[b].double().abs().amax()
        bound[b] += (2 * step * a * vmax).T[..., None]
    assert_close(got, want, bound)


# ---------------------------------------------------------------- pages
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 90])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("page", [16, 64])
def test_entries_outside_the_pool_are_invisible(T, bad, page):
    """Pages in the middle of a row that the table no longer names: as if their keys did not exist; the append
    writes nothing there."""
    g = gen(1)
    cache = Paged(g, [300 + T, 40 + T], 8, 128, page, BF)
    for b, j in ((0, 0), (0, 2), (1, 0)):
        cache.table[b, j] = bad
        cache.held[b][j * page:(j + 1) * page] = False
    q = torch.randn(2, T, 16, 128, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([300, 40]), scale=0.09)
    assert_close(got, *cache.want(q, [300, 40], [T, T], 0, 0, 0.09))
    # the write: row 1 starts inside its missing page where pages hold 64
    kp, vp = cache.kp.cuda(), cache.vp.cuda()
    new = torch.randn(2, T, 8, 128, generator=g).to(BF).transpose(1, 2).cuda()
    ops.kv_append_paged(new, new, kp, vp, cache.table.cuda(), i32([300, 40]))
    named = set(cache.table.flatten().tolist())
    for i in range(kp.shape[0]):
        if i not in named:
            assert torch.equal(kp[i].cpu().nan_to_num(7.0), cache.kp[i].nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32])
def test_missing_pages_at_head_dim_512(page):
    """The same where every wave looks up both groups of 16 keys of a tile: one of them missing, the other, both."""
    g = gen(21)
    T, pasts = 21, [500, 70]
    cache = Paged(g, [p + T for p in pasts], 1, 512, page, BF)
    for b, j in ((0, 0), (0, 3), (0, 6), (0, 7), (1, 1)):
        cache.table[b, j] = -1 - j
        cache.held[b][j * page:(j + 1) * page] = False
    q = torch.randn(2, T, 16, 512, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts), scale=0.04)
    assert_close(got, *cache.want(q, pasts, [T, T], 0, 0, 0.04))


@pytest.mark.gpu
def test_a_row_without_any_page_is_zero():
    g = gen(1)
    for T in (1, 80):
        cache = Paged(g, [20 + T, 30 + T], 4, 64, 16, HF)
        cache.table[0] = -1
        cache.held[0][:] = False
        q = torch.randn(2, T, 12, 64, generator=g).to(HF).transpose(1, 2)
        got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([20, 30]), scale=0.1)
        assert not got[0].any()
        assert_close(got, *cache.want(q, [20, 30], [T, T], 0, 0, 0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70])
def test_rows_may_share_pages(T):
    """Two rows with one prefix in the same pages, their own pages after it."""
    g = gen(2)
    one = Paged(g, [64 + T], 8, 128, 16, BF, extra=0)
    table = one.table.repeat(2, 1)
    q = torch.randn(2, T, 16, 128, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_paged(q.cuda(), one.kp.cuda(), one.vp.cuda(), table.cuda(), i32([64, 64]), scale=0.1)
    for b in range(2):
        want, bound = one.want(q[b:b + 1], [64], [T], 0, 0, 0.1)
        assert_close(got[b:b + 1], want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 66])
def test_pool_offsets_past_32_bits(T):
    """Pages at the end of pools of more than 2^32 bytes (and 2^31 elements)."""
    g = gen(4)
    n = (2 ** 31 + 2 ** 27) // (8 * 64 * 128)
    cache = Paged(g, [200 + T, 3 + T], 8, 128, 64, BF)
    held = cache.kp.shape[0]
    kp, vp = (torch.zeros(n, 8, 64, 128, dtype=BF, device="cuda") for _ in range(2))
    kp[-held:], vp[-held:] = cache.kp.cuda(), cache.vp.cuda()
    table = torch.where(cache.table >= 0, cache.table + (n - held), cache.table)
    q = torch.randn(2, T, 16, 128, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_paged(q.cuda(), kp, vp, table.cuda().int(), i32([200, 3]), scale=0.1)
    assert_close(got, *cache.want(q, [200, 3], [T, T], 0, 0, 0.1))
    new = torch.randn(2, T, 8, 128, generator=g).to(BF).transpose(1, 2)
    ops.kv_append_paged(new.cuda(), new.cuda(), kp, vp, table.cuda().int(), i32([200, 3]))
    for t in (0, T - 1):
        page = int(table[0, (200 + t) // 64])
        assert torch.equal(kp[page, :, (200 + t) % 64].cpu(), new[0, :, t])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70])
def test_a_long_contiguous_cache_past_32_bits(T):
    """Batch rows more than 2^32 bytes apart, the window at the end of the last one."""
    H, K, D, cap = 4, 2, 64, 2 ** 24 + 4096
    kc, vc = (torch.zeros(2, K, cap, D, dtype=BF, device="cuda") for _ in range(2))
    assert kc.stride(0) * 2 > 2 ** 31 and kc.numel() * 2 > 2 ** 32
    g = gen(6)
    n, window, sinks = cap - T - 5, 200, 6
    for c in (kc, vc):
        c[:, :, :64] = torch.randn(2, K, 64, D, generator=g).to(BF).cuda()
        c[:, :, n - 400:n + T] = torch.randn(2, K, 400 + T, D, generator=g).to(BF).cuda()
    q = torch.randn(2, T, H, D, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_sinks(q.cuda(), kc, vc, scale=0.2, window=window, sinks=sinks, pos=n)
    where = torch.tensor([*range(sinks), *range(n - window + 1, n + T)])
    for b in range(2):
        k, v = (c[b][:, where.cuda()].cpu() for c in (kc, vc))
        see = visible(torch.arange(n, n + T), where, window, sinks)
        want, bound = attend64(q[b], k, v, see, 0.2)
        assert_close(got[b], want, bound)


# ---------------------------------------------------------------- how it is called
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 100])
def test_strided_and_unaligned_inputs(T):
    """Head-major q, an odd offset into a buffer, pools inside a larger one, an output slice: same values."""
    g = gen(7)
    cache = Paged(g, [90 + T, 8 + T], 4, 64, 16, BF)
    q = torch.randn(2, T, 12, 64, generator=g).to(BF).transpose(1, 2)
    args = (cache.table.cuda(), i32([90, 8]))
    kp, vp = cache.kp.cuda(), cache.vp.cuda()
    ref = ops.attn_paged(q.cuda(), kp, vp, *args, scale=0.1)
    assert_close(ref, *cache.want(q, [90, 8], [T, T], 0, 0, 0.1))
    head_major = q.cuda().contiguous()
    odd = torch.empty(q.numel() + 3, dtype=BF, device="cuda")[3:].view(q.shape).copy_(q)
    wide_k, wide_v = (torch.full((kp.shape[0], 4, 16, 128), math.nan, dtype=BF, device="cuda") for _ in range(2))
    wide_k[..., 64:], wide_v[..., 64:] = kp, vp
    for qq, kk, vv in ((head_major, kp, vp), (odd, kp, vp), (q.cuda(), wide_k[..., 64:], wide_v[..., 64:])):
        assert torch.equal(ops.attn_paged(qq, kk, vv, *args, scale=0.1), ref)
    table = torch.full((2, 2 * cache.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    table[:, ::2] = cache.table.cuda()
    assert torch.equal(ops.attn_paged(q.cuda(), kp, vp, table[:, ::2], i32([90, 8]), scale=0.1), ref)
    big = torch.full((3, T + 1, 20, 64), 7.0, dtype=BF, device="cuda")
    out = big[:2, :T, 4:16]
    assert ops.attn_paged(q.cuda(), kp, vp, *args, scale=0.1, out=out) is out
    assert torch.equal(out, ref)
    out.fill_(7.0)
    assert bool((big == 7.0).all())   # nothing around it was touched


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 90])
def test_same_bits_again_and_with_other_bounds(T):
    """The same call gives the same bits; bounds that only size the launch stay within the error bound."""
    g = gen(8)
    pasts = [3000, 10, 700]
    cache = Paged(g, [p + T for p in pasts], 8, 128, 16, BF, extra=200)
    q = torch.randn(3, T, 16, 128, generator=g).to(BF).transpose(1, 2).cuda()
    args = (cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts))
    want, bound = cache.want(q.cpu(), pasts, [T] * 3, 0, 0, 0.09)
    for most in (3000 + T, 4000, None):
        a = ops.attn_paged(q, *args, scale=0.09, max_kv_len=most)
        assert_close(a, want, bound)
        for _ in range(5):
            assert torch.equal(ops.attn_paged(q, *args, scale=0.09, max_kv_len=most), a)


@pytest.mark.gpu
@pytest.mark.parametrize("T,window", [(1, 0), (1, 100), (70, 0), (300, 64)])
def test_graph_replays_with_new_lengths_and_tables(T, window):
    """Recorded once, replayed with other positions, lengths and tables in the same buffers, eager work in between."""
    g = gen(9)
    B, H, K, D, page = 3, 16, 8, 128, 16
    table = torch.full((B, 80), -1, dtype=torch.int32, device="cuda")
    row_pos, news = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    kp, vp = (torch.zeros(260, K, page, D, dtype=BF, device="cuda") for _ in range(2))
    q = torch.zeros(B, T, H, D, dtype=BF, device="cuda").transpose(1, 2)
    kn = torch.zeros(B, T, K, D, dtype=BF, device="cuda").transpose(1, 2)
    vn = torch.zeros_like(kn)
    most = 80 * page

    def call():
        ops.kv_append_paged(kn, vn, kp, vp, table, row_pos, new_lens=news)
        return ops.attn_paged(q, kp, vp, table, row_pos, scale=0.09, new_lens=news, max_kv_len=most, window=window,
                              sinks=4 if window else 0)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for pasts, real in (([0, 5, 17], [T, T, T]), ([700, 0, 64], [T, 0, 1]), ([31, 900, 2], [1, T, T]), ([0, 5, 17], [T, T, T])):
        cache = Paged(g, [p + n for p, n in zip(pasts, real)], K, D, page, BF, extra=0)
        table.fill_(-1)
        table[:, :cache.table.shape[1]] = cache.table.cuda()
        kp[:cache.kp.shape[0]], vp[:cache.vp.shape[0]] = cache.kp.cuda(), cache.vp.cuda()
        row_pos.copy_(i32(pasts))
        news.copy_(i32(real))
        qh = torch.randn(B, T, H, D, generator=g).to(BF).transpose(1, 2)
        q.copy_(qh)
        for b, (p, n) in enumerate(zip(pasts, real)):   # the new keys go in through the call
            kn[b, :, :n], vn[b, :, :n] = cache.k[b][:, p:p + n].cuda(), cache.v[b][:, p:p + n].cuda()
            for pos in range(p, p + n):
                kp[int(cache.table[b, pos // page]), :, pos % page] = 0
        graph.replay()
        want, bound = cache.want(qh, pasts, real, window, 4 if window else 0, 0.09)
        assert_close(out, want, bound)
        first = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(call(), first)
        graph.replay()
        assert torch.equal(out, first)


@pytest.mark.gpu
def test_two_graphs_and_streams_at_once():
    """Split calls on two streams and from two recorded graphs have partials of their own."""
    g = gen(10)
    jobs = []
    for T in (1, 60):
        cache = Paged(g, [4000 + T, 900 + T], 8, 128, 16, BF)
        q = torch.randn(2, T, 16, 128, generator=g).to(BF).transpose(1, 2)
        args = (q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([4000, 900]))
        jobs.append((args, *cache.want(q, [4000, 900], [T, T], 0, 0, 0.09)))
    for args, want, bound in jobs:
        assert_close(ops.attn_paged(*args, scale=0.09), want, bound)
    graphs = []
    for args, *_ in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attn_paged(*args, scale=0.09)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = [None] * 4
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i < 2:
                    outs[i] = ops.attn_paged(*jobs[i][0], scale=0.09)
                else:
                    graphs[i - 2][0].replay()
    torch.cuda.synchronize()
    outs[2], outs[3] = graphs[0][1], graphs[1][1]
    for i, o in enumerate(outs):
        assert_close(o, *jobs[i % 2][1:])


@pytest.mark.gpu
def test_without_a_workspace():
    """The C entry points without memory for the partials: unsplit, the same values within the bound."""
    g = gen(11)
    for T in (1, 40, 90):
        cache = Paged(g, [2500 + T], 8, 128, 16, BF)
        q = torch.randn(1, T, 16, 128, generator=g).to(BF).cuda().transpose(1, 2)
        kp, vp, table, rp = cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([2500])
        out = torch.empty(1, T, 16, 128, dtype=BF, device="cuda")
        st = _lib.lib().forge_attn_paged(_lib.BF16, 1, T, 16, 8, 128, q.data_ptr(), *q.stride()[:3], None, 0.0, 0, None, None,
                                         0, 0, kp.data_ptr(), vp.data_ptr(), *kp.stride()[:3], kp.shape[0], 16,
                                         table.data_ptr(), 0, table.shape[1], rp.data_ptr(), None, 2500 + T, 0, 0, 0.09,
                                         out.data_ptr(), *out.stride()[:3], None, 0, 0,
                                         torch.cuda.current_stream().cuda_stream)
        assert st == 0
        assert_close(out, *cache.want(q.cpu(), [2500], [T], 0, 0, 0.09))


@pytest.mark.gpu
def test_positions_past_the_bound_do_not_exist():
    """Rows at or past max_kv_len, and positions below zero: zeros, nothing read."""
    g = gen(12)
    cache = Paged(g, [64, 64, 64], 8, 128, 16, BF, extra=0)
    for T in (1, 70):
        q = torch.randn(3, T, 16, 128, generator=g).to(BF).transpose(1, 2).cuda()
        got = ops.attn_paged(q, cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([64, -5, 2 ** 31 - 1]), scale=0.1)
        assert not got.any()
    kp, vp = cache.kp.cuda(), cache.vp.cuda()
    new = torch.ones(3, 8, 4, 128, dtype=BF, device="cuda")
    ops.kv_append_paged(new, new, kp, vp, cache.table.cuda(), i32([64, -5, 2 ** 31 - 5]))
    same = lambda a, b: bool(((a.cpu() == b) | (a.cpu().isnan() & b.isnan())).all())   # noqa: E731 (spare pages hold NaN)
    assert same(kp, cache.kp) and same(vp, cache.vp)


@pytest.mark.gpu
def test_empty_calls():
    kp = torch.zeros(2, 4, 16, 64, dtype=BF, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    for B, T in ((0, 1), (2, 0)):
        q = torch.zeros(B, 8, T, 64, dtype=BF, device="cuda")
        assert ops.attn_paged(q, kp, kp, table[:B], i32([0] * B), scale=0.1).shape == (B, T, 8, 64)
        k = torch.zeros(B, 4, T, 64, dtype=BF, device="cuda")
        ops.kv_append_paged(k, k, kp, kp, table[:B], i32([0] * B))
        c = torch.zeros(B, 4, 16, 64, dtype=BF, device="cuda")
        assert ops.attn_sinks(q, c, c, scale=0.1, window=4, sinks=1, pos=0).shape == (B, T, 8, 64)


# How a call is cut follows from what its table can hold, so tables far wider than the rows send small calls, in
# every form above, to the kernel of large chunks: cut on the host (4,000 keys), or planned on the device (200,000)
@pytest.fixture(params=[4000, 200000])
def wide_tables(request, monkeypatch):
    plain = Paged.__init__

    def widened(self, *args, **kw):
        plain(self, *args, **kw)
        page = self.kp.shape[2]
        self.table = torch.nn.functional.pad(self.table, (0, request.param // page - self.table.shape[1]), value=-1)

    monkeypatch.setattr(Paged, "__init__", widened)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [c for c in CASES if c[6] > 1], ids=_id)
def test_chunks_with_wide_tables(wide_tables, case):
    got, want, bound = _run_paged(*case)
    assert_close(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["norm", "rope", "both"])
@pytest.mark.parametrize("dtype,H,K,D,T", [(BF, 16, 8, 128, 80), (HF, 8, 4, 256, 40), (BF, 16, 1, 512, 12), (BF, 12, 4, 64, 70), (HF, 8, 4, 32, 60),
                                           (SF, 16, 8, 128, 40), (SF, 8, 1, 256, 12), (SF, 12, 4, 64, 30)])
def test_fused_q_with_wide_tables(wide_tables, dtype, H, K, D, T, what):
    test_fused_q(dtype, H, K, D, T, what)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_pages_with_wide_tables(wide_tables, page):
    for T in (90, 300):
        test_entries_outside_the_pool_are_invisible(T, -1, page)
    test_a_row_without_any_page_is_zero()
    test_rows_may_share_pages(70)
    test_missing_pages_at_head_dim_512(32)
    test_strided_and_unaligned_inputs(100)
    test_large_scores_and_infinite_keys_out_of_sight()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # long enough for the kernel of large chunks with the caches' own lengths
    (BF, 16, 8, 128, 64, [2500, 300], 200, None, 0, 0), (HF, 12, 4, 64, 16, [1500], 700, None, 0, 0),
    (BF, 8, 4, 256, 32, [900, 30], 300, [300, 299], 0, 0), (SF, 16, 8, 128, 64, [700], 260, None, 0, 0),
    (SF, 8, 4, 64, 16, [300, 900, 0], 400, [400, 1, 77], 256, 33), (BF, 28, 4, 128, 16, [1000, 90], 200, None, 300, 20),
    (HF, 16, 1, 512, 32, [600], 150, None, 0, 0), (SF, 8, 1, 256, 16, [1200], 90, None, 0, 0)], ids=_id)
def test_longer_chunks(case):
    got, want, bound = _run_paged(*case)
    assert_close(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    (HF, 12, 4, 64, [0], 2000, 300, 4, "pos"), (BF, 16, 8, 128, [0], 900, 100, 64, "pos"),
    (BF, 16, 8, 128, [500], 700, 129, 1, "dev"), (BF, 8, 4, 256, [40, 40], 500, 70, 9, "pos"), (SF, 8, 4, 64, [0], 1100, 200, 3, "pos"),
    (BF, 16, 1, 512, [0], 220, 250, 3, "pos"), (BF, 16, 16, 64, [100, 900], 400, 5000, 10, "rows"), (BF, 28, 4, 128, [7, 300], 300, 64, 17, "rows"),
    (HF, 8, 4, 32, [5], 3001, 1400, 7, "pos")],
    ids=_id)
def test_longer_windows(case):
    test_attn_sinks(case)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 70)])
def test_planned_chunks_at_head_dim_512(window, sinks):
    """A large call whose rows differ, its parts planned on the device (with a window: too few tiles, not planned)."""
    got, want, bound = _run_paged(BF, 16, 1, 512, 32, [2700, 40, 1500], 130, [130, 128, 0] if window else None, window, sinks)
    assert_close(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(window=1 << 30), dict(window=(1 << 32) + 4), dict(window=4, sinks=1 << 30)])
def test_windows_past_the_range_are_refused(kw):
    q, kp = torch.zeros(2, 8, 1, 64, dtype=BF, device="cuda"), torch.zeros(4, 4, 16, 64, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="2\\^30"):
        ops.attn_paged(q, kp, kp, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), i32([0, 0]), scale=1.0, **kw)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.attn_sinks(q, kp[:2], kp[:2], scale=1.0, pos=0, **{"sinks": 0, **kw})
    widest = ops.attn_paged(q, kp, kp, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), i32([0, 0]), scale=1.0,
                            window=(1 << 30) - 1, sinks=(1 << 30) - 1)
    assert not widest.any()


@pytest.mark.gpu
def test_large_scores_and_infinite_keys_out_of_sight():
    """Scores of hundreds (the running maximum moves), infinities where the mask hides them."""
    g = gen(13)
    for T in (1, 80):
        cache = Paged(g, [500 + T], 8, 128, 16, BF)
        cache.k[0] *= 12
        for j in range(cache.table.shape[1]):
            if cache.table[0, j] >= 0:
                lo, hi = j * 16, min(500 + T, j * 16 + 16)
                cache.kp[cache.table[0, j], :, :hi - lo] = cache.k[0][:, lo:hi]
        # keys behind the window and past the first tokens, on pages that are still held
        for pos in (70, 100, 200):
            at = int(cache.table[0, pos // 16]), slice(None), pos % 16
            cache.kp[at] = math.inf
            cache.k[0][:, pos] = math.inf
        q = torch.randn(1, T, 16, 128, generator=g).to(BF).transpose(1, 2)
        got = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([500]), scale=0.5, window=200,
                             sinks=20)
        assert_close(got, *cache.want(q, [500], [T], 200, 20, 0.5))


# ---------------------------------------------------------------- refusals
def test_python_refusals():
    """Checked before anything touches a GPU."""
    q = torch.zeros(2, 8, 1, 64)
    kp = torch.zeros(4, 4, 16, 64)
    table, rp = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.attn_paged(q, kp, kp, table, rp, scale=1.0)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.kv_append_paged(q[:, :4], q[:, :4], kp, kp, table, rp)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.attn_sinks(q, kp[:2], kp[:2], scale=1.0, window=4, sinks=1, pos=0)
    assert ops.paged_supported(BF, 512) and not ops.paged_supported(SF, 512)
    assert not ops.paged_supported(BF, 96) and not ops.paged_supported(torch.float64, 64)


@pytest.mark.gpu
def test_gpu_refusals():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")   # noqa: E731
    q, kp, table, rp = z(2, 8, 1, 64), z(4, 4, 16, 64), z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32)

    def paged(q=q, kp=kp, vp=None, table=table, rp=rp, **kw):
        return ops.attn_paged(q, kp, kp if vp is None else vp, table, rp, scale=1.0, **kw)

    paged()
    for what, kw in (("power of two", dict(kp=z(4, 4, 8, 64))), ("power of two", dict(kp=z(4, 4, 48, 64))),
                     ("page_table", dict(table=z(2, 2, dtype=torch.int64))), ("page_table", dict(table=z(3, 2, dtype=torch.int32))),
                     ("row_pos", dict(rp=z(2, dtype=torch.int64))), ("row_pos", dict(rp=z(3, dtype=torch.int32))),
                     ("new_lens", dict(new_lens=z(2, dtype=torch.int64))), ("does not fit", dict(q=z(2, 6, 1, 64))),
                     ("does not fit", dict(q=z(2, 8, 1, 128))), ("float16", dict(q=z(2, 8, 1, 64, dtype=HF))),
                     ("window", dict(sinks=3)), ("window", dict(window=-1)), ("window", dict(window=4, sinks=-1)),
                     ("max_kv_len", dict(max_kv_len=0)), ("must be", dict(vp=z(3, 4, 16, 64))),
                     ("one dtype", dict(vp=z(4, 4, 16, 64, dtype=HF))), ("strides", dict(vp=z(4, 4, 64, 16).transpose(2, 3))),
                     ("strides", dict(kp=z(4, 4, 16, 65)[..., 1:], vp=z(4, 4, 16, 65)[..., 1:])),
                     ("out must", dict(out=z(2, 1, 8, 64, dtype=HF))), ("out must", dict(out=z(2, 8, 1, 64))),
                     ("cos", dict(cos=z(3, 64, dtype=SF), sin=z(3, 64, dtype=SF)))):
        with pytest.raises(ValueError, match=what):
            paged(**kw)
    with pytest.raises(ValueError, match="head dim 96"):
        paged(q=z(2, 8, 1, 96), kp=z(4, 4, 16, 96))
    with pytest.raises(ValueError, match="head dim 512"):
        paged(q=z(2, 8, 1, 512, dtype=SF), kp=z(4, 4, 16, 512, dtype=SF))
    c = z(2, 4, 32, 64)
    for what, kw in (("needs a window", dict(window=0, sinks=0)), ("do not fit", dict(pos=32)), ("do not fit", dict(pos=-1)),
                     ("row_pos", dict(row_pos=z(3, dtype=torch.int32))), ("pos_dev", dict(pos_dev=z(1, dtype=torch.int32)))):
        with pytest.raises(ValueError, match=what):
            ops.attn_sinks(q, c, c, scale=1.0, **{"window": 4, "sinks": 1, **kw})
    k = z(2, 4, 1, 64)
    for what, a in (("do not fit", (k[:, :2], k[:, :2], kp, kp, table, rp)), ("must be", (k, k[:, :2], kp, kp, table, rp)),
                    ("row_pos", (k, k, kp, kp, table, rp.long())), ("page_table", (k, k, kp, kp, table[:1], rp))):
        with pytest.raises(ValueError, match=what):
            ops.kv_append_paged(*a)
    with pytest.raises(ValueError, match="head dim 40"):
        ops.kv_append_paged(z(2, 4, 1, 40), z(2, 4, 1, 40), z(4, 4, 16, 40), z(4, 4, 16, 40), table, rp)


# C entry points: every rejection happens before a launch, so host pointers that are never followed will do
_P = 1 << 20   # an aligned, non-null address


def _paged_call(**over):
    a = dict(dtype=_lib.BF16, B=2, T=1, H=8, K=4, D=64, q=_P, sqb=512, sqh=64, sqt=512, qw=None, eps=1e-6, flags=0, cos=None,
             sin=None, scb=0, sct=0, kp=_P, vp=_P, skp=4096, skh=1024, sks=64, n_pages=4, page=16, table=_P, spt=2, max_pages=2,
             row_pos=_P, new=None, max_kv=32, window=0, sinks=0, scale=1.0, out=_P, sob=512, sot=512, soh=64, ws=None, wsb=0,
             wsf=0, stream=None)
    a.update(over)
    return _lib.lib().forge_attn_paged(*a.values())


@pytest.mark.parametrize("what,over", [
    ("dtype", dict(dtype=7)), ("sizes", dict(B=-1)), ("sizes", dict(H=6)), ("sizes", dict(K=0)), ("head dim", dict(D=96)),
    ("head dim", dict(D=512, dtype=_lib.F32)), ("null", dict(q=None)), ("null", dict(vp=None)), ("null", dict(out=None)),
    ("null", dict(table=None)), ("null", dict(row_pos=None)), ("power of two", dict(page=8)), ("power of two", dict(page=24)),
    ("page table", dict(n_pages=0)), ("page table", dict(max_pages=0)), ("page table", dict(spt=-1)),
    ("max_kv_len", dict(max_kv=0)), ("negative", dict(window=-1)), ("negative", dict(window=3, sinks=-1)),
    ("window", dict(sinks=2)), ("strides", dict(sqt=510)), ("strides", dict(skh=1020)), ("strides", dict(sob=4)),
    ("aligned", dict(q=_P + 8)), ("aligned", dict(kp=_P + 2)), ("aligned", dict(out=_P + 4)), ("apart", dict(sks=32)),
    ("apart", dict(sks=1 << 28)), ("gain", dict(flags=_lib.NORM_QK, qw=_P + 4)), ("cos", dict(flags=_lib.ROPE)),
    ("2^31", dict(max_pages=1 << 28, max_kv=1 << 40)), ("query rows", dict(T=1 << 30)),
])
def test_c_refusals(what, over):
    assert _paged_call(**over) < 0
    assert what in _lib.lib().forge_last_error().decode()


def test_c_refusals_of_the_others():
    lib = _lib.lib()
    base = [_lib.BF16, 2, 1, 8, 4, 64, _P, 512, 64, 512, None, 1e-6, 0, None, None, 0, 0, _P, _P, 8192, 2048, 64, 32, _P, None,
            0, 32, 8, 2, 1.0, _P, 512, 512, 64, None, 0, 0, None]
    for what, at, value in (("window", 27, 0), ("max_kv_len", 26, 0), ("max_len", 22, 0), ("head dim", 5, 80)):
        a = list(base)
        a[at] = value
        assert lib.forge_attn_sinks(*a) < 0 and what in lib.forge_last_error().decode(), what
    a = list(base)
    a[23], a[25] = None, 32   # a host position that does not fit
    assert lib.forge_attn_sinks(*a) < 0 and "cache length" in lib.forge_last_error().decode()
    app = [_lib.BF16, 2, 1, 4, 64, _P, 256, 64, 256, _P, 256, 64, 256, _P, _P, 4096, 1024, 64, 4, 16, _P, 2, 2, _P, None, None,
           1e-6, 0, None, None, 0, 0, None]
    for what, at, value in (("sizes", 1, -1), ("head dim", 4, 40), ("null", 5, None), ("null", 20, None), ("null", 23, None),
                            ("power of two", 19, 20), ("page table", 18, 0), ("strides", 8, 252), ("aligned", 13, _P + 8),
                            ("cos", 27, _lib.ROPE)):
        a = list(app)
        a[at] = value
        assert lib.forge_kv_append_paged(*a) < 0 and what in lib.forge_last_error().decode(), what


def test_workspace_bytes():
    f = _lib.lib().forge_attn_paged_workspace_bytes
    assert f(_lib.BF16, 2, 1, 8, 4, 64, 16, 0, 0) == 0                   # one short tile: nothing to split
    assert f(_lib.BF16, 1, 1, 16, 8, 128, 32768, 0, 0) > 0               # eight pairs of a long row: split
    assert f(_lib.BF16, 1, 1, 16, 8, 128, 32768, 16, 0) == 0             # a short window is not
    assert f(_lib.BF16, 1, 1, 16, 8, 96, 32768, 0, 0) == 0 and f(9, 1, 1, 6, 4, 64, 100, 0, 0) == 0
    assert _lib.lib().forge_attn_sinks_workspace_bytes(_lib.F32, 4, 1, 8, 4, 64, 9000, 4096, 4) > 0


@pytest.mark.gpu
def test_merges_by_the_last_part_equal_the_combine_launch():
    """Split decode calls with the stream's workspace (the part that ends last merges) and under a recorded graph (a
    launch of its own merges): the same bits, many times over, and the counters are zero afterwards."""
    g = gen(14)
    for dtype, H, K, D, pasts, T in ((BF, 16, 8, 128, [1500, 700, 0], 1), (HF, 12, 4, 64, [1000] * 4, 1),
                                     (SF, 8, 4, 32, [3000, 12], 2), (BF, 8, 4, 256, [900, 300], 1), (BF, 16, 1, 512, [200], 1)):
        cache = Paged(g, [p + T for p in pasts], K, D, 16, dtype)
        B = len(pasts)
        q = torch.randn(B, T, H, D, generator=g).to(dtype).transpose(1, 2)
        args = (q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts))
        want, bound = cache.want(q, pasts, [T] * B, 0, 0, 0.1)
        first = ops.attn_paged(*args, scale=0.1)
        assert_close(first, want, bound)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attn_paged(*args, scale=0.1)
        for _ in range(20):
            assert torch.equal(ops.attn_paged(*args, scale=0.1), first)
            graph.replay()
            assert torch.equal(out, first)
    key = (0, torch.cuda.current_stream().cuda_stream)
    assert not ops._PAGED_WS[key][:64 * 1024].any()


@pytest.mark.gpu
def test_threads_on_one_stream():
    """Two threads that call on the same stream at once use workspaces of their own."""
    import threading

    g = gen(15)
    cache = Paged(g, [900, 2000], 8, 128, 16, BF)
    q = torch.randn(2, 1, 16, 128, generator=g).to(BF).transpose(1, 2).cuda()
    args = (q, cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([899, 1999]))
    first = ops.attn_paged(*args, scale=0.1)
    torch.cuda.synchronize()
    outs = {}

    def work(i):
        outs[i] = [ops.attn_paged(*args, scale=0.1) for _ in range(200)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for i in range(4) for o in outs[i])


# ---------------------------------------------------------------- keys that no query sees
HIDDEN = [
    # (dtype, H, K, D, page, pasts, T, window, sinks): steps, 32-row blocks, chunks; the window starts in the tile of
    # the first tokens (70, 75), or far behind it
    (BF, 16, 8, 128, 16, [700, 75, 70], 1, 64, 4), (HF, 12, 4, 64, 64, [300, 90], 5, 50, 20), (SF, 8, 4, 32, 16, [200, 40], 3, 33, 2),
    (BF, 8, 1, 256, 32, [333], 4, 100, 33), (BF, 16, 1, 512, 16, [150, 77], 1, 48, 3), (BF, 16, 8, 128, 16, [700], 1, 1, 0),
    (HF, 8, 4, 32, 64, [900], 1500, 700, 4), (BF, 16, 8, 128, 64, [500], 900, 100, 40), (HF, 12, 4, 64, 16, [777], 2000, 300, 4),
    (BF, 8, 4, 256, 32, [400, 90], 500, 70, 9), (SF, 8, 4, 64, 16, [333], 1100, 200, 3), (BF, 16, 1, 512, 32, [600], 220, 250, 3),
    (HF, 8, 4, 32, 16, [1500], 3001, 1400, 7), (BF, 16, 16, 64, 128, [900], 700, 129, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [math.nan, math.inf])
@pytest.mark.parametrize("case", HIDDEN, ids=_id)
def test_keys_that_no_query_sees_are_never_used(case, fill):
    """Between the first tokens and the window, on pages that are held: NaN or Inf in K and V reach no output, over
    pages and over the contiguous cache."""
    dtype, H, K, D, page, pasts, T, window, sinks = case
    g = gen(31)
    B = len(pasts)
    cache = Paged(g, [p + T for p in pasts], K, D, page, dtype)
    cap = max(cache.lens) + 5
    kc, vc = (torch.full((B, K, cap, D), math.nan, dtype=dtype) for _ in range(2))
    for b, n in enumerate(cache.lens):
        hidden = slice(min(sinks, pasts[b]), max(sinks, pasts[b] - window + 1))
        assert hidden.stop > hidden.start
        cache.k[b][:, hidden], cache.v[b][:, hidden] = fill, fill
        kc[b, :, :n], vc[b, :, :n] = cache.k[b], cache.v[b]
        for j in range(-(-n // page)):
            lo, hi = j * page, min(n, (j + 1) * page)
            cache.kp[cache.table[b, j], :, :hi - lo] = cache.k[b][:, lo:hi]
            cache.vp[cache.table[b, j], :, :hi - lo] = cache.v[b][:, lo:hi]
    q = torch.randn(B, T, H, D, generator=g).to(dtype).transpose(1, 2)
    want, bound = cache.want(q, pasts, [T] * B, window, sinks, D ** -0.5)
    kw = dict(scale=D ** -0.5, window=window, sinks=sinks)
    assert_close(ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts), **kw), want, bound,
                 "pages")
    assert_close(ops.attn_sinks(q.cuda(), kc.cuda(), vc.cuda(), row_pos=i32(pasts), **kw), want, bound, "contiguous")


# ---------------------------------------------------------------- scales
BAD_SCALES = [0.0, -0.0, -0.125, math.nan, math.inf, -math.inf, 1e-300, 3e38]


@pytest.mark.parametrize("scale", BAD_SCALES)
def test_c_refuses_scales_that_are_not_positive(scale):
    """A masked score is -inf before it is scaled: -inf times 0 is NaN, times a negative number +inf."""
    assert _paged_call(scale=scale) < 0 and "scale" in _lib.lib().forge_last_error().decode()
    base = [_lib.BF16, 2, 1, 8, 4, 64, _P, 512, 64, 512, None, 1e-6, 0, None, None, 0, 0, _P, _P, 8192, 2048, 64, 32, _P, None,
            0, 32, 8, 2, scale, _P, 512, 512, 64, None, 0, 0, None]
    assert _lib.lib().forge_attn_sinks(*base) < 0 and "scale" in _lib.lib().forge_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", BAD_SCALES)
def test_ops_refuse_scales_that_are_not_positive(scale):
    q, kp = torch.zeros(2, 8, 1, 64, dtype=BF, device="cuda"), torch.zeros(4, 4, 16, 64, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="scale"):
        ops.attn_paged(q, kp, kp, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), i32([0, 0]), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.attn_sinks(q, kp[:2], kp[:2], scale=scale, window=4, sinks=1, pos=0)


# ---------------------------------------------------------------- steps whose sums do not hang on T
FIXED = [(BF, 16, 8, 128, 2, 300, 4), (HF, 12, 4, 64, 1, 1000, 33), (BF, 8, 1, 256, 3, 64, 5), (BF, 16, 1, 512, 1, 200, 3), (SF, 8, 4, 32, 2, 100, 1),
         (SF, 16, 8, 128, 1, 500, 64), (HF, 28, 4, 128, 1, 129, 0), (BF, 32, 8, 32, 70, 90, 70), (BF, 8, 4, 256, 40, 700, 4), (SF, 8, 1, 256, 1, 333, 9),
         (HF, 16, 16, 64, 1, 5000, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", FIXED, ids=_id)
def test_fixed_cut_rows_are_the_decodes_bit_for_bit(case):
    """A verify step's rows equal the decodes of those tokens, wherever the window starts in a tile, with a host
    position, one on the device and one for each row, and under any bound."""
    dtype, H, K, D, B, window, sinks = case
    g = gen(41)
    cap, scale = 2100, D ** -0.5
    kc, vc = ((1.3 * torch.randn(B, K, cap, D, generator=g)).to(dtype).cuda() for _ in range(2))
    kw = dict(scale=scale, window=window, sinks=sinks, fixed_cut=True)
    for T, at in ((2, 0), (5, window - 3), (4, window + 29), (3, 62), (16, 1000), (7, 1721), (5, cap - 5), (9, 1500 + sinks)):
        q = torch.randn(B, T, H, D, generator=g).to(dtype).cuda().transpose(1, 2)
        at = min(max(at, 0), cap - T)
        rows = ops.attn_sinks(q, kc, vc, pos=at, **kw)
        want, bound = _sinks_want(q[:2].cpu(), kc[:2].cpu(), vc[:2].cpu(), [at] * min(B, 2), window, sinks, scale)
        assert_close(rows[:2], want, bound)
        for t in range(T):
            one = ops.attn_sinks(q[:, :, t:t + 1], kc, vc, pos=at + t, **kw)
            assert torch.equal(one[:, 0], rows[:, t]), (T, at, t)
        for other in (dict(pos_dev=torch.tensor([at], device="cuda")), dict(row_pos=i32([at] * B)),
                      dict(row_pos=i32([at] * B), max_kv_len=at + T)):
            assert torch.equal(ops.attn_sinks(q, kc, vc, **other, **kw), rows)
        graph = torch.cuda.CUDAGraph()   # (merged by a launch of its own)
        with torch.cuda.graph(graph):
            out = ops.attn_sinks(q, kc, vc, pos=at, **kw)
        graph.replay()
        assert torch.equal(out, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_fixed_cut_never_uses_keys_that_no_query_sees(fill):
    g = gen(42)
    kc, vc = (torch.randn(1, 8, 800, 128, generator=g).to(BF) for _ in range(2))
    for c in (kc, vc):
        c[:, :, 4:637], c[:, :, 703:] = fill, fill
    q = torch.randn(1, 3, 16, 128, generator=g).to(BF).transpose(1, 2)
    got = ops.attn_sinks(q.cuda(), kc.cuda(), vc.cuda(), scale=0.1, window=64, sinks=4, pos=700, fixed_cut=True)
    assert_close(got, *_sinks_want(q, kc, vc, [700], 64, 4, 0.1))


def test_fixed_cut_refusals():
    lib = _lib.lib()
    base = [_lib.BF16, 2, 17, 8, 4, 64, _P, 512, 64, 512, None, 1e-6, _lib.FIXED_CUT, None, None, 0, 0, _P, _P, 8192, 2048, 64, 32,
            _P, None, 0, 32, 8, 2, 1.0, _P, 512, 512, 64, None, 0, 0, None]
    assert lib.forge_attn_sinks(*base) < 0 and "16 tokens" in lib.forge_last_error().decode()
    f = lib.forge_attn_sinks_fixed_workspace_bytes
    assert f(_lib.BF16, 1, 17, 16, 8, 128, 9000, 1024, 4) == 0 and f(_lib.BF16, 1, 1, 16, 8, 96, 9000, 1024, 4) == 0
    assert f(_lib.BF16, 1, 1, 16, 8, 128, 9000, 1024, 4) > 64 * 1024 and f(_lib.BF16, 1, 1, 16, 8, 128, 64, 16, 4) == 0


@pytest.mark.gpu
def test_fixed_cut_refuses_long_calls():
    c = torch.zeros(1, 4, 64, 64, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="fixed_cut"):
        ops.attn_sinks(torch.zeros(1, 8, 17, 64, dtype=BF, device="cuda"), c, c, scale=1.0, window=4, sinks=1, pos=0, fixed_cut=True)


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [0, -1, -5])
def test_sinks_bounds_below_one_are_refused(bound):
    """Where it is the call that gives the bound: positions on the device."""
    c, q = torch.zeros(2, 4, 32, 64, dtype=BF, device="cuda"), torch.zeros(2, 8, 1, 64, dtype=BF, device="cuda")
    for where in (dict(row_pos=i32([3, 4])), dict(pos_dev=torch.tensor([3], device="cuda"))):
        with pytest.raises(ValueError, match="max_kv_len"):
            ops.attn_sinks(q, c, c, scale=1.0, window=4, sinks=1, max_kv_len=bound, **where)


def test_calls_whose_tiles_pass_32_bits_are_not_planned():
    """The device's plan adds up the tiles of all row blocks in 32 bits; past that it could hand out more parts than its
    list holds. 64 row blocks of 2^25 tiles are cut on the host, which needs no plan (nor, here, partials)."""
    f = _lib.lib().forge_attn_paged_workspace_bytes
    assert f(_lib.BF16, 2, 2048, 16, 8, 128, 100_000, 0, 0) > 0
    assert f(_lib.BF16, 2, 2048, 16, 8, 128, 2 ** 31 - 65537, 0, 0) == 0


def test_partials_of_calls_that_fill_the_device_many_times():
    """Blocks that are many for each that the device holds are not split: their partials would be gigabytes."""
    f = _lib.lib().forge_attn_paged_workspace_bytes
    assert f(_lib.F32, 8, 4096, 32, 8, 32, 32768, 0, 0) == 0
    assert f(_lib.BF16, 64, 1, 16, 8, 128, 32768, 0, 0) > 0 and f(_lib.BF16, 256, 1, 16, 8, 128, 32768, 0, 0) > 0


# ---------------------------------------------------------------- the split kernel's weights
def _pairs(g, dtype, H, K, D, pairs):
    """Keys in pairs whose scores differ a little and whose values are opposite: a row is a small difference of large
    terms, so that half a step on a weight shows beside half a step on the output. Small queries: the bound's part for the
    scores' own roundings, which grows with sum |q k|, is small too."""
    k = torch.randn(K, 2 * pairs, D, generator=g)
    k[:, 1::2] = k[:, ::2] * 1.01
    v = 3 * torch.randn(K, 2 * pairs, D, generator=g)
    v[:, 1::2] = -v[:, ::2].to(dtype).float()
    return k.to(dtype), v.to(dtype), (0.1 * torch.randn(H, 1, D, generator=g)).to(dtype)


def _two_number_bound(q, k, v, see, scale):
    """attend64's bound with weights of two numbers of the type: what the second leaves out is half a step of half a step
    (h * h in place of h)."""
    want, bound = attend64(q, k, v, see, scale)
    h = torch.finfo(q.dtype).eps / 2
    vmax = v.double().abs().masked_fill(~see.any(0)[None, :, None], 0).amax((1, 2))          # [K]
    return want, bound - (vmax * (h - h * h)).repeat_interleave(q.shape[0] // k.shape[0])[None, :, None]


SPLIT = [(BF, 16, 8, 128), (HF, 12, 4, 64), (BF, 8, 1, 256), (BF, 16, 1, 512), (HF, 8, 4, 32)]


@pytest.mark.parametrize("dtype,H,K,D", SPLIT)
def test_the_two_number_bound_tells_weights_rounded_once(dtype, H, K, D):
    """The oracle's own output with weights rounded once lies outside the bound."""
    k, v, q = _pairs(gen(51), dtype, H, K, D, 3)
    see = torch.ones(1, 6, dtype=torch.bool)
    want, bound = _two_number_bound(q, k, v, see, D ** -0.5)
    rep = H // K
    s = (q.double() @ k.double().repeat_interleave(rep, 0).transpose(1, 2)) * D ** -0.5
    w = (s - s.amax(-1, keepdim=True)).exp()
    once = ((w.to(dtype).double() @ v.double().repeat_interleave(rep, 0)) / w.sum(-1, keepdim=True)).transpose(0, 1)
    with pytest.raises(AssertionError, match="outside"):
        assert_close(once.to(dtype), want, bound)
    exact = ((w @ v.double().repeat_interleave(rep, 0)) / w.sum(-1, keepdim=True)).transpose(0, 1)
    assert_close(exact.to(dtype), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H,K,D", SPLIT)
@pytest.mark.parametrize("pairs", [1, 3, 40, 700])
def test_split_weights_are_not_rounded_to_the_type(dtype, H, K, D, pairs):
    g = gen(52)
    k, v, q = _pairs(g, dtype, H, K, D, pairs)
    n = 2 * pairs
    want, bound = _two_number_bound(q, k, v, torch.ones(1, n, dtype=torch.bool), D ** -0.5)
    kc, vc = (torch.nn.functional.pad(x, (0, 0, 0, -n % 16))[None].cuda() for x in (k, v))
    for fixed in (False, True):
        got = ops.attn_sinks(q[None].cuda(), kc, vc, scale=D ** -0.5, window=4096, sinks=2, pos=n - 1, fixed_cut=fixed)
        assert_close(got[0], want, bound)
    kp, vp = (x.view(K, -1, 16, D).transpose(0, 1).contiguous() for x in (kc[0], vc[0]))
    table = torch.arange(kp.shape[0], dtype=torch.int32, device="cuda")[None]
    assert_close(ops.attn_paged(q[None].cuda(), kp, vp, table, i32([n - 1]), scale=D ** -0.5)[0], want, bound)


def test_c_refuses_overlapping_outputs_and_stray_flags():
    for over in (dict(sob=0), dict(sot=0, T=2, sqt=512), dict(soh=0)):
        assert _paged_call(**over) < 0 and "overlap" in _lib.lib().forge_last_error().decode()
    assert _paged_call(flags=_lib.FIXED_CUT) < 0 and "forge_attn_sinks" in _lib.lib().forge_last_error().decode()


@pytest.mark.gpu
def test_ops_refuse_overlapping_outputs_and_q_of_other_ranks():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")   # noqa: E731
    q, kp, table, rp, c = z(2, 8, 1, 64), z(4, 4, 16, 64), z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32), z(2, 4, 32, 64)
    with pytest.raises(ValueError, match="out must"):
        ops.attn_paged(q, kp, kp, table, rp, scale=1.0, out=z(1, 1, 8, 64).expand(2, 1, 8, 64))
    with pytest.raises(ValueError, match="out must"):
        ops.attn_sinks(q, c, c, scale=1.0, window=4, sinks=1, pos=0, out=z(2, 1, 1, 64).expand(2, 1, 8, 64))
    for bad in (z(8, 64), z(2, 8, 64)):
        with pytest.raises(ValueError, match="q "):
            ops.attn_paged(bad, kp, kp, table, rp, scale=1.0)
        with pytest.raises(ValueError, match="q "):
            ops.attn_sinks(bad, c, c, scale=1.0, window=4, sinks=1, pos=0)


@pytest.mark.gpu
def test_fixed_cut_without_memory_for_its_partials_raises(monkeypatch):
    """Unsplit, the call's bits would be others."""
    from types import SimpleNamespace

    c, q = torch.zeros(1, 8, 2000, 128, dtype=BF, device="cuda"), torch.zeros(1, 16, 1, 128, dtype=BF, device="cuda")
    kw = dict(scale=1.0, window=1024, sinks=4, pos=1500)
    monkeypatch.setattr(ops, "host", lambda: SimpleNamespace(attn_sinks=lambda *a: None))
    monkeypatch.setattr(ops, "_PAGED_WS_KEPT", 0)
    monkeypatch.setattr(ops, "_partials", lambda need, dev: None)
    ops.attn_sinks(q, c, c, **kw)   # (not split)
    with pytest.raises(torch.cuda.OutOfMemoryError, match="fixed_cut"):
        ops.attn_sinks(q, c, c, fixed_cut=True, **kw)
