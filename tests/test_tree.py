"""Trees of drafted tokens (ops.tree_mask, attn_tree, attn_tree_paged, verify_drafts, kv_compact, copy_pages) against plain
64-bit forms."""

from __future__ import annotations

import ctypes as C
import itertools
import math
import random
import time

import pytest
import torch

from paged_oracle import Paged, assert_close, attend64, norm_rope64
from sleuth_amd import _lib, ops
from sleuth_amd.rope import rope_tables
from tree_oracle import bits_to_bool, chain_of, compact_row, make_parents, mask_of, tree_see, tree_see_long, verify_row

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def i32(xs, dev="cuda"):
    return torch.tensor(xs, dtype=torch.int32, device=dev)


def _id(c):
    return "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)


# ================================================================ on the CPU: what is refused, what the oracle is
def _refused(status, what):
    assert status == -1
    assert what in _lib.lib().forge_last_error().decode()


FAKE = 1 << 20   # an address that no refused call reads


def test_tree_mask_refusals():
    f = _lib.lib().forge_tree_mask
    _refused(f(1, 1025, FAKE, 0, None, FAKE, FAKE, None), "at most 1024")
    _refused(f(-1, 4, FAKE, 0, None, FAKE, FAKE, None), "bad sizes")
    _refused(f(1, 4, None, 0, None, FAKE, FAKE, None), "null")
    _refused(f(1, 4, FAKE, 0, None, None, FAKE, None), "null")
    assert f(0, 4, None, 0, None, None, None, None) == 0
    assert f(4, 0, None, 0, None, None, None, None) == 0


def _tree_call(**kw):
    a = dict(dtype=_lib.BF16, B=2, T=4, H=4, K=2, D=64, q=FAKE, sqb=1024, sqh=64, sqt=256, qw=None, eps=0.0, flags=0, cos=None,
             sin=None, scb=0, sct=0, k=FAKE, v=FAKE, skp=8192, skh=4096, sks=64, n_pages=8, page_size=64, table=None, s_table=0,
             max_pages=0, row_pos=FAKE, pos_dev=None, pos0=0, news=None, max_kv=64, window=0, sinks=0, scale=0.125, mask=FAKE,
             smb=4, smt=1, depth=None, sdb=0, out=FAKE, sob=1024, sot=256, soh=64, ws=None, wsb=0, wsf=0, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().forge_attn_tree(*a.values())


@pytest.mark.parametrize("bad, why", [
    (dict(T=1025), "at most 1024"), (dict(mask=None), "mask"), (dict(mask=FAKE + 4), "mask"), (dict(smb=-1), "mask"),
    (dict(window=5), "depths"), (dict(window=5, depth=FAKE, sdb=-1), "depths"), (dict(sinks=3), "sinks need a window"),
    (dict(window=-1), "negative"), (dict(row_pos=None, pos0=61), "exceeds"), (dict(row_pos=None, pos0=-1), "exceeds"),
    (dict(max_kv=0), "positive"), (dict(page_size=0), "positive"), (dict(D=48), "head dim"), (dict(D=512, dtype=_lib.F32), "head dim"),
    (dict(H=3), "multiple"), (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q=None), "null"), (dict(q=FAKE + 8), "aligned"), (dict(sqh=60), "16 bytes"), (dict(sot=0), "overlap"),
    (dict(flags=_lib.FIXED_CUT), "FIXED_CUT"), (dict(flags=_lib.ROPE), "cos and sin"), (dict(dtype=7), "dtype"),
    (dict(table=FAKE, page_size=48, max_pages=2), "power of two"), (dict(table=FAKE, max_pages=0), "page table"),
    (dict(table=FAKE, max_pages=2, row_pos=None), "row positions"), (dict(ws=FAKE, wsb=1, B=1, T=64, max_kv=1 << 20, page_size=1 << 20), "workspace"),
    (dict(page_size=1 << 31, max_kv=1 << 31), "2^31"),
], ids=str)
def test_attn_tree_refusals(bad, why):
    _refused(_tree_call(**bad), why)


def test_attn_tree_of_nothing():
    assert _tree_call(B=0, mask=None, q=None) == 0
    assert _tree_call(T=0, mask=None, q=None) == 0


def _verify_call(**kw):
    a = dict(dtype=_lib.BF16, B=2, T=4, V=100, logits=FAKE, slb=400, slt=100, tokens=FAKE, stb=4, parents=None, spb=0, uniform=FAKE,
             sub=4, temps=None, heat=1.0, pdt=0, probs=None, sqb=0, sqt=0, news=None, out=FAKE, path=FAKE, count=FAKE, ws=FAKE,
             wsb=1 << 20, wsf=0, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().forge_verify_drafts(*a.values())


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=5), "dtype"), (dict(T=0), "bad sizes"), (dict(V=0), "bad sizes"), (dict(B=-1), "bad sizes"), (dict(T=1025), "at most"),
    (dict(B=65536), "at most"), (dict(V=1 << 22), "at most"), (dict(tokens=None), "null"), (dict(heat=-1.0), "temperature"),
    (dict(heat=math.nan), "temperature"), (dict(heat=math.inf), "temperature"), (dict(heat=1e-40), "temperature"),
    (dict(uniform=None), "random numbers"), (dict(heat=0.0, temps=FAKE, uniform=None), "random numbers"),
    (dict(probs=FAKE, pdt=_lib.F16), "logits' type"), (dict(slt=-1), "strides"), (dict(wsb=8), "workspace"),
    (dict(ws=None), "workspace"), (dict(ws=FAKE + 16), "aligned"),
], ids=str)
def test_verify_refusals(bad, why):
    _refused(_verify_call(**bad), why)


def test_verify_workspace():
    size = _lib.lib().forge_verify_drafts_workspace_bytes
    assert size(0, 4, 100, 0) == size(1, 1025, 100, 0) == size(1, 4, 1 << 22, 0) == size(1, 4, 0, 0) == 0
    assert 0 < size(2, 4, 100, 0) < size(2, 4, 100, 1) and size(2, 4, 9000, 0) >= 2 * 4 * 3 * 16
    assert _verify_call(B=0, logits=None) == 0


def _pointers(*xs):
    return (C.c_void_p * len(xs))(*xs)


def _compact_call(**kw):
    a = dict(es=2, layers=1, B=1, K=2, D=64, k=_pointers(FAKE), v=_pointers(FAKE), skp=8192, skh=4096, sks=64, n_pages=4, page_size=64,
             table=None, s_table=0, max_pages=0, row_pos=FAKE, pos_dev=None, pos0=0, path=FAKE, s_path=4, T=4, counts=FAKE, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().forge_kv_compact(*a.values())


@pytest.mark.parametrize("bad, why", [
    (dict(es=1), "2 or 4"), (dict(D=4), "16 bytes"), (dict(K=0), "bad sizes"), (dict(layers=-1), "bad sizes"), (dict(k=None), "null"),
    (dict(k=_pointers(FAKE + 8)), "aligned"), (dict(v=_pointers(None)), "aligned"), (dict(sks=60), "strides"), (dict(skh=-64), "strides"),
    (dict(page_size=0), "positive"), (dict(table=FAKE, page_size=24, max_pages=1), "power of two"), (dict(table=FAKE), "page table"),
    (dict(table=FAKE, max_pages=1, row_pos=None), "row positions"), (dict(path=None), "null"), (dict(counts=None), "null"),
    (dict(B=65536), "bad sizes"), (dict(page_size=1 << 31), "2^31"),
], ids=str)
def test_kv_compact_refusals(bad, why):
    _refused(_compact_call(**bad), why)


@pytest.mark.parametrize("k, v", [([1, 2, 3], [4, 5, 1]), ([2, 1, 2], [4, 5, 6]), ([1], [1]), ([3, 2, 1], [6, 4, 4])])
def test_kv_compact_refuses_a_cache_named_twice(k, v):
    k, v = (_pointers(*(FAKE + 4096 * i for i in x)) for x in (k, v))
    _refused(_compact_call(layers=len(k), k=k, v=v), "twice")


def test_moves_of_nothing():
    assert _compact_call(layers=0) == _compact_call(B=0) == _compact_call(T=0, path=None) == 0
    f = _lib.lib().forge_copy_pages
    one = _pointers(FAKE)
    assert f(2, 0, 2, 64, None, None, 8192, 4096, 64, 4, 64, 3, FAKE, FAKE, None) == 0
    assert f(2, 1, 2, 64, one, one, 8192, 4096, 64, 4, 64, 0, None, None, None) == 0
    _refused(f(2, 1, 2, 64, one, one, 8192, 4096, 64, 4, 24, 3, FAKE, FAKE, None), "power of two")
    _refused(f(2, 1, 2, 64, one, one, 8192, 4096, 64, 0, 64, 3, FAKE, FAKE, None), "bad sizes")
    _refused(f(2, 1, 2, 64, one, one, 8192, 4096, 64, 4, 64, 3, None, FAKE, None), "null")
    _refused(f(2, 1, 2, 64, one, one, 8190, 4096, 64, 4, 64, 3, FAKE, FAKE, None), "strides")


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_mask(x)
    with pytest.raises(ValueError, match="GPU"):
        ops.verify_drafts(torch.zeros(1, 4, 8), x.long())
    kv = [torch.zeros(2, 1, 16, 32)]
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_compact(kv, kv, x, x[:, 0])
    with pytest.raises(ValueError, match="GPU"):
        ops.copy_pages(kv, kv, [0], [1])
    with pytest.raises(ValueError, match="GPU"):
        ops.attn_tree(torch.zeros(1, 2, 4, 32), kv[0], kv[0], x.long(), scale=1.0, pos=0)


def test_page_numbers_are_checked_in_one_pass():
    """Lists of 20,000 pages, whose check took 6 s where it built a set for each page, in well under one."""
    src, dst = list(range(20000)), list(range(20000, 40000))
    start = time.perf_counter()
    assert ops._page_numbers(src, dst, 40000) == (src, dst)
    assert time.perf_counter() - start < 1.0
    for bad in ((src, dst[:-1]), (src, dst[:-1] + dst[:1]), (src, dst[:-1] + src[:1]), (src[:1], [40000]), ([-1], dst[:1])):
        with pytest.raises(ValueError):
            ops._page_numbers(*bad, 40000)
    assert ops._page_numbers([], [], 1) == ([], [])
    assert ops._page_numbers([3, 3], [1, 2], 4) == ([3, 3], [1, 2])


def _outcomes(p, q, children, drawn):
    """The distribution of the token behind a node whose children (tokens, in order) are verified: `drawn` by q, or not."""
    out = torch.zeros_like(p)
    left, reach = p.clone(), 1.0
    for x in children:
        W = float(left.sum())
        yes = 1.0 if W <= 0 else min(1.0, float(left[x]) / W / (float(q[x]) if drawn else 1.0))
        out[x] += reach * yes
        reach *= 1 - yes
        if drawn:
            left = (left / W - q).clamp(min=0)   # the textbook's step: normalise, take q out, again
        else:
            left[x] = 0
        if reach < 1e-15:
            return out
    return out + reach * left / left.sum()


@pytest.mark.parametrize("drawn", [False, True])
def test_the_rule_keeps_the_targets_distribution(drawn):
    """Over the drafter's draws and the random numbers, what comes out is the target's distribution; and the rule's closed
    form, max(p - a q, 0) with a growing by what was left, is the repeated step."""
    torch.manual_seed(3)
    p, q = torch.rand(5).double().softmax(0), (2 * torch.rand(5)).double().softmax(0)
    if not drawn:
        for children in itertools.permutations(range(5), 3):
            assert torch.allclose(_outcomes(p, q, children, False), p, atol=1e-14)
        return
    total = torch.zeros(5).double()
    for xs in itertools.product(range(5), repeat=3):
        total += _outcomes(p, q, xs, True) * math.prod(float(q[x]) for x in xs)
    assert torch.allclose(total, p, atol=1e-13)
    left, a = p.clone(), 0.0
    for _ in range(3):
        a += float((p - a * q).clamp(min=0).sum())
        left = (left / left.sum() - q).clamp(min=0)
        closed = (p - a * q).clamp(min=0)
        assert torch.allclose(left / left.sum(), closed / closed.sum(), atol=1e-12)


def test_oracle_row_by_hand():
    logits = torch.tensor([[0.0, math.log(3.0)], [0.0, 0.0]])
    # p(1) = 3/4 behind node 0: accepted up to u = 3/4; behind node 1 the halves are drawn by u[0]
    assert verify_row(logits, [0, 1], [-1, 0], [0.6, 0.74], 1.0, None, 2) == ([1, 1], [0, 1])
    assert verify_row(logits, [0, 1], [-1, 0], [0.4, 0.74], 1.0, None, 2) == ([1, 0], [0, 1])
    assert verify_row(logits, [0, 1], [-1, 0], [0.9, 0.76], 1.0, None, 2) == ([0], [0])
    assert verify_row(logits, [0, 1], [-1, 0], None, 0.0, None, 2) == ([1, 0], [0, 1])
    assert verify_row(logits, [0, 1], [-1, 0], None, 0.0, None, 1) == ([1], [0])


# ================================================================ who sees whom
@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 13, 63, 64, 65, 128, 200, 256, 257, 700, 1024])
@pytest.mark.parametrize("shape", ["chain", "star", "tree", "forest"])
def test_tree_mask(T, shape):
    rng = random.Random(T)
    B = 3
    parents = [make_parents(rng, T, shape) for _ in range(B)]
    wild = list(parents[2])
    for t in range(0, T, 3):   # parents that are none
        wild[t] = rng.choice([t, t + 1, T, 2 ** 31 - 1, -2 ** 31, -7])
    parents[2] = wild
    news = [T, rng.randrange(T + 1), T]
    for new_lens in (None, news):
        mask, depth = ops.tree_mask(i32(parents), None if new_lens is None else i32(new_lens))
        want = [mask_of(p, T if new_lens is None else n) for p, n in zip(parents, news)]
        assert mask.tolist() == [m for m, _ in want]
        assert depth.tolist() == [d for _, d in want]


@pytest.mark.gpu
def test_tree_mask_forms():
    rng = random.Random(0)
    p = make_parents(rng, 30, "tree")
    mask, depth = ops.tree_mask(i32(p))
    want = mask_of(p, 30)
    assert (mask.tolist(), depth.tolist()) == want
    wide = torch.full((4, 60), 99, dtype=torch.int32, device="cuda")
    wide[:, ::2] = i32([p] * 4)
    mask, depth = ops.tree_mask(wide[:, ::2])                       # strided
    assert mask.tolist() == [want[0]] * 4
    mask, depth = ops.tree_mask(i32(p).expand(4, -1), i32([30, -5, 99, 7]))   # lengths outside are taken inside
    assert depth.tolist() == [want[1], [0] * 30, want[1], mask_of(p, 7)[1]]
    mask, depth = ops.tree_mask(torch.zeros(0, 5, dtype=torch.int32, device="cuda"))
    assert mask.shape == (0, 5, 1) and depth.shape == (0, 5)
    mask, depth = ops.tree_mask(torch.zeros(3, 0, dtype=torch.int32, device="cuda"))
    assert mask.shape == (3, 0, 0) and depth.shape == (3, 0)
    for bad in (torch.zeros(2, 4, device="cuda"), torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda"),
                torch.zeros(1, 1025, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            ops.tree_mask(bad)
    with pytest.raises(ValueError):
        ops.tree_mask(i32([p] * 2), i32([1, 2, 3]))


# ================================================================ attention
# (dtype, H, K, D, page or 0, pasts, T, shape, news or None, window, sinks)
ATTEND = [
    # small trees: lengths of zero and one, page and tile ends inside the tree
    (BF, 16, 8, 128, 0, [0, 1, 15, 31, 212], 12, "tree", None, 0, 0),
    (BF, 16, 8, 128, 16, [0, 1, 15, 16, 31, 400], 12, "tree", None, 0, 0),
    (HF, 12, 4, 64, 32, [0, 63, 500], 26, "tree", None, 0, 0),
    (SF, 8, 4, 32, 16, [0, 5, 300], 9, "forest", None, 0, 0),
    (SF, 16, 8, 128, 0, [90, 3], 5, "star", None, 0, 0),
    (SF, 8, 1, 256, 16, [130], 3, "tree", None, 0, 0),
    (BF, 8, 4, 32, 0, [77, 1030], 7, "tree", None, 0, 0),
    (BF, 16, 1, 512, 16, [0, 333], 6, "tree", None, 0, 0),
    (HF, 28, 4, 128, 16, [2500, 9], 8, "tree", None, 0, 0),
    (HF, 8, 1, 256, 0, [61, 5], 1, "tree", None, 0, 0),
    # larger ones, over one row block and several, more bits than a word
    (BF, 16, 8, 128, 64, [700, 20], 64, "tree", None, 0, 0),
    (BF, 16, 8, 128, 0, [3000], 65, "tree", None, 0, 0),
    (HF, 12, 4, 64, 0, [0, 5000], 100, "chain", None, 0, 0),
    (BF, 8, 4, 256, 16, [900, 1], 70, "forest", None, 0, 0),
    (SF, 16, 8, 128, 32, [600], 80, "tree", None, 0, 0),
    (SF, 12, 4, 64, 0, [40, 1500], 66, "tree", None, 0, 0),
    (SF, 8, 1, 256, 0, [700], 40, "tree", None, 0, 0),
    (BF, 16, 1, 512, 32, [800], 40, "tree", None, 0, 0),
    (HF, 8, 4, 32, 16, [4000], 130, "tree", None, 0, 0),
    (BF, 32, 8, 128, 0, [100], 300, "tree", None, 0, 0),
    # padded batches: none, one, some, all
    (BF, 16, 8, 128, 16, [100, 50, 0, 700], 9, "tree", [9, 0, 1, 4], 0, 0),
    (HF, 12, 4, 64, 0, [30, 8, 900], 90, "tree", [90, 1, 0], 0, 0),
    (SF, 8, 4, 64, 16, [30, 8], 40, "tree", [0, 33], 0, 0),
    # windows: beyond the tree, within it, and so small that a branch passes it; first tokens that reach into the tree
    (BF, 16, 8, 128, 16, [0, 10, 700, 2000], 12, "tree", None, 64, 4),
    (BF, 16, 8, 128, 0, [700, 4], 30, "chain", None, 7, 3),
    (HF, 8, 1, 256, 32, [300, 31], 26, "tree", None, 3, 40),
    (SF, 8, 4, 64, 16, [300, 2], 20, "chain", [20, 13], 5, 6),
    (BF, 12, 4, 64, 0, [0, 250], 150, "chain", None, 40, 7),
    (BF, 16, 8, 128, 64, [1000], 140, "tree", None, 300, 64),
    (BF, 8, 4, 256, 16, [4000], 66, "tree", None, 1024, 4),
    (BF, 16, 1, 512, 16, [150], 20, "chain", None, 1, 0),
]


def _dense(cache: Paged, cap: int, fill=math.nan):
    """The same keys as a contiguous cache [B, K, cap, D], the rest poisoned."""
    B, (K, _, D) = len(cache.lens), cache.k[0].shape
    k = torch.full((B, K, cap, D), fill, dtype=cache.k[0].dtype)
    v = k.clone()
    for b, n in enumerate(cache.lens):
        k[b, :, :n], v[b, :, :n] = cache.k[b], cache.v[b]
    return k, v


def _tree_inputs(dtype, H, K, D, page, pasts, T, shape, news, window, sinks, seed=0):
    g, rng = gen(seed), random.Random(seed)
    real = news if news is not None else [T] * len(pasts)

    def freed(b, j):   # pages that no query of the call sees are given back
        P = page or 16
        return bool(window) and j * P >= sinks and (j + 1) * P - 1 <= pasts[b] - window

    cache = Paged(g, [p + n for p, n in zip(pasts, real)], K, D, page or 16, dtype, freed=freed)
    parents = [make_parents(rng, T, shape) for _ in pasts]
    q = (1.3 * torch.randn(len(pasts), T, H, D, generator=g)).to(dtype)
    for b, n in enumerate(real):
        q[b, n:] = math.nan
    return cache, parents, q.transpose(1, 2), real


def _tree_want(cache, q, pasts, real, among, depths, window, sinks, scale):
    B, H, T, D = q.shape
    out, bound = torch.zeros(B, T, H, D, dtype=torch.float64), torch.zeros(B, T, H, 1, dtype=torch.float64)
    for b, n in enumerate(real):
        if n:
            see = tree_see(pasts[b], n, among[b][:n, :n], depths[b], window, sinks) & cache.held[b][None]
            out[b, :n], bound[b, :n] = attend64(q[b, :, :n], cache.k[b], cache.v[b], see, scale)
    return out, bound


def _call(cache, page, q, mask, depth, pasts, scale, **kw):
    if page:
        return ops.attn_tree_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32(pasts), mask, scale=scale,
                                   depth=depth, **kw)
    k, v = _dense(cache, max(cache.lens) + 37)
    return ops.attn_tree(q.cuda(), k.cuda(), v.cuda(), mask, scale=scale, row_pos=i32(pasts), depth=depth, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTEND, ids=_id)
def test_attn_tree(case):
    dtype, H, K, D, page, pasts, T, shape, news, window, sinks = case
    cache, parents, q, real = _tree_inputs(*case)
    mask, depth = ops.tree_mask(i32(parents))
    among = bits_to_bool(mask.cpu(), T)
    got = _call(cache, page, q, mask, depth if window else None, pasts, D ** -0.5, window=window, sinks=sinks,
                new_lens=i32(news) if news is not None else None)
    want, bound = _tree_want(cache, q, pasts, real, among, depth.tolist(), window, sinks, D ** -0.5)
    assert_close(got, want, bound)
    for b, n in enumerate(real):
        assert not got[b, n:].any()


@pytest.mark.parametrize("base, n, window, sinks", [(0, 1, 0, 0), (0, 30, 4, 2), (90, 40, 20, 5), (200, 33, 300, 4), (50, 30, 7, 60)])
def test_who_sees_whom_by_rows(base, n, window, sinks):
    parents = make_parents(random.Random(n), n, "tree")
    among = torch.tensor([[j in chain_of(parents, t) for j in range(n)] for t in range(n)])
    depth = mask_of(parents, n)[1] if window else None
    assert torch.equal(tree_see_long(base, n, among, depth, window, sinks), tree_see(base, n, among, depth, window, sinks))


# What long batches take on 256 CUs: the chunk kernel's parts planned on the device, in one round or two, with windows or not; its
# windowed calls that are not planned; the split kernel's blocks of 32 rows
LONG = [
    (BF, 16, 8, 128, 16, [9000, 200, 4100, 0, 8999, 1500, 6000, 333], 64, "tree", [64, 64, 1, 7, 64, 0, 50, 64], 0, 0),
    (BF, 16, 8, 128, 0, [9000, 5200, 7100, 800, 8999, 9000, 6000, 8333], 60, "forest", None, 0, 0),
    (BF, 16, 8, 128, 16, [1900 - 7 * i for i in range(40)], 64, "tree", [64 - i % 7 for i in range(40)], 0, 0),
    (BF, 16, 8, 128, 16, [2400 - 9 * i if i % 13 else 30 * i for i in range(40)], 64, "tree", [64 - i % 5 * 13 for i in range(40)], 1900, 4),
    (HF, 12, 4, 64, 32, [13000, 12900, 500, 0, 7000, 64, 9000, 13000], 64, "tree", [64, 3, 64, 64, 64, 64, 0, 64], 0, 0),
    (BF, 8, 1, 256, 16, [9000, 8000, 100, 7000, 8500, 5, 31, 4000] * 2, 26, "tree", None, 0, 0),
    (BF, 16, 1, 512, 64, [7000, 10, 6500, 6999], 40, "tree", [40, 40, 9, 40], 0, 0),
    (SF, 16, 8, 128, 16, [4600, 4200, 100, 3000, 4600, 17, 4500, 2000], 64, "tree", None, 0, 0),
    (BF, 8, 1, 256, 16, [5000, 700, 1030, 1100, 3000, 0, 2047, 900], 26, "tree", [26, 26, 1, 26, 0, 26, 13, 26], 1024, 4),
    (HF, 8, 2, 256, 0, [700, 5, 1030, 3000] * 3, 40, "chain", None, 300, 64),
    (HF, 8, 2, 256, 0, [700, 5, 1030, 3000] * 3, 40, "chain", None, 9, 2),
    (SF, 16, 4, 64, 16, [3000, 40, 700, 1200] * 4, 40, "tree", [40, 7, 40, 0] * 4, 250, 10),
    (BF, 16, 1, 512, 16, [900, 31, 1500], 26, "tree", None, 256, 4),
    (BF, 16, 8, 128, 16, [2000 - 97 * i for i in range(16)], 12, "tree", [12 - i % 4 for i in range(16)], 0, 0),
    (SF, 16, 8, 64, 0, [1900 - 90 * i for i in range(16)], 12, "tree", None, 0, 0),
    (HF, 16, 8, 128, 32, [3000 - 101 * i for i in range(24)], 12, "tree", None, 700, 4),
    (BF, 8, 1, 256, 16, [4300 - 100 * i for i in range(16)], 4, "forest", [4 - i % 3 for i in range(16)], 0, 0),
    (BF, 16, 8, 32, 16, [4000 - 60 * i for i in range(16)], 14, "tree", None, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", LONG, ids=lambda c: _id((*c[:5], f"{len(c[5])}x{max(c[5])}", *c[6:8], *c[9:])))
def test_attn_tree_over_long_batches(case):
    dtype, H, K, D, page, pasts, T, shape, news, window, sinks = case
    cache, parents, q, real = _tree_inputs(*case)
    mask, depth = ops.tree_mask(i32(parents))
    among, depths = bits_to_bool(mask.cpu(), T), depth.tolist()
    got = _call(cache, page, q, mask, depth if window else None, pasts, D ** -0.5, window=window, sinks=sinks,
                new_lens=i32(news) if news is not None else None)
    for b, n in enumerate(real):
        assert not got[b, n:].any()
        if n:
            see = tree_see_long(pasts[b], n, among[b][:n, :n], depths[b], window, sinks) & cache.held[b][None]
            assert_close(got[b, :n], *attend64(q[b, :, :n], cache.k[b], cache.v[b], see, D ** -0.5), f"row {b}")
    again = _call(cache, page, q, mask, depth if window else None, pasts, D ** -0.5, window=window, sinks=sinks,
                  new_lens=i32(news) if news is not None else None)
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, heads, page, T", [(BF, (16, 8, 128), 16, 40), (BF, (16, 8, 128), 0, 100), (SF, (8, 4, 32), 0, 33),
                                                   (HF, (8, 1, 256), 64, 24), (BF, (16, 1, 512), 16, 70)])
def test_any_mask(dtype, heads, page, T):
    """Masks that are no trees: later tokens, not oneself, nothing at all; rows without a cache then come out as zeros."""
    H, K, D = heads
    pasts = [0, 45]
    cache, _, q, real = _tree_inputs(dtype, H, K, D, page, pasts, T, "tree", [T, T - 3], 0, 0)
    words = -(-T // 64)
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (2, T, words), generator=gen(5))   # (bits of padding and past T are set too)
    mask[:, 5] = 0
    mask[:, T - 4] = -1
    among = bits_to_bool(mask, T)
    got = _call(cache, page, q, mask.cuda(), None, pasts, D ** -0.5, new_lens=i32(real))
    want, bound = _tree_want(cache, q, pasts, real, among, [None, None], 0, 0, D ** -0.5)
    assert not got[0, 5].any()
    assert_close(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, heads, page, T, past", [
    (BF, (16, 8, 128), 16, 12, 40), (HF, (12, 4, 64), 0, 12, 3), (SF, (8, 4, 32), 0, 12, 21), (SF, (8, 1, 256), 16, 12, 40),
    (BF, (16, 1, 512), 0, 12, 50), (BF, (16, 8, 128), 64, 64, 9000), (BF, (8, 4, 256), 0, 64, 9000), (SF, (16, 8, 128), 0, 80, 6000),
    (BF, (16, 1, 512), 32, 64, 9000), (HF, (12, 4, 64), 0, 80, 9000)])
def test_branches_do_not_see_each_others_infinities(dtype, heads, page, T, past):
    """Keys and values of one branch that are infinite or NaN reach the tokens that hang on it, and no others: those come out
    bit for bit as without them."""
    H, K, D = heads
    B = 1 if past < 1000 else 8   # (8: the chunk kernel's)
    cache, _, q, real = _tree_inputs(dtype, H, K, D, page, [past] * B, T, "tree", None, 0, 0)
    parents = [-1, 0, 0] + [1 + t % 2 for t in range(T - 3)]      # two branches: 1 and 2
    mask, depth = ops.tree_mask(i32([parents] * B))
    clean = _call(cache, page, q, mask, None, [past] * B, D ** -0.5)
    for where, value in (("v", math.nan), ("v", math.inf), ("v", -math.inf), ("k", math.nan)):
        x = cache.v if where == "v" else cache.k
        pool = cache.vp if where == "v" else cache.kp
        kept = [y.clone() for y in x], pool.clone()
        ch = slice(3, 4) if where == "v" else slice(None)
        for b in range(B):
            x[b][:, past + 2, ch] = value
            pool[cache.table[b, (past + 2) // cache.page], :, (past + 2) % cache.page, ch] = value
        got = _call(cache, page, q, mask, None, [past] * B, D ** -0.5)
        hit = torch.tensor([2 in chain_of(parents, t) for t in range(T)])
        assert torch.equal(got[:, ~hit], clean[:, ~hit]), (where, value)
        bad = got[:, hit][..., ch].float().cpu()
        assert (bad == value).all() if math.isinf(value) else bad.isnan().all(), (where, value)
        if where == "v":
            assert torch.equal(got[:, hit][..., 4:], clean[:, hit][..., 4:])
        for b in range(B):
            x[b].copy_(kept[0][b])
        pool.copy_(kept[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, heads, page", [(BF, (16, 8, 128), 16), (SF, (8, 4, 64), 0)])
def test_norm_and_rope_at_the_trees_positions(dtype, heads, page):
    H, K, D = heads
    T, pasts = 11, [37, 4]
    cache, parents, q, real = _tree_inputs(dtype, H, K, D, page, pasts, T, "tree", None, 0, 0)
    mask, depth = ops.tree_mask(i32(parents))
    cos, sin = rope_tables(D, 128, 1e4)
    at = torch.tensor(pasts)[:, None] + depth.cpu()
    gain = 1.0 + 0.1 * torch.randn(D, generator=gen(2))
    got = _call(cache, page, q, mask, None, pasts, D ** -0.5, q_weight=gain.cuda(), eps=1e-6, norm_q=True, cos=cos[at].cuda(),
                sin=sin[at].cuda())
    q64 = norm_rope64(q, gain, 1e-6, cos[at][:, None], sin[at][:, None])
    rounded = q64.to(dtype)   # (a step of the type either way is a change of q: the bound's own slack, below)
    want, bound = _tree_want(cache, rounded, pasts, real, bits_to_bool(mask.cpu(), T), [None] * 2, 0, 0, D ** -0.5)
    # The kernel rounds q once as well, from 32 bits: an element may fall to the neighbour, one step eps |q|. A score then moves by
    # at most eps a, a = scale sum |q k|, and the output by 2 eps a vmax.
    a = max(float((rounded[b].double().abs().amax(1) @ cache.k[b].double().abs().amax(0).T).max()) for b in range(2)) * D ** -0.5
    vmax = max(float(v.double().abs().max()) for v in cache.v)
    assert_close(got, want, bound + 2 * torch.finfo(dtype).eps * a * vmax)


@pytest.mark.gpu
def test_one_tree_for_all_rows_and_other_positions():
    T, B, (H, K, D) = 20, 3, (16, 8, 128)
    pasts = [50] * B
    cache, _, q, real = _tree_inputs(BF, H, K, D, 0, pasts, T, "tree", None, 0, 0)
    parents = make_parents(random.Random(9), T, "tree")
    one, d1 = ops.tree_mask(i32(parents))
    each, dB = ops.tree_mask(i32([parents] * B))
    k, v = (x.cuda() for x in _dense(cache, 100))
    a = dict(scale=D ** -0.5, window=30, sinks=2)
    want = ops.attn_tree(q.cuda(), k, v, each, row_pos=i32(pasts), depth=dB, **a)
    for where in (dict(pos=50), dict(pos_dev=torch.tensor([50], device="cuda")), dict(row_pos=i32(pasts), max_kv_len=71)):
        # (another bound may cut the sums elsewhere)
        got = ops.attn_tree(q.cuda(), k, v, one, depth=d1, **where, **a)
        assert (got.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()
    out = torch.empty_like(want)
    assert ops.attn_tree(q.cuda(), k, v, one, depth=d1, row_pos=i32(pasts), out=out, **a) is out and torch.equal(out, want)
    wide = torch.full((B, T, 5), 3, dtype=torch.int64, device="cuda")
    wide[..., 2] = each[..., 0]
    assert torch.equal(ops.attn_tree(q.cuda(), k, v, wide[..., 2:3], depth=dB, row_pos=i32(pasts), **a), want)
    # q of a width that is not aligned is copied
    odd = torch.zeros(B, T, H, D + 1, dtype=BF, device="cuda")[..., 1:]
    odd.copy_(q.transpose(1, 2))
    assert torch.equal(ops.attn_tree(odd.transpose(1, 2), k, v, each, row_pos=i32(pasts), depth=dB, **a), want)


@pytest.mark.gpu
def test_attn_tree_arguments():
    q = torch.zeros(2, 4, 6, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 2, 64, 64, dtype=BF, device="cuda")
    mask, depth = ops.tree_mask(i32([[-1, 0, 1, 2, 3, 4]] * 2))
    ok = dict(scale=0.1, pos=3)
    ops.attn_tree(q, k, k, mask, **ok)
    for bad in (dict(mask=mask[:1]), dict(mask=mask.int()), dict(mask=mask[:, :5]), dict(mask=mask.cpu()), dict(window=4),
                dict(window=4, depth=depth.long()), dict(window=4, depth=depth[:, :3]), dict(sinks=2), dict(pos=60), dict(pos=-1),
                dict(row_pos=i32([1, 2])), dict(scale=-1.0), dict(new_lens=i32([1])), dict(out=torch.zeros(2, 6, 4, 64, device="cuda")),
                dict(window=1 << 30, depth=depth)):
        a = dict(ok, mask=mask)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.attn_tree(q, k, k, **a)
    with pytest.raises(ValueError):
        ops.attn_tree(q, k.half(), k.half(), mask, **ok)
    with pytest.raises(ValueError):
        ops.attn_tree(q, k, k[:, :, :32], mask, **ok)
    with pytest.raises(ValueError):
        ops.attn_tree_paged(q, k, k, i32([[0], [1]]).long(), i32([0, 0]), mask, scale=0.1)
    with pytest.raises(ValueError):
        ops.attn_tree_paged(q, k[:, :, :24], k[:, :, :24], i32([[0], [1]]), i32([0, 0]), mask, scale=0.1)
    empty = ops.attn_tree(q[:, :, :0], k, k, mask[:, :0, :0], **ok)
    assert empty.shape == (2, 0, 4, 64)


@pytest.mark.gpu
def test_rows_outside_the_cache():
    """Positions, tables and lengths that name nothing: zeros, no access."""
    T, (H, K, D) = 9, (16, 8, 128)
    cache, parents, q, _ = _tree_inputs(BF, H, K, D, 16, [20, 20, 20], T, "tree", None, 0, 0)
    mask, depth = ops.tree_mask(i32(parents))
    table = cache.table.clone()
    table[0] = torch.tensor([-1, 2 ** 31 - 1, 999, -5][:table.shape[1]])
    got = ops.attn_tree_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), table.cuda(), i32([20, -3, 2 ** 31 - 1]), mask,
                              scale=D ** -0.5)
    assert not got.any()


# ================================================================ verification
def _verify_inputs(B, T, V, dtype, shape, probs, seed=0, spread=3.0):
    g, rng = gen(seed), random.Random(seed)
    parents = [make_parents(rng, T, shape) for _ in range(B)]
    draft = spread * torch.randn(B, T, V, generator=g)
    draft[..., torch.randint(V, (3,), generator=g)] += 2.5 * spread
    logits = (draft + 0.5 * torch.randn(B, T, V, generator=g)).to(dtype)
    q = draft.softmax(-1)
    tokens = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for t in range(1, T):
            at = max(0, parents[b][t])
            tokens[b, t] = torch.multinomial(q[b, at], 1, generator=g)[0]
    return parents, logits, q if probs else None, tokens, torch.rand(B, T, generator=g)


def _verify_want(logits, tokens, parents, u, heats, probs, news):
    B, T = tokens.shape
    out, path, count = (torch.full((B, T), -1) for _ in range(3))
    count = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        o, p = verify_row(logits[b], tokens[b].tolist(), parents[b], u[b].double().tolist() if u is not None else None, heats[b],
                          None if probs is None else probs[b], news[b])
        out[b, :len(o)], path[b, :len(p)], count[b] = torch.tensor(o, dtype=torch.int64), torch.tensor(p, dtype=torch.int64), len(p)
    return out, path, count


def _same(got, want):
    for x, y, n in zip(got, want, ("tokens", "path", "count")):
        assert x.cpu().tolist() == y.tolist(), n
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.int32 and got[2].dtype == torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("shape, T", [("chain", 1), ("chain", 6), ("tree", 20), ("star", 9), ("tree", 70), ("forest", 12)])
@pytest.mark.parametrize("V", [1, 7, 1000, 4093, 8192, 20011])
@pytest.mark.parametrize("mode", ["greedy", "sampled", "probs"])
def test_verify_drafts(dtype, shape, T, V, mode):
    if T * V > 500000:
        pytest.skip("large enough elsewhere")
    B = 5
    parents, logits, q, tokens, u = _verify_inputs(B, T, V, dtype, shape, mode == "probs", seed=V + T)
    heat = 0.0 if mode == "greedy" else 1.0 if V % 2 else 0.7
    got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(parents), uniform=None if mode == "greedy" else u.cuda(),
                            temperature=heat, draft_probs=None if q is None else q.cuda())
    _same(got, _verify_want(logits, tokens, parents, u, [heat] * B, q, [T] * B))


@pytest.mark.gpu
@pytest.mark.parametrize("probs", [False, True])
def test_verify_over_a_large_vocabulary(probs):
    parents, logits, q, tokens, u = _verify_inputs(4, 5, 151937, BF, "tree", probs, seed=1)
    got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(parents), uniform=u.cuda(), temperature=0.8,
                            draft_probs=None if q is None else q.cuda())
    _same(got, _verify_want(logits, tokens, parents, u, [0.8] * 4, q, [5] * 4))


@pytest.mark.gpu
@pytest.mark.parametrize("T, B, V, shape", [(1024, 1, 40, "tree"), (600, 2, 9, "chain"), (513, 1, 5000, "star"), (256, 2, 30, "forest")])
@pytest.mark.parametrize("mode", ["greedy", "sampled", "probs"])
def test_verify_large_trees(T, B, V, shape, mode):
    parents, logits, q, tokens, u = _verify_inputs(B, T, V, SF, shape, mode == "probs", seed=T, spread=1.0)
    heat = 0.0 if mode == "greedy" else 1.3
    got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(parents), uniform=None if mode == "greedy" else u.cuda(),
                            temperature=heat, draft_probs=None if q is None else q.cuda())
    _same(got, _verify_want(logits, tokens, parents, u, [heat] * B, q, [T] * B))


@pytest.mark.gpu
def test_verify_on_the_streams_workspace():
    """Calls of one launch and of two, of other operators on the same workspace between them, and again: its counters are zero
    each time."""
    small = _verify_inputs(2, 6, 9000, BF, "tree", True, seed=8)
    large = _verify_inputs(40, 6, 20011, BF, "tree", False, seed=9)
    case = (BF, 16, 8, 128, 16, [0, 400], 12, "tree", None, 0, 0)
    cache, parents, qs, real = _tree_inputs(*case)
    mask, _ = ops.tree_mask(i32(parents))
    first = _call(cache, 16, qs, mask, None, [0, 400], 0.1)
    for _ in range(3):
        for p, logits, q, tokens, u in (small, large):
            got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(p), uniform=u.cuda(), temperature=1.0,
                                    draft_probs=None if q is None else q.cuda())
            _same(got, _verify_want(logits, tokens, p, u, [1.0] * len(p), q, [6] * len(p)))
        assert torch.equal(_call(cache, 16, qs, mask, None, [0, 400], 0.1), first)


@pytest.mark.gpu
def test_greedy_calls_of_one_launch():
    """Greedy calls that walk in the scan's launch (few chunks: up to half the CUs) and ones just above, rows of no node, of some
    and of more than there are, one chunk a row and several, and other operators on the stream's workspace between them: each
    call leaves its counters at zero, whatever its sizes."""
    case = (BF, 16, 8, 128, 16, [0, 400], 12, "tree", None, 0, 0)
    cache, parents, qs, real = _tree_inputs(*case)
    mask, _ = ops.tree_mask(i32(parents))
    first = _call(cache, 16, qs, mask, None, [0, 400], 0.1)
    news, real = [8, 0, 1, 3, 99, -4], [8, 0, 1, 3, 8, 0]
    calls = [(6, 8, 900, BF, "tree", news, real), (6, 8, 5000, SF, "chain", news, real), (6, 8, 9000, HF, "tree", news, real),
             (2, 6, 9000, BF, "tree", None, [6] * 2), (1, 1, 4000, SF, "chain", [0], [0]), (1, 1, 4000, SF, "chain", [1], [1]),
             (1, 100, 300, HF, "tree", None, [100]), (2, 64, 3000, BF, "star", [64, 7], [64, 7]), (128, 1, 50, BF, "chain", None, [1] * 128),
             (1, 5, 32768, BF, "chain", None, [5])]
    inputs = [_verify_inputs(B, T, V, dtype, shape, False, seed=V) for B, T, V, dtype, shape, _, _ in calls]
    wants = [_verify_want(x[1], x[3], x[0], None, [0.0] * c[0], None, c[6]) for c, x in zip(calls, inputs)]
    for _ in range(3):
        for (B, T, V, dtype, shape, lens, _), (p, logits, _, tokens, _), want in zip(calls, inputs, wants):
            for _ in range(2):
                _same(ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(p), new_lens=None if lens is None else i32(lens)), want)
        assert torch.equal(_call(cache, 16, qs, mask, None, [0, 400], 0.1), first)


@pytest.mark.gpu
def test_rejected_tokens_are_taken_out_in_order():
    """A star of 459 drafts, all rejected: 458 of weight 2^-54, then one of weight 1. What is left of 3 + 2^-46 + 458 2^-54 is
    2 + 2^-46 if they are added up in their order: half of it passes the first of what stays, 1, and not 1 + 2^-46, the second.
    With the weight of 1 before others, those are lost to its rounding, half of what is left is up to 2^-45.2 more, and the third
    would be the token."""
    V, T = 1000, 460
    x = torch.full((V,), -math.inf)
    x[[10, 20, 900]] = 0.0
    x[11] = -46 * math.log(2)
    x[100:558] = -54 * math.log(2)
    tokens = torch.tensor([[0, *range(100, 558), 20]])
    logits = x.expand(1, T, V).cuda()
    u = torch.full((1, T), 0.9)
    u[0, 0] = 0.5
    args = logits, tokens.cuda()
    kw = dict(parents=i32([[-1] + [0] * (T - 1)]), uniform=u.cuda(), temperature=1.0)
    for _ in range(50):
        out, path, count = ops.verify_drafts(*args, **kw)
        assert (out[0, 0].item(), count.item()) == (11, 1)


@pytest.mark.gpu
def test_verify_forms():
    """A chain by default, one tree for all, a temperature for each row, short rows, probabilities of 16 bits and of T - 1 nodes,
    strided logits."""
    B, T, V = 6, 8, 515
    _, logits, q, tokens, u = _verify_inputs(B, T, V, BF, "chain", True, seed=4)
    chain = [[t - 1 for t in range(T)]] * B
    news = [T, 0, 1, 3, 99, -4]
    real = [T, 0, 1, 3, T, 0]
    temps = [1.0, 0.5, 0.0, -1.0, math.nan, 2.0]
    heats = torch.tensor(temps, device="cuda")
    a = dict(uniform=u.cuda(), temperature=heats, new_lens=i32(news))
    want = _verify_want(logits, tokens, chain, u, temps, None, real)
    _same(ops.verify_drafts(logits.cuda(), tokens.cuda(), **a), want)
    _same(ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(chain[0]), **a), want)
    wide = torch.zeros(B, T + 2, V + 9, dtype=BF, device="cuda")
    wide[:, 1:T + 1, 5:V + 5] = logits.cuda()
    _same(ops.verify_drafts(wide[:, 1:T + 1, 5:V + 5], tokens.cuda(), **a), want)
    flip = logits.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    _same(ops.verify_drafts(flip, tokens.cuda(), **a), want)
    heats = [1.0, 0.9, 0.8, 0.7, 0.6, 1.5]
    q16 = q.to(BF)
    want = _verify_want(logits, tokens, chain, u, torch.tensor(heats).double().tolist(), q16, real)
    a = dict(uniform=u.cuda(), temperature=torch.tensor(heats, device="cuda"), new_lens=i32(news))
    _same(ops.verify_drafts(logits.cuda(), tokens.cuda(), draft_probs=q16.cuda(), **a), want)
    _same(ops.verify_drafts(logits.cuda(), tokens.cuda(), draft_probs=q16[:, :T - 1].cuda(), **a), want)
    out, path, count = ops.verify_drafts(logits[:0].cuda(), tokens[:0].cuda())
    assert out.shape == (0, T) and count.shape == (0,)


@pytest.mark.gpu
def test_verify_extremes():
    """Infinities and NaN among logits, ties, random numbers at the ends, tokens and parents that are none, siblings alike."""
    inf, nan = math.inf, math.nan
    V = 5000
    base = torch.zeros(V)
    rows = []
    rows.append(torch.full((V,), -inf))                                      # nothing
    rows.append(torch.full((V,), nan))
    x = base.clone(); x[[17, 4500]] = inf; rows.append(x)                    # two share the mass
    x = torch.full((V,), -inf); x[4999] = -3.0; rows.append(x)               # one
    x = torch.full((V,), -inf); x[[0, 4096]] = 1.0; x[2] = nan; rows.append(x)
    rows.append(base)                                                        # all alike: sums are whole numbers
    x = base.clone(); x[4095] = 3e38; rows.append(x)
    x = torch.linspace(-80, 80, V); rows.append(x)
    top = 1.0 - 2.0 ** -24
    for draft in (0, 17, 4095, 4096, 4500, 4999, -1, V, 2 ** 40):
        for u0 in (0.0, 0.5, top):
            for u1 in (0.0, 0.3, top):
                B = len(rows)
                logits = torch.stack([torch.stack([r, r, r, r]) for r in rows])
                tokens = torch.tensor([[7, draft, draft, 4096]] * B)
                parents = [[-1, 0, 0, 1]] * B
                u = torch.tensor([[u0, u1, u1, u1]] * B)
                for heat in (0.0, 1.0, 0.01):
                    got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(parents), uniform=u.cuda(), temperature=heat)
                    _same(got, _verify_want(logits, tokens, parents, u, [heat] * B, None, [4] * B))


@pytest.mark.gpu
def test_verify_residuals_that_are_nothing():
    """A drafter that is the target leaves nothing behind a rejection that rounding alone can bring; one that gave a token no
    probability, or all of it; zero and huge probabilities."""
    V, T = 9000, 3
    logits = torch.full((4, T, V), -math.inf)
    logits[..., :2] = 0.0
    q = torch.zeros(4, T, V)
    q[0, :, :2] = 0.5          # the target's own
    q[1, :, 0] = 1.0           # token 1 is never drawn
    q[2] = 0.0                 # nothing is
    q[3] = 1e30                # everything is taken
    tokens = torch.tensor([[0, 0, 1]] * 4)
    parents = [[-1, 0, 0]] * 4
    for us in ([0.6, 0.9, 0.9], [0.1, 0.0, 0.0], [0.5, 0.5, 0.5], [0.99, 1 - 2.0 ** -24, 1 - 2.0 ** -24]):
        u = torch.tensor([us] * 4)
        got = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32(parents), uniform=u.cuda(), temperature=1.0,
                                draft_probs=q.cuda())
        _same(got, _verify_want(logits, tokens, parents, u, [1.0] * 4, q, [T] * 4))


@pytest.mark.gpu
def test_verify_keeps_the_distribution():
    """20,000 rows of one drafted pair each: how often each token comes out, against the target's probabilities. A count is
    binomial; of 2 x 12 the chance that one is six standard deviations off is below 1e-7."""
    B, V = 20000, 12
    g = gen(11)
    p, q = (1.5 * torch.randn(V, generator=g)), (1.5 * torch.randn(V, generator=g)).softmax(-1)
    logits = p.expand(B, 3, V).contiguous()
    for probs in (False, True):
        tokens = torch.zeros(B, 3, dtype=torch.int64)
        if probs:
            tokens[:, 1:] = torch.multinomial(q, 2 * B, replacement=True, generator=g).view(B, 2)
        else:
            tokens[:, 1:] = q.topk(2).indices
        out, _, _ = ops.verify_drafts(logits.cuda(), tokens.cuda(), parents=i32([-1, 0, 0]), uniform=torch.rand(B, 3, generator=g).cuda(),
                                      temperature=1.0, draft_probs=q.expand(B, 3, V).contiguous().cuda() if probs else None)
        seen = torch.bincount(out[:, 0].cpu(), minlength=V).double()
        want = p.double().softmax(-1)
        assert ((seen - B * want).abs() <= 6 * (B * want * (1 - want)).sqrt()).all(), probs


@pytest.mark.gpu
def test_verify_arguments():
    x = torch.zeros(2, 4, 100, device="cuda")
    t = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    u = torch.zeros(2, 4, device="cuda")
    ops.verify_drafts(x, t)
    ops.verify_drafts(x, t, temperature=1, uniform=u)   # (a whole number is a number)
    for bad in (dict(tokens=t.int()), dict(tokens=t[:, :3]), dict(parents=t), dict(parents=i32([0, 1, 2])), dict(temperature=1.0),
                dict(temperature=-1.0, uniform=u), dict(temperature=math.inf, uniform=u), dict(temperature=math.nan, uniform=u),
                dict(temperature=torch.ones(3, device="cuda"), uniform=u), dict(temperature=torch.ones(2), uniform=u),
                dict(temperature=1.0, uniform=u.double()), dict(temperature=1.0, uniform=u[:, :2]), dict(new_lens=i32([1])),
                dict(draft_probs=x[:, :2]), dict(draft_probs=x.half()), dict(draft_probs=x[..., :5]), dict(logits=x[0]),
                dict(logits=x.long()), dict(logits=x[:, :, :0]), dict(tokens=t.cpu())):
        a = dict(logits=x, tokens=t)
        a.update(bad)
        with pytest.raises((ValueError, TypeError)):
            ops.verify_drafts(**a)


# ================================================================ moves
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, shapes, page, T", [
    (BF, [(8, 128)] * 3, 0, 12), (BF, [(8, 128)] * 3, 16, 26), (SF, [(4, 32)], 16, 9), (HF, [(4, 64)] * 70, 32, 5),
    (BF, [(2, 256), (4, 64), (2, 256)], 16, 40), (SF, [(1, 256)], 0, 64), (BF, [(1, 512)] * 2, 64, 8), (BF, [(3, 8)], 0, 20)])
def test_kv_compact(dtype, shapes, page, T):
    rng, g = random.Random(T), gen(T)
    pasts = [0, 1, 15, 16, 40, 7]
    B = len(pasts)
    paths = []
    for b in range(B):
        parents = make_parents(rng, T, rng.choice(["tree", "chain", "star"]))
        paths.append(chain_of(parents, rng.randrange(T))[::-1])
    paths[4] = list(range(T))                              # nothing to move
    paths[5] = [0, 0, T + 500, 5, 2 ** 31 - 1, -3][:T]     # entries that move nothing, and one that does
    counts = [len(p) for p in paths]
    counts[3] = 0
    path = torch.full((B, T), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    counts_dev = list(counts)
    counts_dev[4] = T + 7                                  # (taken as T)
    cap = max(pasts) + T + 3
    if page:
        caches = [Paged(g, [p + T for p in pasts], K, D, page, dtype) for K, D in shapes]
        for c in caches:
            c.table = caches[0].table
        pools = [(torch.randn(c.kp.shape, generator=g).to(dtype), torch.randn(c.vp.shape, generator=g).to(dtype)) for c in caches]
        table = caches[0].table.clone()
        table[2, (pasts[2] + 2) // page] = -1              # a page that is not there
        n_pages = min(k.shape[0] for k, _ in pools)
        pools = [(k[:n_pages].clone(), v[:n_pages].clone()) for k, v in pools]

        def rows(pool, b):
            ids = table[b].long()
            x = pool[ids.clamp(min=0)].transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])
            return x

        want = []
        for k, v in pools:
            ys = []
            for x in (k, v):
                y = x.clone()
                for b, p in enumerate(pasts):
                    held = lambda s: s // page < table.shape[1] and table[b, s // page] >= 0
                    new = compact_row(rows(x, b), p, paths[b][:counts[b]], table.shape[1] * page, held)
                    for j, i in enumerate(table[b].tolist()):
                        if i >= 0:
                            y[i] = new[:, j * page:(j + 1) * page]
                ys.append(y)
            want.append(ys)
        ks, vs = [k.cuda() for k, _ in pools], [v.cuda() for _, v in pools]
        ops.kv_compact_paged(ks, vs, table.cuda(), i32(pasts), path.cuda(), i32(counts_dev))
    else:
        data = [(torch.randn(B, K, cap, D, generator=g).to(dtype), torch.randn(B, K, cap, D, generator=g).to(dtype)) for K, D in shapes]
        want = [[torch.stack([compact_row(x[b], p, paths[b][:counts[b]], cap) for b, p in enumerate(pasts)]) for x in kv] for kv in data]
        ks, vs = [k.cuda() for k, _ in data], [v.cuda() for _, v in data]
        ops.kv_compact(ks, vs, path.cuda(), i32(counts_dev), row_pos=i32(pasts))
    for l, (k, v) in enumerate(zip(ks, vs)):
        assert torch.equal(k.cpu(), want[l][0]) and torch.equal(v.cpu(), want[l][1]), l


@pytest.mark.gpu
def test_kv_compact_positions_and_arguments():
    x = torch.randn(2, 4, 50, 32, generator=gen(0)).cuda()
    path, count = i32([[0, 2, 5], [0, 1, 4]]), i32([3, 3])
    want = torch.stack([compact_row(x[b].cpu(), 30, path[b].tolist(), 50) for b in range(2)]).cuda()
    for where in (dict(pos=30), dict(pos_dev=torch.tensor([30], device="cuda")), dict(row_pos=i32([30, 30]))):
        k, v = x.clone(), x.clone()
        ops.kv_compact([k], [v], path, count, **where)
        assert torch.equal(k, want) and torch.equal(v, want)
    k = x.clone()
    ops.kv_compact([k], [k.clone()], path, count, pos=2 ** 40)      # beyond the cache: nothing
    ops.kv_compact((k,), (k.clone(),), path, count, row_pos=i32([-1, 2 ** 31 - 1]))
    ops.kv_compact([], [], path, count, pos=0)
    ops.kv_compact([k], [k.clone()], path[:, :0], count, pos=0)
    assert torch.equal(k, x)
    big = torch.zeros(2, 8, 50, 64, device="cuda")[:, ::2, :, :32]   # strided heads and positions
    big.copy_(x)
    ops.kv_compact([big], [torch.zeros(2, 8, 50, 64, device="cuda")[:, ::2, :, :32]], path, count, pos=30)   # (of its strides)
    assert torch.equal(big, want)
    for bad in (dict(v_caches=[]), dict(k_caches=[x[0]]), dict(path=path.long()), dict(path=path[:1]), dict(count=count.long()),
                dict(pos=0, row_pos=i32([0, 0])), dict(pos=-1), dict(v_caches=[x.half()]), dict(k_caches=[x.cpu()]),
                dict(k_caches=[x[..., 1:]], v_caches=[x[..., 1:]]), dict(k_caches=[x.double()], v_caches=[x.double()]),
                dict(k_caches=[x, x[:, :, :20]], v_caches=[x, x[:, :, :20]])):
        a = dict(k_caches=[k], v_caches=[x], path=path, count=count)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.kv_compact(**a)


@pytest.mark.gpu
def test_a_cache_named_twice_stays_as_it_is():
    x, y = (torch.randn(2, 4, 48, 32, generator=gen(i)).cuda() for i in range(2))
    path, count = i32([[0, 2, 5], [0, 1, 4]]), i32([3, 3])
    table = i32([[0], [1]])
    pool = [t[:, :, :32].contiguous() for t in (x, y)]
    before = [t.clone() for t in (x, y, *pool)]
    for ks, vs in (([x], [x]), ([x, x], [y, y.clone()]), ([x, y], [y, x]), ([x, x[:, :2]], [y, y[:, :2]])):
        with pytest.raises(ValueError, match="twice"):
            ops.kv_compact(ks, vs, path, count, pos=10)
    with pytest.raises(ValueError, match="twice"):
        ops.kv_compact_paged([pool[0]] * 2, [pool[1]] * 2, table, i32([10, 10]), path, count)
    assert all(torch.equal(a, b) for a, b in zip(before, (x, y, *pool)))


@pytest.mark.gpu
def test_page_lists_are_not_recorded():
    kp, vp = torch.zeros(4, 2, 16, 32, device="cuda"), torch.ones(4, 2, 16, 32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="recording"):
            ops.copy_pages([kp], [vp], [0], [1])
        out = kp + 1
    g.replay()
    assert torch.equal(out, kp + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, shapes, page, n", [(BF, [(8, 128)] * 3, 16, 1), (SF, [(4, 32)], 32, 7), (HF, [(2, 256), (4, 64)], 64, 3),
                                                    (BF, [(1, 512)] * 70, 16, 2), (BF, [(3, 8)], 128, 5)])
def test_copy_pages(dtype, shapes, page, n):
    g = gen(n)
    pools = 2 * n + 3
    ids = torch.randperm(pools, generator=g).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    src[-1] = src[0]                                          # one page may be copied twice
    ks = [torch.randn(pools, K, page, D, generator=g).to(dtype).cuda() for K, D in shapes]
    vs = [torch.randn(pools, K, page, D, generator=g).to(dtype).cuda() for K, D in shapes]
    want = [[x.clone() for x in xs] for xs in (ks, vs)]
    for xs in want:
        for x in xs:
            x[dst] = x[src].clone()
    for form in ("list", "tensor"):
        k2, v2 = [x.clone() for x in ks], [x.clone() for x in vs]
        if form == "list":
            ops.copy_pages(k2, v2, src, dst)
        else:   # what names no page copies nothing
            ops.copy_pages(k2, v2, i32(src + [-1, pools, 0, 2 ** 31 - 1, 1]), i32(dst + [0, 1, -9, 2, 1]))
        assert all(torch.equal(a, b) for a, b in zip(k2 + v2, want[0] + want[1])), form


@pytest.mark.gpu
def test_copy_pages_arguments():
    x = torch.zeros(6, 2, 16, 32, device="cuda")
    strided = torch.randn(6, 16, 4, 32, generator=gen(0)).cuda().transpose(1, 2)[:, ::2]
    want = strided.clone()
    want[3] = want[1]
    ops.copy_pages([strided], [torch.zeros(6, 16, 4, 32, device="cuda").transpose(1, 2)[:, ::2]], [1], [3])   # (of its strides)
    assert torch.equal(strided, want)
    ops.copy_pages([x], [x], [], [])
    for src, dst in (([0], [6]), ([-1], [0]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]), (i32([0]), [1]),
                     (i32([0]), i32([1, 2])), (i32([0]).long(), i32([1]).long()), (i32([0], "cpu"), i32([1], "cpu"))):
        with pytest.raises(ValueError):
            ops.copy_pages([x], [x.clone()], src, dst)
    with pytest.raises(ValueError):
        ops.copy_pages([x[:, :, :12]], [x[:, :, :12]], [0], [1])


# ================================================================ together
def _step(s):
    """A verify step of a drafted tree: the mask, one layer's cache write and attention, verification, the accepted branch closes
    up."""
    mask, depth = ops.tree_mask(s["parents"])
    at = s["row_pos"][:, None] + depth
    cos, sin = s["cos"][at], s["sin"][at]
    ops.kv_append_paged(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["row_pos"], cos=cos, sin=sin)
    y = ops.attn_tree_paged(s["q"], s["kp"], s["vp"], s["table"], s["row_pos"], mask, scale=0.1, depth=depth, window=40, sinks=2,
                            cos=cos, sin=sin)
    logits = y.flatten(2) @ s["w"]
    out = ops.verify_drafts(logits, s["tokens"], parents=s["parents"], uniform=s["u"], temperature=0.9)
    ops.kv_compact_paged([s["kp"]], [s["vp"]], s["table"], s["row_pos"], out[1], out[2])
    return y, *out


def _step_inputs(seed):
    g, rng = gen(seed), random.Random(seed)
    B, T, H, K, D = 3, 14, 16, 8, 128
    pasts = [rng.randrange(5, 60) for _ in range(B)]
    cache = Paged(g, [p + T for p in pasts], K, D, 16, BF, poison=False, extra=0)
    full = torch.full((B, 6), -1, dtype=torch.int32)
    full[:, :cache.table.shape[1]] = cache.table
    pool = torch.zeros(24, K, 16, D, dtype=BF)
    kp, vp = pool.clone(), pool.clone()
    kp[:cache.kp.shape[0]], vp[:cache.vp.shape[0]] = cache.kp, cache.vp
    cos, sin = rope_tables(D, 256, 1e4)
    rn = lambda *n: torch.randn(*n, generator=g).to(BF)
    s = dict(parents=i32([make_parents(rng, T, "tree") for _ in range(B)]), row_pos=i32(pasts), k=rn(B, K, T, D), v=rn(B, K, T, D),
             q=rn(B, H, T, D), kp=kp, vp=vp, table=full, w=0.1 * rn(H * D, 300), tokens=torch.randint(300, (B, T), generator=g),
             u=torch.rand(B, T, generator=g), cos=cos, sin=sin)
    return {n: x.cuda() for n, x in s.items()}


@pytest.mark.gpu
def test_a_whole_step_recorded_and_replayed():
    """The operators together, eagerly, on another stream, and recorded: replays see other trees, positions, tables and data."""
    live = _step_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step({n: x.clone() for n, x in live.items()})
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = _step(live)
    for seed in (1, 2, 3, 2, 4):
        fresh = _step_inputs(seed)
        eager = {n: x.clone() for n, x in fresh.items()}
        want = [x.clone() for x in _step(eager)]
        for n, x in fresh.items():
            live[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        # (a recorded call may cut its sums elsewhere: its bound is the table's; whole numbers must agree all the same here)
        assert torch.equal(recorded[1], want[1]) and torch.equal(recorded[2], want[2]) and torch.equal(recorded[3], want[3])
        assert torch.equal(recorded[0], want[0])
        assert torch.equal(live["kp"], eager["kp"]) and torch.equal(live["vp"], eager["vp"])
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            again = _step({n: x.clone() for n, x in fresh.items()})
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.gpu
def test_a_chain_is_what_attn_paged_sees():
    """A tree that is a chain: the same visibility as attn_paged, within both bounds; and the same call twice gives the same bits."""
    case = (BF, 16, 8, 128, 16, [700, 31], 40, "chain", None, 100, 5)
    cache, parents, q, real = _tree_inputs(*case)
    mask, depth = ops.tree_mask(i32(parents))
    a = dict(scale=128 ** -0.5, window=100, sinks=5)
    got = _call(cache, 16, q, mask, depth, [700, 31], a["scale"], window=100, sinks=5)
    paged = ops.attn_paged(q.cuda(), cache.kp.cuda(), cache.vp.cuda(), cache.table.cuda(), i32([700, 31]), **a)
    want, bound = cache.want(q, [700, 31], real, 100, 5, a["scale"])
    assert_close(got, want, bound)
    assert_close(paged, want, bound)
    assert torch.equal(got, _call(cache, 16, q, mask, depth, [700, 31], a["scale"], window=100, sinks=5))
