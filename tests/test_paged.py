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
