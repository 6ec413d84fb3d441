"""Plain 64-bit forms of the paged cache write and of attention with windows and first tokens, and the error
bounds that their fp32-accumulating, one-rounding kernels are held to."""

from __future__ import annotations

import math

import torch


def norm_rope64(x, gain, eps, cos, sin):
    """x [..., T, D] -> RMSNorm (gain or None; eps None: no norm) and NEOX RoPE (cos/sin [..., T, D] or None), 64 bits."""
    x = x.double()
    if eps is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        if gain is not None:
            x = x * gain.double()
    if cos is not None:
        h = x.shape[-1] // 2
        x = x * cos.double() + torch.cat([-x[..., h:], x[..., :h]], -1) * sin.double()
    return x


def visible(qpos, keys, window, sinks):
    """[T, S] bool: which positions `keys` the queries at `qpos` see."""
    see = keys[None] <= qpos[:, None]
    if window:
        see &= (keys[None] > qpos[:, None] - window) | (keys[None] < sinks)
    return see


def attend64(q, k, v, see, scale):
    """q [H, T, D], k/v [K, S, D], see [T, S] -> (out [T, H, D], bound [T, H, 1] without the output's rounding), 64
    bits. Rows that see nothing: zeros. Keys nobody sees may hold anything (NaN too): they are left out.

    The bound on a kernel's error before its last rounding, in units of the largest visible |v|:
      - a weight exp2(c s - m): s is a sum of D products (error at most (D + 2) u a, u = 2^-24, a = scale sum |q k|), the
        exponent one fma (u |x|), exp2 a few steps: relative error e = 2 (D + 4) u a + 8 u, and the quotient has it twice;
      - sums of n weights and products: n u each, twice;
      - 16-bit weights for the second product: half a step of the type, h (also where the sum takes the rounded
        weights: the error is then sum w d (v - out), |d| <= h, and sum w |v - out| is at most the largest |v|); in fp16 2^-25 more per key below its range."""
    H, T, D = q.shape
    G = H // k.shape[0]
    keep = see.any(0)
    k, v, see = k[:, keep].double(), v[:, keep].double(), see[:, keep]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    bound = torch.zeros(T, H, 1, dtype=torch.float64)
    u, n = 2.0 ** -24, int(keep.sum())
    if n == 0:
        return out, bound
    h = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2
    under = n * 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    for i in range(H):
        kk, vv, qq = k[i // G], v[i // G], q[i].double()
        s = (qq @ kk.T) * scale
        a = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~see, 0).amax(-1)
        w = s.masked_fill(~see, -math.inf).softmax(-1).nan_to_num(0.0)   # (a row that sees nothing)
        out[:, i] = w @ vv
        vmax = torch.stack([vv.abs().amax(-1).masked_fill(~see[t], 0).max() for t in range(T)])
        e = 2 * (D + 4) * u * a + 8 * u
        bound[:, i, 0] = vmax * (2 * e + 2 * n * u + h + under)
    return out, bound


def assert_close(got, want, bound, what=""):
    """Every element within its bound and half a step of the output's type."""
    got64 = got.detach().cpu().double()
    assert torch.isfinite(got64).all(), f"{what}: not finite"
    tiny = torch.finfo(got.dtype).smallest_normal
    limit = bound + want.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 1e-3) + tiny
    bad = (got64 - want).abs() > limit
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {at}: got {got64[at]}, want "
                             f"{want[at]}, limit {limit[at]}")


class Paged:
    """A paged cache with its dense twin on the CPU: rows of `lens` keys, pages scattered over the pool, NaN in every
    slot and page that holds no key. `freed(b, page_index)` pages are given back (-1, invisible)."""

    def __init__(self, g, lens, K, D, page, dtype, spare=3, extra=2, freed=lambda b, j: False, poison=True):
        self.lens, self.page = lens, page
        B, top = len(lens), max(max(lens), 1)
        self.k = [1.3 * torch.randn(K, n, D, generator=g).to(dtype) for n in lens]
        self.v = [torch.randn(K, n, D, generator=g).to(dtype) for n in lens]
        self.k = [x.to(dtype) for x in self.k]
        held = [[j for j in range(-(-n // page)) if not freed(b, j)] for b, n in enumerate(lens)]
        pool = sum(map(len, held)) + spare
        ids = torch.randperm(pool, generator=g).tolist()
        self.table = torch.full((B, -(-top // page) + extra), -1, dtype=torch.int32)
        fill = math.nan if poison else 0.0
        self.kp = torch.full((pool, K, page, D), fill, dtype=dtype)
        self.vp = torch.full((pool, K, page, D), fill, dtype=dtype)
        self.held = [torch.zeros(n, dtype=torch.bool) for n in lens]
        for b, pages in enumerate(held):
            for j in pages:
                i = ids.pop()
                self.table[b, j] = i
                lo, hi = j * page, min(lens[b], (j + 1) * page)
                self.kp[i, :, :hi - lo] = self.k[b][:, lo:hi]
                self.vp[i, :, :hi - lo] = self.v[b][:, lo:hi]
                self.held[b][lo:hi] = True

    def want(self, q, pasts, news, window, sinks, scale):
        """(out, bound) [B, T, H, D] of attn_paged on q [B, H, T, D] (as the kernel takes it: of the cache's type)."""
        B, H, T, D = q.shape
        out = torch.zeros(B, T, H, D, dtype=torch.float64)
        bound = torch.zeros(B, T, H, 1, dtype=torch.float64)
        for b in range(B):
            n = news[b]
            if not n:
                continue
            qpos = torch.arange(pasts[b], pasts[b] + n)
            see = visible(qpos, torch.arange(self.lens[b]), window, sinks) & self.held[b][None]
            out[b, :n], bound[b, :n] = attend64(q[b, :, :n], self.k[b], self.v[b], see, scale)
        return out, bound
