"""Helpers of the paged-cache tests: ragged batches over a scrambled page pool whose unused slots hold
NaN, and the operators' definitions in 64 bits on the CPU."""
import math

import torch

from oracle import kvcodec


class Ragged:
    """A pool, a batch over it and the values its positions stand for.

    ``lens[b]`` own positions, ``news[b]`` new tokens, ``prefix`` shared positions, ``pad`` token rows
    behind the last sequence.  ``self.own[b]`` / ``self.pre``: (K, V) float64 ``[positions, KV, D]``."""

    def __init__(self, lens, news, KV=2, G=4, D=128, page=16, mode="f16", prefix=0, pad=0, seed=0, cu=None, vscale=1.0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lens, self.news, self.KV, self.G, self.H, self.D = lens, news, KV, G, KV * G, D
        self.page, self.mode, self.prefix, self.pad = page, mode, prefix, pad
        B = len(lens)
        counts = [-(-n // page) for n in lens]
        npre = -(-prefix // page)
        self.pages = pages = sum(counts) + npre + 2
        ids = torch.randperm(pages, generator=g, dtype=torch.int64).tolist()
        width = max(counts + [1]) + 1
        self.table = torch.full((B, width), -7, dtype=torch.int32)  # unused entries: no page at all
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        self.prefix_pages = torch.tensor(ids[at:at + npre], dtype=torch.int32)
        self.cu = [0]
        for n in news:
            self.cu.append(self.cu[-1] + n)
        self.T = self.cu[-1] + pad
        raw = [torch.randn((pages, page, KV, D), generator=g) * s for s in (1.0, vscale)]
        self.data, self.scales, self.values = [], [], []
        used = torch.zeros(pages * page, dtype=torch.bool)
        for b, n in enumerate(lens):
            used[self.rows(b, n)] = True
        if prefix:
            used[self.prefix_rows()] = True
        for x in raw:
            enc, sc = kvcodec.encode(mode, x.numpy())
            val = torch.from_numpy(kvcodec.decode(mode, enc, sc)).double().view(pages * page, KV, D)
            if mode == "q8":  # the reference decode in 64 bits
                val = (torch.from_numpy(enc).double() / 127).clamp(min=-1).view(pages * page, KV, D // 32, 32)
                val = (val * torch.from_numpy(sc).double().view(pages * page, KV, D // 32, 1)).view(pages * page, KV, D)
            enc = torch.from_numpy(enc).reshape(pages * page, KV, D).clone()
            sc = torch.from_numpy(sc).reshape(pages * page, KV, D // 32).clone() if sc is not None else None
            if mode == "q8":
                sc[~used] = math.nan
            else:
                enc[~used] = math.nan
            self.data.append(enc.view(pages, page, KV, D))
            self.scales.append(sc.view(pages, page, KV, D // 32) if sc is not None else None)
            self.values.append(val)

    def rows(self, b, n):
        j = torch.arange(n)
        return self.table[b].long()[j // self.page] * self.page + j % self.page

    def prefix_rows(self):
        j = torch.arange(self.prefix)
        return self.prefix_pages.long()[j // self.page] * self.page + j % self.page

    def kv(self, b):
        """float64 K, V ``[prefix + lens[b], KV, D]``."""
        r = self.rows(b, self.lens[b])
        if self.prefix:
            r = torch.cat([self.prefix_rows(), r])
        return self.values[0][r], self.values[1][r]

    def cache(self, ops):
        dev = [t.cuda() if t is not None else None for t in (*self.data, *self.scales)]
        return ops.PagedKVCache.from_tensors(*dev)

    def batch(self, ops, max_q=None):
        cu = torch.tensor(self.cu, dtype=torch.int32).cuda()
        one = max(self.news) == 1 == min(self.news) and not self.pad
        return ops.PagedBatch(self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                              cu_q=None if one else cu, tokens=self.T, max_q=max_q or max(self.news + [1]),
                              prefix_pages=self.prefix_pages.cuda() if self.prefix else None, prefix_len=self.prefix)

    def queries(self, dtype, scale=1.5):
        return (torch.randn((self.T, self.H, self.D), generator=self.g) * scale).to(dtype)

    def attention(self, q, gate=None, scale=None):
        """(out, A, S): the result, sum p |v| x gate (what errors of p scale with) and the largest
        sum |q k| x scale of any score (what errors of a score scale with), all in 64 bits."""
        sc = scale or self.D ** -0.5
        out = torch.zeros(self.T, self.H, self.D, dtype=torch.float64)
        A, S = torch.zeros_like(out), 0.0
        for b, (L, n) in enumerate(zip(self.lens, self.news)):
            K, V = self.kv(b)
            for i in range(n):
                t = self.cu[b] + i
                m = self.prefix + max(0, L - n + i + 1)
                if m == 0:
                    continue
                qq = q[t].double().view(self.KV, self.G, self.D)
                s = torch.einsum("kgd,jkd->kgj", qq, K[:m]) * sc
                S = max(S, float(torch.einsum("kgd,jkd->kgj", qq.abs(), K[:m].abs()).max()) * sc)
                p = torch.softmax(s, -1)
                out[t] = torch.einsum("kgj,jkd->kgd", p, V[:m]).reshape(self.H, self.D)
                A[t] = torch.einsum("kgj,jkd->kgd", p, V[:m].abs()).reshape(self.H, self.D)
        if gate is not None:
            f = torch.sigmoid(gate.double())
            out, A = out * f, A * f
        return out, A, S


def tolerance(out, A, S, q_f16, out_f16):
    """Largest error of each output value.

    A score is a sum of up to 24 accumulated f32 terms (2^-24 each of at most S) of operands kept to
    2^-22: 28 * 2^-24 * S in all, and p carries it as a relative error; exp2, the sums of p and the
    rounding of the last division add 16 * 2^-24.  f16 rows: p may be rounded to f16 (2^-11) before
    the product with V, and the result is (2^-11, or half the smallest f16 step)."""
    tol = (28 * S + 16) * 2.0 ** -24 * A
    if q_f16 and out_f16:
        tol = tol + 2.0 ** -11 * A
    if out_f16:
        tol = tol + 2.0 ** -11 * out.abs() + 2.0 ** -25
    return tol


def check_attention(got, want, q_f16, what=""):
    out, A, S = want
    err = (got.double().cpu() - out).abs()
    tol = tolerance(out, A, S, q_f16, got.dtype == torch.float16)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = float((err / (tol + 1e-300)).max())
    assert (err <= tol).all(), f"{what}: error {float(err.max()):.3g}, {worst:.3g} of what is allowed"


def norm_rope(x, gamma, cos, sin, pos, eps):
    """RMSNorm and rotation of ``x [T, heads, D]`` in 64 bits."""
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gamma.double()
    if cos is None:
        return y
    r = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a = y[..., :r]
    h = torch.cat([-a[..., r // 2:], a[..., :r // 2]], -1)
    return torch.cat([a * c + h * s, y[..., r:]], -1)
