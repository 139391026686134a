"""Paged attention over the whole range of its values, through each of its kernels: small, large and mixed
q8 block scales, every q8 code, small and large f32 queries, gates, lengths beyond the page table, long runs
of one accumulator.  Definitions in 64 bits and tolerances: tests/paged_util.py."""
import math

import pytest
import torch

from paged_util import Ragged, tolerance
from test_gpu_paged_attention import DT, ops  # noqa: F401  (a fixture)
from test_gpu_paged_matrix import wide

pytestmark = pytest.mark.gpu

# rows of a unit decide the kernel's form: 4, 8 or 16 rows of the decode kernel, a tile of the tcgen05 kernel; "cuda"
# is the CUDA-core kernel
KERNELS = {"cuda": (4, [1, 3, 1]), "decode4": (4, [1, 1, 1]), "decode8": (6, [1, 1, 1]), "decode16": (4, [3, 2, 4]),
           "tc": (4, [40, 1, 70])}
each_kernel = pytest.mark.parametrize("kernel", list(KERNELS))


def make(kernel, mode="q8", D=128, lens=(700, 64, 130), seed=1, **kw):
    G, news = KERNELS[kernel]
    r = Ragged(list(lens), news, KV=2, G=G, D=D, mode=mode, seed=seed, **kw)
    return wide(r) if kernel == "tc" else r


def rescale(r, which, factor):
    """Multiply the block scales of K (0) or V (1) by ``factor`` (broadcast to [slots, KV, D / 32])."""
    sc = r.scales[which]
    sc.copy_((sc.double().view(-1, r.KV, r.D // 32) * factor).float().view(sc.shape))
    revalue(r)


def revalue(r):
    """What codes and scales stand for, in 64 bits."""
    for i in range(2):
        v = (r.data[i].double() / 127).clamp(min=-1).view(-1, r.KV, r.D // 32, 32)
        r.values[i] = (v * r.scales[i].double().view(-1, r.KV, r.D // 32, 1)).view(-1, r.KV, r.D)


def attend(ops, kernel, r, q, out_dtype, **kw):  # noqa: F811
    from bitgpu_b200._lib import lib
    lib().bg_force_generic(int(kernel == "cuda"))
    try:
        out = ops.paged_attention(q.cuda(), r.cache(ops), r.batch(ops), out_dtype=out_dtype, **kw)
    finally:
        lib().bg_force_generic(0)
    assert lib().bg_device_status(None) == 0
    return out.cpu()


def check(r, got, want, q_dtype, extra=0.0):
    """Beside ``tolerance``: weights enter the products as f16 halves at least 2^6 times as large as
    exp(score - largest score), so a weight may be off by 2^-31 of the largest (the smallest f16 step is 2^-24):
    2^-31 * sum |v| of a result."""
    out, A, S = want
    lost = torch.zeros_like(out)
    for b, n in enumerate(r.news):
        v = r.kv(b)[1].abs().nan_to_num(0).sum(0).repeat_interleave(r.G, 0)
        lost[r.cu[b]:r.cu[b] + n] = 2.0 ** -31 * v
    tol = tolerance(out, A, S, q_dtype == torch.float16, got.dtype == torch.float16) + lost + extra
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all(), "not finite"
    assert (err <= tol).all(), f"error {float((err / (out.abs() + 1e-300)).max()):.3g} relative, {float((err / tol).max()):.3g} of what is allowed"


def long_batch(ops, mode, D, length, io, drift=False, n=20, B=40):  # noqa: F811
    """Sequences of n tokens over the same ``length`` positions, V of one sign, a few rows checked."""
    from bitgpu_b200._lib import lib
    KV, G = 8, 4
    H, page = KV * G, 64
    pages = -(-length // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    shape = (pages, page, KV, D)
    if mode == "f16":
        kv = [torch.randn(shape, generator=g, device="cuda").half(),
              (1 + 0.2 * torch.rand(shape, generator=g, device="cuda")).half(), None, None]
        K, V = kv[0].view(-1, KV, D)[:length].double(), kv[1].view(-1, KV, D)[:length].double()
    else:
        sc = [torch.rand(shape[:3] + (D // 32,), generator=g, device="cuda") + s for s in (0.5, 1.0)]
        if drift:
            pos = torch.arange(pages * page, device="cuda").view(pages, page, 1, 1)
            sc[0] *= torch.exp2(torch.round(3 * torch.sin(pos / 900.0)) - 2)
            sc[1] *= torch.exp2(torch.round(10 * torch.cos(pos / 700.0 + torch.arange(D // 32, device="cuda"))))
        kv = [torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8),
              torch.randint(100, 128, shape, generator=g, device="cuda", dtype=torch.int8), *sc]
        K, V = ((kv[i].double() / 127 * sc[i].double().repeat_interleave(32, -1)).view(-1, KV, D)[:length] for i in (0, 1))
    cache = ops.PagedKVCache.from_tensors(*kv)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(B, pages).contiguous()
    lens = torch.full((B,), length, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, n * B + 1, n, dtype=torch.int32, device="cuda")
    q = (torch.randn((n * B, H, D), generator=g, device="cuda") * 0.05).to(DT[io])
    got = ops.paged_attention(q, cache, ops.PagedBatch(table, lens, cu, n * B, n), out_dtype=DT[io])
    assert lib().bg_device_status(None) == 0
    worst = 0.0
    for b, i in ((0, 0), (B // 2 - 3, n - 1), (B - 1, n // 3)):
        m = length - n + i + 1
        t = b * n + i
        for k in range(KV):
            qq = q[t].view(KV, G, D)[k].double()
            s = qq @ K[:m, k].T * D ** -0.5
            S = float((qq.abs() @ K[:m, k].abs().T).max()) * D ** -0.5
            w = torch.softmax(s, -1) @ V[:m, k]
            # f32 rows: 64 steps of a run; f16 rows: 512, beside two roundings to f16
            tol = (28 * S + 16 + 64) * 2.0 ** -24 * w if io == "f32" else (28 * S + 16 + 512) * 2.0 ** -24 * w + 2.0 ** -10 * w
            worst = max(worst, float(((got[t].view(KV, G, D)[k].double() - w).abs() / tol).max()))
    assert worst <= 1, f"{worst:.3g} of what is allowed"


# ---- q8 block scales -----------------------------------------------------------------------------
@each_kernel
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("vs", [1e-20, 1e-6, 1e-4, 1e-2, 1e3, 1e6, 1e20])
def test_value_scales(ops, kernel, D, vs):  # noqa: F811
    """V of any magnitude is read to the same relative error, f32 rows."""
    r = make(kernel, D=D)
    rescale(r, 1, vs)
    q = r.queries(torch.float32)
    check(r, attend(ops, kernel, r, q, torch.float32), r.attention(q), torch.float32)


@each_kernel
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("vs", [1e-3, 1e-1, 1e1, 1e3])
def test_value_scales_f16(ops, kernel, D, vs):  # noqa: F811
    r = make(kernel, D=D)
    rescale(r, 1, vs)
    q = r.queries(torch.float16)
    check(r, attend(ops, kernel, r, q, torch.float16), r.attention(q), torch.float16)


@each_kernel
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("by", ["block", "position", "both"])
def test_mixed_value_scales(ops, kernel, D, by):  # noqa: F811
    """Block scales that differ by up to ten decimal orders between channels, and by three between positions.
    The largest of a channel's scales sets the step of the others: f16 halves of at most 2^15 end at 2^-24, so
    that a value (or a weight times a scale) is off by at most 2^-25 / 2^13 = 2^-38 of the largest scale."""
    r = make(kernel, D=D)
    g = torch.Generator().manual_seed(5)
    n, nb = r.values[1].shape[0], D // 32
    f = torch.ones(n, r.KV, nb, dtype=torch.float64)
    if by != "position":
        f = f * 10.0 ** torch.linspace(-8, 2, nb, dtype=torch.float64)
    if by != "block":
        f = f * 10.0 ** (3 * torch.rand((n, r.KV, nb), generator=g, dtype=torch.float64) - 1.5)
    rescale(r, 1, f)
    q = r.queries(torch.float32)
    top = torch.stack([r.kv(b)[1].abs().amax(0) for b in range(3)]).amax(0).view(r.KV, nb, 32).amax(-1, keepdim=True)
    top = top.expand(r.KV, nb, 32).reshape(r.KV, 1, D).expand(r.KV, r.G, D).reshape(r.H, D)
    check(r, attend(ops, kernel, r, q, torch.float32), r.attention(q), torch.float32, extra=max(r.lens) * 2.0 ** -38 * top)


@each_kernel
@pytest.mark.parametrize("mode_order", ["rising", "falling"])
def test_value_scales_along_a_sequence(ops, kernel, mode_order):  # noqa: F811
    """Scales that grow (or shrink) by a factor of two every 64 positions, over 2^31 in all."""
    r = make(kernel, lens=(2000, 64, 130))
    f = torch.ones(r.values[1].shape[0], dtype=torch.float64)
    for b, n in enumerate(r.lens):
        e = torch.arange(n) // 64 - 16.0
        f[r.rows(b, n)] = 2.0 ** (e if mode_order == "rising" else -e).double()
    rescale(r, 1, f[:, None, None])
    q = r.queries(torch.float32)
    top = torch.stack([r.kv(b)[1].abs().amax() for b in range(3)]).amax()
    check(r, attend(ops, kernel, r, q, torch.float32), r.attention(q), torch.float32, extra=float(2000 * 2.0 ** -38 * top))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("length", [700, 5000, 40001])
def test_drifting_scales_of_long_units(ops, D, io, length):  # noqa: F811
    """Units of many tiles whose K scales rise and fall by 2^6 and V scales by 2^20, each block in its own time."""
    long_batch(ops, "q8", D, length, io, drift=True)


@each_kernel
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("ks", [1e-20, 1e-6, 1e-4, 1e3, 1e6, 1e20])
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_key_scales(ops, kernel, D, ks, io):  # noqa: F811
    """K of any magnitude, with the softmax scale that such keys need."""
    r = make(kernel, D=D)
    rescale(r, 0, ks)
    q = r.queries(DT[io])
    sc = 1 / (ks * math.sqrt(D))
    check(r, attend(ops, kernel, r, q, DT[io], scale=sc), r.attention(q, None, sc), DT[io])


@each_kernel
@pytest.mark.parametrize("D", [128, 256])
def test_mixed_key_scales(ops, kernel, D):  # noqa: F811
    r = make(kernel, D=D)
    g = torch.Generator().manual_seed(6)
    rescale(r, 0, 10.0 ** (5 * torch.rand((r.values[0].shape[0], r.KV, D // 32), generator=g, dtype=torch.float64) - 4.5))
    q = r.queries(torch.float32)
    check(r, attend(ops, kernel, r, q, torch.float32), r.attention(q), torch.float32)


# ---- q8 codes ------------------------------------------------------------------------------------
@each_kernel
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_every_code(ops, kernel, D, io):  # noqa: F811
    """Codes from -128 on: code -128 stands for -1, as -127 does."""
    r = make(kernel, D=D)
    for d in r.data:
        d.copy_(torch.randint(-128, 128, d.shape, generator=r.g))
        d[torch.rand(d.shape, generator=r.g) < 0.3] = -128
    revalue(r)
    q = r.queries(DT[io], 0.5)
    check(r, attend(ops, kernel, r, q, DT[io]), r.attention(q), DT[io])


# ---- f32 queries ---------------------------------------------------------------------------------
@each_kernel
@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("qs", [1e-20, 1e-8, 1e-4, 1e5, 1e20])
def test_query_scales(ops, kernel, mode, D, qs):  # noqa: F811
    """f32 queries of any magnitude, with the softmax scale that such queries need."""
    r = make(kernel, mode, D)
    q = r.queries(torch.float32, 1.5 * qs)
    sc = 1 / (qs * math.sqrt(D))
    for out in DT.values():
        check(r, attend(ops, kernel, r, q, out, scale=sc), r.attention(q, None, sc), torch.float32)


@each_kernel
@pytest.mark.parametrize("mode", ["f16", "q8"])
def test_mixed_query_scales(ops, kernel, mode):  # noqa: F811
    """Rows of one unit that differ by twelve decimal orders, zero rows among them; a row's error is its own."""
    r = make(kernel, mode)
    q = r.queries(torch.float32)
    g = torch.Generator().manual_seed(7)
    q *= 10.0 ** (12 * torch.rand((r.T, r.H, 1), generator=g) - 6)
    q[0, 1] = 0
    got = attend(ops, kernel, r, q, torch.float32, scale=1e-5)
    for t in range(r.T):
        for h in range(r.H):
            one = torch.zeros_like(q)
            one[t, h] = q[t, h]
            b = max(i for i in range(3) if r.cu[i] <= t)
            if t not in (0, r.T - 1) and h % 3:
                continue
            K, V = r.kv(b)
            m = r.lens[b] - r.news[b] + t - r.cu[b] + 1
            k, v, qq = K[:m, h // r.G], V[:m, h // r.G], q[t, h].double()
            s = k @ qq * 1e-5
            p = torch.softmax(s, 0)
            S = float((k.abs() @ qq.abs()).max()) * 1e-5
            tol = tolerance(p @ v, p @ v.abs(), S, False, False) + 2.0 ** -31 * v.abs().sum(0)
            assert ((got[t, h].double() - p @ v).abs() <= tol).all(), (t, h)


# ---- gates ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("kernel", [*KERNELS, "tc whole"])
@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("low,high", [(-80, 80), (-80, -20), (-8, 8)])
def test_gate_range(ops, kernel, mode, D, low, high):  # noqa: F811
    """A shut gate leaves little of a value, and that little as exact as the value: beside the ungated result's
    error 8 * 2^-24 (exp to two units in the last place, a sum, a quotient, a product)."""
    if kernel == "tc whole":  # units that no block's border cuts: gated by the tcgen05 kernel itself
        r = wide(Ragged([30] * 40, [30] * 40, KV=2, G=4, D=D, mode=mode, seed=1))
    else:
        r = make(kernel, mode, D)
    for io in DT.values():
        q = r.queries(io)
        gate = low + (high - low) * torch.rand(q.shape, generator=r.g)
        plain = attend(ops, kernel, r, q, torch.float32).double()
        got = attend(ops, kernel, r, q, torch.float32, gate=gate.cuda()).double()
        want = plain * torch.sigmoid(gate.double())
        err = (got - want).abs()
        assert (err <= 8 * 2.0 ** -24 * want.abs() + 2.0 ** -140).all(), float((err / want.abs()).max() * 2 ** 24)


# ---- lengths beyond the page table ---------------------------------------------------------------
@each_kernel
@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("prefix", [0, 40])
def test_length_beyond_the_table(ops, kernel, mode, prefix):  # noqa: F811
    """kv_len says more than the table holds: positions are what kv_len says, the append drops those that have no
    page, attention reads those that have one, both report it, and the other sequences are served."""
    from bitgpu_b200._lib import BG_EINVAL, lib
    G, news = KERNELS[kernel]
    KV, D, page, over = 2, 128, 16, 6
    r = Ragged([128, 64, 130], news, KV=KV, G=G, D=D, mode=mode, prefix=prefix, seed=3)
    width = 1 << 14 if kernel == "tc" else 9
    cap = width * page
    n = news[2]
    table = torch.zeros(3, width, dtype=torch.int32)
    table[:, :9] = r.table[:, :9].clamp(min=0)
    # the last sequence fills its whole row of the table with one page, over and over
    table[2] = r.table[2, 0]
    kv_len = torch.tensor([128, 64, cap + over], dtype=torch.int32)
    q = r.queries(torch.float32)
    cache = r.cache(ops)
    b = ops.PagedBatch(table.cuda(), kv_len.cuda(), torch.tensor(r.cu, dtype=torch.int32).cuda(), r.T, max(news),
                       r.prefix_pages.cuda() if prefix else None, prefix)
    lib().bg_force_generic(int(kernel == "cuda"))
    try:
        got = ops.paged_attention(q.cuda(), cache, b).cpu().double()
    finally:
        lib().bg_force_generic(0)
    assert lib().bg_device_status(None) == BG_EINVAL
    assert lib().bg_device_status(None) == 0
    # the repeated page: attended floor(m / page) times whole, and its first m % page slots once more
    first = r.table[2, 0].long() * page + torch.arange(page)
    K, V = r.values[0][first], r.values[1][first]
    if prefix:
        pr = r.prefix_rows()
        PK, PV = r.values[0][pr], r.values[1][pr]
    r.lens[2] = page  # the oracle's own rows of the other sequences
    r.news[2] = 0
    out, A, S = r.attention(q)
    r.news[2] = n
    for i in range(n):
        m = min(cap, cap + over - n + i + 1)
        w = (torch.tensor(m // page) + (torch.arange(page) < m % page)).double()
        qq = q[r.cu[2] + i].double().view(KV, G, D)
        s = torch.einsum("kgd,jkd->kgj", qq, K) * D ** -0.5
        S = max(S, float(torch.einsum("kgd,jkd->kgj", qq.abs(), K.abs()).max()) * D ** -0.5)
        v, e = V, s + w.log()
        if prefix:
            e = torch.cat([torch.einsum("kgd,jkd->kgj", qq, PK) * D ** -0.5, e], -1)
            v = torch.cat([PV, V])
        p = torch.softmax(e, -1)
        out[r.cu[2] + i] = torch.einsum("kgj,jkd->kgd", p, v).reshape(r.H, D)
        A[r.cu[2] + i] = torch.einsum("kgj,jkd->kgd", p, v.abs()).reshape(r.H, D)
    # (the tcgen05 kernel's accumulators run over the whole table here: its own test below bounds their error)
    tol = tolerance(out, A, S, False, False) + 64 * 2.0 ** -24 * A
    assert ((got - out).abs() <= tol).all(), float(((got - out).abs() / tol).max())


@pytest.mark.parametrize("n", [1, 10, 40])
def test_append_and_attend_beyond_the_table(ops, n):  # noqa: F811
    """Four pages of 16, kv_len 70: the tokens at 60 to 63 are appended and attend up to themselves, the ones
    behind attend what there is."""
    from bitgpu_b200._lib import BG_EINVAL, lib
    KV, G, D = 2, 4, 128
    H = KV * G
    torch.manual_seed(0)
    for kind in ("cuda", "fast"):
        cache = ops.PagedKVCache(6, 16, KV, D, "f16")
        cache.K.normal_()
        cache.V.normal_()
        table = torch.tensor([[3, 0, 5, 1]], dtype=torch.int32).cuda()
        b = ops.PagedBatch(table, torch.tensor([70], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(),
                           n, n)
        x = torch.randn(n, H + 2 * KV, D, device="cuda")
        ops.paged_append(cache, b, x[:, H:H + KV], x[:, H + KV:])
        assert lib().bg_device_status(None) == BG_EINVAL
        lib().bg_force_generic(int(kind == "cuda"))
        try:
            got = ops.paged_attention(x[:, :H].contiguous(), cache, b).double()
        finally:
            lib().bg_force_generic(0)
        assert lib().bg_device_status(None) == BG_EINVAL
        K, V = (t[table[0].long()].view(64, KV, D).double() for t in (cache.K, cache.V))
        for i in range(n):
            m = min(64, 70 - n + i + 1)
            if 70 - n + i < 64:
                assert torch.equal(V[m - 1].half(), x[i, H + KV:].half())
            qq = x[i, :H].double().view(KV, G, D)
            p = torch.softmax(torch.einsum("kgd,jkd->kgj", qq, K[:m]) * D ** -0.5, -1)
            w = torch.einsum("kgj,jkd->kgd", p, V[:m]).reshape(H, D)
            assert (got[i] - w).abs().max() <= 1e-5, (kind, i)


# ---- long runs of one accumulator ----------------------------------------------------------------
@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("length", [2000, 9000, 40000, 120000])
def test_long_units(ops, mode, D, length):  # noqa: F811
    """Units that stay whole over many tiles, values of one sign: the error of f32 rows does not grow with the
    length.  A run of matrix products into one accumulator has at most 64 steps, each of which may drop less than
    2^-23 of what has been added up; the parts of equal steps add up to 33 / 64 of that: 64 * 2^-24 in all, beside
    the tolerance's other terms."""
    long_batch(ops, mode, D, length, "f32")


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D,n", [(128, 20), (128, 60), (256, 20)])
def test_long_units_f16(ops, mode, D, n):  # noqa: F811
    """(60 tokens of 4 heads fill both query tiles of a unit.)"""
    long_batch(ops, mode, D, 60000, "f16", n=n)
