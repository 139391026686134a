"""Paged attention over tables wide enough for the tensor-core kernels, at the sizes and batches where
they can go wrong: page and group sizes, ragged prompts, padding, rows without positions, bad pages,
captured calls.  (Which kernel runs follows from the room in the page table, not from the lengths.)"""
import pytest
import torch

from paged_util import Ragged, check_attention, tolerance
from test_gpu_paged_attention import DT, ops, run  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def wide(r, positions=1 << 18):
    """The same batch in a table with room for that many positions; the entries behind are no pages."""
    t = torch.full((r.table.shape[0], -(-positions // r.page)), -7, dtype=torch.int32)
    t[:, :r.table.shape[1]] = r.table
    r.table = t
    return r


KINDS = [("f16", "f16"), ("f16", "f32"), ("q8", "f16"), ("q8", "f32")]


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("page", [8, 24, 48, 192, 256])
def test_page_sizes(ops, mode, io, D, page):  # noqa: F811
    run(ops, wide(Ragged([213, 100, 515], [80, 100, 33], D=D, page=page, mode=mode, seed=page)), DT[io], DT[io])


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("G", [1, 3, 5, 6, 12, 20, 40, 65, 100, 128, 130])
def test_head_groups(ops, mode, io, D, G):  # noqa: F811
    """Groups that fill a tile, that leave rows of it empty, and one that has no tile."""
    run(ops, wide(Ragged([190, 33], [60, 33], KV=2, G=G, D=D, mode=mode, seed=G)), DT[io], DT[io], gated=G == 6)


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
def test_prefill_ragged(ops, mode, io, D):  # noqa: F811
    """Prompts beside single tokens; prompts with and without earlier positions."""
    run(ops, wide(Ragged([150, 77, 300, 64, 5, 129], [150, 1, 70, 64, 5, 1], D=D, mode=mode, page=32, seed=5)), DT[io], DT[io])


@pytest.mark.parametrize("io", [("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("D", [128, 256])
def test_mixed_types(ops, io, D):  # noqa: F811
    run(ops, wide(Ragged([150, 77], [150, 33], D=D, seed=6)), DT[io[0]], DT[io[1]], gated=True)


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
def test_scale_and_gate(ops, mode, io, D):  # noqa: F811
    run(ops, wide(Ragged([100, 131], [100, 30], D=D, mode=mode, seed=1)), DT[io], DT[io], scale=0.03, gated=True)


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("G", [4, 6])
def test_padding_rows(ops, mode, io, D, G):  # noqa: F811
    """NaN queries behind the last sequence; the rows are left as they were."""
    run(ops, wide(Ragged([190, 70], [90, 33], D=D, G=G, mode=mode, pad=40, seed=1)), DT[io], DT[io])
    run(ops, wide(Ragged([190, 70, 20], [90, 1, 20], KV=8, D=D, G=G, mode=mode, pad=40, prefix=1500, seed=1)), DT[io], DT[io])


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("D", [128, 256])
def test_no_position(ops, io, D):  # noqa: F811
    """Tokens that the length leaves no position for are zero; a batch whose sequences are all empty."""
    got = run(ops, wide(Ragged([0, 40], [100, 130], D=D, seed=2)), DT[io], DT[io])
    assert not got[:190].any()
    got = run(ops, wide(Ragged([0, 0], [60, 30], D=D, seed=2)), DT[io], DT[io])
    assert not got.any()


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("max_q", [5, 31, 5000])
def test_max_q_is_only_a_hint(ops, mode, max_q):  # noqa: F811
    for io in DT.values():
        run(ops, wide(Ragged([150, 40, 9], [90, 3, 1], mode=mode, seed=6)), io, io, max_q=max_q)


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
def test_large_values(ops, mode, io, D):  # noqa: F811
    """Scores tens of units apart and large V: nothing overflows, small weights are not lost."""
    r = wide(Ragged([700, 64], [40, 30], D=D, mode=mode, seed=12, vscale=30.0))
    q = r.queries(DT[io], 12.0)
    got = ops.paged_attention(q.cuda(), r.cache(ops), r.batch(ops), out_dtype=DT[io])
    # The weights enter the product as f16, one half or two, 64 times as large as exp(score - largest score): the
    # smallest f16 step is 2^-24, so a weight is off by at most 2^-25 / 64 = 2^-31 beside its relative error, and
    # the largest weight, and with it their sum, is 1 or more.  A channel whose values are zero wherever a
    # weight is not tiny (a q8 code may be) shows it: 2^-31 * sum |v| may be missing.
    out, A, S = r.attention(q)
    lost = torch.zeros_like(out)
    for b, n in enumerate(r.news):
        v = r.kv(b)[1].abs().sum(0).repeat_interleave(r.G, 0)
        lost[r.cu[b]:r.cu[b] + n] = 2.0 ** -31 * v
    tol = tolerance(out, A, S, io == "f16", io == "f16") + lost
    err = (got.double().cpu() - out).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
def test_bad_page_reads_zeros(ops, mode, io, D):  # noqa: F811
    from bitgpu_b200._lib import BG_EINVAL, lib
    for bad in (-1, 1 << 30):
        r = wide(Ragged([100, 90], [80, 60], D=D, mode=mode, seed=4))
        for v in r.values:
            v[r.table[0, 2] * 16:(r.table[0, 2] + 1) * 16] = 0
        q = r.queries(DT[io])
        want = r.attention(q)
        cache = r.cache(ops)
        r.table[0, 2] = bad
        got = ops.paged_attention(q.cuda(), cache, r.batch(ops), out_dtype=DT[io])
        assert lib().bg_device_status(None) == BG_EINVAL
        assert lib().bg_device_status(None) == 0
        check_attention(got, want, io == "f16")


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_one_sequence_twice(ops, io):  # noqa: F811
    """Two sequences of a batch over the same pages give the same rows."""
    r = wide(Ragged([100, 90], [50, 50], seed=4))
    r.table[1] = r.table[0]
    r.lens[1] = r.lens[0]
    q = r.queries(DT[io])
    q[50:100] = q[:50]
    got = ops.paged_attention(q.cuda(), r.cache(ops), r.batch(ops), out_dtype=DT[io])
    check_attention(got, r.attention(q), io == "f16")


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
def test_streams_and_graphs(ops, mode, io, D):  # noqa: F811
    """Captured calls follow in-place updates of their batch, beside each other and an eager call."""
    def make():
        return wide(Ragged([300, 20, 90], [100, 1, 30], D=D, mode=mode, seed=7))
    r = make()
    q = r.queries(DT[io])
    cache, b1, b2, qd = r.cache(ops), r.batch(ops), r.batch(ops), q.cuda()

    def call(b):
        return ops.paged_attention(qd, cache, b, out_dtype=DT[io])
    first = call(b1).clone()
    g1, g2 = ops.Graphed(lambda: call(b1)), ops.Graphed(lambda: call(b2))
    lens = [107, 20, 33]
    b2.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    r2 = make()
    r2.lens = lens
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for _ in range(5):
        o1 = g1.replay()
        with torch.cuda.stream(side):
            o2 = g2.replay()
            o3 = call(b1)
    torch.cuda.synchronize()
    want = r.attention(q)
    check_attention(o1, want, io == "f16")
    check_attention(o2, r2.attention(q), io == "f16")
    assert torch.equal(o1, o3) and torch.equal(o1, first)


@pytest.mark.parametrize("mode,io", KINDS)
def test_same_bits_twice(ops, mode, io):  # noqa: F811
    r = wide(Ragged([2000, 300, 40], [170, 1, 33], KV=8, prefix=1700, mode=mode, seed=3))
    q, cache, b = r.queries(DT[io]).cuda(), r.cache(ops), r.batch(ops)
    a = ops.paged_attention(q, cache, b, out_dtype=DT[io])
    for _ in range(5):
        assert torch.equal(a, ops.paged_attention(q, cache, b, out_dtype=DT[io]))


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("room", [64, 1 << 18])
def test_output_in_place(ops, mode, io, D, room):  # noqa: F811
    """out may be q, whichever kernels run."""
    for prefix in (0, 1500):
        r = wide(Ragged([300, 20, 90], [60, 1, 30], KV=4, G=6, D=D, mode=mode, prefix=prefix, page=64, seed=9),
                 max(room, 384))
        q = r.queries(DT[io]).cuda()
        cache, b = r.cache(ops), r.batch(ops)
        want = ops.paged_attention(q, cache, b, out_dtype=DT[io])
        assert torch.equal(ops.paged_attention(q, cache, b, out=q), want)


@pytest.mark.parametrize("mode,io", KINDS)
@pytest.mark.parametrize("room", [320, 1 << 18])
@pytest.mark.parametrize("news", [[1, 1], [60, 30]])
def test_shut_and_open_gates(ops, mode, io, room, news):  # noqa: F811
    r = wide(Ragged([300, 90], news, mode=mode, seed=9), room)
    q = r.queries(DT[io]).cuda()
    cache, b = r.cache(ops), r.batch(ops)
    want = ops.paged_attention(q, cache, b, out_dtype=DT[io])
    inf = torch.full(q.shape, float("inf"), device="cuda")
    assert torch.equal(ops.paged_attention(q, cache, b, gate=inf, out_dtype=DT[io]), want)
    assert not ops.paged_attention(q, cache, b, gate=-inf, out_dtype=DT[io]).any()


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
def test_many_sequences(ops, mode):  # noqa: F811
    """Thousands of short sequences, a few of them without a token."""
    B = 5000
    lens = [i * 7 % 19 + 1 for i in range(B)]
    news = [0 if i % 97 == 5 else min(lens[i], i % 2 + 1) for i in range(B)]
    run(ops, Ragged(lens, news, KV=1, G=2, D=128, page=8, mode=mode, seed=5))


@pytest.mark.parametrize("mode,D,pages", [("f16", 128, 66000), ("q8", 128, 66000), ("q8", 256, 33000), ("f32", 64, 40000)])
@pytest.mark.parametrize("room", [640, 1 << 18])
def test_far_pages(ops, mode, D, pages, room):  # noqa: F811
    """Pages behind the first 2^32 values (f32: bytes) of a pool: the bits of a small pool, appended and read."""
    KV, G, page, n = 8, 4, 64, 20
    far = ops.PagedKVCache.from_tensors(*[
        torch.empty((pages, page, KV, w), dtype=dt, device="cuda")
        for dt, w in [({"f16": torch.float16, "q8": torch.int8, "f32": torch.float32}[mode], D)] * 2
        + [(torch.float32, D // 32)] * 2 * (mode == "q8")])
    near = ops.PagedKVCache(n, page, KV, D, mode)
    torch.manual_seed(1)
    lens, news = [500, 70, 129], [100, 1, 129]
    T = sum(news)
    table = torch.zeros(3, room // page, dtype=torch.int32, device="cuda")
    table[:, :6] = torch.randperm(18)[:18].view(3, 6).int().cuda()
    table[0, 6:8] = torch.tensor([18, 19], dtype=torch.int32)
    qkv = torch.randn(T, (G + 2) * KV, D, device="cuda")
    H = G * KV
    out = []
    for cache, first in ((near, 0), (far, pages - n)):
        args = (table + first, torch.tensor(lens).int().cuda())
        cu = torch.tensor([0, 100, 101, T]).int().cuda()
        if first:  # the positions before the new tokens
            for x in ("K", "V") + ("Ks", "Vs") * (mode == "q8"):
                getattr(far, x)[first:] = before[x]
        else:
            near.K.copy_(torch.randn(near.K.shape, device="cuda") * 20)
            near.V.copy_(torch.randn(near.V.shape, device="cuda") * 20)
            if mode == "q8":
                near.Ks.uniform_(0.5, 1.5)
                near.Vs.uniform_(0.5, 1.5)
            before = {x: getattr(near, x).clone() for x in ("K", "V") + ("Ks", "Vs") * (mode == "q8")}
        b = ops.PagedBatch(*args, cu, T, max(news))
        ops.paged_append(cache, b, qkv[:, H:H + KV], qkv[:, H + KV:])
        out.append(ops.paged_attention(qkv[:, :H].contiguous(), cache, b))
    for x in ("K", "V") + ("Ks", "Vs") * (mode == "q8"):
        assert torch.equal(getattr(far, x)[pages - n:], getattr(near, x)), x
        assert not torch.equal(getattr(near, x), before[x])
    assert torch.isfinite(out[0]).all() and torch.equal(out[0], out[1])
