"""Ragged attention over a paged cache, with and without a shared prefix, against its definition in
64 bits (tests/paged_util.py; unused pool slots and pages hold NaN)."""
import pytest
import torch

from paged_util import Ragged, check_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from bitgpu_b200 import ops
    return ops


def run(ops, r, q_dtype=torch.float32, out_dtype=torch.float32, gated=False, scale=0.0, max_q=None, what=""):
    q = r.queries(q_dtype)
    q[r.cu[-1]:] = float("nan")
    gate = torch.randn(q.shape, generator=r.g) if gated else None
    want = r.attention(q, gate, scale or None)
    out = torch.full(q.shape, 7.0, dtype=out_dtype, device="cuda")
    got = ops.paged_attention(q.cuda(), r.cache(ops), r.batch(ops, max_q), scale=scale,
                              gate=gate.cuda() if gated else None, out=out)
    torch.cuda.synchronize()
    n = r.cu[-1]
    check_attention(got[:n], (want[0][:n], want[1][:n], want[2]), q_dtype == torch.float16, what)
    assert (got[n:] == 7.0).all(), "rows behind the last sequence were written"
    from bitgpu_b200._lib import lib
    assert lib().bg_device_status(None) == 0
    return got


DT = {"f32": torch.float32, "f16": torch.float16}


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_decode_lengths(ops, mode, D, io):
    """One token each over lengths around the tile and page borders, from one position on."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1]
    run(ops, Ragged(lens, [1] * len(lens), D=D, mode=mode, seed=D), DT[io], DT[io])


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 32, 48, 64, 128, 192, 256])
def test_page_sizes(ops, mode, page):
    lens = [3, 200, 65, 513]
    run(ops, Ragged(lens, [1] * 4, page=page, mode=mode, seed=page), what=f"page {page}")


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("page", [5, 8, 24, 48, 64, 192, 256])
def test_page_sizes_prefill(ops, mode, page):
    run(ops, Ragged([213, 100, 515], [80, 100, 33], page=page, mode=mode, prefix=77, seed=page), torch.float16,
        torch.float16, what=f"page {page}")


@pytest.mark.parametrize("G", [1, 2, 3, 6, 8, 12, 16, 20])
@pytest.mark.parametrize("mode", ["f16", "q8"])
def test_head_groups(ops, G, mode):
    run(ops, Ragged([70, 9, 200], [1] * 3, KV=3, G=G, mode=mode, seed=G))


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("io", [("f32", "f32"), ("f16", "f16"), ("f32", "f16"), ("f16", "f32")])
def test_several_tokens(ops, mode, D, io):
    """Verification: a few tokens each, some sequences with one or none, an odd split of rows."""
    run(ops, Ragged([40, 130, 3, 65, 260], [3, 1, 3, 0, 5], D=D, mode=mode, seed=3), DT[io[0]], DT[io[1]])


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_prefill_ragged(ops, mode, D, io):
    """Prompts beside single tokens; prompts with and without earlier positions."""
    run(ops, Ragged([150, 77, 300, 64, 5, 129], [150, 1, 70, 64, 5, 1], D=D, mode=mode, page=32, seed=5), DT[io], DT[io])


@pytest.mark.parametrize("G,KV", [(1, 2), (3, 1), (6, 2), (16, 1), (5, 3)])
def test_prefill_groups(ops, G, KV):
    run(ops, Ragged([190, 33], [120, 33], KV=KV, G=G, seed=G), torch.float16, torch.float16)


def test_prefill_long(ops):
    """Many tiles of both operands: every sequence is cut into pieces."""
    run(ops, Ragged([1500, 900], [700, 333], KV=1, G=4, page=64, seed=8), torch.float16, torch.float16)


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
def test_long_single_stream(ops, mode, D):
    """Few rows and many positions: the work is split and joined."""
    run(ops, Ragged([9001], [1], KV=2, G=4, D=D, mode=mode, page=64, seed=9), gated=True)


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("prefix", [1, 16, 100, 513])
def test_prefix(ops, mode, D, prefix):
    run(ops, Ragged([1, 20, 64, 0, 65], [1] * 5, D=D, mode=mode, prefix=prefix, seed=prefix), gated=D == 256)


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("B", [1, 9, 40, 70])
def test_prefix_many_rows(ops, mode, D, io, B):
    """Enough rows behind one prefix for the matrix kernels, odd row counts, short own parts."""
    lens = [(7 * i) % 90 + 1 for i in range(B)]
    run(ops, Ragged(lens, [1] * B, KV=2, G=4, D=D, mode=mode, prefix=777, page=32, seed=B), DT[io], DT[io])


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("B,G", [(24, 4), (40, 4), (67, 4), (30, 3)])
def test_prefix_many_tiles(ops, mode, io, B, G):
    """A prefix long enough that every block of the matrix kernels walks a dozen tiles of a unit, with
    one unit of rows and with several."""
    lens = [(11 * i) % 70 + 1 for i in range(B)]
    run(ops, Ragged(lens, [1] * B, KV=8, G=G, mode=mode, prefix=13001, page=64, seed=B), DT[io], DT[io])


@pytest.mark.parametrize("mode,io", [("f16", "f16"), ("f16", "f32"), ("q8", "f16"), ("q8", "f32")])
def test_many_tiles_d256(ops, mode, io):
    """head_dim 256, six heads a group: a long prefix and long prompts through the matrix kernels."""
    lens = [(11 * i) % 70 + 1 for i in range(30)]
    run(ops, Ragged(lens, [1] * 30, KV=4, G=6, D=256, mode=mode, prefix=9001, page=64, seed=3), DT[io], DT[io], gated=True)
    run(ops, Ragged([3000, 1001, 150, 9], [130, 300, 150, 1], KV=4, G=6, D=256, mode=mode, page=16, seed=4), DT[io], DT[io],
        gated=True)


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("n", [33, 129, 257])
def test_prefill_many_tiles(ops, mode, io, n):
    """Prompts behind long contexts: units of many tiles in every block, cut ones among them."""
    run(ops, Ragged([9000, 7001, 1500], [n, n // 2, 1], KV=8, G=4, mode=mode, page=16, seed=n), DT[io], DT[io])


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_prefix_tokens(ops, io):
    """Several tokens each behind a prefix (verification and prompts), padding behind them."""
    run(ops, Ragged([4, 30, 90, 200], [4, 2, 90, 150], prefix=333, pad=5, seed=4), DT[io], DT[io])


def test_padding_rows(ops):
    run(ops, Ragged([33, 70], [2, 3], pad=7, seed=1))
    run(ops, Ragged([33, 70], [2, 3], pad=300, prefix=65, seed=1))
    for io in DT.values():
        run(ops, Ragged([190, 70], [90, 33], pad=40, prefix=165, seed=1), io, io)


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_no_position(ops, io):
    """Tokens that the length leaves no position for: zeros, or the prefix alone."""
    for prefix in (0, 50):
        r = Ragged([0, 2, 5], [1, 4, 5], prefix=prefix, seed=2)
        got = run(ops, r, DT[io], DT[io])
        if not prefix:
            assert not got[:3].any()
    r = Ragged([0, 40], [100, 130], seed=2)
    assert not run(ops, r, DT[io], DT[io])[:190].any()


def test_scale_and_gate(ops):
    run(ops, Ragged([100, 31], [1, 1], seed=1), scale=0.03, gated=True)
    run(ops, Ragged([100, 131], [100, 3], seed=1), scale=0.03, gated=True)


def test_max_q_is_only_a_hint(ops):
    """A wrong max_q selects another kernel, not another result."""
    for mq in (1, 500):
        run(ops, Ragged([150, 40], [90, 3], seed=6), torch.float16, torch.float16, max_q=mq)


@pytest.mark.parametrize("mode", ["f16", "q8"])
def test_large_values(ops, mode):
    """Scores tens of units apart and large V: nothing overflows, small weights are not lost."""
    r = Ragged([700, 64], [1, 1], mode=mode, seed=12, vscale=300.0)
    r.queries_scale = 12.0
    q = r.queries(torch.float32, 12.0)
    want = r.attention(q)
    got = ops.paged_attention(q.cuda(), r.cache(ops), r.batch(ops))
    check_attention(got, want, False)


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("news", [[1, 1], [80, 60]])
def test_bad_page_reads_zeros(ops, io, news):
    """A page id outside the pool: zeros instead of its positions, and the status says so."""
    from bitgpu_b200._lib import BG_EINVAL, lib
    for bad in (-1, 1 << 30):
        r = Ragged([100, 90], news, seed=4)
        r.values[0][r.table[0, 2] * 16:(r.table[0, 2] + 1) * 16] = 0
        r.values[1][r.table[0, 2] * 16:(r.table[0, 2] + 1) * 16] = 0
        q = r.queries(DT[io])
        want = r.attention(q)
        cache = r.cache(ops)
        r.table[0, 2] = bad
        got = ops.paged_attention(q.cuda(), cache, r.batch(ops), out_dtype=DT[io])
        assert lib().bg_device_status(None) == BG_EINVAL
        assert lib().bg_device_status(None) == 0
        check_attention(got, want, io == "f16")


def test_streams_and_graphs(ops):
    """A captured step follows in-place updates of its batch; two graphs and an eager call on another
    stream run beside each other."""
    r = Ragged([300, 20, 90], [1, 1, 1], seed=7)
    q = r.queries(torch.float32)
    cache = r.cache(ops)
    b1, b2 = r.batch(ops), r.batch(ops)
    qd = q.cuda()
    ops.paged_attention(qd, cache, b1)
    g1 = ops.Graphed(lambda: ops.paged_attention(qd, cache, b1))
    g2 = ops.Graphed(lambda: ops.paged_attention(qd, cache, b2))
    want = r.attention(q)
    b2.kv_len.copy_(torch.tensor([7, 20, 33], dtype=torch.int32))
    r2 = Ragged([300, 20, 90], [1, 1, 1], seed=7)
    r2.lens = [7, 20, 33]
    want2 = r2.attention(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for _ in range(5):
        o1 = g1.replay()
        with torch.cuda.stream(side):
            o2 = g2.replay()
            o3 = ops.paged_attention(qd, cache, b1)
    torch.cuda.synchronize()
    check_attention(o1, want, False)
    check_attention(o2, want2, False)
    check_attention(o3, want, False)


def test_same_bits_twice(ops):
    for news in ([1, 1, 1], [70, 1, 33]):
        r = Ragged([2000, 300, 40], news, prefix=200, seed=3)
        q, cache, b = r.queries(torch.float32).cuda(), r.cache(ops), r.batch(ops)
        a = ops.paged_attention(q, cache, b)
        for _ in range(3):
            assert torch.equal(a, ops.paged_attention(q, cache, b))


def test_step_together(ops):
    """A serving loop: append and attend, prompt first, then one token at a time, one batch object."""
    torch.manual_seed(0)
    KV, G, D, page, prompt, steps = 2, 4, 128, 16, 37, 30
    H = KV * G
    for mode in ("f32", "f16", "q8"):
        cache = ops.PagedKVCache(20, page, KV, D, mode)
        table = torch.randperm(20)[:16].view(2, 8).int().cuda()
        lens = [prompt, prompt - 6]
        T = sum(lens) + steps
        ang = torch.outer(torch.arange(200.0), 1e4 ** (-torch.arange(0, D, 2) / D))
        cos, sin = (torch.cat([f, f], -1).cuda() for f in (ang.cos(), ang.sin()))
        gam = (1 + 0.1 * torch.randn(D)).cuda()
        x = torch.randn(2, prompt + steps, H + 2 * KV, D, device="cuda")
        outs = [[], []]
        rows = torch.cat([x[0, :lens[0]], x[1, :lens[1]]]).contiguous()
        first = ops.PagedBatch(table, torch.tensor(lens).int().cuda(), torch.tensor([0, lens[0], sum(lens)]).int().cuda(),
                               sum(lens), max(lens))
        step = ops.PagedBatch(table, torch.tensor(lens).int().cuda())
        qn = []

        def go(rows, batch):
            q = ops.paged_append(cache, batch, rows[:, H:H + KV], rows[:, H + KV:], cos, sin, gam, 1e-6, rows[:, :H], gam)
            return q, ops.paged_attention(q, cache, batch)

        q, o = go(rows, first)
        for b, (a, e) in enumerate(((0, lens[0]), (lens[0], sum(lens)))):
            outs[b].append(o[a:e])
            qn.append([q[a:e]])
        for s in range(steps):
            step.kv_len.add_(1)
            q, o = go(torch.stack([x[b, lens[b] + s] for b in range(2)]), step)
            for b in range(2):
                outs[b].append(o[b:b + 1])
                qn[b].append(q[b:b + 1])
        # the same positions through the cache's own values, all at once in 64 bits
        r = Ragged([lens[0] + steps, lens[1] + steps], [lens[0] + steps, lens[1] + steps], KV=KV, G=G, D=D, page=page, mode="f32")
        val = []
        for d, s in ((cache.K, cache.Ks), (cache.V, cache.Vs)):
            v = d.cpu().double().view(-1, KV, D)
            if mode == "q8":
                v = (v / 127).clamp(min=-1) * s.cpu().double().view(-1, KV, D // 32).repeat_interleave(32, -1)
            val.append(v)
        r.values, r.table = val, table.cpu()
        qa = torch.cat([torch.cat(z) for z in qn]).cpu()
        check_attention(torch.cat([torch.cat(z) for z in outs]), r.attention(qa), False, mode)
