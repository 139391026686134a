"""Append to a paged cache: norm, rotation, codec and placement of a ragged batch against the formulas in
64 bits and the oracle's codec."""
import pytest
import torch

from oracle import kvcodec
from paged_util import norm_rope

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    from bitgpu_b200 import ops
    return ops


def build(ops, lens, news, KV, H, D, page, mode, rot, prefix=0, pad=0, seed=0, wide=1):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-max(n, 1) // page) for n in lens]
    pages = sum(counts) + 2
    ids = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    T = cu[-1] + pad
    cache = ops.PagedKVCache(pages, page, KV, D, mode)
    one = set(news) == {1} and not pad
    pre = torch.zeros(-(-prefix // page), dtype=torch.int32).cuda() if prefix else None
    batch = ops.PagedBatch(table.cuda(), torch.tensor(lens).int().cuda(),
                           None if one else torch.tensor(cu).int().cuda(), T, max(news), pre, prefix)
    x = torch.randn((T, H * wide + 2 * KV, D), generator=g)
    ang = torch.outer(torch.arange(prefix + max(lens) + 1.0), 1e4 ** (-torch.arange(0, max(rot, 2), 2) / max(rot, 2)))
    cos, sin = (torch.cat([f, f], -1) for f in (ang.cos(), ang.sin()))
    gam = 1 + 0.1 * torch.randn((2, D), generator=g)
    tok = [(b, L - n + i) for b, (L, n) in enumerate(zip(lens, news)) for i in range(n)]
    return cache, batch, x, cos, sin, gam, table, tok, cu[-1]


def check(ops, lens, news, KV=2, H=6, D=128, page=16, mode="f16", rot=None, norm=True, src=torch.float32,
          out=torch.float32, with_q=True, prefix=0, pad=0, seed=0):
    rot = D if rot is None else rot
    cache, batch, x, cos, sin, gam, table, tok, n = build(ops, lens, news, KV, H, D, page, mode, rot, prefix, pad, seed)
    x = x.to(src)
    if not rot:
        cos = sin = None
    xd = x.cuda()
    c, s = (None, None) if cos is None else (cos.cuda(), sin.cuda())
    gd = gam.cuda()
    kg, qg = (gd[0], gd[1]) if norm else (None, None)
    T = x.shape[0]
    qo = torch.full((T, H, D), 9.0, dtype=out, device="cuda") if with_q else None
    q = ops.paged_append(cache, batch, xd[:, H:H + KV], xd[:, H + KV:], c, s, kg, EPS, xd[:, :H] if with_q else None,
                         qg if with_q else None, q_out=qo)
    torch.cuda.synchronize()
    pos = torch.tensor([prefix + o for _, o in tok])
    live = torch.tensor([o >= 0 for _, o in tok])
    xs = x[:n]
    pc = pos.clamp(min=0)
    wk = norm_rope(xs[:, H:H + KV], gam[0] if norm else None, cos, sin, pc, EPS)
    wv = xs[:, H + KV:].double()
    # a product of the norm's factors, two products and a sum of the rotation: at most 12 f32 roundings
    # of values up to |y| + |partner| <= 2 max|y|
    room = 12 * 2.0 ** -24 * 2
    if with_q:
        wq = norm_rope(xs[:, :H], gam[1] if norm else None, cos, sin, pc, EPS)
        tol = room * wq.abs().amax(-1, keepdim=True).clamp(min=1) + (2.0 ** -11 * wq.abs() + 2.0 ** -25 if out == torch.float16 else 0)
        assert ((q[:n].cpu().double() - wq).abs() <= tol)[live].all()
        assert (q[n:] == 9.0).all() and (q[:n].cpu()[~live] == 9.0).all()
    else:
        assert q is None
    rows = torch.tensor([int(table[b, o // page]) * page + o % page if o >= 0 else 0 for b, o in tok])[live]
    for data, sc, w in ((cache.K, cache.Ks, wk[live]), (cache.V, cache.Vs, wv[live])):
        flat = data.cpu().view(-1, KV, D)
        got = flat[rows]
        big = w.abs().amax(-1, keepdim=True).clamp(min=1)
        if mode == "f32":
            assert ((got.double() - w).abs() <= room * big).all()
        elif mode == "f16":
            assert ((got.double() - w).abs() <= room * big + 2.0 ** -11 * w.abs() + 2.0 ** -25).all()
        else:
            enc, s8 = kvcodec.encode("q8", w.float().numpy())
            gs = sc.cpu().view(-1, KV, D // 32)[rows]
            assert ((gs.double() - torch.from_numpy(s8).double()).abs() <= room * big).all()
            d = (got.int() - torch.from_numpy(enc).int()).abs()
            # a value within rounding of a code's border may take the neighbouring code
            assert d.max() <= 1 and d.float().mean() <= 127 * 2 * room * 4
            if w is wv[live] or not (norm or rot):
                assert d.max() == 0
        other = torch.ones(flat.shape[0], dtype=torch.bool)
        other[rows] = False
        assert not flat[other].float().any(), "slots that belong to no new token were written"
    from bitgpu_b200._lib import lib
    assert lib().bg_device_status(None) == 0


@pytest.mark.parametrize("mode", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_types(ops, mode, D, src):
    check(ops, [1, 40, 17, 33], [1] * 4, D=D, mode=mode, src=src, out=src)
    check(ops, [50, 33, 9], [50, 2, 9], D=D, mode=mode, src=src, pad=3, seed=1)


@pytest.mark.parametrize("rot", [0, 2, 6, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("src", [torch.float32, torch.float16])
def test_rotation_widths(ops, rot, src):
    for mode in ("f16", "q8"):
        check(ops, [30, 9], [7, 9], rot=rot, mode=mode, src=src)


@pytest.mark.parametrize("H,KV", [(1, 1), (3, 1), (5, 5), (24, 4), (7, 3)])
def test_heads(ops, H, KV):
    for norm in (True, False):
        check(ops, [20, 5, 64], [3, 5, 1], H=H, KV=KV, norm=norm, D=64, src=torch.float16)


def test_without_q(ops):
    check(ops, [20, 5], [3, 5], with_q=False)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_pages_and_prefix(ops, page):
    check(ops, [70, 5, 64, 0], [65, 5, 1, 0], page=page, prefix=100)


def test_no_position(ops):
    """Tokens whose length leaves no position are skipped."""
    check(ops, [0, 2, 30], [2, 5, 3])


@pytest.mark.parametrize("B", [1, 31, 32, 33, 100, 1025, 1100])
def test_many_sequences(ops, B):
    """The search over sequences, with empty ones among them."""
    news = [(i * 7) % 3 for i in range(B)]
    news[-1] = 2
    check(ops, [n + i % 5 for i, n in enumerate(news)], news, KV=1, H=1, D=64)


def test_views(ops):
    """q from rows that interleave a gate half, k and v from a fused projection, odd strides and offsets."""
    lens, news, KV, H, D, page = [40, 12], [5, 12], 2, 3, 128, 16
    for off in (0, 1, 4):
        cache, batch, _, cos, sin, gam, table, tok, n = build(ops, lens, news, KV, H, D, page, "f32", D)
        g = torch.Generator().manual_seed(off)
        w = H * 2 * D + 2 * KV * D + off
        x = torch.randn((n, w + off), generator=g)
        xd = x.cuda()
        views = [t[:, off:off + H * 2 * D].view(n, H, 2 * D)[..., :D] if off == 0 else
                 t[:, off:off + H * 2 * D].unflatten(1, (H, 2 * D))[..., :D] for t in (x, xd)]
        kv = [t[:, off + H * 2 * D:off + H * 2 * D + 2 * KV * D].unflatten(1, (2 * KV, D)) for t in (x, xd)]
        q = ops.paged_append(cache, batch, kv[1][:, :KV], kv[1][:, KV:], cos.cuda(), sin.cuda(), q=views[1])
        pos = torch.tensor([o for _, o in tok])
        want = norm_rope(views[0], None, cos, sin, pos, EPS)
        assert (q.cpu().double() - want).abs().max() <= 24 * 2.0 ** -24 * want.abs().max()
        rows = torch.tensor([int(table[b, o // page]) * page + o % page for b, o in tok])
        wk = norm_rope(kv[0][:, :KV], None, cos, sin, pos, EPS)
        assert (cache.K.cpu().view(-1, KV, D)[rows].double() - wk).abs().max() <= 24 * 2.0 ** -24 * wk.abs().max()
        assert torch.equal(cache.V.cpu().view(-1, KV, D)[rows], kv[0][:, KV:])


def test_bad_pages_and_positions(ops):
    """A page id outside the pool, a table that is too narrow and a position behind the rotation table:
    the row is dropped, nothing else is touched, and the status says so."""
    from bitgpu_b200._lib import BG_EINVAL, lib
    for what in ("page", "low", "narrow", "rope"):
        cache, batch, x, cos, sin, gam, table, tok, n = build(ops, [20, 20], [1, 1], 2, 4, 128, 16, "f16", 128)
        if what == "page":
            batch.page_table[1, 1] = 1 << 30
        elif what == "low":
            batch.page_table[1, 1] = -5
        elif what == "narrow":
            batch.kv_len[1] = 33
        rows = 19 if what == "rope" else cos.shape[0]
        if what == "rope":
            batch.kv_len[0] = 19
        if what == "narrow":
            cos, sin = (torch.cat([t, t]) for t in (cos, sin))
            rows = cos.shape[0]
        q = torch.full((2, 4, 128), 9.0, device="cuda")
        ops.paged_append(cache, batch, x[:, 4:6].cuda(), x[:, 6:].cuda(), cos[:rows].contiguous().cuda(),
                         sin[:rows].contiguous().cuda(), q=x[:, :4].cuda(), q_out=q)
        assert lib().bg_device_status(None) == BG_EINVAL
        assert lib().bg_device_status(None) == 0
        row = int(table[0, 1]) * 16 + (2 if what == "rope" else 3)
        assert torch.equal(cache.V.cpu().view(-1, 2, 128)[row], x[0, 6:].half())
        flat = cache.V.cpu().view(-1, 256).clone()
        flat[row] = 0
        assert not flat.any()
        assert (q[1] == 9.0).all() == (what == "rope")


def test_graph_and_stream(ops):
    """A captured append follows kv_len; a side stream's append is ordered by that stream."""
    cache, batch, x, cos, sin, gam, table, tok, n = build(ops, [20, 40], [1, 1], 2, 4, 128, 16, "f16", 128)
    xd, c, s = x.cuda(), cos.cuda(), sin.cuda()
    g = ops.Graphed(lambda: ops.paged_append(cache, batch, xd[:, 4:6], xd[:, 6:], c, s, q=xd[:, :4]))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache.V.zero_()
        batch.kv_len.copy_(torch.tensor([5, 33]).int())
        q = g.replay()
    torch.cuda.synchronize()
    flat = cache.V.cpu().view(-1, 2, 128)
    for b, o in ((0, 4), (1, 32)):
        assert torch.equal(flat[int(table[b, o // 16]) * 16 + o % 16], x[b, 6:].half())
    want = norm_rope(x[:, :4], None, cos, sin, torch.tensor([4, 32]), EPS)
    assert (q.cpu().double() - want).abs().max() <= 24 * 2.0 ** -24 * want.abs().max()
