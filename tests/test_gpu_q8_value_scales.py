"""Decode over dense q8 caches whose V is small, large or of mixed magnitude, against 64 bits: block scales are f32,
and the weights (p times V's scale) that enter the tensor cores as f16 keep 11 bits whatever the scales."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from bitgpu_b200 import ops
    return ops


def case(ops, D, B, G, factor, roll=False, gate=False, L=1500, KV=2, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, dev = KV * G, "cuda"
    cache = ops.KVCache(B, L, KV, D, "q8")
    cache.K.copy_(torch.randint(-127, 128, cache.K.shape, generator=g, device=dev))
    cache.Ks.copy_(torch.rand(cache.Ks.shape, generator=g, device=dev) + 0.5)
    cache.V.copy_(torch.randint(-127, 128, cache.V.shape, generator=g, device=dev))
    cache.Vs.copy_((torch.rand(cache.Vs.shape, generator=g, device=dev) + 1.0) * factor(cache.Vs.shape, g))
    q = torch.randn((B, 1, H, D), generator=g, device=dev) * 0.1
    gt = torch.randn(q.shape, generator=g, device=dev) if gate else None
    cos = sin = None
    if roll:
        a = torch.outer(torch.arange(L + 8, device=dev).double(), 1e6 ** (-torch.arange(0, D, 2, device=dev).double() / D))
        cos, sin = a.cos().float(), a.sin().float()
    out = ops.attention(q, cache, L - 1, gate=gt, cos_t=cos, sin_t=sin).double()
    K, V = (c.double() / 127 * s.double().repeat_interleave(32, -1) for c, s in ((cache.K, cache.Ks), (cache.V, cache.Vs)))
    if roll:
        c, s, h = cos[:L, None].double(), sin[:L, None].double(), D // 2
        K = torch.cat([K[..., :h] * c - K[..., h:] * s, K[..., h:] * c + K[..., :h] * s], -1)
    qq = q.double().view(B, KV, G, D)
    sc = torch.einsum("bkgd,bjkd->bkgj", qq, K) * D ** -0.5
    S = float(torch.einsum("bkgd,bjkd->bkgj", qq.abs(), K.abs()).max()) * D ** -0.5
    p = torch.softmax(sc, -1)

    def mix(x):
        y = torch.einsum("bkgj,bjkd->bkgd", p, x).reshape(q.shape)
        return y * torch.sigmoid(gt.double()) if gate else y
    want, A = mix(V), mix(V.abs())
    scale = mix(cache.Vs.double().repeat_interleave(32, -1))
    # a weight is rounded to 11 bits; scores are f32 sums of 22-bit products (rope at read: of K rounded to f16 once
    # more, 2^-11 of at most S); codes enter as code + 1152, which the accumulator holds and loses again: two roundings
    # of 1152 / 127 scales at 2^-23; a weight below 2^-14 / 2^13 of a block's largest has f16's absolute step, 2^-38 of it
    tol = (2.0 ** -11 + (28 * S + 16) * 2.0 ** -24) * A + 20 * 2.0 ** -23 * scale
    if roll:
        tol = tol + 2 * 2.0 ** -11 * S * A
    top = cache.Vs.double().amax((0, 1)).repeat_interleave(32, -1).repeat_interleave(G, 0).view(1, 1, H, D)
    err = (out - want).abs()
    assert torch.isfinite(out).all()
    worst = float((err / (tol + L * 2.0 ** -38 * top)).max())
    assert worst <= 1, f"{worst:.3g} of what is allowed, {float((err.norm() / want.norm())):.3g} of the norm"


@pytest.mark.parametrize("vs", [1e-20, 1e-6, 1e-4, 1e-3, 1.0, 1e4, 1e8, 1e20])
@pytest.mark.parametrize("D,B,G", [(128, 1, 4), (128, 3, 8), (128, 2, 12), (256, 2, 6), (256, 40, 4)])
def test_decode(ops, vs, D, B, G):
    case(ops, D, B, G, lambda shape, g: vs, gate=D == 256)


@pytest.mark.parametrize("vs", [1e-20, 1e-4, 1.0, 1e8])
@pytest.mark.parametrize("B,G", [(1, 4), (16, 8), (3, 2)])
def test_rope_at_read(ops, vs, B, G):
    case(ops, 128, B, G, lambda shape, g: vs, roll=True)


@pytest.mark.parametrize("roll", [False, True])
@pytest.mark.parametrize("by", ["block", "position"])
def test_mixed(ops, by, roll):
    """Blocks ten decimal orders apart, and positions three."""
    def factor(shape, g):
        if by == "block":
            return 10.0 ** torch.linspace(-8, 2, shape[-1], device="cuda")
        return 10.0 ** (3 * torch.rand(shape, generator=g, device="cuda") - 1.5)
    case(ops, 128, 2, 4, factor, roll=roll)


def test_rising(ops):
    """Scales that double every 50 positions, and halve."""
    for sign in (1, -1):
        case(ops, 128, 2, 4, lambda shape, g: torch.exp2(sign * (torch.arange(shape[1], device="cuda") // 50 - 15.0))[None, :, None, None])
