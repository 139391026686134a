"""Decode kernels stream K and V through a ring in shared memory: a stage that were refilled before all of it is read
would show as results that change from call to call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from bitgpu_b200 import ops
    return ops


def same(call, times=60):
    first = call().clone()
    assert torch.isfinite(first).all()
    assert sum(not torch.equal(call(), first) for _ in range(times)) == 0


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("B,H,KV,D,L,roll", [(64, 32, 8, 128, 16384, False), (8, 32, 8, 128, 32768, False),
                                             (2, 24, 4, 256, 32768, False), (16, 32, 8, 128, 8192, True)])
def test_dense_decode(ops, mode, B, H, KV, D, L, roll):
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = ops.KVCache(B, L, KV, D, mode)
    for which in (0, 1):
        cache.append(which, torch.randn((B, L, KV, D), generator=g, device="cuda"), 0)
    q = torch.randn((B, 1, H, D), generator=g, device="cuda")
    cos = sin = None
    if roll:
        a = torch.outer(torch.arange(L + 8, device="cuda").double(), 1e6 ** (-torch.arange(0, D, 2, device="cuda").double() / D))
        cos, sin = a.cos().float(), a.sin().float()
    same(lambda: ops.attention(q, cache, L - 1, cos_t=cos, sin_t=sin))


@pytest.mark.parametrize("mode", ["f16", "q8"])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("D,G,new", [(128, 4, 1), (128, 6, 1), (128, 4, 3), (256, 6, 1), (128, 4, 60)])
def test_paged(ops, mode, io, D, G, new):
    KV, page, L, B = 8, 16, 16384, 12
    g = torch.Generator(device="cuda").manual_seed(6)
    pages = B * L // page
    cache = ops.PagedKVCache(pages, page, KV, D, mode)
    if mode == "q8":
        cache.K.random_(-127, 128, generator=g)
        cache.V.random_(-127, 128, generator=g)
        cache.Ks.uniform_(0.5, 1.5, generator=g)
        cache.Vs.uniform_(0.5, 1.5, generator=g)
    else:
        cache.K.normal_(generator=g)
        cache.V.normal_(generator=g)
    table = torch.randperm(pages, generator=g, device="cuda").int().view(B, L // page)
    lens = torch.tensor([L - 997 * b for b in range(B)], dtype=torch.int32, device="cuda")
    batch = ops.PagedBatch(table, lens, torch.arange(0, new * B + 1, new, dtype=torch.int32, device="cuda"), new * B, new)
    q = torch.randn((new * B, KV * G, D), generator=g, device="cuda").to(io)
    same(lambda: ops.paged_attention(q, cache, batch, out_dtype=io), 30)
