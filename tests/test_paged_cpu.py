"""Refusals of the paged-cache operators, checked before any CUDA call: the C entry points on made-up
pointers, and the Python objects."""
import ctypes as C

import pytest
import torch

from bitgpu_b200 import _lib, ops
from bitgpu_b200._lib import BG_EINVAL, BG_ENOMEM, BG_EUNSUPPORTED, BG_OK, PagedBatchDesc, PagedCacheDesc, Rows, lib

A = 1 << 20  # an aligned address that nothing is at


def cache(**kw):
    d = dict(K=A, V=A, Ks=None, Vs=None, num_pages=8, page_size=16, mode=_lib.KV_F16)
    d.update(kw)
    return PagedCacheDesc(*[d[n] for n, _ in PagedCacheDesc._fields_])


def batch(**kw):
    d = dict(cu_q=None, kv_len=A, page_table=A, prefix_pages=None, batch=2, tokens=2, max_q=1, table_stride=64, prefix_len=0)
    d.update(kw)
    return PagedBatchDesc(*[d[n] for n, _ in PagedBatchDesc._fields_])


def attend(c, b, H=8, KV=2, D=128, q=A, qd=0, gate=None, out=A, od=0, ws=A, wb=0):
    return lib().bg_paged_attention(C.byref(c) if c else None, C.byref(b) if b else None, H, KV, D, q, qd, 0.0, gate, out,
                                    od, ws, wb, None)


def append(c, b, H=8, KV=2, D=128, q=None, k=A, v=A, sd=0, cos=None, sin=None, rot=0, q_out=None, od=0):
    r = [C.byref(Rows(x, 1, 1)) if x is not None else None for x in (q, k, v)]
    return lib().bg_paged_append(C.byref(c), C.byref(b), H, KV, D, *r, sd, None, None, 1e-6, cos, sin, rot, 64, q_out, od,
                                 None)


BAD_SHARED = [
    (dict(K=None), {}, BG_EINVAL), (dict(V=None), {}, BG_EINVAL), (dict(K=A + 8), {}, BG_EINVAL),
    (dict(num_pages=0), {}, BG_EINVAL), (dict(num_pages=1 << 31), {}, BG_EINVAL), (dict(page_size=0), {}, BG_EINVAL),
    (dict(mode=_lib.KV_Q8), {}, BG_EINVAL), (dict(mode=_lib.KV_Q8, Ks=A, Vs=A + 4), {}, BG_EINVAL),
    (dict(mode=_lib.KV_Q8R, Ks=A, Vs=A), {}, BG_EUNSUPPORTED), (dict(mode=9), {}, BG_EINVAL),
    ({}, dict(kv_len=None), BG_EINVAL), ({}, dict(page_table=None), BG_EINVAL), ({}, dict(table_stride=0), BG_EINVAL),
    ({}, dict(max_q=0), BG_EINVAL), ({}, dict(tokens=3), BG_EINVAL), ({}, dict(prefix_len=1), BG_EINVAL),
    ({}, dict(table_stride=1 << 27), BG_EINVAL), ({}, dict(prefix_len=(1 << 31) - 64, prefix_pages=A), BG_EINVAL),
]


@pytest.mark.parametrize("ckw,bkw,code", BAD_SHARED)
def test_shared_refusals(ckw, bkw, code):
    assert attend(cache(**ckw), batch(**bkw)) == code
    assert append(cache(**ckw), batch(**bkw)) == code
    assert lib().bg_paged_attention_workspace_size(C.byref(cache(**ckw)), C.byref(batch(**bkw)), 8, 2, 128) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(H=7), BG_EINVAL), (dict(H=0), BG_EINVAL), (dict(KV=0), BG_EINVAL), (dict(D=96), BG_EUNSUPPORTED),
    (dict(q=None), BG_EINVAL), (dict(out=None), BG_EINVAL), (dict(qd=2), BG_EINVAL), (dict(od=2), BG_EINVAL),
    (dict(q=A + 4), BG_EINVAL), (dict(out=A + 8), BG_EINVAL), (dict(gate=A + 4), BG_EINVAL), (dict(ws=A + 4), BG_EINVAL),
    (dict(wb=0), BG_ENOMEM), (dict(ws=None, wb=1 << 30), BG_ENOMEM),
])
def test_attention_refusals(kw, code):
    assert attend(cache(), batch(), **kw) == code


def test_workspace_is_needed_whole():
    n = lib().bg_paged_attention_workspace_size(C.byref(cache()), C.byref(batch()), 8, 2, 128)
    assert n > 0 and attend(cache(), batch(), wb=n - 1) == BG_ENOMEM


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), BG_EINVAL), (dict(v=None), BG_EINVAL), (dict(sd=2), BG_EINVAL), (dict(od=2), BG_EINVAL),
    (dict(q=A), BG_EINVAL), (dict(q=A, q_out=A, H=0), BG_EINVAL), (dict(q=A, q_out=A + 4), BG_EINVAL),
    (dict(cos=A), BG_EINVAL), (dict(cos=A, sin=A), BG_EINVAL), (dict(cos=A, sin=A, rot=3), BG_EINVAL),
    (dict(cos=A, sin=A, rot=130), BG_EINVAL), (dict(cos=A + 4, sin=A, rot=64), BG_EINVAL), (dict(D=80), BG_EUNSUPPORTED),
    (dict(KV=0), BG_EINVAL),
])
def test_append_refusals(kw, code):
    assert append(cache(), batch(), **kw) == code


def test_empty_calls():
    for b in (batch(batch=0, tokens=0), batch(batch=3, tokens=0, cu_q=A)):
        assert attend(cache(), b, q=None, out=None) == BG_OK
        assert append(cache(), b) == BG_OK


def test_python_refusals():
    with pytest.raises(ValueError):
        ops.PagedKVCache(4, 16, 2, 128, "q8r", device="cpu")
    with pytest.raises(ValueError):
        ops.PagedKVCache(0, 16, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKVCache.from_tensors(torch.zeros(2, 16, 2, 128), torch.zeros(2, 16, 2, 128))
    with pytest.raises(ValueError):
        ops.PagedKVCache.from_tensors(torch.zeros(2, 16, 2, 128).bfloat16(), torch.zeros(2, 16, 2, 128).bfloat16())
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_find_seq_search():
    """The kernels' 32-way search over cu_q, step by step on the CPU: every probe stays inside the
    array and the last sequence that begins at or before the token is found."""
    def find(cu, t):
        lo, n, B = 0, len(cu), len(cu) - 1
        while True:
            step = (n + 31) // 32
            probe = [lo + i * step for i in range(32)]
            le = [i < lo + n and cu[i] <= t for i in probe]
            assert all(i < len(cu) for i in probe if i < lo + n)
            cnt = sum(le)
            if cnt == 0:
                return -1
            lo += (cnt - 1) * step
            if step == 1:
                return lo if lo < B else -1
            n = min(step, B + 1 - lo)

    for B in (1, 2, 31, 32, 33, 100, 1023, 1024, 1025, 5000):
        cu = [0]
        for i in range(B):
            cu.append(cu[-1] + (i * 7) % 3)
        for t in list(range(0, cu[-1] + 2, max(1, cu[-1] // 50))) + [cu[-1] - 1, cu[-1]]:
            want = max((b for b in range(B) if cu[b] <= t), default=-1) if t < cu[-1] else -1
            assert find(cu, t) == want or t < 0, (B, t)


@pytest.mark.parametrize("scale", [-0.1, float("nan"), float("inf"), -float("inf")])
def test_scale_refusals(scale):
    assert lib().bg_paged_attention(C.byref(cache()), C.byref(batch()), 8, 2, 128, A, 0, scale, None, A, 0, A, 1 << 30,
                                    None) == BG_EINVAL
