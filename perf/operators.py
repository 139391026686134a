"""Measured cases of the paged-cache operators: append with norm and rotation, attention over a paged
cache, and attention of a batch that shares a long prefix.

Layout.  A pool holds ``K, V [pages, page, kv_heads, head_dim]`` (f16, or int8 codes with one f32
scale per 32 values).  Sequence b's own position j lives in slot ``j % page`` of page
``table[b, j // page]``; with a shared prefix, position j < prefix lives in ``prefix_pages[j // page]``
and the own positions follow it.  ``cu[b] : cu[b + 1]`` are the token rows of sequence b, its newest.

Formulas, for token i of the n new tokens of a sequence with ``len`` own positions (the new ones
among them), own position ``o = len - n + i``:
  append     y = x / sqrt(mean(x^2) + eps) * gamma;  r = y * cos[p] + rotate_half(y) * sin[p] over the
             first ``rot`` dims, p = prefix + o;  K[slot(o)] = codec(r),  V[slot(o)] = codec(v)
  attention  out = softmax_j(q . K[j] * scale) . V[j] over the prefix and the own positions j <= o,
             times 1 / (1 + exp(-gate)) where a gate is given.

With ``own`` false the operators run as plain torch operations in 32 bits; with ``own`` true they run
through ``bitgpu_b200.ops``.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6


# ---- cases ---------------------------------------------------------------------------------------
def _case(op, name=None, batch=1, heads=32, kv=8, dim=128, page=16, mode="f16", io="f32", lo=1, hi=1, new=1,
          prefix=0, gate=False, norm=False, rot=0):
    c = dict(op=op, batch=batch, heads=heads, kv=kv, dim=dim, page=page, mode=mode, io=io, lo=lo, hi=hi, new=new,
             prefix=prefix, gate=gate, norm=norm, rot=rot)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of 32 streams: q and k normed and rotated, k and v into their pages
        _case("append", "append decode b32", batch=32, lo=40, hi=2000, norm=True, rot=128),
        # four prompts prefilled together into a q8 cache
        _case("append", "append prefill q8 8k", batch=4, page=64, mode="q8", io="f16", lo=2048, hi=2048, new=2048,
              norm=True, rot=128),
        # the gated hybrid layer: 256 wide heads of which 64 dims rotate, an odd ragged batch
        _case("append", "append hybrid d256", batch=7, heads=24, kv=4, dim=256, page=32, lo=301, hi=611, new=211,
              norm=True, rot=64),
        # one short chat turn, one stream: latency
        _case("attend", "decode b1 short", batch=1, lo=777, hi=777),
        # a full server: 64 streams of every length up to 32768
        _case("attend", "decode b64 32k", batch=64, io="f16", lo=64, hi=32768),
        # 32 streams over the quantised cache, the engine's own f32 rows
        _case("attend", "decode b32 q8 8k", batch=32, page=64, mode="q8", lo=500, hi=8192),
        # verification of drafted tokens, four at a time, 16 query heads over 8
        _case("attend", "verify b8 s4", batch=8, heads=16, page=32, lo=1000, hi=4100, new=4),
        # the gated hybrid layer over one long document
        _case("attend", "decode d256 gated 128k", batch=1, heads=24, kv=4, dim=256, page=64, lo=131072, hi=131072,
              gate=True),
        # chunked prefill beside running streams: three prompts and a few single tokens
        _case("attend", "prefill mixed 4k", batch=6, page=64, io="f16", lo=1500, hi=4096, new=2048),
        # a few streams behind one system prompt of odd length
        _case("prefix", "prefix b8 1k", batch=8, lo=3, hi=60, prefix=1000),
        # 64 answers drawn from one 8192 token prompt
        _case("prefix", "prefix b64 8k", batch=64, io="f16", page=64, lo=1, hi=512, prefix=8192),
        # 128 streams over one long quantised document
        _case("prefix", "prefix b128 q8 32k", batch=128, io="f16", page=64, mode="q8", lo=16, hi=1024, prefix=32768),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (24, 4, 256)])
    c = _case(op, heads=heads, kv=kv, dim=dim, page=rng.choice([16, 32, 64, 128]), mode=rng.choice(["f16", "q8"]),
              io=rng.choice(["f32", "f16"]))
    c["gate"] = op != "append" and dim == 256
    if op == "append":
        c["norm"] = rng.random() < 0.7
        c["rot"] = 64 if dim == 256 else dim
        c["new"] = _log(rng, 1, 2048)
        c["batch"] = _log(rng, 1, max(1, min(128, 8192 // c["new"])))
        c["lo"] = c["new"] + _log(rng, 1, 500) - 1
        c["hi"] = c["lo"] + _log(rng, 1, 1000)
    elif op == "attend":
        kind = rng.choice(["decode", "decode", "verify", "prefill"])
        c["new"] = 1 if kind == "decode" else rng.randint(2, 8) if kind == "verify" else _log(rng, 32, 1024)
        c["hi"] = _log(rng, 16, 32768 if kind == "decode" else 4096)
        c["hi"] = max(c["hi"], c["new"])
        room = 400000 if kind != "prefill" else 8192
        c["batch"] = _log(rng, 1, max(1, min(64 if kind != "prefill" else 8, room // c["hi"])))
        c["lo"] = max(c["new"], _log(rng, 1, c["hi"]))
    else:
        c["prefix"] = _log(rng, 100, 16384)
        c["batch"] = _log(rng, 2, 128)
        c["hi"] = _log(rng, 4, 512)
        c["lo"] = _log(rng, 1, c["hi"])
        c["new"] = 1 if rng.random() < 0.7 else min(c["lo"], rng.randint(2, 4))
    return c


def _lengths(c):
    """(own positions, new tokens) of every sequence: spread evenly over [lo, hi] in a scrambled order;
    the longest has ``hi``.  A mixed prefill (many new tokens) has single tokens between its prompts."""
    B = c["batch"]
    order = sorted(range(B), key=lambda i: (i * 0.6180339887498949) % 1.0)
    lens, news = [0] * B, [0] * B
    for rank, i in enumerate(order):
        f = rank / (B - 1) if B > 1 else 1.0
        lens[i] = int(round(c["lo"] + f * (c["hi"] - c["lo"])))
        n = c["new"]
        if n > 8:  # ragged prompts; a single token now and then
            n = 1 if c["op"] == "attend" and i % 2 else max(1, n - (i * n) // (4 * B))
        news[i] = min(n, lens[i])
    return lens, news


def work(c):
    lens, news = _lengths(c)
    H, KV, D, P, T = c["heads"], c["kv"], c["dim"], c["prefix"], sum(news)
    io = 4 if c["io"] == "f32" else 2
    row = KV * (D * 2 if c["mode"] == "f16" else D + D // 8)  # bytes of one position of K or V
    if c["op"] == "append":
        b = T * ((2 * H + 2 * KV) * D * io + 2 * row + c["rot"] * 8)
        return {"bytes": b, "flops": T * (H + KV) * (3 * c["rot"] + (4 * D if c["norm"] else 0))}
    pairs = sum(P * n + sum(length - n + i + 1 for i in range(n)) for length, n in zip(lens, news))
    b = 2 * row * (P + sum(lens)) + T * H * D * (2 * io + (4 if c["gate"] else 0))
    return {"bytes": b, "flops": 4 * D * H * pairs}


# ---- inputs --------------------------------------------------------------------------------------
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    lens, news = _lengths(c)
    B, H, KV, D, page = c["batch"], c["heads"], c["kv"], c["dim"], c["page"]
    T, P = sum(news), c["prefix"]
    counts = [-(-n // page) for n in lens]
    npre = -(-P // page)
    pages = sum(counts) + npre + 3
    ids = list(range(pages))
    rnd.shuffle(ids)
    table = torch.zeros(B, max(counts), dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    s = {"case": c, "lens": lens, "news": news}
    s["table"] = table.cuda()
    s["prefix_pages"] = torch.tensor(ids[at:at + npre], dtype=torch.int32).cuda() if P else None
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    s["cu"] = torch.tensor(cu, dtype=torch.int32).cuda()
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(news)).cuda()
    s["seq"] = seq                                                                    # sequence of each token
    s["own_pos"] = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, news)]).cuda()
    shape = (pages, page, KV, D)
    for name in ("K", "V"):
        if c["mode"] == "f16":
            s[name] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
            s[name + "s"] = None
        else:
            s[name] = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
            s[name + "s"] = torch.rand((pages, page, KV, D // 32), generator=g, device="cuda") + 1.0
    dt = torch.float32 if c["io"] == "f32" else torch.float16
    s["dtype"] = dt
    if c["op"] != "append":
        s["q"] = (1.5 * torch.randn((T, H, D), generator=g, device="cuda")).to(dt)
        s["gate"] = torch.randn((T, H, D), generator=g, device="cuda") if c["gate"] else None
        return s
    # one fused projection row per token: q heads (the hybrid's interleave a gate half), then k, then v
    qw = 2 * D if D == 256 else D
    x = torch.randn((T, H * qw + 2 * KV * D), generator=g, device="cuda").to(dt)
    s["q"] = x[:, :H * qw].view(T, H, qw)[..., :D]
    s["k"] = x[:, H * qw:H * qw + KV * D].view(T, KV, D)
    s["v"] = x[:, H * qw + KV * D:].view(T, KV, D)
    s["q_gamma"] = s["k_gamma"] = None
    if c["norm"]:
        s["q_gamma"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
        s["k_gamma"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    rot = c["rot"]
    inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    ang = torch.outer(torch.arange(max(lens) + P, dtype=torch.float64, device="cuda"), inv)
    s["cos"], s["sin"] = (torch.cat([f, f], -1).float() for f in (ang.cos(), ang.sin()))
    s["rows"] = s["table"][seq, s["own_pos"] // page].long() * page + s["own_pos"] % page  # pool row of each token
    return s


# ---- the framework's calls -----------------------------------------------------------------------
def _handles(s):
    """The cache and batch objects that a program builds once and keeps."""
    if "cache" not in s:
        from bitgpu_b200 import ops
        c = s["case"]
        s["ops"] = ops
        s["cache"] = ops.PagedKVCache.from_tensors(s["K"], s["V"], s["Ks"], s["Vs"])
        s["batch"] = ops.PagedBatch(s["table"], s["kv_len"], cu_q=None if max(s["news"]) == 1 else s["cu"],
                                    tokens=sum(s["news"]), max_q=max(s["news"]), prefix_pages=s["prefix_pages"],
                                    prefix_len=c["prefix"])
    return s["ops"], s["cache"], s["batch"]


def run(s):
    c = s["case"]
    if own:
        ops, cache, batch = _handles(s)
        if c["op"] == "append":
            q = ops.paged_append(cache, batch, s["k"], s["v"], cos=s["cos"], sin=s["sin"], k_gamma=s["k_gamma"],
                                 eps=EPS, q=s["q"], q_gamma=s["q_gamma"], q_dtype=s["dtype"])
        else:
            return ops.paged_attention(s["q"], cache, batch, gate=s["gate"], out_dtype=s["dtype"])
    else:
        if c["op"] != "append":
            return _plain_attention(s)
        q = _plain_append(s)
    if c["mode"] == "f16":
        return {"q": q, "K": s["K"], "V": s["V"]}
    return {"q": q, "K": _read_rows(s, "K").half(), "V": _read_rows(s, "V").half()}


# ---- plain forms ---------------------------------------------------------------------------------
def _read_rows(s, name):
    """The values that the written q8 rows stand for."""
    codes = s[name].flatten(0, 1)[s["rows"]].float()
    scale = s[name + "s"].flatten(0, 1)[s["rows"]]
    return (codes / 127).clamp(min=-1) * scale.repeat_interleave(32, -1)


def _plain_norm_rope(s, x, gamma):
    rot = s["case"]["rot"]
    y = x.float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma
    pos = s["own_pos"] + s["case"]["prefix"]
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    a = y[..., :rot]
    half = torch.cat([-a[..., rot // 2:], a[..., :rot // 2]], -1)
    return torch.cat([a * cos + half * sin, y[..., rot:]], -1)


def _plain_append(s):
    rows = s["rows"]
    for name, x in (("K", _plain_norm_rope(s, s["k"], s["k_gamma"])), ("V", s["v"].float())):
        pool = s[name].flatten(0, 1)
        if s["case"]["mode"] == "f16":
            pool[rows] = x.half()
        else:
            blocks = x.unflatten(-1, (-1, 32))
            scale = blocks.abs().amax(-1).clamp(min=1e-30)
            code = torch.floor(0.5 + 127 * (blocks / scale[..., None]).clamp(-1, 1)).flatten(-2)
            pool[rows] = code.to(torch.int8)
            s[name + "s"].flatten(0, 1)[rows] = scale
    return _plain_norm_rope(s, s["q"], s["q_gamma"]).to(s["dtype"])


def _plain_gather(s, name, rows):
    x = s[name].flatten(0, 1)[rows].float()
    if s["case"]["mode"] == "q8":
        x = (x / 127).clamp(min=-1) * s[name + "s"].flatten(0, 1)[rows].repeat_interleave(32, -1)
    return x


def _plain_attention(s):
    c = s["case"]
    B, H, KV, D, page, P = c["batch"], c["heads"], c["kv"], c["dim"], c["page"], c["prefix"]
    N, L, G = max(s["news"]), max(s["lens"]), H // KV
    dev = s["q"].device
    # queries padded to [B, N]
    step = torch.arange(N, device=dev)
    n = (s["cu"][1:] - s["cu"][:-1])[:, None]
    there = step < n
    rows = (s["cu"][:-1, None] + step).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(B, N, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * N, D)
    # own positions padded to [B, L]
    j = torch.arange(L, device=dev)
    slot = s["table"][:, j // page].long() * page + j % page
    slot = torch.where(j < s["kv_len"][:, None], slot, 0)
    k = _plain_gather(s, "K", slot).permute(0, 2, 3, 1)                              # [B, KV, D, L]
    score = torch.matmul(q, k) / math.sqrt(D)
    last = s["kv_len"][:, None] - n + step                                           # own position of a query
    score = score.view(B, KV, G, N, L).masked_fill((j > last[..., None])[:, None, None], -math.inf).flatten(2, 3)
    del k
    if P:
        i = torch.arange(P, device=dev)
        pslot = s["prefix_pages"][i // page].long() * page + i % page
        pk = _plain_gather(s, "K", pslot).permute(1, 2, 0)                           # [KV, D, P]
        qs = q.transpose(0, 1).reshape(KV, B * G * N, D)
        pscore = (torch.matmul(qs, pk) / math.sqrt(D)).view(KV, B, G * N, P).transpose(0, 1)
        score = torch.cat([pscore, score], -1)
        del pk, pscore
    p = torch.exp(score - score.amax(-1, keepdim=True))
    del score
    total = p.sum(-1, keepdim=True)
    v = _plain_gather(s, "V", slot).transpose(1, 2)                                  # [B, KV, L, D]
    out = torch.matmul(p[..., P:], v)
    del v
    if P:
        pv = _plain_gather(s, "V", pslot).transpose(0, 1)                            # [KV, P, D]
        front = p[..., :P].transpose(0, 1).reshape(KV, B * G * N, P)
        out = out + torch.matmul(front, pv).view(KV, B, G * N, D).transpose(0, 1)
    out = (out / total).view(B, KV, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)[there]
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"]))
    return out.to(s["dtype"])


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_values(s, name, rows):
    """Pool rows as the numbers that they stand for, in 64 bits."""
    c = s["case"]
    data = s[name].reshape(-1, c["kv"], c["dim"])[rows].double()
    if c["mode"] == "f16":
        return data
    scale = s[name + "s"].reshape(-1, c["kv"], c["dim"] // 32, 1)[rows].double()
    return (torch.clamp(data / 127.0, min=-1.0).view(-1, c["kv"], c["dim"] // 32, 32) * scale).view_as(data)


def _exact_row(s, x, gamma, t):
    """One token's heads [n, D], normed and rotated pair by pair."""
    rot = s["case"]["rot"]
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * gamma.double()
    h = rot // 2
    cos, sin = s["cos"][t].double()[..., None, :h], s["sin"][t].double()[..., None, :h]
    first, second = y[..., :h].clone(), y[..., h:rot].clone()
    y[..., :h] = first * cos - second * sin
    y[..., h:rot] = second * cos + first * sin
    return y


def exact(c, seed):
    s = prepare(c, seed)
    lens, news, page, P = s["lens"], s["news"], c["page"], c["prefix"]
    table = s["table"].tolist()
    if c["op"] == "append":
        pos = torch.cat([torch.arange(P + L - n, P + L) for L, n in zip(lens, news)]).cuda()
        rows = torch.tensor([table[b][o // page] * page + o % page for b, (L, n) in enumerate(zip(lens, news))
                             for o in range(L - n, L)], device="cuda")
        out = {"q": _exact_row(s, s["q"], s["q_gamma"], pos)}
        for name, x in (("K", _exact_row(s, s["k"], s["k_gamma"], pos)), ("V", s["v"].double())):
            if c["mode"] == "f16":
                pool = s[name].double()
                pool.view(-1, c["kv"], c["dim"])[rows] = x
                out[name] = pool
            else:
                blk = x.reshape(x.shape[0], c["kv"], -1, 32)
                scale = blk.abs().max(-1, keepdim=True).values.clamp(min=1e-30)
                code = torch.floor(127.0 * (blk / scale) + 0.5)
                out[name] = (torch.clamp(code / 127.0, min=-1.0) * scale).reshape(x.shape)
        return out
    if work(c)["flops"] > 3e12:
        return None
    G, D = c["heads"] // c["kv"], c["dim"]
    pre = s["prefix_pages"].tolist() if P else []
    prow = torch.tensor([pre[j // page] * page + j % page for j in range(P)], dtype=torch.long, device="cuda")
    pk = _exact_values(s, "K", prow).permute(1, 2, 0)
    pv = _exact_values(s, "V", prow).transpose(0, 1)
    outs, t = [], 0
    for b, (L, n) in enumerate(zip(lens, news)):
        idx = torch.arange(L, device="cuda")
        rows = s["table"][b].long()[idx // page] * page + idx % page
        k = torch.cat([pk, _exact_values(s, "K", rows).permute(1, 2, 0)], -1)         # [KV, D, P + L]
        v = torch.cat([pv, _exact_values(s, "V", rows).transpose(0, 1)], 1)           # [KV, P + L, D]
        for a in range(0, n, 256):                                                   # a block of tokens at a time
            m = min(256, n - a)
            q = s["q"][t + a:t + a + m].double().view(m, c["kv"], G, D).permute(1, 2, 0, 3).reshape(c["kv"], G * m, D)
            z = (q @ k * D ** -0.5).view(c["kv"], G, m, P + L)
            lim = P + L - n + a + torch.arange(m, device="cuda")
            z = torch.where(torch.arange(P + L, device="cuda") <= lim[:, None], z, -math.inf)
            w = torch.softmax(z, -1).view(c["kv"], G * m, P + L)
            o = (w @ v).view(c["kv"], G, m, D).permute(2, 0, 1, 3).reshape(m, c["heads"], D)
            if c["gate"]:
                o = o * torch.sigmoid(s["gate"][t + a:t + a + m].double())
            outs.append(o)
        t += n
    return torch.cat(outs)
