"""What the 8-bit key/value cache is timed on: the write behind the QKV projection (rotation, then one
power-of-two scale per row), the read back, decode attention and chunk attention over its pages.

The cache.  A row is the D values of one token and kv head.  With amax its largest magnitude, e is the
smallest whole number for which amax / 2^e <= 448, held to [-100, 119]; the row is kept as the e4m3 codes of
x / 2^e (nearest, ties to even) and one byte e + 127.  Pages: keys ``k[page, head, token, D]``, values
``v[page, head, token // 16, D, token % 16]``, one byte a row ``k_scale`` / ``v_scale[page, head, token]``.

A case names a direction (``"op"``) and the layer's sizes; ``"mix"`` says how lengths spread.  Activations are
bf16, the type models are served in.  Sizes are those of the model catalogue's layers.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BF = torch.bfloat16
F8 = torch.float8_e4m3fn


def listed():
    return [
        # one decode step of 32 chat users writes its keys and values: latency
        dict(name="append_32", op="append", heads=32, kv_heads=8, dim=128, page=128, tokens=32, past=700,
             bias=False, norm=False, mix=1),
        # a prompt portion of 4096 tokens, the usual budget of a step
        dict(name="append_4096", op="append", heads=32, kv_heads=8, dim=128, page=128, tokens=4096, past=4096,
             bias=False, norm=False, mix=2),
        # an odd portion of a layer with a bias and per-head norms of queries and keys
        dict(name="append_norm_777", op="append", heads=28, kv_heads=4, dim=128, page=64, tokens=777, past=130,
             bias=True, norm=True, mix=3),
        # a cached prefix of about a page and a half, handed on in the model's type
        dict(name="read_200", op="read", heads=32, kv_heads=8, dim=128, page=128, tokens=200, mix=4),
        # a cached document, handed on
        dict(name="read_32768", op="read", heads=32, kv_heads=8, dim=128, page=128, tokens=32768, mix=5),
        # one interactive user in a long conversation
        dict(name="decode_1", op="decode", heads=32, kv_heads=8, dim=128, page=128, rows=1, ctx=4000, window=0, mix=6),
        # 65 chat users, ragged
        dict(name="decode_65", op="decode", heads=32, kv_heads=8, dim=128, page=128, rows=65, ctx=2000, window=0, mix=7),
        # 32 users with long documents
        dict(name="decode_long", op="decode", heads=32, kv_heads=8, dim=128, page=128, rows=32, ctx=16384, window=0, mix=8),
        # a layer with a sliding window and heads of 64, small pages
        dict(name="decode_window", op="decode", heads=16, kv_heads=4, dim=64, page=16, rows=48, ctx=5000, window=1024, mix=9),
        # eight users whose five drafted tokens are scored over their contexts
        dict(name="chunk_drafts", op="chunk", heads=32, kv_heads=8, dim=128, page=128, seqs=8, tokens=5, past=3000, window=0,
             causal=True, mix=10),
        # one long prompt in one step
        dict(name="chunk_8192", op="chunk", heads=32, kv_heads=8, dim=128, page=128, seqs=1, tokens=8192, past=0, window=0,
             causal=True, mix=11),
        # ragged portions behind cached contexts, seven heads to a kv head
        dict(name="chunk_ragged", op="chunk", heads=28, kv_heads=4, dim=128, page=64, seqs=6, tokens=701, past=1500, window=0,
             causal=True, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "chunk", "chunk"])
    h, g, d = rng.choice([(32, 8, 128), (28, 4, 128), (40, 8, 128), (16, 4, 128), (8, 1, 128), (12, 12, 64), (16, 4, 64), (12, 4, 256)])
    c = dict(op=op, heads=h, kv_heads=g, dim=d, page=rng.choice([128, 128, 64, 16]), mix=rng.randrange(1 << 16))
    if op == "append":
        c.update(tokens=_log(rng, 1, 4096 * 4096 // (h * d)), past=_log(rng, 1, 20000), bias=rng.random() < 0.3, norm=rng.random() < 0.3)
    elif op == "read":
        c.update(tokens=_log(rng, 1, (1 << 25) // (g * d)))
    elif op == "decode":
        rows = _log(rng, 1, 128)
        c.update(rows=rows, ctx=_log(rng, 1, min(32768, (1 << 28) // (rows * g * d))), window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))
    else:
        seqs = _log(rng, 1, 16)
        tokens = _log(rng, 1, 4096 // seqs)
        past = rng.choice([0, _log(rng, 1, min(16000, (1 << 24) // (seqs * tokens)))])
        c.update(seqs=seqs, tokens=tokens, past=past, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), causal=rng.random() < 0.9)
        if not c["causal"]:
            c["window"] = 0
    return c


# ------------------------------------------------------------------------------ inputs
def _lens(c):
    """(new tokens, tokens in the cache with them) of every sequence."""
    r = random.Random(c["mix"])
    if c["op"] == "decode":
        ctx = [c["ctx"]] + [r.randint(max(1, c["ctx"] // 2), c["ctx"]) for _ in range(c["rows"] - 1)]
        return [1] * c["rows"], ctx
    new = [c["tokens"]] + [r.randint(max(1, c["tokens"] // 2), c["tokens"]) for _ in range(c["seqs"] - 1)]
    past = [c["past"]] + [r.randint(c["past"] // 2, c["past"]) for _ in range(c["seqs"] - 1)]
    return new, [n + p for n, p in zip(new, past)]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _two_to(e):
    """2^e in fp32 for whole e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _rows8(x):
    """fp32 rows -> (e4m3 codes, a byte a row)."""
    mant, ex = torch.frexp(x.abs().amax(-1))
    e = (ex - 9 + (mant > 0.875)).clamp(-100, 119)
    return (x * _two_to(-e).unsqueeze(-1)).clamp(-448, 448).to(F8), (e + 127).to(torch.uint8)


def _pages(c, g, pages):
    """Key and value pages as earlier steps have left them: channels of unlike size, tokens of unlike size."""
    hk, d, bs = c["kv_heads"], c["dim"], c["page"]
    k = torch.empty(pages, hk, bs, d, dtype=F8, device="cuda")
    v = torch.empty(pages, hk, bs // 16, d, 16, dtype=F8, device="cuda")
    ks, vs = (torch.empty(pages, hk, bs, dtype=torch.uint8, device="cuda") for _ in range(2))
    wide = torch.exp(0.5 * _randn(g, hk, 1, d))
    step = max(1, (1 << 26) // (hk * bs * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        k[p:p + n], ks[p:p + n] = _rows8(_randn(g, n, hk, bs, d) * wide)
        code, vs[p:p + n] = _rows8(_randn(g, n, hk, bs, d) * torch.exp(0.7 * _randn(g, n, hk, bs, 1)))
        v[p:p + n] = code.view(torch.uint8).view(n, hk, bs // 16, 16, d).transpose(3, 4).contiguous().view(F8)
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def _tables(c, g, lens):
    """Every sequence's pages, at random places of the pool -> (tables, pages of the pool)."""
    bs = c["page"]
    need = [-(-n // bs) for n in lens]
    total = sum(need) + 2
    order = torch.randperm(total, generator=torch.Generator().manual_seed(c["mix"])).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    return table, total


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:                          # what a program keeps: its layer's cache, its model's table, a step's work list
        from enterprise_inference_amd.ops import quant_cache as Q
        from enterprise_inference_amd.ops.rotary import RotaryCache
        c = case
        s["cache"] = Q.QuantKVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if c["op"] == "append":
            s["rotary"] = RotaryCache.from_table(s["cos_sin"])
        if c["op"] == "chunk":
            s["plan"] = Q.quant_prefill_plan(*_lens(c), c["heads"], c["kv_heads"], c["dim"], "cuda", causal=c["causal"],
                                             sliding_window=c["window"] or None)
    return s


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, hk, d, bs = c["heads"], c["kv_heads"], c["dim"], c["page"]
    s = dict(case=c)
    if c["op"] in ("append", "read"):
        n = c["tokens"]
        table, pages = _tables(c, g, [n])
        t = torch.arange(n)
        slots = (torch.tensor(table[0])[t // bs] * bs + t % bs).to(torch.int32).cuda()
        s.update(slots=slots)
        if c["op"] == "read":
            return s | _pages(c, g, pages)
        s.update(k=torch.zeros(pages, hk, bs, d, dtype=torch.uint8, device="cuda").view(F8),
                 v=torch.zeros(pages, hk, bs // 16, d, 16, dtype=torch.uint8, device="cuda").view(F8),
                 k_scale=torch.zeros(pages, hk, bs, dtype=torch.uint8, device="cuda"),
                 v_scale=torch.zeros(pages, hk, bs, dtype=torch.uint8, device="cuda"))
        s["qkv"] = (_randn(g, n, (h + 2 * hk) * d) * torch.exp(0.5 * _randn(g, (h + 2 * hk) * d))).to(BF)
        s["positions"] = torch.arange(c["past"], c["past"] + n, dtype=torch.int32, device="cuda")
        ang = torch.arange(c["past"] + n, dtype=torch.float64, device="cuda")[:, None] * torch.pow(
            500000.0, -torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        s["bias"] = _randn(g, (h + 2 * hk) * d).to(BF) if c["bias"] else None
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * _randn(g, d)).to(BF) if c["norm"] else None for _ in range(2))
        return s
    new, lens = _lens(c)
    table, pages = _tables(c, g, lens)
    s |= _pages(c, g, pages)
    s["tables"], s["lens"] = _i32(table), _i32(lens)
    s["q"] = (1.3 * _randn(g, sum(new), h, d)).to(BF)
    if c["op"] == "chunk":
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu_q"], s["most"] = _i32(cu), max(new)
    return s


# ------------------------------------------------------------------------------ plain forms
def _values(code, scale):
    """Codes [..., D] and a byte a row -> fp32 values."""
    return code.float() * _two_to(scale.to(torch.int32) - 127).unsqueeze(-1)


def _read(s):
    bs = s["case"]["page"]
    p, t = s["slots"].long() // bs, s["slots"].long() % bs
    k = s["k"].view(torch.uint8)[p, :, t].view(F8)
    v = s["v"].view(torch.uint8)[p, :, t // 16, :, t % 16].view(F8)
    return _values(k, s["k_scale"][p, :, t]).to(BF), _values(v, s["v_scale"][p, :, t]).to(BF)


def _append(s):
    c = s["case"]
    h, hk, d, bs = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].float()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    x = x.view(-1, h + 2 * hk, d)
    qk, v = x[:, :h + hk], x[:, h + hk:]
    if s["q_norm"] is not None:
        w = torch.cat([s["q_norm"].float().expand(h, d), s["k_norm"].float().expand(hk, d)])
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * w
    cs = s["cos_sin"][s["positions"].long()].unsqueeze(1)
    cos, sin = cs[..., :d // 2], cs[..., d // 2:]
    a, b = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    p, t = s["slots"].long() // bs, s["slots"].long() % bs
    code, byte = _rows8(qk[:, h:])
    s["k"].view(torch.uint8)[p, :, t] = code.view(torch.uint8)
    s["k_scale"][p, :, t] = byte
    code, byte = _rows8(v)
    s["v"].view(torch.uint8)[p, :, t // 16, :, t % 16] = code.view(torch.uint8)
    s["v_scale"][p, :, t] = byte
    return (qk[:, :h].to(BF), *_read(s))


def _attend(q, s, kmax, klo):
    """q fp32 [S, Q, H, D] over the pages; a query sees the keys klo <= j <= kmax ([S, Q])."""
    c = s["case"]
    hk, d, bs = c["kv_heads"], c["dim"], c["page"]
    S, Q, H, _ = q.shape
    at = s["tables"].long()
    n = at.shape[1] * bs
    k = _values(s["k"].view(torch.uint8)[at].view(F8), s["k_scale"][at]).transpose(1, 2).reshape(S, hk, n, d)
    v = s["v"].view(torch.uint8)[at].transpose(-1, -2).contiguous().view(F8).view(S, -1, hk, bs, d)
    v = _values(v, s["v_scale"][at]).transpose(1, 2).reshape(S, hk, n, d)
    q = q.view(S, Q, hk, H // hk, d).permute(0, 2, 3, 1, 4).reshape(S, hk, -1, d)
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(d ** -0.5).view(S, hk, H // hk, Q, n)
    j = torch.arange(n, device="cuda")
    seen = (j <= kmax.unsqueeze(-1)) & (j >= klo.unsqueeze(-1))
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    sc = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(sc.view(S, hk, -1, n), v).view(S, hk, H // hk, Q, d) / sc.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(S, Q, H, d)


def _first(c, at):
    return (at - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(at)


def _decode(s):
    at = s["lens"].long().unsqueeze(1) - 1
    return _attend(s["q"].float().unsqueeze(1), s, at, _first(s["case"], at)).squeeze(1).to(BF)


def _chunk(s):
    c = s["case"]
    cu, lens = s["cu_q"].long(), s["lens"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["most"], device="cuda")
    row = torch.minimum(cu[:-1, None] + i, cu[1:, None] - 1)
    at = (lens - new)[:, None] + torch.minimum(i, new[:, None] - 1)
    kmax = at if c["causal"] else (lens[:, None] - 1).expand_as(at)
    o = _attend(s["q"].float()[row], s, kmax, _first(c, at)).to(BF)
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.bucketize(t, cu[1:], right=True)
    return o[seq, t - cu[seq]]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _append, "read": _read, "decode": _decode, "chunk": _chunk}[c["op"]](s)
    from enterprise_inference_amd.ops import quant_cache as Q
    cache = s["cache"]
    if c["op"] == "append":
        q = Q.rope_qkv_quant(s["qkv"], s["positions"], s["rotary"], s["slots"], cache, c["heads"], c["kv_heads"], c["dim"],
                             bias=s["bias"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], norm_eps=1e-6)
        return (q, *Q.quant_read(cache, s["slots"]))
    if c["op"] == "read":
        return Q.quant_read(cache, s["slots"])
    if c["op"] == "decode":
        return Q.quant_decode(s["q"], cache, s["tables"], s["lens"], c["dim"] ** -0.5, sliding_window=c["window"] or None)
    return Q.quant_prefill(s["q"], cache, s["tables"], s["lens"], s["cu_q"], s["plan"], c["dim"] ** -0.5)


# ------------------------------------------------------------------------------ what a pass cannot do without
def _seen(c):
    """(keys that some query of a sequence sees, query-key pairs) over all sequences."""
    keys = pairs = 0
    for n, total in zip(*_lens(c)):
        past, w = total - n, c["window"] or total
        if not c.get("causal", True):
            keys, pairs = keys + total, pairs + n * total
            continue
        keys += total - max(0, past - w + 1)
        full = max(0, min(n, w - 1 - past))                      # queries that see all before them
        pairs += full * past + full * (full + 1) // 2 + (n - full) * w
    return keys, pairs


def work(case):
    c = case
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] in ("append", "read"):
        n = c["tokens"]
        back = n * (4 + 2 * hk * (d + 1) + 2 * hk * d * 2)        # slots, rows, values
        if c["op"] == "read":
            return {"bytes": back, "flops": 2 * n * hk * d}
        new = n * ((h + 2 * hk) * d * 2 + 4 * d + 8 + h * d * 2 + 2 * hk * (d + 1))
        return {"bytes": new + back, "flops": n * (h + hk) * d * 3 + 4 * n * hk * d}
    new, _ = _lens(c)
    keys, pairs = _seen(c)
    return {"bytes": keys * 2 * hk * (d + 1) + 2 * sum(new) * h * d * 2 + 4 * keys // c["page"], "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------------------ 64 bits
def _pow2(e):
    """2^e in float64, from its bits (a power function may be off by its last one)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _e4m3(byte):
    """The number an e4m3 byte stands for, from its bits."""
    b = byte.to(torch.int64)
    ex, m = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(ex == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * _pow2(ex - 7))
    return torch.where(b >= 128, -mag, mag)


def _kept(x):
    """What a row of float64 values reads back as."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -100)))
    e = torch.where(amax > 448 * _pow2(e), e + 1, torch.where((amax <= 224 * _pow2(e)) & (e > -100), e - 1, e))
    y = x / _pow2(e)
    step = _pow2(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return torch.round(y / step) * step * _pow2(e)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    h, hk, d, bs = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["op"] == "append":
        n = c["tokens"]
        x = s["qkv"].double()
        x = (x + s["bias"].double() if c["bias"] else x).reshape(n, h + 2 * hk, d)
        parts = []
        for head in range(h + hk):
            y = x[:, head]
            if c["norm"]:
                y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + 1e-6) * (s["q_norm"] if head < h else s["k_norm"]).double()
            turn = torch.complex(*s["cos_sin"].double()[s["positions"].long()].chunk(2, 1))
            z = torch.complex(y[:, :d // 2].contiguous(), y[:, d // 2:].contiguous()) * turn
            parts.append(torch.cat([z.real, z.imag], 1))
        return torch.stack(parts[:h], 1), _kept(torch.stack(parts[h:], 1)), _kept(x[:, h + hk:])
    k = _e4m3(s["k"].view(torch.uint8)) * _pow2(s["k_scale"].int() - 127).unsqueeze(-1) if c["op"] != "read" else None
    if c["op"] == "read":
        got = []
        for name in ("k", "v"):
            byte, sc = s[name].view(torch.uint8), s[name + "_scale"]
            if name == "v":
                byte = byte.permute(0, 1, 2, 4, 3)
            byte, sc = (t.reshape(t.shape[0], hk, bs, -1).permute(0, 2, 1, 3).reshape(-1, hk, t.numel() // (t.shape[0] * hk * bs)) for t in (byte, sc))
            at = s["slots"].long()
            got.append(_e4m3(byte[at]) * _pow2(sc[at].int() - 127))
        return tuple(got)
    v = _e4m3(s["v"].view(torch.uint8)).transpose(3, 4).reshape(k.shape) * _pow2(s["v_scale"].int() - 127).unsqueeze(-1)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    new, lens = _lens(c)
    t0 = 0
    for i, (n, total) in enumerate(zip(new, lens)):
        used = s["tables"][i, :-(-total // bs)].long()
        q_at = torch.arange(total - n, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None]
        hidden = j > q_at if c.get("causal", True) else torch.zeros(n, total, dtype=torch.bool, device="cuda")
        if c["window"]:
            hidden = hidden | (q_at - j >= c["window"])
        for head in range(h):
            kh, vh = (t[used, head * hk // h].reshape(-1, d)[:total] for t in (k, v))
            sc = (s["q"][t0:t0 + n, head].double() @ kh.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[t0:t0 + n, head] = torch.softmax(sc, -1) @ vh
        t0 += n
    return out
