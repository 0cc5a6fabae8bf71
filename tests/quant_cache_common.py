"""What the tests of the 8-bit key/value cache share: caches made byte by byte, and a 64-bit implementation per sequence and
head that shares nothing with the product."""

import math

import torch

F8 = torch.float8_e4m3fn


def e4m3_values():
    """The 256 values of e4m3 by their bits (no infinities; 0x7f and 0xff are no numbers)."""
    v = []
    for b in range(256):
        ex, m = b >> 3 & 15, b & 7
        x = math.nan if ex == 15 and m == 7 else (1 + m / 8) * 2.0 ** (ex - 7) if ex else m / 8 * 2.0 ** -6
        v.append(-x if b & 128 else x)
    return torch.tensor(v, dtype=torch.float64)


def tables(g, lens, bs, spare=1):
    """Pages of sequences at random places of a pool -> (block tables, pages)."""
    need = [-(-n // bs) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    bt = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = order[at:at + n]
        at += n
    return bt, sum(need) + spare


def raw_cache(g, pages, hk, bs, d, low=122, high=128):
    """Random codes (numbers all) and bytes, as cpu tensors k, v, k_scale, v_scale of the documented layout."""
    def codes(*shape):
        c = torch.randint(0, 256, shape, generator=g, dtype=torch.int64)
        return torch.where(c & 127 >= 112, c & 143, c).to(torch.uint8).view(F8)      # magnitudes below 128
    scale = lambda: torch.randint(low, high, (pages, hk, bs), generator=g, dtype=torch.int64).to(torch.uint8)
    return codes(pages, hk, bs, d), codes(pages, hk, bs // 16, d, 16), scale(), scale()


def spoil_behind(parts, bt, lens, bs):
    """Slots behind the sequences' last tokens hold what is no number."""
    k, v, ks, vs = parts
    for s, n in enumerate(lens):
        if n % bs:
            p = int(bt[s, n // bs])
            for t in range(n % bs, bs):
                k.view(torch.uint8)[p, :, t] = 0x7f
                v.view(torch.uint8)[p, :, t // 16, :, t % 16] = 0xff
                ks[p, :, t] = vs[p, :, t] = 255


def row64(parts, bt_row, n, head):
    """float64 (k, v) [n, D] of a sequence's first n tokens."""
    k, v, ks, vs = parts
    bs, val = k.shape[2], e4m3_values()
    t = torch.arange(n)
    p, o = bt_row[t // bs].long(), t % bs
    kk = val[k.view(torch.uint8)[p, head, o].long()] * torch.pow(2.0, ks[p, head, o].double() - 127).unsqueeze(1)
    vv = val[v.view(torch.uint8)[p, head, o // 16, :, o % 16].long()] * torch.pow(2.0, vs[p, head, o].double() - 127).unsqueeze(1)
    bad = ks[p, head, o] == 255
    return kk.masked_fill(bad.unsqueeze(1), math.nan), vv.masked_fill(bad.unsqueeze(1), math.nan)


def attend64(q, parts, bt, q_lens, lens, scale, causal=True, window=0, chunk=0):
    """(out, sum of weight * |value|) float64 [T, Hq, D], query by query over the keys that it sees."""
    T, H, D = q.shape
    hk = parts[0].shape[1]
    out, mag = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    for h in range(H):
        t0 = 0
        for s, (n, L) in enumerate(zip(q_lens, lens)):
            k, v = row64(parts, bt[s], L, h * hk // H)
            for i in range(n):
                at = L - n + i
                hi = min(at + 1, L) if causal else L
                lo = max(0, at - window + 1) if window else 0
                lo = max(lo, at // chunk * chunk) if chunk else lo
                if hi <= lo:
                    continue
                sc = k[lo:hi] @ q[t0 + i, h].double() * scale
                w = torch.softmax(sc, 0)
                out[t0 + i, h], mag[t0 + i, h] = w @ v[lo:hi], w @ v[lo:hi].abs()
            t0 += n
    return out, mag


def check_attention(got, want, mag):
    """Weights w are rounded to bf16 once: w (1 + d), |d| <= 2^-8, half a step.  Their sum is that of the weights before or after
    the rounding, a factor 1 + D, |D| <= 2^-8.  So out = sum w (1 + d) v / (sum w (1 + D)) is off by at most 2^-8 sum w |v| / sum w from the
    first and 2^-8 |out| from the second, and the output's own rounding adds 2^-8 |out|.  Scores and sums are fp32 (2^-12 of the weighted
    magnitudes covers scores of some hundreds and thousands of terms, and the products of the roundings).  A weight under 2^-126 of the
    largest becomes 0 in fp32: with at most 2^10 such keys here, of values under 2^7, that is less than 2^-109."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    off = (got - want).abs()[fine] - (2 ** -8 * (2 * want.abs() + mag) + 2 ** -12 * mag + 2.0 ** -109)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0.0, float(off.max())
