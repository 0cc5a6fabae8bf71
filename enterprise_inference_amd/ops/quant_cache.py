"""The 8-bit key/value cache: write, read back, decode and chunk attention -> csrc/kernels/quant_*.hip.

A row is the D values of one token and kv head.  With amax its largest magnitude, e is the smallest whole number for which
amax <= 448 * 2^e, held to [-100, 119]; the row is kept as the e4m3 codes of x / 2^e (nearest, ties to even, at most 448) and one
byte e + 127.  Every value code * 2^e is exact in bf16.  A token and head of which a key or a value is not finite is marked in
``k_scale`` by byte 255: both rows read back as NaN, and a query that sees the token becomes NaN.

Step layout, block tables, slots and lengths are those of ``ops.attention`` and ``ops.rotary``.
"""

from __future__ import annotations

import dataclasses
import functools
import heapq
import itertools
from typing import List, Optional, Sequence, Tuple

import torch

from ._dispatch import check, lib, ptr, require, use_hip

F8 = torch.float8_e4m3fn
GROUP = 16                    # tokens of a value tile
ROW_BYTES = 1                 # beside a row's D codes
HEAD_DIMS = (64, 128, 256)
UNIT = 64                     # keys that the kernels take at a time
CUS = 256


class QuantKVCache:
    """One layer's pages: ``k`` [pages, Hkv, page, D] and ``v`` [pages, Hkv, page / 16, D, 16] in e4m3, ``k_scale`` and
    ``v_scale`` [pages, Hkv, page] bytes.  Pages may lie apart (strides of the first dimension, the same for keys and values);
    inside a page everything is contiguous."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "num_kv_heads", "block_size", "head_dim", "device", "_hip", "_args")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        require(k.dim() == 4 and v.dim() == 5, "QuantKVCache: k [pages, Hkv, page, D], v [pages, Hkv, page / 16, D, 16]")
        n, h, bs, d = k.shape
        require(bs % GROUP == 0 and bs > 0 and d in HEAD_DIMS, f"QuantKVCache: pages of a multiple of 16 tokens, heads of {HEAD_DIMS}")
        require(v.shape == (n, h, bs // GROUP, d, GROUP) and k_scale.shape == v_scale.shape == (n, h, bs), "QuantKVCache: shapes")
        require(k.dtype == v.dtype == F8 and k_scale.dtype == v_scale.dtype == torch.uint8, "QuantKVCache: e4m3 codes, bytes as scales")
        require(k.device == v.device == k_scale.device == v_scale.device, "QuantKVCache: one device")
        require(n == 0 or all(t[0].is_contiguous() for t in (k, v, k_scale, v_scale)), "QuantKVCache: a page is contiguous")
        require(n < 2 or (k.stride(0) == v.stride(0) >= h * bs * d and k_scale.stride(0) == v_scale.stride(0) >= h * bs),
                "QuantKVCache: keys and values step alike from page to page")
        require(n * bs < 1 << 31, "QuantKVCache: slots are 32-bit")
        require(all(t.data_ptr() % 16 == 0 and (n < 2 or t.stride(0) % 16 == 0) for t in (k, v, k_scale, v_scale)),
                "QuantKVCache: pages begin on 16 bytes")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.num_kv_heads, self.block_size, self.head_dim = n, h, bs, d
        self.device, self._hip = k.device, use_hip(k)
        self._args = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.stride(0), k_scale.stride(0))

    @classmethod
    def allocate(cls, pages: int, num_kv_heads: int, block_size: int, head_dim: int, device=None) -> "QuantKVCache":
        half = num_kv_heads * block_size * (head_dim + ROW_BYTES)
        require(block_size > 0 and block_size % GROUP == 0, "QuantKVCache: pages of a multiple of 16 tokens")
        return cls.of_halves(*torch.zeros(2, pages, half, dtype=torch.uint8, device=device), num_kv_heads, block_size, head_dim)

    @classmethod
    def of_halves(cls, keys: torch.Tensor, values: torch.Tensor, num_kv_heads: int, block_size: int, head_dim: int) -> "QuantKVCache":
        """Over two byte buffers [pages, Hkv * page * (D + 1)]: a page's codes, then its scales, so that a page is one piece."""
        h, bs, d = num_kv_heads, block_size, head_dim
        split = h * bs * d
        require(keys.dim() == values.dim() == 2 and keys.shape == values.shape and keys.shape[1] == h * bs * (d + ROW_BYTES)
                and keys.dtype == values.dtype == torch.uint8, "QuantKVCache.of_halves: [pages, Hkv * page * (D + 1)] bytes")
        codes = [t[:, :split].view(F8) for t in (keys, values)]
        scales = [t[:, split:].unflatten(1, (h, bs)) for t in (keys, values)]
        return cls(codes[0].unflatten(1, (h, bs, d)), codes[1].unflatten(1, (h, bs // GROUP, d, GROUP)), *scales)

    @staticmethod
    def bytes_per_page(num_kv_heads: int, block_size: int, head_dim: int) -> int:
        return 2 * num_kv_heads * block_size * (head_dim + ROW_BYTES)


# ------------------------------------------------------------------------------ plain forms (CPU, and types without kernels)
def _two_to(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantise_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """fp32 rows [..., D] -> (codes, bytes, whether a value is not finite [...]); rows that are not finite: codes 0, byte 127."""
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad.unsqueeze(-1), torch.zeros((), dtype=x.dtype, device=x.device), x)
    mant, ex = torch.frexp(x.abs().amax(-1))
    e = (ex - 9 + (mant > 0.875)).clamp(-100, 119)
    e = torch.where(bad, torch.zeros_like(e), e)
    return (x * _two_to(-e).unsqueeze(-1)).clamp(-448, 448).to(F8), (e + 127).to(torch.uint8), bad


def row_values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Codes [..., D] and their bytes -> fp32 values."""
    e = scale.to(torch.int32) - 127
    x = codes.float() * _two_to(e.clamp(-100, 119)).unsqueeze(-1)
    return torch.where((scale == 255).unsqueeze(-1), torch.full((), float("nan"), device=x.device), x)


def _write_rows(cache: QuantKVCache, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    keep = (slots >= 0) & (slots < cache.pages * cache.block_size)
    slots, k, v = slots[keep].long(), k[keep], v[keep]
    p, t = slots // cache.block_size, slots % cache.block_size
    kc, kb, kbad = quantise_rows(k)
    vc, vb, vbad = quantise_rows(v)
    bad = kbad | vbad
    kc, vc = (torch.where(bad.unsqueeze(-1), torch.zeros((), dtype=torch.uint8, device=c.device), c.view(torch.uint8)) for c in (kc, vc))
    cache.k.view(torch.uint8)[p, :, t] = kc
    cache.v.view(torch.uint8)[p, :, t // GROUP, :, t % GROUP] = vc
    cache.k_scale[p, :, t] = torch.where(bad, torch.full((), 255, dtype=torch.uint8, device=kb.device), kb)
    cache.v_scale[p, :, t] = torch.where(bad, torch.full((), 127, dtype=torch.uint8, device=kb.device), vb)


def _read_rows(cache: QuantKVCache, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows of slots (zeros where a slot is outside the cache)."""
    there = (slots >= 0) & (slots < cache.pages * cache.block_size)
    at = torch.where(there, slots, torch.zeros_like(slots)).long()
    p, t = at // cache.block_size, at % cache.block_size
    ks = cache.k_scale[p, :, t]
    vs = torch.where(ks == 255, ks, cache.v_scale[p, :, t])
    k = row_values(cache.k.view(torch.uint8)[p, :, t].view(F8), ks)
    v = row_values(cache.v.view(torch.uint8)[p, :, t // GROUP, :, t % GROUP].contiguous().view(F8), vs)
    gone = ~there[:, None, None]
    return k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)


def _rope_rows(qkv, positions, rotary, num_heads, num_kv_heads, head_dim, bias, q_norm_w, k_norm_w, eps):
    """fp32 (q, k, v) rows of a projection, rotated."""
    x = qkv.float()
    if bias is not None:
        x = x + bias.float()
    x = x.view(x.shape[0], num_heads + 2 * num_kv_heads, head_dim)
    qk, v = x[:, :num_heads + num_kv_heads], x[:, num_heads + num_kv_heads:]
    if q_norm_w is not None:
        w = torch.cat([q_norm_w.float().expand(num_heads, head_dim), k_norm_w.float().expand(num_kv_heads, head_dim)])
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + eps) * w
    if rotary is not None:
        cs = rotary.cos_sin[positions.long()].unsqueeze(1)
        c, s = cs[..., :head_dim // 2], cs[..., head_dim // 2:]
        a, b = (qk[..., :head_dim // 2], qk[..., head_dim // 2:]) if rotary.is_neox else (qk[..., 0::2], qk[..., 1::2])
        a, b = a * c - b * s, b * c + a * s
        qk = torch.cat([a, b], -1) if rotary.is_neox else torch.stack([a, b], -1).flatten(-2)
    return qk[:, :num_heads], qk[:, num_heads:], v


def _attend_plain(q, cache, table, L, scale, causal, window, chunk):
    """q [n, Hq, D], the last n tokens of a sequence of L -> fp32 [n, Hq, D]."""
    n, Hq, D = q.shape
    if L <= 0:
        return torch.zeros(n, Hq, D, device=q.device)
    j = torch.arange(L, device=q.device)
    k, v = _read_rows(cache, table[j // cache.block_size].long() * cache.block_size + j % cache.block_size)
    at = torch.arange(L - n, L, device=q.device).unsqueeze(1)
    seen = (j <= at) if causal else torch.ones(n, L, dtype=torch.bool, device=q.device)
    if window:
        seen = seen & (j > at - window)
    if chunk:
        seen = seen & (j >= torch.div(at, chunk, rounding_mode="floor") * chunk)
    g = Hq // cache.num_kv_heads
    out = torch.empty(n, Hq, D, device=q.device)
    for h in range(Hq):
        s = (q[:, h].float() @ k[:, h // g].T * scale).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1)
        p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
        # a value that nobody sees may be anything
        vh = torch.where(seen.any(0).unsqueeze(1), v[:, h // g], torch.zeros_like(v[:, h // g]))
        bad = torch.isnan(vh).any(1)
        o = p @ vh.masked_fill(bad.unsqueeze(1), 0.0)
        out[:, h] = o.masked_fill((seen & bad).any(-1, keepdim=True), float("nan"))
    return out


# ------------------------------------------------------------------------------ write and read
# Calls of few tokens are bound by the host: a launch takes it 3 us, torch.empty 1.65 (empty_strided 1.26, empty_like 1.15), a tensor's
# attribute 0.05 to 0.1.
def _empty(shape, device) -> torch.Tensor:
    """bf16 [n, heads, D]."""
    d = shape[2]
    return torch.empty_strided(shape, (shape[1] * d, d, 1), dtype=torch.bfloat16, device=device)


def _launch(name: str, call, device: torch.device, *args) -> None:
    """``call`` on the device's current stream.  A launch belongs to the device that is current: the tensors' one."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        check(call(*args, torch._C._cuda_getCurrentRawStream(index)), name)
    else:
        with torch.cuda.device(index):
            check(call(*args, torch._C._cuda_getCurrentRawStream(index)), name)


def rope_qkv_quant(qkv, positions: Optional[torch.Tensor], rotary, slot_mapping: torch.Tensor, cache: QuantKVCache, num_heads: int,
                   num_kv_heads: int, head_dim: int, bias: Optional[torch.Tensor] = None, q_norm_w: Optional[torch.Tensor] = None,
                   k_norm_w: Optional[torch.Tensor] = None, norm_eps: float = 1e-6) -> torch.Tensor:
    """qkv [T, (Hq + 2 Hkv) D] -> q [T, Hq, D]; keys and values go into the 8-bit cache (``rope_qkv_cache`` for it).

    ``qkv`` may be a ``gemm.SplitK``, summed here.  Bias, per-head norms and rotation are rounded once: queries, formed in
    fp32, to bf16, keys (fp64 in the kernel) and values to their codes.  Slots are distinct; tokens whose slot is outside the cache write nothing.  Positions lie in the
    rotary table."""
    part = None
    if not isinstance(qkv, torch.Tensor):
        from .gemm import SplitK
        require(isinstance(qkv, SplitK), "rope_qkv_quant: a tensor or split-K sums")
        if qkv.bias is not None:
            require(bias is None, "rope_qkv_quant: bias given twice")
        if cache._hip and qkv.part.is_cuda:
            part, bias = qkv, qkv.bias if qkv.bias is not None else bias
            require(part.part.is_contiguous() and part.part.dtype == torch.float32, "rope_qkv_quant: split-K sums")
        else:
            qkv = qkv.materialize()
    T, N = (part.M, part.N) if part is not None else qkv.shape
    width = (num_heads + 2 * num_kv_heads) * head_dim
    if not (N == width and cache.num_kv_heads == num_kv_heads and cache.head_dim == head_dim):
        raise ValueError("rope_qkv_quant: qkv width, cache layout")
    if (q_norm_w is None) != (k_norm_w is None):
        raise ValueError("rope_qkv_quant: norms of queries and keys together")
    if not (slot_mapping.dtype is torch.int32 and slot_mapping.numel() >= T and slot_mapping.is_contiguous()):
        raise ValueError("rope_qkv_quant: slot_mapping int32[T]")
    table, neox = None, True
    if rotary is not None:
        table, neox = rotary.cos_sin, rotary.is_neox
        if not (positions is not None and positions.dtype is torch.int32 and positions.numel() >= T and positions.is_contiguous()):
            raise ValueError("rope_qkv_quant: positions int32[T]")
        if not (table.shape[0] > 0 and table.shape[1] == head_dim and table.dtype is torch.float32 and table.is_contiguous()):
            raise ValueError("rope_qkv_quant: cos | sin fp32 [positions, D]")
    src = part.part if part is not None else qkv
    if part is None and not (cache._hip and qkv.is_cuda and qkv.dtype is torch.bfloat16):
        q, k, v = _rope_rows(qkv, None if positions is None else positions[:T], rotary, num_heads, num_kv_heads, head_dim, bias,
                             q_norm_w, k_norm_w, norm_eps)
        _write_rows(cache, slot_mapping[:T], k, v)
        return q.to(qkv.dtype)
    if part is None and not (qkv.stride(1) == 1 and qkv.stride(0) % 8 == 0 and qkv.data_ptr() % 16 == 0):
        raise ValueError("rope_qkv_quant: rows on 16 bytes")
    for w, n in ((bias, width), (q_norm_w, head_dim), (k_norm_w, head_dim)):
        if w is not None and not (w.dtype is torch.bfloat16 and w.numel() == n and w.is_contiguous() and w.data_ptr() % 16 == 0):
            raise ValueError("rope_qkv_quant: bf16 weights on 16 bytes")
    device = src.device
    if not all(t is None or t.device == device for t in (cache, slot_mapping, positions if table is not None else None, table, bias, q_norm_w,
                                                         k_norm_w)):
        raise ValueError("rope_qkv_quant: one device")
    q = _empty((T, num_heads, head_dim), device)
    _launch("rope_qkv_quant", lib().eia_quant_write, device, None if part is not None else ptr(qkv),
            0 if part is not None else qkv.stride(0), ptr(src) if part is not None else None, part.sk if part is not None else 0,
            ptr(positions), ptr(table), 0 if table is None else table.shape[0], ptr(slot_mapping), *cache._args, cache.pages, ptr(q), ptr(bias), ptr(q_norm_w), ptr(k_norm_w),
            float(norm_eps), T, num_heads, num_kv_heads, head_dim, cache.block_size, 1 if neox else 0)
    return q


def quant_read(cache: QuantKVCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache's slots (int32 [n]) as (k, v) [n, Hkv, D]: exactly the values kept, zeros where a slot is outside."""
    if not (slots.dtype is torch.int32 and slots.dim() == 1 and slots.is_contiguous() and slots.device == cache.device):
        raise ValueError("quant_read: slots int32 [n] on the cache's device")
    if not (cache._hip and dtype is torch.bfloat16):
        return tuple(t.to(dtype) for t in _read_rows(cache, slots))
    shape = (slots.shape[0], cache.num_kv_heads, cache.head_dim)
    device = cache.device
    k = _empty(shape, device)
    v = torch.empty_like(k)
    _launch("quant_read", lib().eia_quant_read, device, *cache._args, cache.pages, slots.data_ptr(), shape[0], k.data_ptr(),
            v.data_ptr(), shape[1], shape[2], cache.block_size)
    return k, v


# ------------------------------------------------------------------------------ attention
def _check_attention(name, q, cache, block_tables, seq_lens, n, scale, window, chunk, out):
    """(whether the kernels take it, tokens, heads); ``n`` sequences."""
    T, Hq, D = q.shape
    if not (D == cache.head_dim and Hq % cache.num_kv_heads == 0):
        raise ValueError(f"{name}: q [tokens, Hq, D]")
    if not (block_tables.dtype is torch.int32 and seq_lens.dtype is torch.int32 and block_tables.dim() == 2):
        raise ValueError(f"{name}: int32 metadata")
    if not (block_tables.shape[0] >= n and seq_lens.numel() >= n):
        raise ValueError(f"{name}: metadata rows < sequences")
    if not scale > 0.0:
        raise ValueError(f"{name}: scale > 0")
    if (window or 0) < 0 or (chunk or 0) < 0:
        raise ValueError(f"{name}: window, chunk size >= 0")
    if out is not None and not (out.shape == q.shape and out.dtype == q.dtype and out.device == q.device):
        raise ValueError(f"{name}: out like q")
    if not (cache._hip and q.is_cuda and q.dtype is torch.bfloat16):
        return False, T, Hq
    for t in (q, out) if out is not None else (q,):
        s = t.stride()
        if not (s[2] == 1 and s[1] == D and s[0] % 8 == 0 and t.data_ptr() % 16 == 0):
            raise ValueError(f"{name}: rows of q and out on 16 bytes")
    device = cache.device
    if not (q.device == device and block_tables.device == device and seq_lens.device == device):
        raise ValueError(f"{name}: one device")
    if not (block_tables.stride(1) == 1 and seq_lens.is_contiguous()):
        raise ValueError(f"{name}: contiguous metadata")
    return True, T, Hq


def _row_tiles(rows: int, head_dim: int) -> int:
    """16-row tiles of the few-rows kernel for so many (query, head) rows; 0: it does not take them."""
    tiles = -(-rows // 16)
    return tiles if 1 <= tiles <= (1 if head_dim == 256 else 2) else 0


ROW_SHARE = 512               # workgroups that share out a launch of the few-rows kernel: two a CU, or by _row_share
ROW_HELD = {(1, 64): 1024, (2, 64): 768, (1, 128): 768, (2, 128): 512, (1, 256): 512}     # (row tiles, D): what the chip holds of them
ROW_LEAST = 4                 # units a part at least
ROW_LONG = 48                 # longer parts are halved


def _launch_rows(name, q, out, cache, block_tables, seq_lens, cu, seqs, n, sequences, scale, causal, window, chunk, tiles, parts, per,
                 share):
    Hq, D, device = q.shape[1], cache.head_dim, cache.device
    ws = torch.empty_strided((parts * cache.num_kv_heads * 16 * tiles * (D + 2) + 2 * sequences,), (1,), dtype=torch.float32,
                             device=device) if parts > n else None
    _launch(name, lib().eia_quant_rows, device, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), *cache._args,
            cache.pages, block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1], seq_lens.data_ptr(), cu, seqs, n, float(scale), Hq,
            cache.num_kv_heads, D, cache.block_size, 1 if causal else 0, window or 0, chunk or 0, tiles, parts, per, ROW_LEAST, *share,
            ptr(ws))


def _row_share(n: int, num_kv_heads: int, tiles: int, head_dim: int) -> Tuple[int, int]:
    """(Workgroups to share out n sequences over, waves of one): as many as run at a time, without those that rounding adds (half a part a
    sequence and head).  us shared over 512 / so, decode, 32 heads on 8 of 128: 32 rows of 8192 to 16384 keys 143 / 138, 15 of 3209 to 6418 39.4 /
    34.2, 4 of 8301 to 16602 32.1 / 28.5, of 2483 to 4966 14.2 / 14.9, 65 of 1000 to 2000 42.9 / 43.0; 12 on 4 of 256, 32 of 2000 to 4000
    51.9 / 44.1; chunks of 6 tokens, 32 on 8 of 128, 16 behind 1000 to 2000 27.4 / 21.4.  Workgroups of two waves where the heads and rows
    alone are more than that (csrc/kernels/quant_rows.hip has the times)."""
    held, alone = ROW_HELD.get((tiles, head_dim), ROW_SHARE), n * num_kv_heads
    two = tiles == 1 and head_dim <= 128 and alone > held
    return max(ROW_SHARE // 2, (held * 3 // 2 if two else held) - alone // 2), 2 if two else 4


def _rows_per(units: int, share: int = ROW_SHARE) -> int:
    """Units a part for so many of all sequences and kv heads (rows_per in csrc/kernels/quant_rows.hip)."""
    one = -(-units // share)
    return max(ROW_LEAST, min(one, max((one + 1) // 2, ROW_LONG)))


def _row_parts(n: int, units: int, num_kv_heads: int, share: int = ROW_SHARE) -> int:
    """Room for the parts of n sequences of at most ``units`` each, whatever their lengths: below one per ``least`` units, and
    fewer than n more than the workgroups that the units are shared out over."""
    rounds = 2 if n * units * num_kv_heads > ROW_LONG * share else 1
    return min(n * max(1, -(-units // ROW_LEAST)), rounds * share // num_kv_heads + n)


@functools.lru_cache(maxsize=256)
def _decode_grid(B: int, span: int, group: int, num_kv_heads: int, head_dim: int, window, chunk) -> Tuple[int, Tuple[int, int], int]:
    """(row tiles, workgroups to share and their waves, room for parts) of B rows of at most ``span`` tokens."""
    units = -(-span // UNIT)
    for w in (window, chunk):
        if w:
            units = min(units, -(-w // UNIT) + 1)
    tiles = _row_tiles(group, head_dim)
    share = _row_share(B, num_kv_heads, tiles, head_dim)
    return tiles, share, _row_parts(B, units, num_kv_heads, share[0])


def quant_decode(q: torch.Tensor, cache: QuantKVCache, block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                 sliding_window: Optional[int] = None, chunk_size: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [B, Hq, D], one token a sequence, the last of ``seq_lens`` [B] -> out [B, Hq, D] (``paged_decode`` for the 8-bit cache).

    Rows of length 0 become zeros.  Nothing is read back: lengths and tables may change under a captured graph, up to the
    tables' width.  The launch has room for what the width allows, and a second one to put parts together unless the width rules parts
    out: no difference where rows are cut, 3 us where none is (csrc/kernels/quant_rows.hip)."""
    B = q.shape[0]
    hip, _, Hq = _check_attention("quant_decode", q, cache, block_tables, seq_lens, B, scale, sliding_window, chunk_size, out)
    if not hip:
        rows = [_attend_plain(q[b:b + 1], cache, block_tables[b], int(seq_lens[b]), scale, True, sliding_window, chunk_size) for b in range(B)]
        r = torch.cat(rows).to(q.dtype) if B else q.clone()
        return r if out is None else out.copy_(r)
    tiles, share, parts = _decode_grid(B, block_tables.shape[1] * cache.block_size, Hq // cache.num_kv_heads, cache.num_kv_heads,
                                       cache.head_dim, sliding_window, chunk_size)
    if tiles == 0:
        raise ValueError("quant_decode: too many query heads a kv head")
    o = _empty((B, Hq, cache.head_dim), cache.device) if out is None else out
    if B == 0:
        return o
    _launch_rows("quant_decode", q, o, cache, block_tables, seq_lens, None, None, B, B, scale, True, sliding_window, chunk_size, tiles, parts,
                 0, share)
    return o


@dataclasses.dataclass
class QuantPrefillPlan:
    """What a step's chunks have to do, laid out once for all of its layers (``quant_prefill_plan``)."""
    q_lens: List[int]
    kv_lens: List[int]
    num_heads: int
    num_kv_heads: int
    head_dim: int
    causal: bool
    sliding_window: Optional[int]
    chunk_size: Optional[int]
    lists: Optional[torch.Tensor]          # int32: blocks of 8, merges of 8, sequences of few rows
    n_items: int = 0
    n_merge: int = 0
    slots: int = 0
    n_rows: int = 0
    row_tiles: int = 1
    row_parts: int = 1
    row_per: int = 0
    row_waves: int = 4

    stream = ready = None                  # of the lists' upload

    def __post_init__(self):
        self.tokens, self.longest = sum(self.q_lens), max(self.kv_lens, default=0)


FLASH_ROWS = {64: 128, 128: 256, 256: 128}      # (query, head) rows of a workgroup of csrc/kernels/quant_flash.hip
FLASH_HELD = {64: 2, 128: 1, 256: 1}            # workgroups on a CU


def _first_key(at: int, window, chunk) -> int:
    lo = max(0, at - window + 1) if window else 0
    return max(lo, at // chunk * chunk) if chunk and at > 0 else lo


def quant_prefill_plan(q_lens: Sequence[int], kv_lens: Sequence[int], num_heads: int, num_kv_heads: int, head_dim: int, device,
                       causal: bool = True, sliding_window: Optional[int] = None, chunk_size: Optional[int] = None) -> QuantPrefillPlan:
    """Work lists of ``quant_prefill`` for chunks of ``q_lens`` new tokens that end at ``kv_lens`` cached ones.

    Sequences of few (query, head) rows go to the kernel that streams the cache for one block of them; the others are cut into
    blocks of rows, the long ones along the keys too where else the launch would wait for them.  The lists are uploaded behind the
    current stream's work.  ``quant_prefill`` waits for them on another stream, but a capture cannot: a program that replays a captured
    ``quant_prefill`` keeps the plan, and captures when its upload is through (``torch.cuda.graph`` waits for the device before it begins;
    who calls ``capture_begin`` synchronises first).  Host time: 20 to 500 us a plan, by blocks and by whether the launch is cut."""
    q_lens, kv_lens = [int(n) for n in q_lens], [int(n) for n in kv_lens]
    require(len(q_lens) == len(kv_lens) and all(n >= 0 for n in q_lens + kv_lens), "quant_prefill_plan: lengths")
    require(num_kv_heads > 0 and num_heads % num_kv_heads == 0 and head_dim in HEAD_DIMS, "quant_prefill_plan: heads")
    require((sliding_window or 0) >= 0 and (chunk_size or 0) >= 0, "quant_prefill_plan: window, chunk size >= 0")
    device = torch.device(device)
    # (a replay would read host memory that is another's by then)
    require(not (device.type == "cuda" and torch.cuda.is_current_stream_capturing()), "quant_prefill_plan: before a graph is captured")
    plan = QuantPrefillPlan(q_lens, kv_lens, num_heads, num_kv_heads, head_dim, causal, sliding_window, chunk_size, None)
    G = num_heads // num_kv_heads
    few, blocks, first = [], [], [0, *itertools.accumulate(q_lens)]
    R = FLASH_ROWS[head_dim]
    units = []
    for s, (n, L) in enumerate(zip(q_lens, kv_lens)):
        if n == 0:
            continue
        if _row_tiles(n * G, head_dim):
            few.append(s)
            plan.row_tiles = max(plan.row_tiles, _row_tiles(n * G, head_dim))
            units.append(-(-L // UNIT) - _first_key(max(L - n, 0), sliding_window, chunk_size) // UNIT if L else 0)
            continue
        for r in range(0, n * G, R):
            a, b = L - n + r // G, L - n + (min(r + R, n * G) - 1) // G          # positions of the block's first and last query
            hi = min(L, b + 1) if causal else L
            lo = _first_key(a, sliding_window, chunk_size) // UNIT * UNIT
            blocks.append((max(0, -(-(hi - lo) // UNIT)), s, r, lo))
    if few:
        plan.n_rows = len(few)
        share, plan.row_waves = _row_share(len(few), num_kv_heads, plan.row_tiles, head_dim)
        plan.row_per = _rows_per(sum(units) * num_kv_heads, share)
        plan.row_parts = sum(max(1, -(-u // plan.row_per)) for u in units)
    blocks.sort(key=lambda b: -b[0])
    items, merges = [], []
    if blocks:
        per = _flash_per([b[0] for b in blocks], num_kv_heads, head_dim)
        for tiles, s, r, lo in blocks:
            parts = max(1, -(-tiles // per))
            if parts == 1:
                items.append((tiles, (s, r, lo, tiles, -1, first[s], q_lens[s], kv_lens[s])))
                continue
            each = -(-tiles // parts)
            parts = -(-tiles // each)
            merges += [r, plan.slots, parts, first[s], q_lens[s], 0, 0, 0]
            for p in range(parts):
                t = min(each, tiles - p * each)
                items.append((t, (s, r, lo + p * each * UNIT, t, plan.slots + p, first[s], q_lens[s], kv_lens[s])))
            plan.slots += parts
        items.sort(key=lambda b: -b[0])
        plan.n_items, plan.n_merge = len(items), len(merges) // 8
    flat = [x for _, it in items for x in it] + merges + few
    plan.lists = torch.tensor(flat, dtype=torch.int32, pin_memory=device.type == "cuda").to(device, non_blocking=True)
    if device.type == "cuda":                     # (a copy behind the stream's work: other streams wait for it)
        plan.stream = torch.cuda.current_stream(plan.lists.device)
        plan.ready = torch.cuda.Event()
        plan.ready.record(plan.stream)
    return plan


# MI355X, us: a tile of 64 keys of a workgroup with the chip full, what a workgroup takes besides, a part's sums written and read.
# (Tiles of 32 workgroups alone take 1.45, 1.8 and 3.1: clocks fall under load.)
FLASH_TILE = {64: 1.4, 128: 2.1, 256: 3.2}
FLASH_FIXED = 4.0
FLASH_PART = {64: 0.02, 128: 0.033, 256: 0.033}
FLASH_MERGE = 3.0


def _makespan(sizes: List[int], slots: int, tile: float) -> float:
    """Time of a launch whose workgroups of so many tiles (longest first) go to the next slot that is free."""
    if len(sizes) <= slots:
        return sizes[0] * tile + FLASH_FIXED
    ends = [n * tile + FLASH_FIXED for n in sizes[:slots]]
    heapq.heapify(ends)
    for n in sizes[slots:]:
        heapq.heapreplace(ends, ends[0] + n * tile + FLASH_FIXED)
    return max(ends)


def _flash_per(tiles: List[int], num_kv_heads: int, head_dim: int) -> int:
    """Key tiles of a part at most, for blocks of so many tiles (longest first): what makes the launch shortest, a second kernel
    and the parts' sums counted.  The kv heads are alike, so one is laid out on its share of the CUs."""
    slots, tile = max(1, CUS * FLASH_HELD[head_dim] // num_kv_heads), FLASH_TILE[head_dim]
    longest, work = max(tiles[0], 1), sum(tiles)
    best, took = longest, _makespan(tiles, slots, tile)
    if len(tiles) >= 4 * slots:                   # many rounds: they even themselves out
        return best
    for rounds in (1, 2, 3, 4, 6):
        per = max(2, -(-work // (slots * rounds)))
        if per >= longest:
            continue
        sizes, parts = [], 0
        for n in tiles:
            k = max(1, -(-n // per))
            parts += k if k > 1 else 0
            sizes += [-(-n // k)] * k
        sizes.sort(reverse=True)
        t = _makespan(sizes, slots, tile) + FLASH_MERGE + parts * num_kv_heads * FLASH_PART[head_dim]
        if t < took:
            best, took = per, t
    return best


def quant_prefill(q: torch.Tensor, cache: QuantKVCache, block_tables: torch.Tensor, seq_lens: torch.Tensor, cu_q: torch.Tensor,
                  plan: QuantPrefillPlan, scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, Hq, D], chunks of new tokens at the end of their sequences (rows cu_q[s] .. cu_q[s + 1]), whose keys and values the
    cache already holds -> out [T, Hq, D] (``paged_prefill`` for the 8-bit cache).  ``plan`` holds the lengths that ``cu_q`` and
    ``seq_lens`` hold on the device; rows that see no key become zeros.  In a capture the plan is one that is there
    (``quant_prefill_plan``)."""
    n = len(plan.q_lens)
    hip, T, Hq = _check_attention("quant_prefill", q, cache, block_tables, seq_lens, n, scale, plan.sliding_window, plan.chunk_size, out)
    D = cache.head_dim
    if not (plan.num_heads == Hq and plan.num_kv_heads == cache.num_kv_heads and plan.head_dim == D):
        raise ValueError("quant_prefill: plan of other heads")
    if not (plan.tokens == T and cu_q.numel() >= n + 1 and cu_q.dtype is torch.int32 and cu_q.is_contiguous()):
        raise ValueError("quant_prefill: plan of other chunks")
    if plan.longest > block_tables.shape[1] * cache.block_size:
        raise ValueError("quant_prefill: tables shorter than the sequences")
    if plan.longest > 0 and cache.pages == 0:       # (tiles are the plan's: the kernel would look for them)
        raise ValueError("quant_prefill: a cache without pages holds no tokens")
    if not hip:
        at, rows = 0, []
        for s, (m, L) in enumerate(zip(plan.q_lens, plan.kv_lens)):
            rows.append(_attend_plain(q[at:at + m], cache, block_tables[s], L, scale, plan.causal, plan.sliding_window, plan.chunk_size))
            at += m
        r = torch.cat(rows).to(q.dtype) if rows else q.clone()
        return r if out is None else out.copy_(r)
    if not (plan.lists.device == cu_q.device == cache.device):
        raise ValueError("quant_prefill: plan and chunks on the cache's device")
    if plan.stream.cuda_stream != torch._C._cuda_getCurrentRawStream(cache.device.index) and not torch.cuda.is_current_stream_capturing():
        here = torch.cuda.current_stream(cache.device)
        here.wait_event(plan.ready)
        plan.lists.record_stream(here)
    o = _empty((T, Hq, D), cache.device) if out is None else out
    base, window, chunk = plan.lists.data_ptr(), plan.sliding_window or 0, plan.chunk_size or 0
    if plan.n_items:
        ws = torch.empty(plan.slots * cache.num_kv_heads * FLASH_ROWS[D] * (D + 2), dtype=torch.float32, device=cache.device) if plan.slots else None
        _launch("quant_prefill", lib().eia_quant_flash, cache.device, q.data_ptr(), q.stride(0), o.data_ptr(), o.stride(0), *cache._args,
                cache.pages, block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1], base, plan.n_items,
                base + 32 * plan.n_items, plan.n_merge, plan.slots, ptr(ws), float(scale), Hq, cache.num_kv_heads, D, cache.block_size,
                1 if plan.causal else 0, window, chunk)
    if plan.n_rows:
        _launch_rows("quant_prefill", q, o, cache, block_tables, seq_lens, cu_q.data_ptr(), base + 32 * (plan.n_items + plan.n_merge),
                     plan.n_rows, n, scale, plan.causal, window, chunk, plan.row_tiles, plan.row_parts,
                     plan.row_per, (1, plan.row_waves))
    return o


def quant_attention(q: torch.Tensor, cache: QuantKVCache, md, scale: float, sliding_window: Optional[int] = None,
                    chunk_size: Optional[int] = None) -> torch.Tensor:
    """The step's decode and prefill parts (``attention.attention`` for the 8-bit cache). q [T, Hq, D]."""
    nd = md.num_decode
    out = None
    if md.num_prefill_tokens:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        key = ("quant", q.shape[1], cache.num_kv_heads, cache.head_dim, sliding_window, chunk_size)
        plan = md.work_cache.get(key)                # once a step: its layers are alike
        if plan is None:
            lens, cu = md.prefill_q_lens, md.prefill_cu_q
            if lens is None:
                cu = cu.tolist()
                lens = [b - a for a, b in zip(cu, cu[1:])]
            kv = md.prefill_kv_lens
            if kv is None:
                kv = md.prefill_seq_lens.tolist()
            plan = quant_prefill_plan(lens, kv, q.shape[1], cache.num_kv_heads, cache.head_dim, q.device, md.causal, sliding_window,
                                      chunk_size)
            md.work_cache[key] = plan
        quant_prefill(q[nd:], cache, md.prefill_block_tables, md.prefill_seq_lens, md.prefill_cu_q, plan, scale, out=out[nd:])
    if nd:
        part = None if out is None else out[:nd]
        o = quant_decode(q if nd == q.shape[0] else q[:nd], cache, md.decode_block_tables, md.decode_seq_lens, scale, sliding_window,
                         chunk_size, out=part)
        out = o if out is None else out
    return out if out is not None else torch.empty_like(q)
