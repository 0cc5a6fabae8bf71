"""The 8-bit key/value cache on the CPU: its format, the plain paths of write, read, decode and chunk attention against a 64-bit
implementation, work lists, and what is refused."""

import math

import pytest
import torch

from enterprise_inference_amd.ops import quant_cache as Q
from enterprise_inference_amd.ops.rotary import RotaryCache

import quant_cache_common as C


def test_every_code_times_its_scale():
    x = Q.row_values(torch.arange(256, dtype=torch.int64).to(torch.uint8).view(Q.F8).view(2, 128), torch.tensor([127, 130], dtype=torch.uint8))
    want = C.e4m3_values().view(2, 128) * torch.tensor([[1.0], [8.0]], dtype=torch.float64)
    assert torch.equal(torch.isnan(x), torch.isnan(want)) and torch.equal(x.nan_to_num().double(), want.nan_to_num())


def test_rows_take_the_smallest_power_of_two():
    # 448 * 2^e is the last magnitude of a byte, in fp32 the next number is the next byte's
    for e in (-100, -30, 0, 7, 119):
        top = torch.tensor(448.0 * 2.0 ** e)
        x = torch.stack([top, torch.nextafter(top, torch.tensor(math.inf)), top * 0.50001]).unsqueeze(1).expand(3, 64)
        _, byte, bad = Q.quantise_rows(x.contiguous())
        assert byte.tolist() == [e + 127, min(e + 128, 246), e + 127] and not bad.any()
    codes, byte, _ = Q.quantise_rows(torch.zeros(1, 64))
    assert not codes.view(torch.uint8).any()
    _, byte, _ = Q.quantise_rows(torch.full((1, 64), 1e-38))
    assert byte.item() == 27
    codes, byte, _ = Q.quantise_rows(torch.full((1, 64), 3.3e38))
    assert byte.item() == 246 and bool((codes.float() == 448).all())


def test_nearest_even():
    g = torch.Generator().manual_seed(1)
    x = (torch.randint(-(1 << 12), 1 << 12, (50, 64), generator=g) * 2.0 ** -4)         # ties among them
    x[:, 0] = 256.0 + 1
    codes, byte, _ = Q.quantise_rows(x)
    v = C.e4m3_values()[codes.view(torch.uint8).long()]
    step = torch.pow(2.0, torch.floor(torch.log2(x.double().abs().clamp(min=2.0 ** -6))) - 3)
    e = torch.pow(2.0, byte.double() - 127).unsqueeze(1)
    y = x.double() / e
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    assert torch.equal(v, torch.round(y / step) * step)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("norm,bias", [(False, False), (True, True)])
def test_write_and_read(neox, norm, bias):
    g = torch.Generator().manual_seed(3)
    H, hk, D, bs, T = 4, 2, 64, 32, 37
    cache = Q.QuantKVCache.allocate(4, hk, bs, D)
    rot = RotaryCache(D, 300, 10000.0, None, torch.device("cpu"), neox)
    qkv = torch.randn(T, (H + 2 * hk) * D, generator=g)
    b = torch.randn((H + 2 * hk) * D, generator=g) if bias else None
    qn, kn = ((1 + 0.1 * torch.randn(D, generator=g)) if norm else None for _ in range(2))
    slots = torch.randperm(4 * bs, generator=g)[:T].to(torch.int32)
    slots[5] = -1
    pos = torch.randint(0, 300, (T,), generator=g).to(torch.int32)
    q = Q.rope_qkv_quant(qkv, pos, rot, slots, cache, H, hk, D, b, qn, kn)
    k, v = Q.quant_read(cache, slots, torch.float32)
    x = (qkv + b if bias else qkv).double().view(T, H + 2 * hk, D)
    for h in range(H + hk):
        y = x[:, h]
        if norm:
            y = y / torch.sqrt(y.square().mean(1, keepdim=True) + 1e-6) * (qn if h < H else kn).double()
        cs = rot.cos_sin[pos.long()].double()
        i = torch.arange(D // 2)
        lo, hi = (i, i + D // 2) if neox else (2 * i, 2 * i + 1)
        z = y.clone()
        z[:, lo] = y[:, lo] * cs[:, :D // 2] - y[:, hi] * cs[:, D // 2:]
        z[:, hi] = y[:, hi] * cs[:, :D // 2] + y[:, lo] * cs[:, D // 2:]
        if h < H:
            assert torch.allclose(q[:, h].double(), z, rtol=1e-5, atol=1e-5)
        else:
            kept = k[:, h - H].double()
            assert not kept[5].any()
            # half a step of e4m3: 2^-4 of the value, or 2^-10 of the row's scale
            amax = z.abs().amax(1, keepdim=True)
            tol = torch.maximum(2.0 ** -4 * z.abs(), 2.0 ** -10 * amax / 224) * (1 + 1e-4)
            keep = torch.arange(T) != 5
            assert bool(((kept - z).abs() <= tol)[keep].all())
    amax = x[:, H + hk:].abs().amax(-1, keepdim=True)
    off = (v.double() - x[:, H + hk:]).abs()
    assert bool((off <= torch.maximum(2.0 ** -4 * x[:, H + hk:].abs(), 2.0 ** -10 * amax / 224) * (1 + 1e-4))[torch.arange(T) != 5].all())


def test_a_value_that_is_not_finite_marks_its_token():
    cache = Q.QuantKVCache.allocate(2, 2, 16, 64)
    qkv = torch.ones(4, 4 * 64 + 2 * 64)
    qkv = torch.ones(4, (2 + 4) * 64)
    qkv[1, 2 * 64 + 3] = math.inf                  # a key of head 0
    qkv[2, 5 * 64 + 7] = math.nan                  # a value of head 1
    slots = torch.arange(4, dtype=torch.int32)
    Q.rope_qkv_quant(qkv, None, None, slots, cache, 2, 2, 64)
    k, v = Q.quant_read(cache, slots)
    want = torch.zeros(4, 2, dtype=torch.bool)
    want[1, 0] = want[2, 1] = True
    for t in (k, v):
        assert torch.equal(torch.isnan(t).all(-1), want) and torch.equal(torch.isnan(t).any(-1), want)
    q = torch.ones(2, 2, 64)
    table = torch.zeros(2, 1, dtype=torch.int32)
    o = Q.quant_decode(q, cache, table, torch.tensor([1, 2], dtype=torch.int32), 0.1)
    assert bool(torch.isfinite(o[0]).all()) and torch.isnan(o[1]).any(-1).tolist() == [True, False]


@pytest.mark.parametrize("causal,window,chunk", [(True, 0, 0), (True, 9, 0), (True, 0, 16), (False, 0, 0), (True, 1, 0)])
def test_attention(causal, window, chunk):
    g = torch.Generator().manual_seed(5)
    H, hk, D, bs = 6, 2, 64, 16
    q_lens, lens = [3, 1, 20, 0, 2], [40, 1, 20, 7, 0]
    bt, pages = C.tables(g, lens, bs)
    parts = C.raw_cache(g, pages, hk, bs, D)
    C.spoil_behind(parts, bt, lens, bs)
    cache = Q.QuantKVCache(*parts)
    q = torch.randn(sum(q_lens), H, D, generator=g)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    plan = Q.quant_prefill_plan(q_lens, lens, H, hk, D, "cpu", causal, window or None, chunk or None)
    got = Q.quant_prefill(q, cache, bt, torch.tensor(lens, dtype=torch.int32), cu, plan, 0.05)
    want, mag = C.attend64(q, parts, bt, q_lens, lens, 0.05, causal, window, chunk)
    C.check_attention(got, want, mag)
    if causal:
        lens = [40, 1, 20, 7, 0]
        q = q[:5].contiguous()
        got = Q.quant_decode(q, cache, bt, torch.tensor(lens, dtype=torch.int32), 0.05, window or None, chunk or None)
        want, mag = C.attend64(q, parts, bt, [1] * 5, lens, 0.05, True, window, chunk)
        C.check_attention(got, want, mag)


@pytest.mark.parametrize("heads,hk,d", [(32, 8, 128), (28, 4, 128), (12, 12, 64), (12, 4, 256), (8, 1, 128)])
@pytest.mark.parametrize("q_lens,lens,causal,window", [([1, 700, 3, 0, 64], [9, 900, 3000, 5, 64], True, 0), ([5000], [5000], True, 0),
                                                       ([300, 20], [9000, 20], True, 500), ([300, 2], [400, 9000], False, 0), ([40], [20], True, 0)])
def test_work_lists(heads, hk, d, q_lens, lens, causal, window):
    """Every key tile that a block of rows sees lies in one part, parts have places of their own, every row is in one block."""
    plan = Q.quant_prefill_plan(q_lens, lens, heads, hk, d, "cpu", causal, window or None)
    flat, G, R = plan.lists.tolist(), heads // hk, Q.FLASH_ROWS[d]
    items = [flat[8 * i:8 * i + 5] for i in range(plan.n_items)]
    at = 8 * plan.n_items
    merges = [flat[at + 8 * i:at + 8 * i + 5] for i in range(plan.n_merge)]
    rows = flat[at + 8 * plan.n_merge:]
    starts = [sum(q_lens[:s]) for s in range(len(q_lens))]
    for i in range(plan.n_items):
        s, _, _, _, _, *rest = flat[8 * i:8 * i + 8]
        assert rest == [starts[s], q_lens[s], lens[s]]
    assert len(rows) == plan.n_rows
    span = lambda s: -(-lens[s] // 64) - (max(0, lens[s] - q_lens[s] - window + 1) // 64 if window else 0)
    assert plan.row_parts == sum(max(1, -(-span(s) // plan.row_per)) for s in rows) if rows else plan.row_parts == 1
    used = sorted(it[4] for it in items if it[4] >= 0)
    assert used == list(range(plan.slots)) == sorted(m[1] + p for m in merges for p in range(m[2]))
    for s, (n, L) in enumerate(zip(q_lens, lens)):
        assert (s in rows) == (0 < n and -(-n * G // 16) <= (1 if d == 256 else 2))
        if s in rows:
            continue
        for r in range(0, n * G, R):
            mine = sorted([it for it in items if it[:2] == [s, r]], key=lambda it: it[2])
            assert mine and all(it[2] % 64 == 0 for it in mine)
            for a, b in zip(mine, mine[1:]):
                assert a[2] + 64 * a[3] == b[2] and a[4] + 1 == b[4]
            first, last = L - n + r // G, L - n + (min(r + R, n * G) - 1) // G
            hi = min(L, last + 1) if causal else L
            assert mine[0][2] <= (max(0, first - window + 1) if window else 0) and mine[-1][2] + 64 * mine[-1][3] >= hi
            assert (len(mine) > 1) == any(m == [r, mine[0][4], len(mine), starts[s], n] for m in merges)
    assert len(items) == sum(len([it for it in items if it[0] == s]) for s, n in enumerate(q_lens) if n and s not in rows)


def test_room_for_parts():
    """Decode launches are sized by the tables' width; whatever lengths the kernel finds, its parts have room."""
    import random
    r = random.Random(0)
    for _ in range(20000):
        n, hk, w = r.choice([1, 2, 3, 8, 65, 200]), r.choice([1, 2, 3, 4, 8, 12, 40, 600]), r.choice([1, 3, 4, 5, 16, 100, 512, 3001])
        units = [r.choice([0, 1, w, r.randint(0, w)]) for _ in range(n)]
        per = Q._rows_per(sum(units) * hk)
        assert sum(max(1, -(-u // per)) for u in units) <= Q._row_parts(n, w, hk)


@pytest.mark.parametrize("share", [256, 300, 448])
def test_room_for_parts_of_fewer_workgroups(share):
    import random
    r = random.Random(share)
    for _ in range(5000):
        n, hk, w = r.choice([1, 2, 3, 8, 65, 200]), r.choice([1, 2, 3, 4, 8, 12, 40, 600]), r.choice([1, 3, 4, 5, 16, 100, 512, 3001])
        units = [r.choice([0, 1, w, r.randint(0, w)]) for _ in range(n)]
        per = Q._rows_per(sum(units) * hk, share)
        assert sum(max(1, -(-u // per)) for u in units) <= Q._row_parts(n, w, hk, share)


def test_pages_of_two_buffers():
    half = 3 * 32 * 65
    buf = torch.zeros(2, 5, half, dtype=torch.uint8)
    c = Q.QuantKVCache.of_halves(buf[0], buf[1], 3, 32, 64)
    assert c.k.shape == (5, 3, 32, 64) and c.v.shape == (5, 3, 2, 64, 16) and c.k_scale.shape == (5, 3, 32)
    c.k_scale[4, 2, 31] = 9
    c.v.view(torch.uint8)[4, 2, 1, 63, 15] = 7
    assert buf[0, 4, -1] == 9 and buf[1, 4, 3 * 32 * 64 - 1] == 7
    assert Q.QuantKVCache.bytes_per_page(3, 32, 64) * 5 == buf.numel()


def test_what_is_refused():
    ok = lambda: list(C.raw_cache(torch.Generator().manual_seed(0), 2, 2, 16, 64))
    Q.QuantKVCache(*ok())
    bad = ok()
    bad[0] = bad[0].view(torch.uint8)
    with pytest.raises(ValueError):
        Q.QuantKVCache(*bad)
    bad = ok()
    bad[1] = bad[1].transpose(3, 4)
    with pytest.raises(ValueError):
        Q.QuantKVCache(*bad)
    bad = ok()
    bad[3] = bad[3][:1]
    with pytest.raises(ValueError):
        Q.QuantKVCache(*bad)
    with pytest.raises(ValueError):
        Q.QuantKVCache.allocate(2, 2, 40, 64)
    with pytest.raises(ValueError):
        Q.QuantKVCache.allocate(2, 2, 16, 80)
    c = Q.QuantKVCache.allocate(2, 2, 16, 64)
    qkv, slots = torch.zeros(3, 8 * 64), torch.zeros(3, dtype=torch.int32)
    rot = RotaryCache(64, 10, 10000.0, None, torch.device("cpu"))
    for kw in (dict(num_heads=3), dict(head_dim=128), dict(slot_mapping=slots[:2]), dict(slot_mapping=slots.long()), dict(q_norm_w=torch.ones(64)),
               dict(positions=None)):
        args = dict(qkv=qkv, positions=slots, rotary=rot, slot_mapping=slots, cache=c, num_heads=4, num_kv_heads=2, head_dim=64) | kw
        with pytest.raises(ValueError):
            Q.rope_qkv_quant(**args)
    with pytest.raises(ValueError):
        Q.quant_read(c, slots.long())
    q, bt, lens = torch.zeros(3, 4, 64), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for args in ((q[:, :3], c, bt, lens, 0.1), (q, c, bt[:2], lens, 0.1), (q, c, bt, lens.long(), 0.1), (q, c, bt, lens, 0.0), (q[..., :32], c, bt, lens, 0.1)):
        with pytest.raises(ValueError):
            Q.quant_decode(*args)
    plan = Q.quant_prefill_plan([1, 2], [5, 6], 4, 2, 64, "cpu")
    cu = torch.tensor([0, 1, 3], dtype=torch.int32)
    Q.quant_prefill(q, c, bt, lens, cu, plan, 0.1)
    with pytest.raises(ValueError):
        Q.quant_prefill(q[:2], c, bt, lens, cu, plan, 0.1)
    with pytest.raises(ValueError):
        Q.quant_prefill(q, c, bt, lens, cu[:2], plan, 0.1)
    with pytest.raises(ValueError):                # tables too short for the plan's lengths
        Q.quant_prefill(q, c, bt, lens, cu, Q.quant_prefill_plan([1, 2], [5, 40], 4, 2, 64, "cpu"), 0.1)
    with pytest.raises(ValueError):
        Q.quant_prefill_plan([1], [5, 6], 4, 2, 64, "cpu")
    for kw in (dict(sliding_window=-1), dict(chunk_size=-8)):
        with pytest.raises(ValueError):
            Q.quant_decode(q, c, bt, lens, 0.1, **kw)
        with pytest.raises(ValueError):
            Q.quant_prefill_plan([1], [5], 4, 2, 64, "cpu", **kw)


@pytest.mark.parametrize("n", [2, 90])
def test_a_cache_without_pages_holds_no_tokens(n):
    """Tables that are wide enough, of a pool that is empty: chunks of few rows and of blocks."""
    c = Q.QuantKVCache.allocate(0, 2, 16, 64)
    q, bt, lens = torch.zeros(n, 4, 64), torch.zeros(1, 8, dtype=torch.int32), torch.full((1,), 100, dtype=torch.int32)
    cu = torch.tensor([0, n], dtype=torch.int32)
    with pytest.raises(ValueError, match="without pages"):
        Q.quant_prefill(q, c, bt, lens, cu, Q.quant_prefill_plan([n], [100], 4, 2, 64, "cpu"), 0.1)
    assert not Q.quant_prefill(q, c, bt, lens * 0, cu, Q.quant_prefill_plan([n], [0], 4, 2, 64, "cpu"), 0.1).any()


def test_columns_of_wider_metadata_are_refused():
    """[n, 1] of [n, 2]: the last dimension's stride is 1, and the rows are not neighbours."""
    c = Q.QuantKVCache.allocate(2, 2, 16, 64)
    column = torch.zeros(4, 2, dtype=torch.int32)[:, :1]
    assert column.stride(-1) == 1 and not column.is_contiguous()
    rot, slots = RotaryCache(64, 10, 10000.0, None, torch.device("cpu")), torch.arange(3, dtype=torch.int32)
    for kw in (dict(slot_mapping=column), dict(positions=column)):
        args = dict(qkv=torch.zeros(3, 8 * 64), positions=slots, rotary=rot, slot_mapping=slots, cache=c, num_heads=4, num_kv_heads=2, head_dim=64)
        Q.rope_qkv_quant(**args)
        with pytest.raises(ValueError):
            Q.rope_qkv_quant(**(args | kw))
    q, bt, lens = torch.zeros(3, 4, 64), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    plan = Q.quant_prefill_plan([1, 1, 1], [1, 1, 1], 4, 2, 64, "cpu")
    with pytest.raises(ValueError):
        Q.quant_prefill(q, c, bt, lens, column, plan, 0.1)
