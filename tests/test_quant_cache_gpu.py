"""The kernels of the 8-bit key/value cache against a 64-bit implementation: write, read, decode and chunks, apart and together."""

import math

import pytest
import torch

import quant_cache_common as C

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _q():
    from enterprise_inference_amd.ops import quant_cache as Q
    return Q


def _on_gpu(parts):
    return _q().QuantKVCache(*(t.cuda() for t in parts))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize("D,H,hk,bs", [(128, 32, 8, 128), (64, 6, 2, 16), (256, 12, 4, 48), (128, 7, 1, 64), (64, 3, 3, 32)])
@pytest.mark.parametrize("T", [0, 1, 19, 300])
@pytest.mark.parametrize("neox,extra,order", [(True, False, "run"), (True, True, "run"), (False, True, "mixed")])
def test_write(D, H, hk, bs, T, neox, extra, order):
    Q = _q()
    from enterprise_inference_amd.ops.gemm import SplitK
    from enterprise_inference_amd.ops.rotary import RotaryCache
    g = torch.Generator().manual_seed(T + D)
    pages = -(-(T + 40) // bs) + 1
    cache = Q.QuantKVCache.allocate(pages, hk, bs, D, "cuda")
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x33)
    cache.k_scale.fill_(120), cache.v_scale.fill_(121)
    width = (H + 2 * hk) * D
    qkv = (torch.randn(T, width + 8, generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(BF)[:, :width]
    bias = torch.randn(width, generator=g).to(BF) if extra else None
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g)).to(BF) if extra else None for _ in range(2))
    pos = torch.randint(0, 5000, (T,), generator=g).to(torch.int32)
    free = torch.randperm(pages * bs, generator=g)[:T] if order == "mixed" else torch.arange(T) + 21
    slots = free.to(torch.int32)
    if T > 2:
        slots[2] = -1
    rot = RotaryCache(D, 5000, 10000.0, None, torch.device("cuda"), neox)
    d = lambda t: None if t is None else t.cuda()
    wide = torch.zeros(T, width + 8, dtype=BF, device="cuda")
    wide[:, :width] = qkv.cuda()
    q = Q.rope_qkv_quant(wide[:, :width], d(pos), rot, d(slots), cache, H, hk, D, d(bias), d(qn), d(kn)).cpu().double()
    k, v = (t.cpu().double() for t in Q.quant_read(cache, d(slots)))
    x = (qkv.double() + (bias.double() if extra else 0)).view(T, H + 2 * hk, D)
    qk = x[:, :H + hk]
    if extra:
        w = torch.cat([qn.double().expand(H, D), kn.double().expand(hk, D)])
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    cs = rot.cos_sin.cpu()[pos.long()].double().unsqueeze(1)
    c, s = cs[..., :D // 2], cs[..., D // 2:]
    a, b = (qk[..., :D // 2], qk[..., D // 2:]) if neox else (qk[..., 0::2], qk[..., 1::2])
    a, b = a * c - b * s, b * c + a * s
    qk = torch.cat([a, b], -1) if neox else torch.stack([a, b], -1).flatten(-2)
    size = qk.abs().amax(-1, keepdim=True)
    # one rounding to bf16 (2^-8); fp32 sums and a norm: some 2^-20 of the row's largest
    assert bool(((q - qk[:, :H]).abs() <= 2 ** -8 * qk[:, :H].abs() + 2 ** -20 * size[:, :H]).all())
    keep = slots >= 0
    for got, want in ((k, qk[:, H:]), (v, x[:, H + hk:])):
        amax = want.abs().amax(-1, keepdim=True)
        # half a step of e4m3: 2^-4 of the value, or 2^-10 of the row's scale, which is at most amax / 224 and a rounding
        tol = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * amax / 224 * 1.01) + 2 ** -20 * amax
        assert bool(((got - want).abs() <= tol)[keep].all())
        assert not got[~keep].any()
    # no other slot was touched
    rest = torch.ones(pages * bs, dtype=torch.bool)
    rest[slots[keep].long()] = False
    k, v = Q.quant_read(cache, torch.arange(pages * bs, dtype=torch.int32, device="cuda")[rest.cuda()])
    code = C.e4m3_values()[0x33]
    assert bool((k.double() == code * 2.0 ** -7).all()) and bool((v.double() == code * 2.0 ** -6).all())
    # sums of a split GEMM give the same as their sum in fp32
    if T:
        part = torch.stack([qkv.float() * 0.5, qkv.float() * 0.25, qkv.float() * 0.25]).cuda().contiguous()
        other = Q.QuantKVCache.allocate(pages, hk, bs, D, "cuda")
        q2 = Q.rope_qkv_quant(SplitK(part=part, bias=d(bias), M=T, N=width, sk=3), d(pos), rot, d(slots), other, H, hk, D, None, d(qn), d(kn))
        assert torch.equal(q2.cpu().double(), q)
        assert torch.equal(Q.quant_read(other, d(slots))[0], Q.quant_read(cache, d(slots))[0])


def test_write_keeps_codes_of_bf16_values():
    """Without rotation every value is exact before its code, so codes, ties among them, are those of the plain path."""
    Q = _q()
    g = torch.Generator().manual_seed(2)
    qkv = (torch.randn(500, 6 * 128, generator=g) * torch.exp(8 * torch.randn(500, 1, generator=g))).to(BF)
    qkv[3] = 0
    qkv[4] = 3e38
    qkv[5] = 1e-37
    qkv[6, 300] = math.inf                                              # (of a query: the cache sees nothing of it)
    qkv[7, 700] = math.nan
    slots = torch.arange(500, dtype=torch.int32) + 3
    a, b = Q.QuantKVCache.allocate(9, 1, 64, 128), Q.QuantKVCache.allocate(9, 1, 64, 128, "cuda")
    Q.rope_qkv_quant(qkv, None, None, slots, a, 4, 1, 128)
    Q.rope_qkv_quant(qkv.cuda(), None, None, slots.cuda(), b, 4, 1, 128)
    for name in ("k_scale", "v_scale"):
        x, y = getattr(a, name), getattr(b, name).cpu()
        x[0, 0, 6], y[0, 0, 6] = 0, 0                                   # (a row of zeros: any byte)
        assert torch.equal(x, y)
    zero = lambda t: torch.where(t == 128, torch.zeros_like(t), t)       # (a zero's sign)
    for name in ("k", "v"):
        assert torch.equal(zero(getattr(a, name).view(torch.uint8)), zero(getattr(b, name).cpu().view(torch.uint8)))
    for t in Q.quant_read(b, slots.cuda()):
        assert torch.isnan(t.cpu()).any(-1).nonzero()[:, 0].tolist() == [7]


@pytest.mark.parametrize("T", [4, 300])
def test_a_key_or_value_that_is_not_finite_marks_its_token(T):
    Q = _q()
    qkv = torch.ones(T, (2 + 4) * 64, dtype=BF, device="cuda")
    qkv[1, 2 * 64 + 3] = math.inf                                       # a key of head 0
    qkv[2, 5 * 64 + 7] = -math.inf                                      # a value of head 1
    cache = Q.QuantKVCache.allocate(10, 2, 32, 64, "cuda")
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    Q.rope_qkv_quant(qkv, None, None, slots, cache, 2, 2, 64)
    want = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    want[1, 0] = want[2, 1] = True
    for t in Q.quant_read(cache, slots):
        assert torch.equal(torch.isnan(t).all(-1), want) and torch.equal(torch.isnan(t).any(-1), want)


@pytest.mark.parametrize("D,hk,bs", [(64, 5, 16), (128, 8, 128), (256, 1, 80), (128, 3, 64)])
def test_read(D, hk, bs):
    Q = _q()
    g = torch.Generator().manual_seed(D)
    parts = C.raw_cache(g, 7, hk, bs, D, 27, 247)
    parts[2][1, hk - 1, 3] = 255
    cache = _on_gpu(parts)
    for slots in (torch.arange(0, 6 * bs), torch.arange(5, 5 + 37), torch.randperm(7 * bs, generator=g)[:50], torch.tensor([-1, bs + 3, 7 * bs, 0]),
                  torch.arange(16, 32), torch.zeros(0)):
        slots = slots.to(torch.int32)
        k, v = Q.quant_read(cache, slots.cuda())
        assert k.shape == v.shape == (len(slots), hk, D)
        for i, t in enumerate(slots.tolist()):
            there = 0 <= t < 7 * bs
            for h in {0, hk - 1} if there else ():
                wk, wv = C.row64(parts, torch.full((t % bs + 1,), t // bs), t % bs + 1, h)
                for got, want in ((k, wk), (v, wv)):
                    assert torch.allclose(got[i, h].cpu().double(), want[-1], rtol=0, atol=0, equal_nan=True)
            if not there:
                assert not k[i].any() and not v[i].any()


# ------------------------------------------------------------------------------ attention
def _attend(H, hk, D, bs, q_lens, lens, causal=True, window=0, chunk=0, poison=False, wide=False, scale=0.02, seed=0):
    Q = _q()
    g = torch.Generator().manual_seed(seed + sum(lens))
    bt, pages = C.tables(g, lens, bs)
    parts = C.raw_cache(g, pages, hk, bs, D)
    C.spoil_behind(parts, bt, lens, bs)
    if poison:
        s = max(range(len(lens)), key=lambda i: lens[i])
        t = lens[s] - max(1, q_lens[s] // 2)
        parts[2][int(bt[s, t // bs]), hk - 1, t % bs] = 255
    T = sum(q_lens)
    q = torch.randn(T, H, D, generator=g).to(BF)
    want, mag = C.attend64(q, parts, bt, q_lens, lens, scale, causal, window, chunk)
    cache, bt, cl = _on_gpu(parts), bt.cuda(), _i32(lens)
    cu = _i32([0] + q_lens).cumsum(0).to(torch.int32)
    dq, out = q.cuda(), None
    if wide:                                                            # rows of wider tensors
        dq = torch.cat([dq.view(T, H * D), torch.zeros(T, 8, dtype=BF, device="cuda")], 1)[:, :H * D].unflatten(1, (H, D))
        room = torch.full((T + 1, H * D + 16), 7.0, dtype=BF, device="cuda")
        out = room[:T, :H * D].unflatten(1, (H, D))
    plan = Q.quant_prefill_plan(q_lens, lens, H, hk, D, "cuda", causal, window or None, chunk or None)
    got = Q.quant_prefill(dq, cache, bt, cl, cu, plan, scale, out=out)
    C.check_attention(got.cpu(), want, mag)
    if wide:
        assert got is out and bool((room[T] == 7).all()) and bool((room[:, H * D:] == 7).all())
    if causal and all(n == 1 for n in q_lens) and H // hk <= (16 if D == 256 else 32):
        got = Q.quant_decode(dq, cache, bt, cl, scale, window or None, chunk or None, out=out)
        C.check_attention(got.cpu(), want, mag)
    return plan


@pytest.mark.parametrize("H,hk,D,bs", [(8, 2, 128, 128), (4, 4, 64, 16), (12, 4, 256, 48), (32, 1, 128, 64), (5, 1, 64, 32), (7, 1, 128, 16),
                                       (16, 1, 256, 64), (20, 1, 64, 192)])
@pytest.mark.parametrize("lens", [[1], [64], [0, 65, 1, 130], [700, 3, 255, 256, 257]])
@pytest.mark.parametrize("window,chunk", [(0, 0), (1, 0), (70, 0), (0, 64)])
def test_decode(H, hk, D, bs, lens, window, chunk):
    _attend(H, hk, D, bs, [1] * len(lens), lens, True, window, chunk)


@pytest.mark.parametrize("H,hk,D,bs", [(4, 1, 128, 128), (12, 4, 256, 64), (8, 8, 64, 16)])
def test_decode_long(H, hk, D, bs):
    _attend(H, hk, D, bs, [1, 1], [9001, 130])
    _attend(H, hk, D, bs, [1, 1], [9001, 130], window=5000, wide=True)


@pytest.mark.parametrize("H,hk,D,bs", [(8, 2, 128, 128), (4, 4, 64, 16), (6, 2, 256, 48), (7, 1, 128, 64), (5, 1, 64, 32), (32, 1, 128, 16)])
@pytest.mark.parametrize("q_lens,lens", [([3], [3]), ([5, 2], [200, 70]), ([65], [65]), ([33, 1, 0, 90], [100, 5, 9, 90]), ([70], [400])])
@pytest.mark.parametrize("causal,window,chunk", [(True, 0, 0), (True, 20, 0), (True, 0, 32), (False, 0, 0), (False, 20, 0)])
def test_chunks(H, hk, D, bs, q_lens, lens, causal, window, chunk):
    _attend(H, hk, D, bs, q_lens, lens, causal, window, chunk)


@pytest.mark.parametrize("H,hk,D,bs", [(8, 2, 128, 128), (3, 3, 64, 16), (6, 2, 256, 64)])
def test_chunks_cut_along_the_keys(H, hk, D, bs):
    plan = _attend(H, hk, D, bs, [150], [3500], wide=True)
    assert plan.n_merge > 0
    plan = _attend(H, hk, D, bs, [150, 2, 40], [1500, 2500, 40])
    assert plan.n_merge > 0 and plan.n_rows > 0


@pytest.mark.parametrize("D,H,hk,q_lens,lens", [(128, 8, 2, [90], [300]), (64, 4, 4, [1, 1], [80, 200]), (128, 4, 1, [3], [90]), (256, 4, 2, [70], [70])])
def test_a_token_that_is_no_number(D, H, hk, q_lens, lens):
    """Rows that see it are no numbers, the others know nothing of it."""
    _attend(H, hk, D, 64, q_lens, lens, poison=True)


def test_queries_before_the_first_key():
    """More new tokens than the sequence holds: those that see nothing become zeros."""
    for q_lens, lens in (([6], [2]), ([90], [20])):
        _attend(4, 1, 128, 64, q_lens, lens)


def test_large_scores_and_values():
    """Scores of thousands: one key takes the weight."""
    _attend(8, 2, 128, 64, [40, 1], [300, 500], scale=1.0)


# ------------------------------------------------------------------------------ together
def test_a_step_after_another():
    """Prompt, portions and single tokens through write, chunk and decode, as a layer calls them: what a query sees is what was
    written, whatever the portions."""
    Q = _q()
    from enterprise_inference_amd.ops.rotary import RotaryCache
    H, hk, D, bs, n = 8, 2, 128, 64, 150
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(n, (H + 2 * hk) * D, generator=g, device="cuda").to(BF)
    rot = RotaryCache(D, 400, 10000.0, None, torch.device("cuda"))
    bt = _i32([[3, 0, 4]])
    t = torch.arange(n, device="cuda")
    slots = (bt[0][t // bs] * bs + t % bs).to(torch.int32)
    pos = t.to(torch.int32)

    def go(portions):
        cache, outs, at = Q.QuantKVCache.allocate(5, hk, bs, D, "cuda"), [], 0
        for m in portions:
            rows = slice(at, at + m)
            q = Q.rope_qkv_quant(qkv[rows], pos[rows], rot, slots[rows], cache, H, hk, D)
            at += m
            if m == 1:
                outs.append(Q.quant_decode(q, cache, bt, _i32([at]), D ** -0.5))
            else:
                plan = Q.quant_prefill_plan([m], [at], H, hk, D, "cuda")
                outs.append(Q.quant_prefill(q, cache, bt, _i32([at]), _i32([0, m]), plan, D ** -0.5))
        return torch.cat(outs), cache

    whole, cache = go([n])
    k, v = (x.double() for x in Q.quant_read(cache, slots))
    fresh = Q.rope_qkv_quant(qkv, pos, rot, slots, cache, H, hk, D).double()
    s = torch.einsum("qhd,khd->hqk", fresh, k.repeat_interleave(H // hk, 1)) * D ** -0.5
    s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    w = torch.softmax(s, -1)
    vv = v.repeat_interleave(H // hk, 1)
    want, mag = torch.einsum("hqk,khd->qhd", w, vv), torch.einsum("hqk,khd->qhd", w, vv.abs())
    C.check_attention(whole.cpu(), want.cpu(), mag.cpu())
    for portions in ([100, 50], [64, 1, 1, 7, 77], [1] * 10 + [140]):
        out, other = go(portions)
        C.check_attention(out.cpu(), want.cpu(), mag.cpu())
        assert all(torch.equal(a, b) for a, b in zip(Q.quant_read(other, slots), Q.quant_read(cache, slots)))


def test_graph_replays_follow_lengths_and_tables():
    Q = _q()
    H, hk, D, bs, B = 8, 2, 128, 64, 3
    g = torch.Generator().manual_seed(9)
    bt, pages = C.tables(g, [900, 640, 900], bs)
    parts = C.raw_cache(g, pages, hk, bs, D)
    cache, dbt, lens = _on_gpu(parts), bt.cuda(), _i32([5, 0, 70])
    q = torch.randn(B, H, D, generator=g).to(BF).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Q.quant_decode(q, cache, dbt, lens, 0.02)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):                                                  # two graphs have workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(Q.quant_decode(q, cache, dbt, lens, 0.02))
        graphs.append(graph)
    for now in ([900, 640, 900], [1, 0, 0], [64, 65, 63], [899, 1, 513]):
        lens.copy_(_i32(now))
        want, mag = C.attend64(q.cpu(), parts, bt, [1] * B, now, 0.02)
        eager = Q.quant_decode(q, cache, dbt, lens, 0.02)
        for graph, out in zip(graphs, outs):
            out.fill_(1)
            graph.replay()
            torch.cuda.synchronize()
            C.check_attention(out.cpu(), want, mag)
            assert torch.equal(out, eager)


def test_another_stream_and_the_same_bits_again():
    Q = _q()
    g = torch.Generator().manual_seed(11)
    lens, q_lens = [700, 300], [200, 3]
    bt, pages = C.tables(g, lens, 64)
    parts = C.raw_cache(g, pages, 2, 64, 128)
    cache, q = _on_gpu(parts), torch.randn(203, 8, 128, generator=g).to(BF).cuda()
    plan = Q.quant_prefill_plan(q_lens, lens, 8, 2, 128, "cuda")
    args = (q, cache, bt.cuda(), _i32(lens), _i32([0, 200, 203]), plan, 0.02)
    first = Q.quant_prefill(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = Q.quant_prefill(*args)
    side.synchronize()
    assert torch.equal(first, other) and torch.equal(first, Q.quant_prefill(*args))


def test_what_is_refused_on_the_gpu():
    Q = _q()
    cache = Q.QuantKVCache.allocate(2, 1, 64, 128, "cuda")
    lens, bt = _i32([3, 3]), _i32([[0], [1]])
    q = torch.zeros(2, 4, 128, dtype=BF, device="cuda")
    with pytest.raises(ValueError):
        Q.quant_decode(torch.zeros(2, 4, 136, dtype=BF, device="cuda")[..., 4:132], cache, bt, lens, 0.1)
    with pytest.raises(ValueError):
        Q.quant_decode(torch.zeros(2, 33, 128, dtype=BF, device="cuda"), cache, bt, lens, 0.1)
    with pytest.raises(ValueError):
        Q.quant_decode(q, cache, bt.cpu(), lens, 0.1)
    with pytest.raises(ValueError):
        Q.quant_decode(q, cache, bt, lens, 0.1, out=torch.zeros(2, 4, 128, device="cuda"))
    plan = Q.quant_prefill_plan([1, 1], [3, 3], 4, 1, 128, "cpu")
    with pytest.raises(ValueError):
        Q.quant_prefill(q, cache, bt, lens, _i32([0, 1, 2]), plan, 0.1)
    with pytest.raises(ValueError):
        Q.rope_qkv_quant(torch.zeros(2, 6 * 128 + 4, dtype=BF, device="cuda")[:, :768], None, None, lens, cache, 4, 1, 128)
    with pytest.raises(ValueError):
        Q.quant_read(cache, lens.cpu())


def test_large_writes_and_reads():
    """Rows that are read past the caches: the same bytes as in portions that are not."""
    Q = _q()
    from enterprise_inference_amd.ops.rotary import RotaryCache
    H, hk, D, bs, T = 32, 8, 128, 128, 5600                              # 65.6 MiB of rows
    g = torch.Generator(device="cuda").manual_seed(21)
    qkv = torch.randn(T, (H + 2 * hk) * D, generator=g, device="cuda").to(BF)
    rot = RotaryCache(D, T, 10000.0, None, torch.device("cuda"))
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    a, b = (Q.QuantKVCache.allocate(44, hk, bs, D, "cuda") for _ in range(2))
    q = Q.rope_qkv_quant(qkv, pos, rot, pos, a, H, hk, D)
    parts = [Q.rope_qkv_quant(qkv[s], pos[s], rot, pos[s], b, H, hk, D) for s in (slice(0, 2800), slice(2800, 5500), slice(5500, T))]
    assert torch.equal(q, torch.cat(parts))
    for name in ("k", "v"):
        assert torch.equal(getattr(a, name).view(torch.uint8), getattr(b, name).view(torch.uint8))
    assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
    slots = torch.randint(0, T, (17000,), generator=g, device="cuda").to(torch.int32)       # 33 MiB of codes
    slots[100:8000] = torch.arange(7900 - 5000, 7900 - 5000 + 7900, device="cuda").clamp(max=T - 1).to(torch.int32)
    whole, half = Q.quant_read(a, slots), [Q.quant_read(a, slots[:8000]), Q.quant_read(a, slots[8000:])]
    for i in range(2):
        assert torch.equal(whole[i], torch.cat([h[i] for h in half]))


def _dense64(q, parts, bt_row, L, n, causal=True, scale=0.02):
    """float64 on the GPU for one sequence's n last tokens: (out, weighted magnitudes) [n, H, D]."""
    H, hk = q.shape[1], parts[0].shape[1]
    out, mag = [], []
    for h in range(H):
        k, v = (x.cuda() for x in C.row64(parts, bt_row, L, h * hk // H))
        s = q[:, h].double() @ k.T * scale
        if causal:
            s = s.masked_fill(torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None], -math.inf)
        w = torch.softmax(s, -1)
        out.append(w @ v), mag.append(w @ v.abs())
    return torch.stack(out, 1).cpu(), torch.stack(mag, 1).cpu()


@pytest.mark.parametrize("bs", [16, 48, 128])
def test_decode_parts_of_many_pages(bs):
    """Enough rows that a part is longer than 64 small pages."""
    Q = _q()
    g = torch.Generator().manual_seed(bs)
    lens = [4000 - 37 * i for i in range(40)]
    bt, pages = C.tables(g, lens, bs)
    parts = C.raw_cache(g, pages, 8, bs, 64)
    C.spoil_behind(parts, bt, lens, bs)
    q = torch.randn(40, 16, 64, generator=g).to(BF).cuda()
    got = Q.quant_decode(q, _on_gpu(parts), bt.cuda(), _i32(lens), 0.02)
    for s in (0, 17, 39):
        C.check_attention(got[s:s + 1].cpu(), *_dense64(q[s:s + 1], parts, bt[s], lens[s], 1))


@pytest.mark.parametrize("D,H,hk", [(128, 8, 2), (64, 4, 4), (256, 4, 2)])
def test_long_chunks(D, H, hk):
    """Several rounds of blocks; more than one block of rows behind a long context."""
    Q = _q()
    g = torch.Generator().manual_seed(D)
    q_lens, lens = [700, 9, 333], [5200, 3000, 333]
    bt, pages = C.tables(g, lens, 32)
    parts = C.raw_cache(g, pages, hk, 32, D)
    C.spoil_behind(parts, bt, lens, 32)
    q = torch.randn(sum(q_lens), H, D, generator=g).to(BF).cuda()
    plan = Q.quant_prefill_plan(q_lens, lens, H, hk, D, "cuda")
    got = Q.quant_prefill(q, _on_gpu(parts), bt.cuda(), _i32(lens), _i32([0, 700, 709, 1042]), plan, 0.02)
    at = 0
    for s, (n, L) in enumerate(zip(q_lens, lens)):
        C.check_attention(got[at:at + n].cpu(), *_dense64(q[at:at + n], parts, bt[s], L, n))
        at += n


def test_pools_past_32_bits():
    """More than 4 GiB of keys, and of values: the last pages."""
    Q = _q()
    H, hk, D, bs, pages, n = 8, 8, 128, 128, 33000, 300
    cache = Q.QuantKVCache.allocate(pages, hk, bs, D, "cuda")
    assert cache.k.stride(0) * (pages - 3) > 1 << 32
    bt = _i32([[pages - 1, pages - 3, pages - 2], [0, 1, 2]])
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(2 * n, (H + 2 * hk) * D, generator=g, device="cuda").to(BF)
    t = torch.arange(n, device="cuda")
    slots = torch.cat([(bt[s][t // bs] * bs + t % bs) for s in range(2)]).to(torch.int32)
    q = Q.rope_qkv_quant(qkv, None, None, slots, cache, H, hk, D)
    # the same tokens in a small pool
    small = Q.QuantKVCache.allocate(6, hk, bs, D, "cuda")
    st = _i32([[0, 1, 2], [3, 4, 5]])
    ss = torch.cat([(st[s][t // bs] * bs + t % bs) for s in range(2)]).to(torch.int32)
    Q.rope_qkv_quant(qkv, None, None, ss, small, H, hk, D)
    for a, b in zip(Q.quant_read(cache, slots), Q.quant_read(small, ss)):
        assert torch.equal(a, b)
    lens, cu = _i32([n, n]), _i32([0, n, 2 * n])
    plan = Q.quant_prefill_plan([n, n], [n, n], H, hk, D, "cuda")
    assert torch.equal(Q.quant_prefill(q, cache, bt, lens, cu, plan, 0.1), Q.quant_prefill(q, small, st, lens, cu, plan, 0.1))
    last = q[[n - 1, 2 * n - 1]].contiguous()
    assert torch.equal(Q.quant_decode(last, cache, bt, lens, 0.1), Q.quant_decode(last, small, st, lens, 0.1))


def test_a_captured_step_replays():
    """Write, chunk and decode in one graph, replayed with other inputs and eager work between."""
    Q = _q()
    from enterprise_inference_amd.ops.rotary import RotaryCache
    H, hk, D, bs = 8, 2, 128, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    rot = RotaryCache(D, 2000, 10000.0, None, torch.device("cuda"))
    q_lens, lens, B = [150, 3], [1500, 700], 2
    bt = torch.randperm(60, generator=g, device="cuda")[:50].view(2, 25).to(torch.int32)
    dbt = torch.randperm(60, generator=g, device="cuda")[:30].view(2, 15).to(torch.int32)
    cache = Q.QuantKVCache.allocate(60, hk, bs, D, "cuda")
    fill = torch.randint(0, 100, cache.k.shape, generator=g, device="cuda").to(torch.uint8)
    cache.k.view(torch.uint8).copy_(fill), cache.v.view(torch.uint8).copy_(fill.view(cache.v.shape))
    cache.k_scale.fill_(124), cache.v_scale.fill_(125)
    T = B + sum(q_lens)
    qkv = torch.randn(T, (H + 2 * hk) * D, generator=g, device="cuda").to(BF)
    pos, slots = torch.randint(0, 2000, (T,), generator=g, device="cuda").to(torch.int32), torch.randperm(60 * bs, generator=g, device="cuda")[:T].to(torch.int32)
    dlens, plens, cu = _i32([900, 33]), _i32(lens), _i32([0, 150, 153])
    plan = Q.quant_prefill_plan(q_lens, lens, H, hk, D, "cuda")

    def step():
        q = Q.rope_qkv_quant(qkv, pos, rot, slots, cache, H, hk, D)
        return torch.cat([Q.quant_decode(q[:B], cache, dbt, dlens, 0.05), Q.quant_prefill(q[B:], cache, bt, plens, cu, plan, 0.05)])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step()) and bool(torch.isfinite(got).all())


def test_two_streams_at_once():
    Q = _q()
    g = torch.Generator().manual_seed(13)
    lens = [3000, 2500, 1]
    bt, pages = C.tables(g, lens, 64)
    parts = C.raw_cache(g, pages, 2, 64, 128)
    cache, dbt, dl = _on_gpu(parts), bt.cuda(), _i32(lens)
    qs = [torch.randn(3, 8, 128, generator=g).to(BF).cuda() for _ in range(2)]
    chunk = torch.randn(90, 8, 128, generator=g).to(BF).cuda()
    args = (chunk, cache, dbt[:1], dl[:1], _i32([0, 90]))
    first = [Q.quant_decode(q, cache, dbt, dl, 0.02) for q in qs]
    plan = Q.quant_prefill_plan([90], [3000], 8, 2, 128, "cuda")
    whole = Q.quant_prefill(*args, plan, 0.02)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(Q.quant_decode(qs[i], cache, dbt, dl, 0.02))
    other = Q.quant_prefill_plan([90], [3000], 8, 2, 128, "cuda")              # made on this stream, used on another
    with torch.cuda.stream(streams[0]):
        late = Q.quant_prefill(*args, other, 0.02)
    torch.cuda.synchronize()
    assert torch.equal(late, whole)
    for i in range(2):
        assert all(torch.equal(x, first[i]) for x in got[i])


def test_a_query_that_is_no_number_stays_alone():
    Q = _q()
    g = torch.Generator().manual_seed(17)
    for q_lens, lens, hk in (([1, 1], [70, 300], 1), ([5], [300], 1), ([90], [300], 2)):
        bt, pages = C.tables(g, lens, 64)
        parts = C.raw_cache(g, pages, hk, 64, 128)
        q = torch.randn(sum(q_lens), 4, 128, generator=g).to(BF)
        bad = q.clone()
        bad[1, 2, 5] = math.nan
        plan = Q.quant_prefill_plan(q_lens, lens, 4, hk, 128, "cuda")
        cu = _i32([0] + q_lens).cumsum(0).to(torch.int32)
        a, b = (Q.quant_prefill(x.cuda(), _on_gpu(parts), bt.cuda(), _i32(lens), cu, plan, 0.02) for x in (q, bad))
        assert bool(torch.isnan(b[1, 2]).all())
        b[1, 2] = a[1, 2]
        assert torch.equal(a, b)


def test_entries_outside_the_pool_and_positions_outside_the_table():
    """Held to the last page, to the last row and to the table's width: nothing outside is read."""
    Q = _q()
    from enterprise_inference_amd.ops.rotary import RotaryCache
    g = torch.Generator().manual_seed(21)
    for bs in (48, 64):
        cache = _on_gpu(C.raw_cache(g, 5, 2, bs, 128))
        q = torch.randn(3, 8, 128, generator=g).to(BF).cuda()
        bad, held = _i32([[0, -1, 2], [1 << 30, 3, 1], [5, 0, 0]]), _i32([[0, 4, 2], [4, 3, 1], [4, 0, 0]])
        lens, long = _i32([3 * bs, 2 * bs + 1, 7]), _i32([1 << 30, 2 * bs + 1, 7])
        want = Q.quant_decode(q, cache, held, lens, 0.02)
        for bt in (bad, held):
            for n in (lens, long):
                assert torch.equal(Q.quant_decode(q, cache, bt, n, 0.02), want)
        chunk, cu = torch.randn(100, 8, 128, generator=g).to(BF).cuda(), _i32([0, 2, 100])
        plan = Q.quant_prefill_plan([2, 98], [3 * bs, 2 * bs + 1], 8, 2, 128, "cuda")
        assert torch.equal(*(Q.quant_prefill(chunk, cache, bt, lens, cu, plan, 0.02) for bt in (bad, held)))
    rot = RotaryCache(128, 50, 10000.0, None, torch.device("cuda"))
    qkv, slots = torch.randn(3, 12 * 128, generator=g).to(BF).cuda(), _i32([1, 2, 3])
    a, b = (Q.rope_qkv_quant(qkv, _i32(p), rot, slots, cache, 8, 2, 128) for p in ([49, 49, 7], [-1, 1 << 30, 7]))
    assert torch.equal(a, b)


def test_no_pages_and_no_width():
    Q = _q()
    q, cu = torch.ones(2, 4, 64, dtype=BF, device="cuda"), _i32([0, 2])
    for pages, width in ((0, 1), (1, 0)):
        cache = Q.QuantKVCache.allocate(pages, 2, 16, 64, "cuda")
        bt = torch.zeros(2, width, dtype=torch.int32, device="cuda")
        assert not Q.quant_decode(q, cache, bt, _i32([0, 0]), 0.1).any()
        assert not Q.quant_decode(q, cache, bt, _i32([9, 9]), 0.1).any()
        assert not Q.quant_prefill(q, cache, bt, _i32([0]), cu, Q.quant_prefill_plan([2], [0], 4, 2, 64, "cuda"), 0.1).any()


def test_a_plan_is_made_before_the_capture():
    Q = _q()
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(ValueError):
            Q.quant_prefill_plan([90], [3000], 8, 2, 128, "cuda")
    graph.replay()
    assert x.sum().item() == 4


def test_more_decode_rows_than_lanes():
    """The sequences' lengths are found 64 at a time."""
    Q = _q()
    g = torch.Generator().manual_seed(130)
    lens = [int(x) for x in torch.randint(0, 700, (130,), generator=g)]
    lens[64], lens[65], lens[129] = 0, 699, 1
    bt, pages = C.tables(g, lens, 64)
    parts = C.raw_cache(g, pages, 2, 64, 128)
    q = torch.randn(130, 8, 128, generator=g).to(BF)
    got = Q.quant_decode(q.cuda(), _on_gpu(parts), bt.cuda(), _i32(lens), 0.02)
    C.check_attention(got.cpu(), *C.attend64(q, parts, bt, [1] * 130, lens, 0.02))


def test_blocks_of_plan_and_kernel():
    Q = _q()
    from enterprise_inference_amd.ops._dispatch import lib
    assert {d: lib().eia_quant_flash_rows(d) for d in Q.HEAD_DIMS} == Q.FLASH_ROWS


@pytest.mark.parametrize("norm", [False, True])
def test_codes_are_the_nearest(norm):
    """A million rotated keys: every code is what rounding the 64-bit value once gives (values so near to a border that 64 bits
    miss it are some 2^-45 of them)."""
    Q = _q()
    from enterprise_inference_amd.ops.rotary import RotaryCache
    H, hk, D, T, bs = 4, 2, 128, 4096, 128
    g = torch.Generator(device="cuda").manual_seed(31)
    rot = RotaryCache(D, 9000, 10000.0, None, torch.device("cuda"))
    qkv = torch.randn(T, (H + 2 * hk) * D, generator=g, device="cuda").to(BF)
    pos, slots = torch.randint(0, 9000, (T,), generator=g, device="cuda").to(torch.int32), torch.arange(T, device="cuda", dtype=torch.int32)
    w = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(BF) if norm else None
    cache = Q.QuantKVCache.allocate(T // bs, hk, bs, D, "cuda")
    Q.rope_qkv_quant(qkv, pos, rot, slots, cache, H, hk, D, None, w, w)
    x = qkv.view(T, H + 2 * hk, D)[:, H:H + hk].double()
    if norm:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    c, s = rot.cos_sin[pos.long()].double().unsqueeze(1).chunk(2, -1)
    a, b = x.chunk(2, -1)
    x = torch.cat([a * c - b * s, b * c + a * s], -1)
    two_to = lambda n: ((n.long() + 1023) << 52).view(torch.float64)            # (torch.ldexp takes a power of 2.0, which is not exact)
    mant, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = e - 9 + (mant > 0.875).int()
    y = x * two_to(-e)
    step = two_to(torch.frexp(y)[1].clamp(min=-5) - 4)
    want = torch.round(y / step) * step * two_to(e)
    assert torch.equal(Q.quant_read(cache, slots)[0].double(), want)


@pytest.mark.parametrize("H,hk,D,bs,B", [(32, 8, 128, 64, 100), (12, 12, 64, 48, 90), (16, 16, 128, 16, 70)])
def test_more_rows_and_heads_than_run_at_a_time(H, hk, D, bs, B):
    Q = _q()
    assert Q._row_share(B, hk, 1, D)[1] == 2 and Q._row_share(B // 2, hk, 1, D)[1] == 4
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.randint(0, 200, (B,), generator=g)]
    lens[3], lens[4], lens[B - 1] = 2900, 0, 64
    bt, pages = C.tables(g, lens, bs)
    parts = C.raw_cache(g, pages, hk, bs, D)
    C.spoil_behind(parts, bt, lens, bs)
    q = torch.randn(B, H, D, generator=g).to(BF)
    args = _on_gpu(parts), bt.cuda(), _i32(lens), 0.02
    got = Q.quant_decode(q.cuda(), *args)
    for s in (0, 1, 2, 3, 4, 5, B - 2, B - 1):
        if lens[s]:
            C.check_attention(got[s:s + 1].cpu(), *_dense64(q[s:s + 1].cuda(), parts, bt[s], lens[s], 1))
        else:
            assert not got[s].any()
    # chunks of two tokens, the same rule
    plan = Q.quant_prefill_plan([1, 2] * (B // 2), lens, H, hk, D, "cuda")
    assert plan.row_waves == 2 and plan.n_rows == B
    cu = _i32([0] + [1, 2] * (B // 2)).cumsum(0).to(torch.int32)
    q2 = torch.randn(int(cu[-1]), H, D, generator=g).to(BF).cuda()
    got = Q.quant_prefill(q2, *args[:3], cu, plan, 0.02)
    for s in (1, 3, B - 1):
        a = int(cu[s])
        C.check_attention(got[a:a + 2].cpu(), *_dense64(q2[a:a + 2], parts, bt[s], lens[s], 2))


def test_lengths_that_are_a_column_are_refused():
    """[n, 1] of [n, 2]: the last dimension's stride is 1, and the rows are not neighbours."""
    Q = _q()
    cache = Q.QuantKVCache.allocate(2, 1, 64, 128, "cuda")
    q, bt, column = torch.zeros(2, 4, 128, dtype=BF, device="cuda"), _i32([[0], [1]]), _i32([[3, 0], [3, 0]])[:, :1]
    plan = Q.quant_prefill_plan([1, 1], [3, 3], 4, 1, 128, "cuda")
    with pytest.raises(ValueError):
        Q.quant_decode(q, cache, bt, column, 0.1)
    with pytest.raises(ValueError):
        Q.quant_prefill(q, cache, bt, column, _i32([0, 1, 2]), plan, 0.1)
