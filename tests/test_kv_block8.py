"""Block-scaled 8-bit KV cache (int8 / e4m3 codes, one power-of-two scale per block and head): write, decode
attention with accumulated weights, prompt attention, eviction; against plain 64-bit restatements.

Tolerances, where the result is rounded: an output element is sum(p v) with p held in f16 (half a step 2^-11, the
products and sums in fp32) and stored in bf16 (half a step 2^-8 relative), so
|error| <= 2^-8 |out| + 2^-10 sum(p |v|). A softmax weight comes from an fp32 score of D products (each
rounded by at most D 2^-24 of sum |q k|) and an exponential of relative error 2^-20 at most."""
import math

import pytest
import torch

from gollek_b200 import ops
from gollek_b200.ops import reference as ref

KINDS = {"int8": torch.int8, "e4m3": torch.uint8}


def numbers(codes):
    """64-bit numbers of the codes, from their bits."""
    if codes.dtype == torch.int8:
        return codes.double()
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2((e - 7).double()))
    v = torch.where((c & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(c >= 128, -v, v)


def values(cache, scales):
    return numbers(cache) * scales.double()[..., None, None]


def least_scale(top, kind):
    y = max(top / (127.0 if kind == "int8" else 448.0), 2.0 ** -100)
    m, e = math.frexp(y)
    return 2.0 ** (e - 1 if m == 0.5 else e)


def nearest(y, kind):
    """y rounded to the type's numbers, ties to even."""
    if kind == "int8":
        return y.round().clamp(-127, 127)
    step = torch.exp2(torch.frexp(y).exponent.clamp(min=-5).double() - 4)
    return ((y / step).round() * step).clamp(-448, 448)


def tables_for(lens, bs, gen, spare=4):
    nb = [(l + bs - 1) // bs for l in lens]
    NB = sum(nb) + spare
    ids = (torch.randperm(NB - 1, generator=gen) + 1).int()   # block 0 belongs to nobody: tables are padded with it
    bt = torch.zeros(len(lens), max(1, max(nb)), dtype=torch.int32)
    k = 0
    for b, n in enumerate(nb):
        bt[b, :n] = ids[k:k + n]
        k += n
    return bt, NB


def filled(kind, lens, Hk, D, bs, seed, layers=1):
    """A cache whose tokens are random; everything behind a sequence's end is poison."""
    g = torch.Generator().manual_seed(seed)
    bt, NB = tables_for(lens, bs, g)
    code = torch.randint(-127, 128, (layers, NB, 2, Hk, bs, D), generator=g)
    cache = code.to(torch.int8) if kind == "int8" else (code.float() / 8).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.exp2(torch.randint(-9, -4, (layers, NB, 2, Hk), generator=g).float())
    if kind == "e4m3":
        scales *= 8
    used = set(bt.flatten().tolist()) - {0}
    for i in range(NB):
        if i not in used:
            scales[:, i] = math.nan
    for b, l in enumerate(lens):
        if l % bs:
            cache[:, bt[b, l // bs].item(), :, :, l % bs:] = 127     # e4m3: NaN
    mass = torch.rand(layers, NB, Hk, bs, generator=g)
    return cache, scales, mass, bt, torch.tensor(lens, dtype=torch.int32)


def attend(q, cache, scales, bt, lens, scale, window=0, softcap=0.0):
    """64-bit attention of one query per row: out, weights per (row, kv head, token), sum(p |v|), sum |q k|."""
    B, H, D = q.shape
    Hk, bs = cache.shape[2], cache.shape[3]
    out = torch.zeros(B, H, D, dtype=torch.float64)
    absv = torch.zeros_like(out)
    weights, big = [], 0.0
    for b in range(B):
        L = int(lens[b])
        lo = max(0, L - window) if window else 0
        at = torch.arange(lo, L)
        w = torch.zeros(Hk, L, dtype=torch.float64)
        if L:
            ids = bt[b].long()[at // bs]
            x = numbers(cache[ids, :, :, at % bs]) * scales[ids].double()[..., None]
            for h in range(H):
                k, v, qq = x[:, 0, h // (H // Hk)], x[:, 1, h // (H // Hk)], q[b, h].double()
                s = k @ qq * scale
                big = max(big, float((k.abs() @ qq.abs()).max()) * scale)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                p = torch.softmax(s, 0)
                out[b, h], absv[b, h] = p @ v, p @ v.abs()
                w[h // (H // Hk), lo:] += p
        weights.append(w)
    return out, weights, absv, big


def check_out(got, out, absv):
    err = (got.double().cpu() - out).abs()
    assert bool((err <= 2.0 ** -8 * out.abs() + 2.0 ** -10 * absv + 1e-30).all()), float((err / (absv + 1e-30)).max())


def check_mass(got, before, weights, bt, lens, bs, D, big, cap=0.0):
    """The weights' sums; everything else untouched to the bit."""
    want, seen = before.double().clone(), torch.zeros_like(before, dtype=torch.bool)
    # the cap's tanh has an absolute error of 2^-20 at most, times the cap
    rel = 2.0 ** -20 + 2 * D * 2.0 ** -24 * big + cap * 2.0 ** -20
    tol = torch.zeros_like(want)
    for b, w in enumerate(weights):
        for t in range(w.shape[1]):
            blk = int(bt[b, t // bs])
            want[blk, :, t % bs] += w[:, t]
            tol[blk, :, t % bs] += rel * w[:, t] + 2.0 ** -23 * want[blk, :, t % bs]
            seen[blk, :, t % bs] |= w[:, t] > 0
    got = got.double().cpu()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
    assert torch.equal(got[~seen], before.double()[~seen])


# ------------------------------------------------------------------------------------------- write
def write_oracle(kv, slots, cache, scales, mass, kind):
    num, sc, ms = numbers(cache), scales.double().clone(), mass.clone()
    bs = cache.shape[3]
    by = {}
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            by.setdefault(s // bs, []).append((t, s % bs))
    x = kv.double().nan_to_num(0.0, 3.3895313892515355e38, -3.3895313892515355e38)
    for blk, rows in by.items():
        for w in range(2):
            for h in range(kv.shape[2]):
                need = least_scale(max(float(x[t, w, h].abs().max()) for t, _ in rows), kind)
                old = float(sc[blk, w, h])
                s = need if any(o == 0 for _, o in rows) else max(old, need)
                if s > old and not any(o == 0 for _, o in rows):
                    num[blk, w, h] = nearest(num[blk, w, h] * (old / s), kind)
                sc[blk, w, h] = s
                for t, o in rows:
                    num[blk, w, h, o] = nearest(x[t, w, h] / s, kind)
        for _, o in rows:
            ms[blk, :, o] = 0
    return num, sc, ms


def write_case(kind, Hk, D, bs, seed):
    """Rows that fill blocks from their start, go on in the middle, sit alone; skipped rows; odd values."""
    g = torch.Generator().manual_seed(seed)
    cache, scales, mass, bt, _ = filled(kind, [3 * bs + 5, 2 * bs], Hk, D, bs, seed)
    scales = scales.nan_to_num(0.25)
    if kind == "e4m3":
        cache = torch.where((cache & 127) == 127, torch.zeros_like(cache), cache)
    slots = []
    slots += [int(bt[0, 0]) * bs + i for i in range(bs)]                   # a whole block
    slots += [-1, int(bt[0, 1]) * bs + 0, -1, int(bt[0, 1]) * bs + 1]      # a block begun, skipped rows around
    slots += [int(bt[0, 2]) * bs + i for i in (3, 4, 5)]                   # in the middle
    slots += [int(bt[0, 3]) * bs + 7, int(bt[1, 0]) * bs + 9, int(bt[1, 1]) * bs + bs - 1, -1]
    kv = torch.randn(len(slots), 2, Hk, D, generator=g)
    kv[-2] *= 1000.0                                                       # its block's scale has to grow
    kv[-3] = 0.0                                                           # nothing to add
    kv[2, 0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, -0.0])
    kv[5, 1] = 1e-38
    return kv.bfloat16(), torch.tensor(slots, dtype=torch.int32), cache[0], scales[0], mass[0]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("Hk,D,bs", [(2, 64, 16), (1, 96, 32), (3, 32, 64)])
def test_write_cpu(kind, Hk, D, bs):
    kv, slots, cache, scales, mass = write_case(kind, Hk, D, bs, 1)
    num, sc, ms = write_oracle(kv, slots, cache, scales, mass, kind)
    ops.kv_quant_blocks(kv, slots, cache, scales, mass=mass)
    assert torch.equal(numbers(cache), num) and torch.equal(scales.double(), sc) and torch.equal(mass, ms)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("Hk,D,bs", [(2, 64, 16), (1, 96, 32), (3, 32, 64), (8, 128, 16), (2, 256, 32)])
def test_write_gpu(kind, Hk, D, bs):
    kv, slots, cache, scales, mass = write_case(kind, Hk, D, bs, 2)
    num, sc, ms = write_oracle(kv, slots, cache, scales, mass, kind)
    c, s, m = cache.cuda(), scales.cuda(), mass.cuda()
    wide = torch.zeros(kv.shape[0], 3, Hk + 1, D + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:, 1:, :D] = kv.cuda()
    ops.kv_quant_blocks(wide[:, 1:, 1:, :D], slots.cuda(), c, s, mass=m)     # a strided view of K / V
    assert torch.equal(numbers(c.cpu()), num) and torch.equal(s.cpu().double(), sc) and torch.equal(m.cpu(), ms)
    c2, s2 = cache.cuda(), scales.cuda()
    ops.kv_quant_blocks(kv.cuda(), slots.cuda(), c2, s2)                     # without weights
    assert torch.equal(c2, c) and torch.equal(s2, s)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("T", [0, 1, 1023, 1024, 2500])
def test_write_long_runs_gpu(kind, T):
    """Prompts of many blocks, the last one part-filled, starting in the middle of a block."""
    Hk, D, bs = 2, 128, 16
    g = torch.Generator().manual_seed(T)
    lens = [T + 21, 40]
    cache, scales, mass, bt, _ = filled(kind, lens, Hk, D, bs, 3)
    scales = scales.nan_to_num(0.5)
    if kind == "e4m3":
        cache = torch.where((cache & 127) == 127, torch.zeros_like(cache), cache)
    pos = torch.arange(21, 21 + T)
    slots = torch.cat([bt[0].long()[pos // bs] * bs + pos % bs, torch.full((5,), -1)]).int()
    kv = torch.randn(T + 5, 2, Hk, D, generator=g).bfloat16()
    want = [x[0].clone() for x in (cache, scales, mass)]
    ops.kv_quant_blocks(kv, slots, *want[:2], mass=want[2])
    got = [x[0].cuda() for x in (cache, scales, mass)]
    ops.kv_quant_blocks(kv.cuda(), slots.cuda(), *got[:2], mass=got[2])
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 5, 40])
def test_write_same_slot_twice_gpu(n):
    """Of rows with the same slot the last one stays (and all of them count for the scale)."""
    g = torch.Generator().manual_seed(n)
    kv = torch.randn(n, 2, 2, 64, generator=g).bfloat16()
    slots = torch.tensor([16 + (i // 2) % 16 for i in range(n)], dtype=torch.int32)
    want = [torch.zeros(3, 2, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2, 2)]
    got = [x.cuda() for x in want]
    ops.kv_quant_blocks(kv, slots, *want)
    ops.kv_quant_blocks(kv.cuda(), slots.cuda(), *got)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# ------------------------------------------------------------------------------------------- decode
LENS = [0, 1, 15, 16, 17, 31, 300, 700]


def test_decode_cpu():
    cache, scales, mass, bt, lens = filled("int8", LENS, 2, 32, 16, 5)
    q = torch.randn(len(LENS), 6, 32, generator=torch.Generator().manual_seed(1))
    m = mass[0].clone()
    got = ops.paged_decode_attention(q, cache[0], bt, lens, 0.2, kv_scales=scales[0], mass=m, window=100, softcap=5.0)
    out, w, absv, big = attend(q, cache[0], scales[0], bt, lens, 0.2, 100, 5.0)
    check_out(got, out, absv)
    check_mass(m, mass[0], w, bt, lens, 16, 32, big, 5.0)
    assert bool((got[0] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D,G,bs", [(128, 4, 16), (64, 8, 32), (96, 1, 16), (32, 7, 64), (256, 2, 16), (256, 12, 32),
                                    (128, 16, 16), (64, 24, 16), (96, 9, 16), (128, 1, 64)])
@pytest.mark.parametrize("splits,weigh", [(0, True), (1, False), (1, True), (5, True), (64, False)])
def test_decode_gpu(kind, D, G, bs, splits, weigh):
    Hk = 2
    cache, scales, mass, bt, lens = filled(kind, LENS, Hk, D, bs, D + G)
    g = torch.Generator().manual_seed(D * G)
    q = (torch.randn(len(LENS), Hk * G, D, generator=g) * 0.5).bfloat16()
    q[3] = 0.0
    q[5] *= 2.0 ** -30
    scale = 1 / math.sqrt(D)
    m = mass[0].cuda()
    dev = [x.cuda() for x in (q, cache[0], bt, lens)]
    got = ops.paged_decode_attention(*dev, scale, num_splits=splits, kv_scales=scales[0].cuda(),
                                     mass=m if weigh else None)
    out, w, absv, big = attend(q, cache[0], scales[0], bt, lens, scale)
    check_out(got, out, absv)
    assert bool((got[0] == 0).all())
    if weigh:
        check_mass(m, mass[0], w, bt, lens, bs, D, big)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (33, 3.0), (5000, 30.0), (0, 0.5)])
def test_decode_window_and_cap_gpu(kind, window, softcap):
    cache, scales, mass, bt, lens = filled(kind, LENS, 2, 64, 16, 9)
    q = torch.randn(len(LENS), 8, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    m = mass[0].cuda()
    got = ops.paged_decode_attention(q.cuda(), cache[0].cuda(), bt.cuda(), lens.cuda(), 0.125, num_splits=0,
                                     kv_scales=scales[0].cuda(), mass=m, window=window, softcap=softcap)
    out, w, absv, big = attend(q, cache[0], scales[0], bt, lens, 0.125, window, softcap)
    check_out(got, out, absv)
    check_mass(m, mass[0], w, bt, lens, 16, 64, big, softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D", [64, 128])
def test_decode_queries_out_of_the_ordinary_gpu(kind, D):
    """A NaN or an infinity in a head's query spoils that head alone; queries of any size keep their precision."""
    cache, scales, _, bt, lens = filled(kind, [50, 300, 129], 2, D, 16, 71)
    q = torch.randn(3, 8, D, generator=torch.Generator().manual_seed(9))
    q[0, 1, 3], q[0, 6, 5], q[1, 2, 0] = math.nan, math.inf, -math.inf
    q[2] *= 2.0 ** torch.tensor([-60, -20, -3, 0, 2, 3, -110, -133]).view(8, 1)     # the last two below the smallest kept size
    q[2, 4, ::2] *= 2.0 ** -12                                                       # a wide spread within a head
    q = q.bfloat16()
    got = ops.paged_decode_attention(q.cuda(), cache[0].cuda(), bt.cuda(), lens.cuda(), 0.1, num_splits=0,
                                     kv_scales=scales[0].cuda())
    bad = torch.zeros(3, 8, dtype=torch.bool)
    bad[0, 1] = bad[0, 6] = bad[1, 2] = True
    assert bool(got.cpu()[bad].isnan().all())
    out, _, absv, _ = attend(q.nan_to_num(0.0, 0.0, 0.0), cache[0], scales[0], bt, lens, 0.1)
    check_out(torch.where(bad[..., None].cuda(), out.cuda().float(), got.float()), out, absv)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [33, 100, 1100])
def test_decode_many_rows_gpu(B):
    """More rows than lanes (and than lanes of lanes), a third of them empty, tables wider than any row."""
    g = torch.Generator().manual_seed(B)
    lens = (torch.randint(-20, 60, (B,), generator=g).clamp(min=0)).tolist()
    cache, scales, mass, bt, sl = filled("int8", lens, 1, 32, 16, B)
    bt = torch.nn.functional.pad(bt, (0, 70))
    q = torch.randn(B, 4, 32, generator=g).bfloat16()
    m = mass[0].cuda()
    got = ops.paged_decode_attention(q.cuda(), cache[0].cuda(), bt.cuda(), sl.cuda(), 0.2, num_splits=0,
                                     kv_scales=scales[0].cuda(), mass=m)
    out, w, absv, big = attend(q, cache[0], scales[0], bt, sl, 0.2)
    check_out(got, out, absv)
    check_mass(m, mass[0], w, bt, sl, 16, 32, big)
    assert not bool(got[sl.cuda() == 0].any())


@pytest.mark.gpu
def test_no_rows_and_no_blocks_gpu():
    cache, scales = torch.zeros(3, 2, 2, 16, 64, dtype=torch.int8, device="cuda"), torch.ones(3, 2, 2, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    out = ops.paged_decode_attention(q[:0], cache, torch.zeros(0, 4, **i32), torch.zeros(0, **i32), 1.0, num_splits=0, kv_scales=scales)
    assert out.shape == (0, 4, 64)
    out = ops.paged_decode_attention(q, cache, torch.zeros(2, 0, **i32), torch.ones(2, **i32), 1.0, num_splits=0, kv_scales=scales)
    assert not bool(out.any())
    kept = ops.kv_evict(cache, scales, torch.zeros(3, 2, 16, device="cuda"), torch.zeros(0, 4, **i32), torch.zeros(0, **i32),
                        torch.zeros(0, **i32), 1, 1, max_keep=3)
    assert kept.shape == (0, 2, 3)
    out = ops.paged_prefill_attention(q[:0], cache, torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32), 1.0,
                                      kv_scales=scales)
    assert out.shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_decode_uneven_scales_gpu(kind):
    """Value scales 2^-100 .. 2^90 apart from block to block, a dominant token in a block of tiny values, all-zero
    blocks, scores of +-200: nothing may overflow or drown."""
    Hk, D, bs = 2, 64, 16
    cache, scales, _, bt, lens = filled(kind, [90, 64, 48], Hk, D, bs, 11)
    cache, scales = cache[0], scales[0]
    q = torch.randn(3, 8, D, generator=torch.Generator().manual_seed(3)).bfloat16() * 8
    scales[bt[0, 0], 1] = 2.0 ** -100
    scales[bt[0, 2], 1] = 2.0 ** 90
    cache[bt[1, 1], 1] = 0
    scales[bt[1, 1], 1] = 2.0 ** -100
    scales[bt[2, 0], 1] = 2.0 ** -60
    scales[bt[2, 0], 0] *= 64                        # its scores decide the softmax
    got = ops.paged_decode_attention(q.cuda(), cache.cuda(), bt.cuda(), lens.cuda(), 1.0, num_splits=0,
                                     kv_scales=scales.cuda())
    out, _, absv, _ = attend(q, cache, scales, bt, lens, 1.0)
    # scores of up to some thousand: an fp32 score is off by up to 2 D 2^-24 of sum |q k|, and so is a weight
    big = max(attend(q[b:b + 1], cache, scales, bt[b:b + 1], lens[b:b + 1], 1.0)[3] for b in range(3))
    err = (got.double().cpu() - out).abs()
    # p * scale is held in f16 over a reference no larger than its largest value among the tokens: below
    # 2^-14 of it f16 steps are 2^-24, so a token's term is off by up to 2^-25 qmax max(p scale) even where its
    # own p is far smaller (sums in which only such tokens have a non-zero code)
    floor = torch.zeros_like(out)
    for b in range(3):
        at = torch.arange(int(lens[b]))
        ids = bt[b].long()[at // bs]
        for h in range(8):
            k = numbers(cache[ids, 0, h // 4, at % bs]) * scales[ids, 0, h // 4].double()[:, None]
            p = torch.softmax(k @ q[b, h].double(), 0)
            floor[b, h] = len(at) * 2.0 ** -25 * 448 * float((p * scales[ids, 1, h // 4].double()).max())
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -10 + 4 * D * 2.0 ** -24 * big) * absv + floor
    assert bool((err <= tol).all())


@pytest.mark.gpu
def test_decode_strides_stream_graph_and_shared_blocks_gpu():
    cache, scales, mass, bt, lens = filled("int8", [200, 333, 64], 2, 128, 16, 13)
    qkv = torch.randn(3, (8 + 4) * 128, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    q = qkv[:, :8 * 128].view(3, 8, 128)
    wide = torch.zeros(5, bt.shape[1] + 9, dtype=torch.int32, device="cuda")
    wide[:3, :bt.shape[1]] = bt.cuda()
    c, s, l = cache[0].cuda(), scales[0].cuda(), lens.cuda()
    base = ops.paged_decode_attention(q, c, wide[:, :bt.shape[1]], l, 0.09, num_splits=0, kv_scales=s)
    out, w, absv, big = attend(q.cpu(), cache[0], scales[0], bt, lens, 0.09)
    check_out(base, out, absv)
    # another stream gives the same bits
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = ops.paged_decode_attention(q, c, wide, l, 0.09, num_splits=3, kv_scales=s)
    torch.cuda.current_stream().wait_stream(st)
    check_out(other, out, absv)
    # captured with other lengths, replayed twice, weights added twice
    m = mass[0].cuda()
    lg = torch.zeros_like(l)
    g = torch.cuda.CUDAGraph()
    res = ops.paged_decode_attention(q, c, wide, lg, 0.09, num_splits=0, kv_scales=s, mass=m)
    with torch.cuda.graph(g):
        res = ops.paged_decode_attention(q, c, wide, lg, 0.09, num_splits=0, kv_scales=s, mass=m)
    lg.copy_(l)
    g.replay()
    g.replay()
    check_out(res, out, absv)
    check_mass(m, mass[0], [2 * x for x in w], bt, lens, 16, 128, big)
    # two rows over the same blocks: both rows' weights arrive
    bt2, l2 = bt.clone(), torch.tensor([200, 200, 64], dtype=torch.int32)
    bt2[1] = bt2[0]
    m = mass[0].cuda()
    got = ops.paged_decode_attention(q, c, bt2.cuda(), l2.cuda(), 0.09, num_splits=0, kv_scales=s, mass=m)
    out, w, absv, big = attend(q.cpu(), cache[0], scales[0], bt2, l2, 0.09)
    check_out(got, out, absv)
    check_mass(m, mass[0], w, bt2, l2, 16, 128, big)


@pytest.mark.gpu
def test_large_workspace_offsets_gpu():
    """64 CTAs a sequence over 8200 sequences: the parts' sums lie up to 2^32 floats and more behind the workspace's start."""
    B, L, G, D = 8200, 4096, 16, 256
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    cache, scales, _, bt, sl = filled("int8", [L], 1, D, 16, 97)
    q = torch.randn(8, G, D, generator=torch.Generator().manual_seed(5)).bfloat16()
    out, _, absv, _ = attend(q, cache[0], scales[0], bt.expand(8, -1), sl.expand(8), 0.05)
    rows = torch.arange(B) % 8
    got = ops.paged_decode_attention(q[rows].cuda(), cache[0].cuda(), bt.cuda().expand(B, -1).contiguous(),
                                     torch.full((B,), L, dtype=torch.int32, device="cuda"), 0.05, 64, kv_scales=scales[0].cuda())
    check_out(got[:8], out, absv)
    assert torch.equal(got.view(-1, 8, G, D), got[:8].expand(B // 8, -1, -1, -1))   # every row splits alike
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_large_pool_offsets_gpu():
    """Blocks whose byte offsets pass 2^32."""
    Hk, D, bs = 8, 128, 16
    NB = (1 << 32) // (2 * Hk * bs * D) + 200
    cache = torch.zeros(NB, 2, Hk, bs, D, dtype=torch.int8, device="cuda")
    scales = torch.full((NB, 2, Hk), 0.01, device="cuda")
    mass = torch.zeros(NB, Hk, bs, device="cuda")
    small, ssc, _, sbt, lens = filled("int8", [100, 50], Hk, D, bs, 17)
    bt = torch.where(sbt > 0, NB - 1 - sbt, torch.zeros_like(sbt))
    for i in set(sbt.flatten().tolist()) - {0}:
        cache[NB - 1 - i], scales[NB - 1 - i] = small[0, i].cuda(), ssc[0, i].cuda()
    q = torch.randn(2, 32, D, generator=torch.Generator().manual_seed(5)).bfloat16()
    got = ops.paged_decode_attention(q.cuda(), cache, bt.cuda(), lens.cuda(), 0.09, num_splits=0, kv_scales=scales,
                                     mass=mass)
    out, w, absv, _ = attend(q, small[0], ssc[0], sbt, lens, 0.09)
    check_out(got, out, absv)
    assert abs(float(mass.double().sum()) - 64) < 1e-3
    want = [small, ssc.clone(), torch.zeros(1, small.shape[1], Hk, bs)]
    for i in set(sbt.flatten().tolist()) - {0}:
        want[2][0, i] = mass[NB - 1 - i].cpu()
    keep = torch.tensor([40, 33], dtype=torch.int32)
    k1 = ops.kv_evict(*want, sbt, lens, keep, 4, 8, max_keep=40)
    k2 = ops.kv_evict(cache, scales, mass, bt.cuda(), lens.cuda(), keep.cuda(), 4, 8, max_keep=40)
    assert torch.equal(k2.cpu(), k1[0])
    for i in set(sbt.flatten().tolist()) - {0}:
        assert torch.equal(cache[NB - 1 - i].cpu(), want[0][0, i])


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 3])
def test_weights_share_their_work_by_the_lengths_gpu(G):
    """More pieces of 1024 tokens than the join has CTAs for them, rows of no and of one token among them; and a table
    64 times wider than the rows need gives the same, to the bit."""
    g = torch.Generator().manual_seed(87)
    lens = [0, 1, 1023, 1024, 1025] + torch.randint(1, 2600, (420,), generator=g).tolist() + [0]
    Hk, D = 4, 32
    cache, scales, mass, bt, sl = filled("int8", lens, Hk, D, 16, 89)
    q = torch.randn(len(lens), Hk * G, D, generator=g).bfloat16()
    out, weights, absv, big = attend(q, cache[0], scales[0], bt, sl, 0.2)
    wide = torch.zeros(len(lens), bt.shape[1] * 64, dtype=torch.int32, device="cuda")
    wide[:, :bt.shape[1]] = bt.cuda()
    ends = []
    for table in (bt.cuda(), wide):
        m = mass[0].cuda()
        got = ops.paged_decode_attention(q.cuda(), cache[0].cuda(), table, sl.cuda(), 0.2, 0, kv_scales=scales[0].cuda(), mass=m)
        ends.append((got.cpu(), m.cpu()))
    check_out(ends[0][0], out, absv)
    want, tol, seen = mass[0].double(), torch.zeros_like(mass[0], dtype=torch.float64), torch.zeros_like(mass[0], dtype=torch.bool)
    for b, w in enumerate(weights):                                    # as check_mass, a row at a time
        at = torch.arange(w.shape[1])
        ids, off = bt[b].long()[at // 16], at % 16
        want[ids, :, off] += w.T
        tol[ids, :, off] = (2.0 ** -20 + 2 * D * 2.0 ** -24 * big) * w.T + 2.0 ** -23 * want[ids, :, off]
        seen[ids, :, off] = True
    got = ends[0][1].double()
    assert bool(((got - want).abs() <= tol).all()) and torch.equal(got[~seen], mass[0].double()[~seen])
    assert torch.equal(ends[0][0], ends[1][0]) and torch.equal(ends[0][1], ends[1][1])


# ------------------------------------------------------------------------------------------- prompts
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D,G,bs,window", [(128, 4, 16, 0), (64, 7, 16, 0), (128, 2, 32, 0), (64, 1, 64, 50),
                                           (32, 2, 16, 0), (256, 2, 16, 0)])
def test_prefill_gpu(kind, D, G, bs, window):
    Hk = 2
    lens, new = [1, 130, 257, 40, 500], [1, 130, 2, 17, 133]
    cache, scales, _, bt, sl = filled(kind, lens, Hk, D, bs, 19)
    cache, scales = cache[0], scales[0]
    qs = torch.tensor([0] + new).cumsum(0).int()
    q = (torch.randn(int(qs[-1]), Hk * G, D, generator=torch.Generator().manual_seed(6)) * 0.5).bfloat16()
    scale = 1 / math.sqrt(D)
    got = ops.paged_prefill_attention(q.cuda(), cache.cuda(), bt.cuda(), sl.cuda(), qs.cuda(), scale, window=window,
                                      kv_scales=scales.cuda()).double().cpu()
    for b, n in enumerate(new):
        rows = torch.arange(lens[b] - n + 1, lens[b] + 1, dtype=torch.int32)
        out, _, absv, _ = attend(q[qs[b]:qs[b + 1]], cache, scales, bt[b:b + 1].expand(n, -1), rows, scale, window)
        # the prompt kernels hold p in bf16 (half a step 2^-8)
        err = (got[qs[b]:qs[b + 1]] - out).abs()
        assert bool((err <= 2.0 ** -8 * out.abs() + 2.0 ** -7 * absv).all()), (b, float((err / absv).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D,G,bs,window,softcap", [(64, 4, 16, 0, 0.0), (128, 8, 16, 0, 0.0), (128, 7, 32, 300, 0.0),
                                                   (64, 12, 16, 129, 20.0), (64, 1, 64, 1, 0.0), (128, 2, 16, 0, 5.0)])
def test_prefill_long_prefixes_gpu(kind, D, G, bs, window, softcap):
    """Items that several CTAs share, sequences without new tokens, more CTAs than tiles; sampled rows."""
    for lens, new in (([2000, 5, 3100, 64, 700], [50, 0, 1, 0, 700]), ([40, 129], [3, 129]), ([6000], [90])):
        cache, scales, _, bt, sl = filled(kind, lens, 1, D, bs, 61)
        cache, scales = cache[0], scales[0]
        qs = torch.tensor([0] + new).cumsum(0).int()
        g = torch.Generator().manual_seed(7)
        wide = (torch.randn(int(qs[-1]), G * D + 64, generator=g) * 0.5).bfloat16().cuda()
        q = wide[:, :G * D].view(-1, G, D)                                        # rows of a wider projection
        scale = 1 / math.sqrt(D)
        got = ops.paged_prefill_attention(q, cache.cuda(), bt.cuda(), sl.cuda(), qs.cuda(), scale, window=window,
                                          softcap=softcap, kv_scales=scales.cuda()).double().cpu()
        for b, n in enumerate(new):
            rows = sorted({0, n - 1, n // 2, *torch.randint(0, max(n, 1), (6,), generator=g).tolist()}) if n else []
            for r in rows:
                at = lens[b] - n + r + 1
                out, _, absv, _ = attend(q[qs[b] + r: qs[b] + r + 1].cpu(), cache, scales, bt[b:b + 1],
                                         torch.tensor([at]), scale, window, softcap)
                err = (got[qs[b] + r] - out[0]).abs()
                # p in bf16 (half a step 2^-8), and the cap's tanh in hardware (2^-11 relative, on a score of at most the cap)
                tol = 2.0 ** -8 * out[0].abs() + (2.0 ** -7 + 2 * softcap * 2.0 ** -11) * absv[0]
                assert bool((err <= tol).all()), (lens, b, r, float((err / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tiles", [False, True])
def test_prefill_lengths_beside_the_queries_gpu(D, tiles):
    """Queries in front of their sequence's first token get zeros; a length beyond the table is cut to it. With its short
    table the work list is taken where there is one."""
    lens, new, H = [0, 100, 7, 300], [150, 400, 7, 20], 40 if tiles else 4
    cache, scales, _, bt, sl = filled("int8", lens, 2, D, 16, 73)
    bt, sl[3] = bt[:, :16], 1000                                       # 256 tokens fit the table
    qs = torch.tensor([0] + new).cumsum(0).int()
    q = torch.randn(int(qs[-1]), H, D, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    work = torch.tensor([[b, r, -1, h] for b, n in enumerate(new) for r in range(0, n, 128) for h in range(H)],
                        dtype=torch.int32)
    got = ops.paged_prefill_attention(q, cache[0].cuda(), bt.cuda(), sl.cuda(), qs.cuda(), 0.1, tiles=work.cuda() if tiles else None,
                                      out=torch.full_like(q, math.nan), kv_scales=scales[0].cuda()).double().cpu()
    assert not bool(got[:150].any()) and not bool(got[150:450].any())
    for b, n in enumerate(new):
        L = min(lens[b] if b < 3 else 1000, 256)
        rows = torch.arange(L - n + 1, L + 1).clamp(min=0).int()
        out, _, absv, _ = attend(q[qs[b]:qs[b + 1]].cpu(), cache[0], scales[0], bt[b:b + 1].expand(n, -1), rows, 0.1)
        assert bool(((got[qs[b]:qs[b + 1]] - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -7 * absv).all())


@pytest.mark.parametrize("device,D", [("cpu", 32), ("cpu", 64), *(pytest.param("cuda", D, marks=pytest.mark.gpu) for D in (32, 256))])
def test_prefill_lengths_beside_the_queries_elsewhere(device, D):
    """The same on the CPU and at the head sizes that go through the work list over a copy."""
    lens, new, H = [0, 100, 7, 300], [150, 400, 7, 20], 4
    cache, scales, _, bt, sl = filled("int8", lens, 2, D, 16, 79)
    bt, sl[3] = bt[:, :16], 1000                                       # 256 tokens fit the table
    qs = torch.tensor([0] + new).cumsum(0).int()
    q = torch.randn(int(qs[-1]), H, D, generator=torch.Generator().manual_seed(6)).bfloat16()
    c, s, t, l, st = (x.to(device) for x in (cache[0], scales[0], bt, sl, qs))
    got = ops.paged_prefill_attention(q.to(device), c, t, l, st, 0.1, out=torch.full_like(q, math.nan, device=device),
                                      kv_scales=s).double().cpu()
    assert not bool(got[:150].any()) and not bool(got[150:450].any())
    for b, n in enumerate(new):
        L = min(lens[b] if b < 3 else 1000, 256)
        rows = torch.arange(L - n + 1, L + 1).clamp(min=0).int()
        out, _, absv, _ = attend(q[qs[b]:qs[b + 1]], cache[0], scales[0], bt[b:b + 1].expand(n, -1), rows, 0.1)
        assert bool(((got[qs[b]:qs[b + 1]] - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -7 * absv).all())


@pytest.mark.gpu
def test_prefill_captured_gpu():
    """A captured step replayed with other lengths and chunk borders."""
    lens, new = [300, 50, 210], [100, 50, 3]
    cache, scales, _, bt, sl = filled("int8", lens, 2, 64, 16, 67)
    c, s, t = cache[0].cuda(), scales[0].cuda(), bt.cuda()
    qs = torch.tensor([0] + new).cumsum(0).int().cuda()
    q = torch.randn(int(qs[-1]), 8, 64, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    lg, qg = torch.tensor([160, 40, 200], dtype=torch.int32).cuda(), torch.tensor([0, 40, 80, 153], dtype=torch.int32).cuda()
    ops.paged_prefill_attention(q, c, t, lg, qg, 0.1, kv_scales=s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.paged_prefill_attention(q, c, t, lg, qg, 0.1, kv_scales=s)
    lg.copy_(sl.cuda())
    qg.copy_(qs)
    g.replay()
    assert torch.equal(out, ops.paged_prefill_attention(q, c, t, sl.cuda(), qs, 0.1, kv_scales=s))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 32, 256])
def test_prefill_copy_of_a_wide_table_is_bounded_gpu(D):
    """Tables far wider than their rows need: the copy stays within 1 GiB and the sequences go in groups; without a work
    list and with one (which the groups leave unused), a row without queries and one without tokens among them."""
    lens, new, H = [700, 0, 2100, 40, 333], [60, 0, 130, 40, 1], 8
    cache, scales, _, bt, sl = filled("int8", lens, 2, D, 16, 83)
    qs = torch.tensor([0] + new).cumsum(0).int()
    q = torch.randn(int(qs[-1]), H, D, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    c, s, l = cache[0].cuda(), scales[0].cuda(), sl.cuda()
    width = 400 * 2 ** 20 // (4 * D * 2) // 16                          # a row's copy takes 400 MiB: two rows a group
    wide = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    wide[:, :bt.shape[1]] = bt.cuda()
    work = ops.prefill_schedule(qs.tolist(), lens, H, 2, D).cuda()
    want = ops.paged_prefill_attention(q, c, bt.cuda(), l, qs.cuda(), 0.1, kv_scales=s)
    for tiles in (None, work):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = ops.paged_prefill_attention(q, c, wide, l, qs.cuda(), 0.1, tiles=tiles, kv_scales=s)
        assert torch.cuda.max_memory_allocated() - before < 2 ** 30 + 2 ** 27
        got = got.double().cpu()
        for b, n in enumerate(new):
            rows = torch.arange(lens[b] - n + 1, lens[b] + 1, dtype=torch.int32)
            out, _, absv, _ = attend(q[qs[b]:qs[b + 1]].cpu(), cache[0], scales[0], bt[b:b + 1].expand(n, -1), rows, 0.1)
            for x in (got, want.double().cpu()):
                assert bool(((x[qs[b]:qs[b + 1]] - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -7 * absv).all())


def infinite_values(kind, D=64):
    """80 tokens written through the operator, the 41st with infinities in V (and a NaN), and 64-bit values of them all."""
    g = torch.Generator().manual_seed(31)
    kv = torch.randn(80, 2, 2, D, generator=g)
    kv[40, 1, 0, 3], kv[40, 1, 0, 4], kv[40, 1, 1, 5] = math.inf, -math.inf, math.nan
    cache = torch.zeros(6, 2, 2, 16, D, dtype=KINDS[kind])
    scales, bt = torch.zeros(6, 2, 2), torch.tensor([[3, 5, 1, 0, 4]], dtype=torch.int32)
    at = torch.arange(80)
    ops.kv_quant_blocks(kv.bfloat16(), (bt[0].long()[at // 16] * 16 + at % 16).int(), cache, scales)
    return cache, scales, bt, g


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", list(KINDS))
def test_infinities_stay_finite_when_read(kind, device):
    """The code of the largest bf16 rounds to 2^128. Read as an infinity it would spoil queries that it is masked from (0 times
    infinity), and an eviction's scales."""
    cache, scales, bt, g = infinite_values(kind)
    big = values(cache, scales).abs().max()
    assert float(big) == 2.0 ** 128
    c, s, t = cache.clone().to(device), scales.clone().to(device), bt.to(device)
    copy, _ = ops.kv_dequant_blocks(c, s, t)
    assert float(copy.double().abs().max()) == float(torch.finfo(torch.bfloat16).max)
    assert torch.equal(copy.double().cpu().sign(), values(cache, scales)[bt[0].long()].sign().view_as(copy))
    # prompts: the queries of tokens 30 .. 79; p in bf16, and 2^128 as the largest bf16: half a step 2^-8 each, and the output's
    q = torch.randn(50, 4, 64, generator=g).bfloat16()
    lens = torch.arange(31, 81, dtype=torch.int32)
    out, _, absv, _ = attend(q, cache, scales, bt.expand(50, -1), lens, 0.2)
    got = ops.paged_prefill_attention(q.to(device), c, t, torch.tensor([80], dtype=torch.int32, device=device),
                                      torch.tensor([0, 50], dtype=torch.int32, device=device), 0.2, kv_scales=s)
    err = (got.double().cpu() - out).abs()
    assert bool(torch.isfinite(got).all()) and bool((err <= 2.0 ** -8 * out.abs() + (2.0 ** -7 + 2.0 ** -8) * absv).all())
    # eviction: token 40's block keeps its code and gets the scale that holds it
    mass = torch.rand(6, 2, 16, generator=g)
    mass[1, :, 8] = 2.0
    m = mass.to(device)
    kept = ops.kv_evict(c, s, m, t, torch.tensor([80], dtype=torch.int32, device=device),
                        torch.tensor([50], dtype=torch.int32, device=device), 4, 8).cpu()
    for h in range(2):
        src = kept[0, h, :50].long()
        x = values(cache, scales)[bt[0].long()[src // 16], :, h, src % 16]                  # [50, 2, D]
        for j in range(0, 50, 16):
            for w in range(2):
                scale = least_scale(min(float(x[j:j + 16, w].abs().max()), 2.0 ** 128 * (1 - 2.0 ** -8)), kind)
                blk = int(bt[0, j // 16])
                n = len(x[j:j + 16])
                assert float(s[blk, w, h]) == scale
                assert torch.equal(numbers(c.cpu()[blk, w, h, :n]), nearest(x[j:j + 16, w] / scale, kind))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("splits", [0, 64])
def test_decode_over_the_largest_values(kind, splits, device):
    """Value scales up to 2^122 beside ordinary ones: the weights of the block's own tokens may not drown, down to 2^-20 of
    the largest, nor the sum they are divided by; a token of the largest bf16 alone reads as that."""
    cache, scales, bt, g = infinite_values(kind)
    q = torch.randn(50, 4, 64, generator=g).bfloat16()
    lens = torch.arange(31, 81, dtype=torch.int32)
    out, _, absv, _ = attend(q, cache, scales, bt.expand(50, -1), lens, 0.2)
    dev = [x.to(device) for x in (q, cache, bt.expand(50, -1).contiguous(), lens)]
    got = ops.paged_decode_attention(*dev, 0.2, splits, kv_scales=scales.to(device)).double().cpu()
    # p times its block's scale is held in f16 against the largest of them: rows that see a token of token 40's block (32 .. 47)
    # are off by up to 2^-25 of that a token and unit of code (as in test_decode_uneven_scales_gpu); the codes there are
    # zero but for token 40's, at most 64 (256 in e4m3), whose product 2^128 stands for, so 2^-25 2^128 a token; and 2^128
    # reads as the largest bf16, 2^-8 less
    floor = torch.where(lens > 32, 80 * 2.0 ** -25 * 2.0 ** 128, 0.0)[:, None, None]
    assert bool(((got - out).abs() <= 2.0 ** -8 * out.abs() + (2.0 ** -10 + 2.0 ** -8) * absv + floor).all())
    one = torch.full((1,), 41, dtype=torch.int32, device=device)
    got = ops.paged_decode_attention(dev[0][:1], dev[1], dev[2][:1], one, 0.2, splits, kv_scales=scales.to(device), window=1)
    top = float(torch.finfo(torch.bfloat16).max)
    assert float(got[0, 0, 3]) == top and float(got[0, 1, 4]) == -top and float(got[0, 2, 5]) == 0.0


def test_gather_cpu_behind_the_end():
    cache, scales, _, bt, lens = filled("e4m3", [5, 70], 2, 32, 32, 23)
    tmp, table = ops.kv_dequant_blocks(cache[0], scales[0], bt, lens)
    x = tmp[table.long()].permute(0, 3, 2, 1, 4, 5)                    # [n, Hk, 2, mb16, 16, D]
    flat = x.reshape(2, 2, 2, -1, 32)
    want = values(cache[0], scales[0])[bt.long()].permute(0, 3, 2, 1, 4, 5).reshape(2, 2, 2, -1, 32)
    for b, l in enumerate([5, 70]):
        assert torch.equal(flat[b, :, :, :l].double(), want[b, :, :, :l]) and not bool(flat[b, :, :, l:].any())


# ------------------------------------------------------------------------------------------- eviction
def evict_oracle(cache, scales, mass, bt, lens, keep, sink, recent, max_keep, kind):
    num, sc, ms = numbers(cache), scales.double().clone(), mass.clone()
    n0, s0, m0 = num.clone(), sc.clone(), ms.clone()
    Ly, _, _, Hk, bs, D = cache.shape
    kept = torch.full((Ly, len(lens), Hk, max_keep), -1, dtype=torch.int32)
    for b, L in enumerate(lens.tolist()):
        K = min(max(int(keep[b]), 0), L)
        if K == L:
            kept[:, b, :, : min(L, max_keep)] = torch.arange(min(L, max_keep), dtype=torch.int32)
            continue
        K = min(K, max_keep)
        a = min(sink, K)
        r = min(recent, K - a)
        for ly in range(Ly):
            for h in range(Hk):
                w = [float(m0[ly, bt[b, t // bs], h, t % bs]) for t in range(L)]
                mid = sorted(range(a, L - r), key=lambda t: (-(w[t] if w[t] == w[t] else 0.0), t))[: K - a - r]
                take = list(range(a)) + sorted(mid) + list(range(L - r, L))
                kept[ly, b, h, :K] = torch.tensor(take, dtype=torch.int32)
                for j0 in range(0, K, bs):
                    part = take[j0:j0 + bs]
                    blk = int(bt[b, j0 // bs])
                    for kvi in range(2):
                        v = torch.stack([n0[ly, bt[b, t // bs], kvi, h, t % bs] * s0[ly, bt[b, t // bs], kvi, h] for t in part])
                        s = least_scale(float(v.abs().max()), kind)
                        sc[ly, blk, kvi, h] = s
                        num[ly, blk, kvi, h, : len(part)] = nearest(v / s, kind)
                    for i, t in enumerate(part):
                        ms[ly, blk, h, i] = m0[ly, bt[b, t // bs], h, t % bs]
    return kept, num, sc, ms


def same(a, b):
    return torch.equal(a.nan_to_num(1.25e33), b.nan_to_num(1.25e33))


def evict_case(kind, D, bs, seed, layers=2, Hk=2):
    lens = [5 * bs + 3, 40, 1, 0, 2 * bs, 100]
    keep = [2 * bs + 5, 39, 0, 0, 5 * bs, 1]
    cache, scales, mass, bt, sl = filled(kind, lens, Hk, D, bs, seed, layers)
    g = torch.Generator().manual_seed(seed)
    mass = torch.where(torch.rand(mass.shape, generator=g) < 0.4, torch.round(mass * 4) / 4, mass)   # many ties
    mass[0, bt[0, 1], 0, 2] = math.nan
    mass[0, bt[0, 2], 1, 1] = math.inf
    mass[0, bt[0, 2], 0, 3] = -0.0
    return cache, scales, mass, bt, sl, torch.tensor(keep, dtype=torch.int32)


EVICT = [(4, 8, None), (0, 0, None), (1000, 3, None), (2, 1000, None), (3, 5, 20)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("sink,recent,max_keep", EVICT)
def test_evict_cpu(kind, sink, recent, max_keep):
    c = evict_case(kind, 32, 16, 29)
    want = evict_oracle(*c, sink, recent, max_keep or c[3].shape[1] * 16, kind)
    got = ops.kv_evict(*c, sink, recent, max_keep=max_keep)
    assert torch.equal(got, want[0]) and same(numbers(c[0]), want[1])
    assert same(c[1].double(), want[2]) and same(c[2], want[3])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("K", [4, 20])
def test_evict_zeros_out_of_a_large_scale(kind, K, device):
    """The neighbours of an infinity are zeros at a scale of 2^120 or more. Once that token is dropped they go to a scale of 2^-100
    (among themselves) or of ordinary tokens, and stay zeros."""
    g = torch.Generator().manual_seed(37)
    kv = torch.randn(48, 2, 2, 128, generator=g)
    kv[5, :, :, 7] = math.inf
    cache, scales, bt = torch.zeros(4, 2, 2, 16, 128, dtype=KINDS[kind]), torch.zeros(4, 2, 2), torch.tensor([[2, 0, 3]], dtype=torch.int32)
    at = torch.arange(48)
    ops.kv_quant_blocks(kv.bfloat16(), (bt[0].long()[at // 16] * 16 + at % 16).int(), cache, scales)
    mass = torch.rand(4, 2, 16, generator=g)
    mass[2, :, 5] = 0.0
    x = values(cache, scales)[bt[0].long()].permute(1, 2, 0, 3, 4).reshape(2, 2, 48, 128)
    c, s = cache.clone().to(device), scales.clone().to(device)
    kept = ops.kv_evict(c, s, mass.clone().to(device), bt.to(device), torch.tensor([48], dtype=torch.int32, device=device),
                        torch.tensor([K], dtype=torch.int32, device=device), 4, 0).cpu()
    for h in range(2):
        src = kept[0, h, :K].long()
        assert 5 not in src.tolist() and src[:4].tolist() == [0, 1, 2, 3]
        for w in range(2):
            for j in range(0, K, 16):
                y = x[w, h, src[j:j + 16]]
                scale, blk = least_scale(float(y.abs().max()), kind), int(bt[0, j // 16])
                assert float(s[blk, w, h]) == scale
                assert torch.equal(numbers(c.cpu()[blk, w, h, :len(y)]), nearest(y / scale, kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32), (64, 16), (96, 16), (256, 64), (32, 16), (160, 16), (192, 32), (224, 16)])
@pytest.mark.parametrize("sink,recent,max_keep", EVICT)
def test_evict_gpu(kind, D, bs, sink, recent, max_keep):
    c = evict_case(kind, D, bs, 31)
    want = evict_oracle(*c, sink, recent, max_keep or c[3].shape[1] * bs, kind)
    d = [x.cuda() for x in c]
    got = ops.kv_evict(*d, sink, recent, max_keep=max_keep)
    assert torch.equal(got.cpu(), want[0]) and same(numbers(d[0].cpu()), want[1])
    assert same(d[1].cpu().double(), want[2]) and same(d[2].cpu(), want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("L,K,ties", [(3000, 2000, False), (20000, 5000, True), (40000, 39999, False)])
def test_evict_long_gpu(L, K, ties):
    """Many chunks moved over one another; sequences whose weights do not fit on chip; a single layer's tensors."""
    Hk, D, bs = 1, 64, 16
    c = filled("int8", [L], Hk, D, bs, 37)
    cache, scales, mass, bt, sl = c[0][0], c[1][0], c[2][0], c[3], c[4]
    mass = torch.round(mass * 50) / 50 if ties else mass
    keep = torch.tensor([K], dtype=torch.int32)
    d = [x.cuda() for x in (cache, scales, mass, bt, sl, keep)]
    want = ops.kv_evict(cache, scales, mass, bt, sl, keep, 16, 100, max_keep=K)
    got = ops.kv_evict(*d, 16, 100, max_keep=K)
    assert torch.equal(got.cpu(), want) and torch.equal(d[0].cpu(), cache)
    assert same(d[1].cpu(), scales) and same(d[2].cpu(), mass)


# ------------------------------------------------------------------------------------------- together
def together(kind, dev, steps=40):
    """A sequence grows token by token, is weighed, evicted and grows on; returns every output and the final cache."""
    Hk, G, D, bs = 2, 4, 64, 16
    g = torch.Generator().manual_seed(41)
    NB = 12
    cache = torch.zeros(NB, 2, Hk, bs, D, dtype=KINDS[kind], device=dev)
    scales = torch.zeros(NB, 2, Hk, device=dev)
    mass = torch.zeros(NB, Hk, bs, device=dev)
    bt = torch.tensor([[7, 3, 9, 1, 5, 2]], dtype=torch.int32)
    n, outs = 0, []

    def put(k):
        nonlocal n
        pos = torch.arange(n, n + k)
        slots = (bt[0].long()[pos // bs] * bs + pos % bs).int()
        kv = (torch.randn(k, 2, Hk, D, generator=g) * torch.exp2(torch.rand(k, 2, Hk, 1, generator=g) * 4)).bfloat16()
        ops.kv_quant_blocks(kv.to(dev), slots.to(dev), cache, scales, mass=mass)
        n += k

    put(37)
    for i in range(steps):
        q = (torch.randn(1, Hk * G, D, generator=g) * 0.3).bfloat16()
        outs.append(ops.paged_decode_attention(q.to(dev), cache, bt.to(dev), torch.tensor([n], dtype=torch.int32).to(dev),
                                               0.125, num_splits=0, kv_scales=scales, mass=mass).float().cpu())
        if n > 60:
            kept = ops.kv_evict(cache, scales, mass, bt.to(dev), torch.tensor([n], dtype=torch.int32).to(dev),
                                torch.tensor([35], dtype=torch.int32).to(dev), 4, 10, max_keep=35)
            outs.append(kept.float().cpu())
            n = 35
        put(1)
    return outs, cache.cpu(), scales.cpu(), mass.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_write_weigh_evict_together_gpu(kind):
    a, b = together(kind, "cpu"), together(kind, "cuda")
    # the same tokens stay (weights differ in their last bits only), so codes and scales are equal
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    torch.testing.assert_close(b[3], a[3], rtol=1e-4, atol=1e-6)
    for x, y in zip(b[0], a[0]):
        # both sides round to bf16 (half a step 2^-8 each)
        torch.testing.assert_close(x, y, rtol=2 * 2.0 ** -8, atol=2.0 ** -6)


# ------------------------------------------------------------------------------------------- refusals
def refusals(dev):
    cache, scales, mass, bt, lens = [x.to(dev) for x in filled("int8", [20, 30], 2, 64, 16, 43)]
    cache, scales, mass = cache[0], scales[0], mass[0]
    dt = torch.bfloat16
    q, kv = torch.zeros(2, 4, 64, dtype=dt, device=dev), torch.zeros(2, 2, 2, 64, dtype=dt, device=dev)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    keep = torch.tensor([5, 5], dtype=torch.int32, device=dev)
    bad = (ValueError, RuntimeError)

    def no(f, *a, **k):
        with pytest.raises(bad):
            f(*a, **k)

    dec, wr, ev = ops.paged_decode_attention, ops.kv_quant_blocks, ops.kv_evict
    no(dec, q, cache.float(), bt, lens, 1.0, kv_scales=scales)                      # not 8 bits
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales[:-1].contiguous())            # fewer blocks
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales.double())
    no(dec, q[..., :32].contiguous(), cache, bt, lens, 1.0, kv_scales=scales)       # another head size
    no(dec, q[:, :3].contiguous(), cache, bt, lens, 1.0, kv_scales=scales)          # heads not a multiple
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales, mass=mass[:, :1].contiguous())
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales, mass=mass.half())
    no(dec, q, torch.zeros(8, 2, 2, 16, 64, dtype=dt, device=dev), bt, lens, 1.0, mass=mass)   # weights of a bf16 cache
    no(dec, q, cache[:, :, :, :8].contiguous(), bt, lens, 1.0, kv_scales=scales)    # blocks of 8 tokens
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales, window=-1)
    no(dec, q, cache, bt, lens, 1.0, kv_scales=scales, softcap=-1.0)
    no(wr, kv[..., :32].contiguous(), slots, cache, scales)
    no(wr, kv, slots[:1], cache, scales)
    no(wr, kv, slots, cache.float(), scales)
    no(wr, kv, slots, cache, scales, mass=mass[:-1].contiguous())
    no(ev, cache, scales, mass, bt, lens, keep, -1, 3)
    no(ev, cache, scales, mass, bt, lens, keep, 1, -3)
    no(ev, cache, scales, mass, bt, lens, keep, 1, 3, max_keep=-1)
    no(ev, cache, scales, mass.double(), bt, lens, keep, 1, 3)
    no(ev, cache, scales[None], mass, bt, lens, keep, 1, 3)
    return cache, scales, mass, bt, lens, q, kv, slots, keep, no


def test_refusals_cpu():
    refusals("cpu")
    cache, scales, mass, bt, lens = filled("int8", [40], 2, 64, 16, 43)
    with pytest.raises(ValueError):      # rows of one block that are not neighbours
        ops.kv_quant_blocks(torch.zeros(3, 2, 2, 64), torch.tensor([16, 32, 17], dtype=torch.int32), cache[0], scales[0])


@pytest.mark.gpu
def test_refusals_gpu():
    cache, scales, mass, bt, lens, q, kv, slots, keep, no = refusals("cuda")
    dec = ops.paged_decode_attention
    no(dec, q.float(), cache, bt, lens, 1.0, kv_scales=scales)
    no(dec, q, cache, bt.long(), lens, 1.0, kv_scales=scales)
    no(dec, q, cache, bt, lens.cpu(), 1.0, kv_scales=scales)
    no(dec, q, cache, bt[:1], lens, 1.0, kv_scales=scales)
    no(dec, q, cache, bt, lens, 1.0, num_splits=65, kv_scales=scales)
    no(dec, q, cache, bt, lens, 1.0, num_splits=4, kv_scales=scales, workspace=torch.empty(8, device="cuda"))
    no(dec, q, cache.transpose(0, 2), bt, lens, 1.0, kv_scales=scales)
    no(ops.kv_quant_blocks, kv.float(), slots, cache, scales)
    no(ops.kv_quant_blocks, kv, slots.long(), cache, scales)
    no(ops.kv_evict, cache, scales, mass, bt, lens, keep.long(), 1, 3)
    no(ops.kv_evict, cache, scales, mass, bt, lens.cpu(), keep, 1, 3)
    z = torch.zeros(4, 2, 2, 16, 48, dtype=torch.int8, device="cuda")
    no(dec, torch.zeros(2, 4, 48, dtype=torch.bfloat16, device="cuda"), z, bt * 0, lens, 1.0, kv_scales=scales[:4].contiguous())


@pytest.mark.gpu
def test_bad_indices_are_reported_gpu():
    """With bounds checking on, block ids and slots outside the pool are reported and nothing else is written."""
    cache, scales, mass, bt, lens = [x.cuda() for x in filled("int8", [40, 33], 2, 64, 16, 47)]
    cache, scales, mass = cache[0], scales[0].nan_to_num(0.5), mass[0]
    NB = cache.shape[0]
    before = cache.clone()
    with ops.BoundsCheck() as bc:
        kv = torch.randn(2, 2, 2, 64, device="cuda").bfloat16()
        ops.kv_quant_blocks(kv, torch.tensor([NB * 16, -1], dtype=torch.int32, device="cuda"), cache, scales)
        torch.cuda.synchronize()
        assert bc.status() == (4, NB) and torch.equal(cache, before)
        bc.reset()
        bad = bt.clone()
        bad[0, 1] = NB + 7
        out = ops.paged_decode_attention(torch.randn(2, 4, 64, device="cuda").bfloat16(), cache, bad, lens, 0.1,
                                         num_splits=0, kv_scales=scales)
        assert bc.status() == (4, NB + 7) and bool(torch.isfinite(out).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_bad_indices_write_to_no_other_block_gpu(kind):
    """With bounds checking on, a block id beyond the pool is reported, and neither weights nor an eviction's tokens go to
    block 0 in its place, which may be somebody's."""
    cache, scales, mass, bt, lens = [x.cuda() for x in filled(kind, [100, 90], 2, 64, 16, 53)]
    cache, scales, mass = cache[0].clamp(max=126), scales[0].nan_to_num(0.5), mass[0]
    NB, mine = cache.shape[0], bt[1, :6].long()
    bad = bt.clone()
    bad[0, 1] = NB + 7
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    keep = torch.tensor([50, 50], dtype=torch.int32).cuda()
    good = [x.clone() for x in (cache, scales, mass)]
    ops.paged_decode_attention(q, good[0], bt, lens, 0.1, 0, kv_scales=good[1], mass=good[2])
    ops.kv_evict(*good, bt, lens, keep, 4, 8)
    with ops.BoundsCheck() as bc:
        got = [x.clone() for x in (cache, scales, mass)]
        ops.paged_decode_attention(q, got[0], bad, lens, 0.1, 0, kv_scales=got[1], mass=got[2])
        assert bc.status() == (4, NB + 7) and torch.equal(got[2][0], mass[0])
        bc.reset()
        ops.kv_evict(*got, bad, lens, keep, 4, 8)
        assert bc.status() == (4, NB + 7)
    for x, y, z in zip(got, (cache, scales, mass), good):
        assert torch.equal(x[0], y[0]) and torch.equal(x[mine], z[mine])
