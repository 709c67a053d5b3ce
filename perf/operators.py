"""Workloads of the block-scaled 8-bit KV cache: what is timed and compared for its operators.

The cache of one layer holds 8-bit codes ``[NB, 2, Hk, bs, D]`` (0 = K, 1 = V; int8, or uint8 with
e4m3 bit patterns) and one fp32 scale per block, K/V and head ``[NB, 2, Hk]``: value = code * scale.
The scales that are written are powers of two. Beside it may lie the attention weight that each
cached token has drawn, summed over the queries of its head group: ``mass [NB, Hk, bs]`` fp32.

    write    the step's K/V rows into their slots; a block whose largest value grows gets a larger
             scale and its older codes are rounded to it; the written tokens' weight starts at zero
    decode   attention of one query token per sequence over the cache, on request adding each
             token's softmax weight to ``mass``
    prefill  causal attention of several new tokens per sequence (they are in the cache already)
    evict    of each sequence, layer and head: keep the first and the latest tokens and those of the
             rest that drew the most weight, moved together at the front of the sequence's blocks

``run`` computes them with elementary torch operations, or, where ``own`` is set, through the
public calls of ``gollek_b200.ops``. ``exact`` restates the definitions in 64 bits.
"""
import math

import torch

own = False

FLOOR_EXP = -100                 # the smallest scale is 2^-100
QMAX = {"int8": 127.0, "e4m3": 448.0}
BF16_MAX = 3.3895313892515355e38


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's rows of 48 running sequences, in a captured batch of 64 (16 padding rows)
        dict(name="write_step_64", op="write", kind="int8", B=48, pad=16, new=1, L=1200, Hk=8, D=128, bs=16,
             mass=True),
        # a prompt step at the engine's token budget: five prompts that start anew or go on mid-block
        dict(name="write_prompt_8k", op="write", kind="e4m3", B=5, pad=0, new=1638, L=300, Hk=8, D=128, bs=16,
             mass=False),
        # a single chat turn: latency of one sequence
        dict(name="decode_one_1k", op="decode", kind="int8", B=1, L=1000, ragged=False, H=32, Hk=8, D=128, bs=16,
             window=0, softcap=0.0, mass=False),
        # the ordinary serving batch: 64 conversations of mixed length
        dict(name="decode_64x4k", op="decode", kind="e4m3", B=64, L=4096, ragged=True, H=32, Hk=8, D=128, bs=16,
             window=0, softcap=0.0, mass=False),
        # long documents on the 64-head configuration: the largest pass over the cache
        dict(name="decode_16x32k", op="decode", kind="int8", B=16, L=32768, ragged=False, H=64, Hk=8, D=128, bs=16,
             window=0, softcap=0.0, mass=False),
        # head size 256 with a sliding window and capped scores, larger blocks
        dict(name="decode_d256_window", op="decode", kind="e4m3", B=33, L=5000, ragged=True, H=16, Hk=8, D=256, bs=32,
             window=4096, softcap=50.0, mass=False),
        # decoding that also weighs the tokens for eviction: few short rows, odd head group of 7
        dict(name="weigh_3x700_g7", op="decode", kind="e4m3", B=3, L=700, ragged=True, H=28, Hk=4, D=128, bs=16,
             window=0, softcap=0.0, mass=True),
        # the ordinary serving batch, weighed
        dict(name="weigh_64x4k", op="decode", kind="int8", B=64, L=4096, ragged=True, H=32, Hk=8, D=128, bs=16,
             window=0, softcap=0.0, mass=True),
        # one prompt from its first token
        dict(name="prefill_4k", op="prefill", kind="int8", B=1, L=4096, new=4096, H=32, Hk=8, D=128, bs=16),
        # chunks of eight prompts over what earlier steps have cached, head size 64
        dict(name="prefill_chunk_8x100", op="prefill", kind="e4m3", B=8, L=6000, new=100, H=32, Hk=8, D=64, bs=16),
        # one layer's share of relieving two sequences
        dict(name="evict_2x1k", op="evict", kind="int8", layers=1, B=2, L=1000, Hk=8, D=128, bs=16, keep=0.6, sink=16,
             recent=0.2),
        # all layers' heads of four long sequences at once (an eight-layer slice of the pool)
        dict(name="evict_8x4x8k", op="evict", kind="e4m3", layers=8, B=4, L=8192, Hk=8, D=128, bs=16, keep=0.6,
             sink=16, recent=0.2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["int8", "e4m3"])
    bs = rng.choice([16, 16, 32, 64])
    op = rng.choice(["write", "decode", "decode", "decode", "prefill", "evict"])
    Hk = rng.choice([1, 2, 4, 8])
    if op == "write":
        if rng.random() < 0.5:
            return dict(op=op, kind=kind, B=_log(rng, 1, 256), pad=rng.randint(0, 8), new=1, L=_log(rng, 1, 2000), Hk=Hk,
                        D=rng.choice([64, 96, 128, 256]), bs=bs, mass=rng.random() < 0.5)
        B = rng.randint(1, 8)
        return dict(op=op, kind=kind, B=B, pad=0, new=_log(rng, 2, 8000 // B), L=_log(rng, 1, 2000), Hk=Hk,
                    D=rng.choice([64, 96, 128]), bs=bs, mass=rng.random() < 0.5)
    if op == "decode":
        B = _log(rng, 1, 128)
        D = rng.choice([64, 96, 128, 128, 256])
        G = rng.choice([1, 2, 3, 4, 7, 8, 12, 16])
        L = _log(rng, 1, min(32768, (1 << 21) // (B * Hk) * 128 // D))
        return dict(op=op, kind=kind, B=B, L=L, ragged=rng.random() < 0.6, H=Hk * G, Hk=Hk, D=D, bs=bs,
                    window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0]),
                    mass=rng.random() < 0.4)
    if op == "prefill":
        D = rng.choice([64, 128])
        G = rng.choice([1, 2, 4, 7])
        if rng.random() < 0.5:
            L = _log(rng, 2, 3000)
            return dict(op=op, kind=kind, B=1, L=L, new=L, H=Hk * G, Hk=Hk, D=D, bs=16)
        new = _log(rng, 2, 200)
        return dict(op=op, kind=kind, B=rng.randint(1, 8), L=new + _log(rng, 16, 6000), new=new, H=Hk * G, Hk=Hk, D=D,
                    bs=16)
    return dict(op="evict", kind=kind, layers=rng.randint(1, 8), B=rng.randint(1, 4), L=_log(rng, 40, 8192), Hk=Hk,
                D=rng.choice([64, 96, 128]), bs=bs, keep=rng.uniform(0.2, 0.9), sink=rng.choice([4, 16, 32]),
                recent=rng.uniform(0.05, 0.3))


# ------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Cached tokens of each sequence and new tokens of each: they go by the case, not by the seed."""
    B, L, gen = case["B"], case["L"], torch.Generator().manual_seed(case["B"] * 977 + case["L"])
    new = torch.full((B,), case.get("new", 1))
    if case["op"] == "write":
        return torch.randint(0, L, (B,), generator=gen) + new, new
    if case["op"] == "prefill" and B > 1:  # chunks of mixed length
        new = (new.double() * (0.3 + 0.7 * torch.rand(B, generator=gen))).long().clamp(min=1)
    if not case.get("ragged"):
        return torch.full((B,), L), new
    return (L * (0.1 + 0.9 * torch.rand(B, generator=gen))).long().clamp(1, L), new  # a serving batch


def _tables(lens, bs, gen, spare=5):
    """Blocks of the sequences scattered over the pool, as an allocator leaves them; padded with 0."""
    nb = (lens + bs - 1) // bs
    mb, total = int(nb.max()), int(nb.sum())
    ids = torch.randperm(total + spare, generator=gen)[:total]
    rows = torch.arange(len(lens)).repeat_interleave(nb)
    cols = torch.arange(total) - (nb.cumsum(0) - nb).repeat_interleave(nb)
    bt = torch.zeros(len(lens), mb, dtype=torch.int32)
    bt[rows, cols] = ids.int()
    return bt, total + spare


def _pool(case, layers, NB, dev, gen):
    """Codes and scales of a filled pool: K with a few strong channels, V with a spread of row sizes."""
    Hk, bs, D, kind = case["Hk"], case["bs"], case["D"], case["kind"]
    strong = 1.0 + 3.0 * (torch.rand(2, Hk, 1, D, device=dev, generator=gen) < 0.05)
    codes = torch.empty(layers, NB, 2, Hk, bs, D, dtype=torch.int8 if kind == "int8" else torch.uint8, device=dev)
    scales = torch.empty(layers, NB, 2, Hk, device=dev)
    step = max(1, (1 << 27) // (2 * Hk * bs * D))
    for l in range(layers):
        for n in range(0, NB, step):
            x = torch.randn(min(step, NB - n), 2, Hk, bs, D, device=dev, generator=gen) * strong
            x = x * (0.5 + torch.rand(x.shape[0], 2, Hk, bs, 1, device=dev, generator=gen))
            s = _pow2_scale(x.abs().amax((-1, -2)), kind)
            codes[l, n:n + step] = _encode(x / s[..., None, None], kind)
            scales[l, n:n + step] = s
    return codes, scales


def prepare(case, seed):
    dev = "cuda"
    hg = torch.Generator().manual_seed(seed * 1000003 + 17)
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 3)
    Hk, D, bs, op = case["Hk"], case["D"], case["bs"], case["op"]
    st = dict(case=case, op=op, kind=case["kind"])
    lens, new = _lengths(case)
    if op == "write":
        bt, NB = _tables(lens, bs, hg)
        pos = ((lens - new)[:, None] + torch.arange(case["new"])).reshape(-1)
        row = torch.arange(case["B"]).repeat_interleave(case["new"])
        slots = bt[row, pos // bs].long() * bs + pos % bs
        slots = torch.cat([slots, torch.full((case["pad"],), -1)])
        st["slots"] = slots.int().to(dev)
        grow = torch.exp2(2.0 * torch.rand(slots.numel(), 2, Hk, 1, device=dev, generator=gen))
        st["kv"] = (torch.randn(slots.numel(), 2, Hk, D, device=dev, generator=gen) * grow).bfloat16()
        codes, scales = _pool(case, 1, NB, dev, gen)
        st["cache"], st["scales"] = codes[0], scales[0]
        st["mass"] = torch.rand(NB, Hk, bs, device=dev, generator=gen) if case["mass"] else None
        return st
    bt, NB = _tables(lens, bs, hg)
    layers = case.get("layers", 1)
    codes, scales = _pool(case, layers, NB, dev, gen)
    st["tables"], st["lens"] = bt.to(dev), lens.int().to(dev)
    if op == "evict":
        st["cache"], st["scales"] = codes, scales
        # weights drawn over many steps: a few tokens draw most of it, the newest have drawn none
        u = torch.rand(layers, NB, Hk, bs, device=dev, generator=gen)
        st["mass"] = torch.where(u < 0.02, torch.zeros_like(u), u.pow(-1.5) * 0.01)
        keep = (lens.double() * case["keep"]).long().clamp(min=1)
        st["keep"] = keep.int().to(dev)
        st["max_keep"] = int(keep.max())
        st["recent"] = max(1, int(case["recent"] * case["L"] * case["keep"]))
        st["sink"] = case["sink"]
        return st
    st["cache"], st["scales"] = codes[0], scales[0]
    st["scale"] = 1.0 / math.sqrt(D)
    if op == "decode":
        st["q"] = (torch.randn(case["B"], case["H"], D, device=dev, generator=gen) * 0.7).bfloat16()
        st["mass"] = torch.rand(NB, Hk, bs, device=dev, generator=gen) if case["mass"] else None
        return st
    qs = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
    T = int(qs[-1])
    st["q"] = (torch.randn(T, case["H"], D, device=dev, generator=gen) * 0.7).bfloat16()
    st["query_start"] = qs.int().to(dev)
    st["row_seq"] = torch.arange(case["B"]).repeat_interleave(new).to(dev)    # sequence of each query row
    st["row_pos"] = (torch.arange(T) - qs[:-1].repeat_interleave(new)).to(dev)  # its place in the chunk
    st["max_new"] = int(new.max())
    if own:  # the work list a program makes once for a step and hands to every layer
        from gollek_b200 import ops
        st["tiles"] = ops.prefill_schedule(qs.tolist(), lens.tolist(), case["H"], Hk, D).to(dev)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _pow2_scale(amax, kind):
    """The smallest power of two s with amax <= qmax * s, at least 2^-100."""
    m, e = torch.frexp(amax.float())
    bits, top = (7, 127.0 / 128.0) if kind == "int8" else (9, 0.875)
    e = (e - bits + (m > top).int()).clamp(min=FLOOR_EXP)
    e = torch.where(amax > 0, e, torch.full_like(e, FLOOR_EXP))
    return ((e + 127) << 23).view(torch.float32)


def _encode(y, kind):
    """8-bit codes of y = value / scale, to nearest, ties to even."""
    if kind == "int8":
        return y.round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes):
    return codes.float() if codes.dtype == torch.int8 else codes.view(torch.float8_e4m3fn).float()


def _shown(codes):
    """The codes as the numbers they stand for, in units of their scale (no copy)."""
    return codes if codes.dtype == torch.int8 else codes.view(torch.float8_e4m3fn)


def _plain_write(st):
    kv, slots, cache, scales, kind = st["kv"], st["slots"].long(), st["cache"], st["scales"], st["kind"]
    NB, bs = cache.shape[0], cache.shape[3]
    ok = slots >= 0
    x = kv[ok].float().nan_to_num(0.0, BF16_MAX, -BF16_MAX)
    blk, off = slots[ok] // bs, slots[ok] % bs
    amax = torch.zeros(NB, 2, cache.shape[2], device=kv.device)
    amax.scatter_reduce_(0, blk[:, None, None].expand(-1, 2, cache.shape[2]), x.abs().amax(-1), "amax")
    touched = torch.zeros(NB, dtype=torch.bool, device=kv.device).index_fill_(0, blk, True)
    fresh = torch.zeros(NB, dtype=torch.bool, device=kv.device).index_fill_(0, blk[off == 0], True)
    need = _pow2_scale(amax, kind)
    new = torch.where(fresh[:, None, None], need, torch.maximum(scales, need))
    new = torch.where(touched[:, None, None], new, scales)
    grown = (new > scales) & touched[:, None, None] & ~fresh[:, None, None]
    again = _encode(_decode(cache) * (scales / new)[..., None, None], kind)
    cache.copy_(torch.where(grown[..., None, None], again, cache))
    scales.copy_(new)
    cache[blk, :, :, off] = _encode(x / new[blk][..., None], kind)
    if st["mass"] is not None:
        st["mass"][blk, :, off] = 0.0


def _values(st, which, mb, valid):
    """K or V of every sequence, [B, Hk, mb * bs, D] fp32, zero where no token is."""
    bt = st["tables"].long()
    cache, scales = st["cache"], st["scales"]
    x = _decode(cache[bt, which]) * scales[bt, which][..., None, None]
    x = x.permute(0, 2, 1, 3, 4).reshape(bt.shape[0], cache.shape[2], mb * cache.shape[3], cache.shape[4])
    return torch.where(valid[:, None, :, None], x, torch.zeros((), device=x.device))


def _plain_decode(st):
    case, q, cache = st["case"], st["q"], st["cache"]
    B, H, D = q.shape
    Hk, bs = cache.shape[2], cache.shape[3]
    mb = st["tables"].shape[1]
    pos = torch.arange(mb * bs, device=q.device)
    lens = st["lens"][:, None]
    valid = pos[None] < lens
    if case["window"]:
        valid &= pos[None] >= lens - case["window"]
    k = _values(st, 0, mb, valid)
    s = torch.matmul(q.float().view(B, Hk, H // Hk, D), k.transpose(2, 3)) * st["scale"]
    del k
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    p = torch.softmax(s.masked_fill(~valid[:, None, None], -math.inf), -1)
    out = torch.matmul(p, _values(st, 1, mb, valid)).reshape(B, H, D).to(q.dtype)
    if st["mass"] is not None:
        w = p.sum(2).view(B, Hk, mb, bs).permute(0, 2, 1, 3).reshape(B * mb, Hk, bs)
        st["mass"].index_add_(0, st["tables"].long().view(-1), w)
    return out


def _plain_prefill(st):
    q, cache = st["q"], st["cache"]
    T, H, D = q.shape
    B, mb = st["tables"].shape
    Hk, bs, Tq = cache.shape[2], cache.shape[3], st["max_new"]
    pos = torch.arange(mb * bs, device=q.device)
    valid = pos[None] < st["lens"][:, None]
    grid = torch.zeros(B, Tq, H, D, device=q.device)
    grid[st["row_seq"], st["row_pos"]] = q.float()
    new = (st["query_start"][1:] - st["query_start"][:-1])[:, None]
    last = (st["lens"][:, None] - new) + torch.arange(Tq, device=q.device)[None]      # each row's position
    seen = valid[:, None] & (pos[None, None] <= last[:, :, None])
    x = grid.view(B, Tq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * Tq, D)
    s = torch.matmul(x, _values(st, 0, mb, valid).transpose(2, 3)) * st["scale"]
    s = s.view(B, Hk, H // Hk, Tq, mb * bs).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.softmax(s, -1).view(B, Hk, H // Hk * Tq, mb * bs)
    o = torch.matmul(p, _values(st, 1, mb, valid)).view(B, Hk, H // Hk, Tq, D).permute(0, 3, 1, 2, 4)
    return o.reshape(B, Tq, H, D)[st["row_seq"], st["row_pos"]].to(q.dtype)


def _plain_evict(st):
    cache, scales, mass, kind = st["cache"], st["scales"], st["mass"], st["kind"]
    Ly, NB, _, Hk, bs, D = cache.shape
    B, mb = st["tables"].shape
    bt, lens = st["tables"].long(), st["lens"].long()
    keep = torch.minimum(st["keep"].long(), lens)
    cut = keep < lens                                                        # the others stay as they are
    n = torch.where(cut, keep.clamp(max=st["max_keep"]), lens)
    sink = torch.clamp(n, max=st["sink"])
    recent = torch.clamp(n - sink, max=st["recent"])
    pos = torch.arange(mb * bs, device=cache.device)
    key = mass[:, bt].permute(0, 1, 3, 2, 4).reshape(Ly, B, Hk, mb * bs).nan_to_num(0.0)
    here = pos[None] < lens[:, None]
    always = here & ((pos[None] < sink[:, None]) | (pos[None] >= (lens - recent)[:, None]))
    key = key.masked_fill(always[None, :, None], math.inf).masked_fill(~here[None, :, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, pos.expand_as(order))
    chosen = (rank < n[None, :, None, None]) & here[None, :, None]
    src = torch.sort(torch.where(chosen, pos, mb * bs), -1).values[..., :st["max_keep"]]
    kept = torch.where(src < mb * bs, src, torch.full_like(src, -1)).int()
    # the kept tokens' values, at the places they move to (whole blocks)
    mk = (st["max_keep"] + bs - 1) // bs * bs
    src = torch.nn.functional.pad(src, (0, mk - st["max_keep"]), value=mb * bs)
    live = (src < mb * bs) & cut[None, :, None, None]
    src = src.clamp(max=mb * bs - 1)
    li = torch.arange(Ly, device=cache.device)[:, None, None, None]
    hi = torch.arange(Hk, device=cache.device)[None, None, :, None]
    bi = torch.arange(B, device=cache.device)[None, :, None, None]
    sb = bt[bi, src // bs]                                                     # [Ly, B, Hk, mk]
    x = _decode(cache[li, sb, :, hi, src % bs]) * scales[li, sb, :, hi][..., None]  # [Ly, B, Hk, mk, 2, D]
    x = torch.where(live[..., None, None], x, torch.zeros((), device=x.device))
    s = _pow2_scale(x.abs().amax(-1).view(Ly, B, Hk, mk // bs, bs, 2).amax(4), kind)
    codes = _encode(x / s.repeat_interleave(bs, 3)[..., None], kind)
    weight = mass[li, sb, hi, src % bs]
    to = torch.arange(mk, device=cache.device)
    lx, bx, hx, tx = live.nonzero(as_tuple=True)
    db = bt[bx, tx // bs]
    cache[lx, db, :, hx, tx % bs] = codes[lx, bx, hx, tx]
    mass[lx, db, hx, tx % bs] = weight[lx, bx, hx, tx]
    scales[lx, db, :, hx] = s[lx, bx, hx, tx // bs]
    return kept


def run(state):
    st, op = state, state["op"]
    if own:
        from gollek_b200 import ops
    if op == "write":
        if own:
            ops.kv_quant_blocks(st["kv"], st["slots"], st["cache"], st["scales"], mass=st["mass"])
        else:
            _plain_write(st)
        return {"codes": _shown(st["cache"]), "scales": st["scales"], "mass": st["mass"]}
    if op == "decode":
        if own:
            out = ops.paged_decode_attention(st["q"], st["cache"], st["tables"], st["lens"], st["scale"], num_splits=0,
                                             window=st["case"]["window"], softcap=st["case"]["softcap"],
                                             kv_scales=st["scales"], mass=st["mass"])
        else:
            out = _plain_decode(st)
        return {"out": out, "mass": st["mass"]}
    if op == "prefill":
        if own:
            return ops.paged_prefill_attention(st["q"], st["cache"], st["tables"], st["lens"], st["query_start"],
                                               st["scale"], tiles=st["tiles"], kv_scales=st["scales"])
        return _plain_prefill(st)
    if own:
        kept = ops.kv_evict(st["cache"], st["scales"], st["mass"], st["tables"], st["lens"], st["keep"], st["sink"],
                            st["recent"], max_keep=st["max_keep"])
    else:
        kept = _plain_evict(st)
    return {"kept": kept, "codes": _shown(st["cache"]), "scales": st["scales"], "mass": st["mass"]}


def work(case):
    """Bytes that have to cross memory (each input once, each output once) and the products' operations."""
    Hk, D, op, bs = case["Hk"], case["D"], case["op"], case["bs"]
    lens, new = _lengths(case)
    if op == "write":
        T = int(new.sum())
        return {"bytes": T * 2 * Hk * D * 3 + 4 * T * (1 + Hk * bool(case["mass"])), "flops": 0}
    if op == "decode":
        n = int((lens.clamp(max=case["window"]) if case["window"] else lens).sum())
        tok = 2 * D + 8 / bs + (8 if case["mass"] else 0)
        return {"bytes": Hk * n * tok + 4 * case["B"] * case["H"] * D, "flops": 4 * case["H"] * n * D}
    if op == "prefill":
        seen = int((new * (lens - new) + new * (new + 1) // 2).sum())
        return {"bytes": Hk * int(lens.sum()) * (2 * D + 8 / bs) + 4 * int(new.sum()) * case["H"] * D,
                "flops": 4 * case["H"] * seen * D}
    n, kept = int(lens.sum()), int((lens.double() * case["keep"]).long().clamp(min=1).sum())
    return {"bytes": case["layers"] * Hk * (4 * n + 8 * kept + 4 * D * kept), "flops": 0}


# ------------------------------------------------------------------------------------ in 64 bits
def _number(codes):
    """The codes' numbers in 64 bits, from their bits."""
    if codes.dtype == torch.int8:
        return codes.double()
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * torch.exp2((e - 7).double()))
    v = torch.where((c & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(c >= 128, -v, v)


def _least_scale(top, kind):
    """2^k, the least power of two that is no less than top / qmax and 2^-100 (top: a Python float)."""
    y = max(top / QMAX[kind], 2.0 ** FLOOR_EXP)
    m, e = math.frexp(y)
    return 2.0 ** (e - 1 if m == 0.5 else e)


def _nearest(y, kind):
    """y (64 bits) rounded to the type's numbers, ties to even."""
    if kind == "int8":
        return torch.round(y).clamp(-127, 127)
    e = torch.frexp(y).exponent.clamp(min=-5).double() - 1.0                     # |y| in [2^e, 2^(e+1)), e >= -6
    step = torch.exp2(e - 3.0)
    return (torch.round(y / step) * step).clamp(-448, 448)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    kind, bs, Hk, D, op = case["kind"], case["bs"], case["Hk"], case["D"], case["op"]
    e4m3 = kind == "e4m3"
    if op == "write":
        num, sc = _number(st["cache"]), st["scales"].double()
        mass = None if st["mass"] is None else st["mass"].double()
        slots = [s for s in st["slots"].tolist()]
        of = {}
        for t, s in enumerate(slots):
            if s >= 0:
                of.setdefault(s // bs, []).append((t, s % bs))
        tops = st["kv"].double().abs().amax(-1).cpu()
        old = sc.cpu()
        for b, rows in of.items():
            ts, offs = [t for t, _ in rows], [o for _, o in rows]
            top = tops[ts].amax(0)
            need = torch.tensor([[_least_scale(float(top[w, h]), kind) for h in range(Hk)] for w in range(2)],
                                dtype=torch.float64)
            s = need if 0 in offs else torch.maximum(need, old[b])
            if 0 not in offs and bool((s > old[b]).any()):
                wide = (s > old[b]).to(num.device)[..., None, None]
                num[b] = torch.where(wide, _nearest(num[b] * (old[b] / s).to(num.device)[..., None, None], kind), num[b])
            s = s.to(num.device)
            sc[b] = s
            num[b][:, :, offs] = _nearest(st["kv"][ts].double() / s[None, ..., None], kind).permute(1, 2, 0, 3)
            if mass is not None:
                mass[b][:, offs] = 0.0
        return {"codes": num if e4m3 else None, "scales": sc, "mass": mass}
    if op == "evict":
        tables, lens, keeps = st["tables"].cpu(), st["lens"].tolist(), st["keep"].tolist()
        num, sc, mass = _number(st["cache"]), st["scales"].double(), st["mass"].double()
        num0, sc0, mass0 = num.clone(), sc.clone(), mass.clone()
        for b in range(case["B"]):
            L, K = lens[b], min(keeps[b], lens[b])
            if K == L:
                continue
            ids = tables[b, torch.arange(L) // bs].long().to(num.device)
            off = torch.arange(L, device=num.device) % bs
            a = min(st["sink"], K)
            r = min(st["recent"], K - a)
            for l in range(case["layers"]):
                for h in range(Hk):
                    w = mass0[l, ids, h, off]
                    mid = torch.sort(w[a:L - r], dim=0, descending=True, stable=True).indices[:K - a - r] + a
                    take = torch.cat([torch.arange(a, device=mid.device), mid.sort().values,
                                      torch.arange(L - r, L, device=mid.device)])
                    v = num0[l, ids[take], :, h, off[take]] * sc0[l, ids[take], :, h][..., None]    # [K, 2, D]
                    top = torch.zeros((K + bs - 1) // bs * bs, 2, dtype=torch.float64, device=v.device)
                    top[:K] = v.abs().amax(-1)
                    y = (top.view(-1, bs, 2).amax(1) / QMAX[kind]).clamp(min=2.0 ** FLOOR_EXP)
                    f = torch.frexp(y)
                    s = torch.exp2((f.exponent - (f.mantissa == 0.5).int()).double())
                    num[l, ids[:K], :, h, off[:K]] = _nearest(v / s.repeat_interleave(bs, 0)[:K, :, None], kind)
                    mass[l, ids[:K], h, off[:K]] = w[take]
                    sc[l, ids[:K], :, h] = s.repeat_interleave(bs, 0)[:K]
        return {"kept": None, "codes": num if e4m3 else None, "scales": sc, "mass": mass}
    q, H = st["q"].double(), case["H"]
    G = H // Hk
    out = torch.zeros_like(q)
    mass = None if st.get("mass") is None else st["mass"].double()
    lens, tables = st["lens"].tolist(), st["tables"].long()
    start = st["query_start"].tolist() if op == "prefill" else list(range(len(lens) + 1))
    for b, L in enumerate(lens):
        ids = tables[b, :(L + bs - 1) // bs]
        n = start[b + 1] - start[b]
        at = torch.arange(L, device=q.device)
        row = torch.arange(L - n, L, device=q.device)[:, None]
        seen = at[None] <= row
        if case.get("window"):
            seen &= at[None] > row - case["window"]
        for h in range(Hk):
            k = (_number(st["cache"][ids, 0, h]) * st["scales"][ids, 0, h].double()[:, None, None]).view(-1, D)[:L]
            v = (_number(st["cache"][ids, 1, h]) * st["scales"][ids, 1, h].double()[:, None, None]).view(-1, D)[:L]
            for g in range(h * G, (h + 1) * G):
                s = q[start[b]:start[b + 1], g] @ k.T * st["scale"]
                if case.get("softcap"):
                    s = torch.tanh(s / case["softcap"]) * case["softcap"]
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                p = torch.exp(s - s.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                out[start[b]:start[b + 1], g] = p @ v
                if mass is not None:
                    mass[ids[at // bs], h, at % bs] += p[0]
    return out if op == "prefill" else {"out": out, "mass": mass}
