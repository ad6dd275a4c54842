"""Measured cases of the operators over a paged KV cache that is held in 8 or 4 bits.

Three operators of `infinicore_b200`:
  quant_paged_caching     quantises new K/V rows as it writes them to their slots
  quant_paged_cache_read  gathers rows by slot and turns them back into values
  quant_paged_attention   decode attention, one query token per sequence, over the quantised pools

Storage.  8 bits: int8 codes [blocks, kv_heads, block_size, head], one scale for a token's whole row of a head.
4 bits: two codes a byte (uint8 [blocks, kv_heads, block_size, head / 2], the even element in the low half, two's
complement), one scale for each 32 elements.  Scales are bfloat16 [blocks, kv_heads, block_size, groups].  With
Q = 127 or 7 and A the largest magnitude of a group,
  s = bfloat16(A / Q)  (0 where that is below 2^-126),   code = x / s to the nearest, halves away from zero,
and a code stands for the value code * s.

`run` returns what is held in few bits as the values it stands for: a pass that appends rows reads the same rows
back, which is what a prefill in chunks does with them next.
"""
import math
import random

import torch

own = False

GROUP = 32  # elements that share a scale in the 4-bit form
TINY = 2.0 ** -126


# ---- cases ------------------------------------------------------------------------------------------------

def _case(name, kind, bits, dtype, heads, kv_heads, head, block, seqs, lo, hi, empty=0, shape_seed=0):
    """`seqs` sequences of lengths spread over lo..hi (over their logarithm), the last `empty` of them empty; for
    "append" and "read" the same numbers give the chunks of tokens that are written or gathered."""
    c = dict(kind=kind, bits=bits, dtype=dtype, heads=heads, kv_heads=kv_heads, head=head, block=block, seqs=seqs, lo=lo, hi=hi,
             empty=empty, shape_seed=shape_seed)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few short chats of a small model: the time of one call
        _case("attend8 small", "attend", 8, "fp16", 8, 2, 64, 16, 4, 1, 256, shape_seed=1),
        # a full decode batch of the 32/8-head, head-128 shape, both widths
        _case("attend8 batch", "attend", 8, "bf16", 32, 8, 128, 16, 64, 4096, 4096),
        _case("attend4 batch", "attend", 4, "bf16", 32, 8, 128, 16, 64, 4096, 4096),
        # a ragged batch of the 64/8-head shape, padded with empty slots as a captured step is
        _case("attend4 ragged", "attend", 4, "bf16", 64, 8, 128, 16, 40, 1, 16384, empty=3, shape_seed=2),
        # two long documents: few rows, a long axis
        _case("attend4 long", "attend", 4, "fp16", 32, 8, 128, 16, 2, 131072, 131072),
        # wide heads, one kv head for 16 query heads, pages of 32, odd lengths
        _case("attend8 wide", "attend", 8, "bf16", 16, 1, 256, 32, 13, 1, 30001, shape_seed=3),
        # one decode step's new rows
        _case("append8 step", "append", 8, "bf16", 32, 8, 128, 16, 64, 1, 1),
        # a prefill's rows: 8 prompts of 2048 tokens, each width
        _case("append4 prompts", "append", 4, "bf16", 32, 8, 128, 16, 8, 2048, 2048),
        # odd prompts of a small model, some rows padding
        _case("append8 odd", "append", 8, "fp16", 8, 2, 64, 16, 7, 31, 3001, empty=5, shape_seed=4),
        # the history of a prefix, gathered for a prefill that goes on from it
        _case("read4 history", "read", 4, "bf16", 32, 8, 128, 16, 16, 4096, 4096),
        _case("read8 small", "read", 8, "fp16", 8, 2, 64, 16, 3, 100, 777, shape_seed=5),
        # one layer's decode step: append the newest row, attend over all
        _case("step4 batch", "step", 4, "bf16", 32, 8, 128, 16, 64, 200, 2000, empty=2, shape_seed=6),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "read", "step"])
    bits = rng.choice([4, 8])
    dtype = rng.choice(["bf16", "fp16"])
    head = rng.choice([64, 64, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 16])
    block = rng.choice([8, 16, 16, 32, 64, 128])
    if kind in ("append", "read"):
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 67_000_000 // (seqs * kv_heads * head)))
        hi = min(hi, 8192)
        lo = _log(rng, 1, hi)
        empty = rng.choice([0, 0, rng.randint(1, 9)])
    else:
        seqs = _log(rng, 1, 200)
        hi = _log(rng, 1, max(1, 260_000_000 // (seqs * kv_heads * head)))
        hi = min(hi, 131072)
        lo = _log(rng, 1, hi)
        empty = rng.choice([0, 0, rng.randint(1, 9)])
    return _case(None, kind, bits, dtype, heads, kv_heads, head, block, seqs, lo, hi, empty, rng.randrange(1 << 20))


def _lengths(c):
    r = random.Random(c["shape_seed"])
    return [_log(r, c["lo"], c["hi"]) for _ in range(c["seqs"])] + [0] * c["empty"]


def _row_bytes(c):
    """Bytes of one token's codes and scales of one kv head, K or V."""
    return c["head"] + 2 if c["bits"] == 8 else c["head"] // 2 + c["head"] // GROUP * 2


def work(c):
    lens = _lengths(c)
    tokens, rows = sum(lens), sum(1 for n in lens if n)
    stored, plain = 2 * c["kv_heads"] * _row_bytes(c), 2 * c["kv_heads"] * c["head"] * 2
    values = tokens * c["kv_heads"] * 2 * c["head"]
    if c["kind"] == "append":  # rows in, codes out; then the codes in and the rows out
        return {"bytes": tokens * (2 * plain + 2 * stored + 16), "flops": 6 * values}
    if c["kind"] == "read":
        return {"bytes": tokens * (plain + stored + 8), "flops": values}
    pages = sum(-(-n // c["block"]) for n in lens)
    moved = tokens * stored + rows * c["heads"] * c["head"] * 2 * 2 + 8 * pages + 8 * len(lens)
    flops = tokens * c["heads"] * c["head"] * 4
    if c["kind"] == "step":
        moved += rows * (plain + stored + 8)
    return {"bytes": moved, "flops": flops}


# ---- inputs -----------------------------------------------------------------------------------------------

def _loud(kv_heads, head, gen):
    """The few channels of each kv head that stand out, as a factor."""
    return torch.where(torch.rand((kv_heads, head), generator=gen, device="cuda") < 0.03, 5.0, 1.0)


def _rows(shape, loud, dtype, gen):
    """Rows as projections give them: normal, with those channels."""
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * loud).to(dtype)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed + 1)
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
    lens, bs, kvh, hd = _lengths(c), c["block"], c["kv_heads"], c["head"]
    pages = [-(-n // bs) for n in lens]
    blocks = sum(pages) + 3
    order = torch.randperm(blocks, generator=host)
    table = torch.zeros((len(lens), max(1, max(pages))), dtype=torch.int64)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    lens_t = torch.tensor(lens, dtype=torch.int64)
    s = dict(kind=c["kind"], bits=c["bits"], dtype=dtype, hd=hd, block=bs, scale=1.0 / math.sqrt(hd), table=table.cuda(), lens=lens_t.cuda())
    # the pools, as a run of appends has left them
    width, groups = (hd, 1) if c["bits"] == 8 else (hd // 2, hd // GROUP)
    loud = {t: _loud(kvh, hd, gen) for t in "kv"}
    for t in "kv":
        codes = torch.empty((blocks, kvh, bs, width), dtype=torch.int8 if c["bits"] == 8 else torch.uint8, device="cuda")
        scales = torch.empty((blocks, kvh, bs, groups), dtype=torch.bfloat16, device="cuda")
        step = max(1, (1 << 26) // (kvh * bs * hd))
        for b in range(0, blocks, step):
            codes[b:b + step], scales[b:b + step] = _quantise(_rows((min(step, blocks - b), kvh, bs, hd), loud[t][:, None], dtype, gen), c["bits"])
        s[t + "_cache"], s[t + "_scales"] = codes, scales
    if c["kind"] in ("attend", "step"):
        s["q"] = torch.randn((len(lens), c["heads"], hd), generator=gen, device="cuda").to(dtype)
        s["out"] = torch.zeros((len(lens), c["heads"], hd), dtype=dtype, device="cuda")
    if c["kind"] == "step":
        last = (lens_t - 1).clamp(min=0)
        slots = torch.where(lens_t > 0, table.gather(1, (last // bs)[:, None])[:, 0] * bs + last % bs, torch.tensor(-1))
    elif c["kind"] != "attend":
        # every token of the chunks, in order; `empty` counts rows of padding here, spread among them
        per = [table[i, torch.arange(n) // bs] * bs + torch.arange(n) % bs for i, n in enumerate(lens) if n]
        slots = torch.cat(per + [torch.full((c["empty"],), -1, dtype=torch.int64)])
        if c["empty"]:
            slots = slots[torch.randperm(slots.numel(), generator=host)]
    if c["kind"] != "attend":
        s["slots"] = slots.cuda()
        s["keep"] = torch.nonzero(slots >= 0)[:, 0].cuda()
        if c["kind"] != "read":
            s["k"], s["v"] = (_rows((slots.numel(), kvh, hd), loud[t], dtype, gen) for t in "kv")
    return s


# ---- the plain form ---------------------------------------------------------------------------------------

def _quantise(x, bits):
    """Codes (packed where two share a byte) and scales of rows [..., head]."""
    q, group = (127, x.shape[-1]) if bits == 8 else (7, GROUP)
    y = x.float().unflatten(-1, (-1, group))
    largest = y.abs().amax(-1)
    s = (largest / q).to(torch.bfloat16).float()
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(largest), s, torch.full_like(s, math.nan))
    r = y / s[..., None]
    codes = (torch.floor(r.abs() + 0.5) * torch.sign(r)).clamp(-q, q)
    codes = torch.where(s[..., None] > 0, codes, torch.zeros_like(codes)).to(torch.int8).flatten(-2)
    if bits == 4:
        codes = ((codes[..., 0::2] & 15) | ((codes[..., 1::2] & 15) << 4)).view(torch.uint8)
    return codes, s.to(torch.bfloat16)


def _values(codes, scales, bits):
    """The 32-bit values that codes [..., width] with scales [..., groups] stand for."""
    if bits == 4:
        low, high = codes & 15, codes >> 4
        both = torch.stack((low, high), -1).flatten(-2).to(torch.float32)
        codes = torch.where(both > 7, both - 16, both)
    s = scales.float()
    return (codes.float().unflatten(-1, (s.shape[-1], -1)) * s[..., None]).flatten(-2)


def _append(s):
    rows = s["keep"]
    at = s["slots"][rows]
    block, off = at // s["block"], at % s["block"]
    for t in "kv":
        codes, scales = _quantise(s[t][rows], s["bits"])
        s[t + "_cache"].transpose(1, 2)[block, off] = codes
        s[t + "_scales"].transpose(1, 2)[block, off] = scales


def _read(s):
    at = s["slots"].clamp(min=0)
    block, off = at // s["block"], at % s["block"]
    here = (s["slots"] >= 0)[:, None, None]
    got = []
    for t in "kv":
        v = _values(s[t + "_cache"].transpose(1, 2)[block, off], s[t + "_scales"].transpose(1, 2)[block, off], s["bits"])
        got.append(torch.where(here, v, torch.zeros_like(v)).to(s["dtype"]))
    return got


def _attend(s):
    q, table, lens, bs = s["q"], s["table"], s["lens"], s["block"]
    pages = table.shape[1]
    n = pages * bs

    def rows(t):  # [seqs, tokens, kv_heads, head]
        codes = s[t + "_cache"][table].transpose(2, 3).flatten(1, 2)
        return _values(codes, s[t + "_scales"][table].transpose(2, 3).flatten(1, 2), s["bits"])

    k = rows("k")
    seqs, heads, hd = q.shape
    kvh = k.shape[2]
    score = torch.einsum("bkgd,blkd->bkgl", q.float().view(seqs, kvh, heads // kvh, hd), k) * s["scale"]
    del k
    seen = (torch.arange(n, device=q.device)[None] < lens[:, None])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - top), torch.zeros_like(score))
    v = rows("v").masked_fill(~(torch.arange(n, device=q.device)[None] < lens[:, None])[:, :, None, None], 0.0)
    o = torch.einsum("bkgl,blkd->bkgd", p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(seqs, heads, hd).to(q.dtype)
    s["out"].copy_(torch.where((lens > 0)[:, None, None], o, s["out"]))  # an empty sequence leaves its row
    return s["out"]


def run(s):
    if own:
        import infinicore_b200 as ib

        pools = (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"])
        if s["kind"] in ("append", "step"):
            ib.quant_paged_caching(*pools, s["k"], s["v"], s["slots"])
        if s["kind"] in ("append", "read"):
            k, v = ib.quant_paged_cache_read(*pools, s["slots"], s["dtype"])
        else:
            o = ib.quant_paged_attention(s["q"], *pools, s["table"], s["lens"], None, s["scale"], out=s["out"])
    else:
        if s["kind"] in ("append", "step"):
            _append(s)
        if s["kind"] in ("append", "read"):
            k, v = _read(s)
        else:
            o = _attend(s)
    if s["kind"] == "read":
        return {"k": k, "v": v}
    if s["kind"] == "append":
        return {"k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if s["kind"] == "step":
        return {"out": o, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    return {"out": o}


# ---- the definition in 64 bits ----------------------------------------------------------------------------

def _decode64(codes, scales, bits):
    """One kv head's [tokens, width] codes and [tokens, groups] scales as float64 [tokens, head]."""
    if bits == 8:
        return codes.double() * scales.double()
    n = codes.to(torch.int16)
    out = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device=codes.device)
    for half, nib in ((0, n % 16), (1, n // 16)):
        out[:, half::2] = (nib - 16 * (nib // 8)).double()
    return out * scales.double().repeat_interleave(GROUP, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    bits, bs = s["bits"], s["block"]
    q_max, group = (127.0, s["hd"]) if bits == 8 else (7.0, GROUP)
    kvh = s["k_cache"].shape[1]
    flat = {t: s[t].permute(0, 2, 1, 3).reshape(-1, kvh, s[t].shape[-1]) for t in ("k_cache", "v_cache", "k_scales", "v_scales")}
    scales = {t: s[t + "_scales"].double() for t in "kv"}
    new = {}
    if s["kind"] in ("append", "step"):
        rows = torch.nonzero(s["slots"] >= 0)[:, 0]
        at = s["slots"][rows]
        for t in "kv":
            x = s[t][rows].double()
            x = x.reshape(x.shape[0], kvh, -1, group)
            step = (x.abs().max(-1).values / q_max).to(torch.bfloat16).double()
            step[step < TINY] = 0.0
            r = (x / step[..., None]).abs()
            code = torch.where(step[..., None] > 0, torch.copysign((2 * r + 1).div(2, rounding_mode="floor").clamp(max=q_max), x), torch.zeros_like(x))
            new[t] = (code * step[..., None]).reshape(rows.numel(), kvh, -1)
            scales[t][at // bs, :, at % bs] = step
    if s["kind"] in ("append", "read"):
        got = {}
        for t in "kv":
            out = torch.zeros((s["slots"].numel(), kvh, s["hd"]), dtype=torch.float64, device="cuda")
            rows = torch.nonzero(s["slots"] >= 0)[:, 0]
            if t in new:
                out[rows] = new[t]
            else:
                for h in range(kvh):
                    at = s["slots"][rows]
                    out[rows, h] = _decode64(flat[t + "_cache"][at, h], flat[t + "_scales"][at, h], bits)
            got[t] = out
        return dict(got, k_scales=scales["k"], v_scales=scales["v"]) if s["kind"] == "append" else got
    seqs, heads, hd = s["q"].shape
    out = torch.zeros((seqs, heads, hd), dtype=torch.float64, device="cuda")
    g = heads // kvh
    owner = {int(r): i for i, r in enumerate(torch.nonzero(s["slots"] >= 0)[:, 0].tolist())} if new else {}
    for i, n in enumerate(_lengths(case)):
        if not n:
            continue
        t = torch.arange(n, device="cuda")
        at = s["table"][i, t // bs] * bs + t % bs
        for h in range(kvh):
            k, v = (_decode64(flat[x + "_cache"][at, h], flat[x + "_scales"][at, h], bits) for x in "kv")
            if i in owner:
                k[n - 1], v[n - 1] = new["k"][owner[i], h], new["v"][owner[i], h]
            w = torch.softmax(k @ s["q"][i, h * g:(h + 1) * g].double().T * s["scale"], dim=0)
            out[i, h * g:(h + 1) * g] = w.T @ v
    return {"out": out, "k_scales": scales["k"], "v_scales": scales["v"]} if s["kind"] == "step" else {"out": out}
