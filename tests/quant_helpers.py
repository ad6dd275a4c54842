"""Plain 64-bit forms of the operators over quantised pools, and the pools the tests run on."""
import torch

GROUP = 32
TINY = 2.0 ** -126


def limits(bits):
    return 127 if bits == 8 else 7


def groups(bits, head):
    return 1 if bits == 8 else head // GROUP


def empty_pools(blocks, kv_heads, block, k_head, v_head, bits, device="cpu", fill=0):
    """k_cache, v_cache, k_scales, v_scales; `fill` is the byte everything starts with."""
    out = []
    for head in (k_head, v_head):
        width = head if bits == 8 else head // 2
        out.append(torch.full((blocks, kv_heads, block, width), fill, dtype=torch.int8 if bits == 8 else torch.uint8, device=device))
    for head in (k_head, v_head):
        raw = torch.full((blocks, kv_heads, block, groups(bits, head), 2), fill, dtype=torch.uint8, device=device)
        out.append(raw.view(torch.bfloat16)[..., 0])
    return out


def quantise(x, bits):
    """int8 codes [..., head] and bfloat16 scales [..., groups] of rows [..., head], by the definition."""
    q = limits(bits)
    g = x.shape[-1] if bits == 8 else GROUP
    y = x.double().unflatten(-1, (-1, g))
    a = y.abs().amax(-1)
    s = (a / q).float().to(torch.bfloat16).double()
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(a), s, torch.full_like(s, float("nan")))
    live = (s > 0)[..., None]
    r = torch.where(live, y, torch.zeros_like(y)) / torch.where(live, s[..., None], torch.ones_like(s[..., None]))
    # r < 2^8 is at least 2^-16 of itself away from a half, or on it: the 53 bits of the quotient and the sum keep the side
    codes = torch.copysign(torch.floor(r.abs() + 0.5), r)
    return codes.to(torch.int8).flatten(-2), s.to(torch.bfloat16)


def pack(codes, bits):
    if bits == 8:
        return codes
    u = codes.to(torch.int16) & 15
    return (u[..., 0::2] | (u[..., 1::2] << 4)).to(torch.uint8)


def unpack(stored, bits):
    if bits == 8:
        return stored
    u = stored.to(torch.int16)
    both = torch.stack((u & 15, u >> 4), -1).flatten(-2)
    return torch.where(both > 7, both - 16, both).to(torch.int8)


def values(stored, scales, bits):
    """float64 values of stored codes [..., width] with scales [..., groups]."""
    s = scales.double()
    return (unpack(stored, bits).double().unflatten(-1, (s.shape[-1], -1)) * s[..., None]).flatten(-2)


def write(pools, k, v, slots, bits):
    """The pools after quant_paged_caching, in place."""
    bs = pools[0].shape[2]
    for codes, scales, rows in ((pools[0], pools[2], k), (pools[1], pools[3], v)):
        c, s = quantise(rows, bits)
        c = pack(c, bits)
        for i, slot in enumerate(slots.tolist()):
            if slot >= 0:
                codes[slot // bs, :, slot % bs] = c[i]
                scales[slot // bs, :, slot % bs] = s[i]


def read(pools, slots, bits):
    bs = pools[0].shape[2]
    out = []
    for codes, scales in ((pools[0], pools[2]), (pools[1], pools[3])):
        at = slots.clamp(min=0)
        rows = values(codes[at // bs, :, at % bs], scales[at // bs, :, at % bs], bits)
        out.append(torch.where((slots >= 0)[:, None, None], rows, torch.zeros_like(rows)))
    return out


def attend(q, pools, tables, lens, scale, bits, alibi=None, out=None):
    """float64 decode attention; rows of empty sequences keep `out`."""
    k_cache, v_cache, k_scales, v_scales = pools
    bs, kvh = k_cache.shape[2], k_cache.shape[1]
    seqs, heads, hd = q.shape
    g = heads // kvh
    res = torch.zeros((seqs, heads, hd), dtype=torch.float64, device=q.device) if out is None else out.double()
    for i in range(seqs):
        n = min(int(lens[i]), tables.shape[1] * bs)
        if n <= 0:
            continue
        t = torch.arange(n, device=q.device)
        block, off = tables[i].long()[t // bs], t % bs
        k = values(k_cache[block, :, off], k_scales[block, :, off], bits)  # [n, kvh, hd]
        v = values(v_cache[block, :, off], v_scales[block, :, off], bits)
        s = torch.einsum("hgd,nhd->hgn", q[i].double().view(kvh, g, hd), k) * scale
        if alibi is not None:
            s = s + alibi.double().view(kvh, g, 1) * (t.double() - (n - 1))
        res[i] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(heads, hd)
    return res


def attend_bound(q, pools, tables, lens, scale, bits, dtype, alibi=None, out=None):
    """attend() and how far a kernel's output may be from it, element by element.

    With p the softmax weights and e_j how far the weight of token j may be off, relatively, an output sum_j p_j v_j is
    off by at most sum_j p_j e_j |v_j| (the numerator) + (sum_j p_j e_j) (sum_j p_j |v_j|) (the denominator).  e_j is
      2^-11                       one rounding of the weight to fp16, where that is normal
      2^-20                       exp2 and the products around it, a few roundings of 2^-22 to 2^-24
      d_j                         the score's error: q . k in fp32 over at most 256 products, in at most 16 steps that may
                                  truncate, is off by 16 * 2^-22 of sum |q k|; q itself may be held in fp16 relative to the
                                  largest |q| of its row, which costs 2^-21 of that where an element is subnormal; a
                                  distance bias counts with its own size
      (n / 4 + 64) 2^-23          sums over the n tokens in fp32, at least four side by side
    A weight that is subnormal in fp16 is off by 2^-25 of the largest p_j max|v_j| instead.  The result is rounded once
    to its type: half a step, finfo.eps / 2, and half of the smallest subnormal."""
    half = torch.finfo(dtype).eps / 2
    k_cache, v_cache, k_scales, v_scales = pools
    bs, kvh = k_cache.shape[2], k_cache.shape[1]
    seqs, heads, hd = q.shape
    g = heads // kvh
    want = attend(q, pools, tables, lens, scale, bits, alibi, out)
    bound = torch.zeros_like(want)
    for i in range(seqs):
        n = min(int(lens[i]), tables.shape[1] * bs)
        if n <= 0:
            continue
        t = torch.arange(n, device=q.device)
        block, off = tables[i].long()[t // bs], t % bs
        k = values(k_cache[block, :, off], k_scales[block, :, off], bits)
        v = values(v_cache[block, :, off], v_scales[block, :, off], bits).abs()
        qq = q[i].double().view(kvh, g, hd)
        s = torch.einsum("hgd,nhd->hgn", qq, k) * scale
        d = torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs()) * abs(scale) * 2.0 ** -18
        d = d + qq.abs().amax(-1, keepdim=True) * k.abs().sum(-1).T[:, None] * abs(scale) * 2.0 ** -21
        if alibi is not None:
            bias = alibi.double().view(kvh, g, 1) * (t.double() - (n - 1))
            s, d = s + bias, d + bias.abs() * 2.0 ** -21
        p = torch.softmax(s, -1)
        e = p * (2.0 ** -11 + 2.0 ** -20 + torch.expm1(2 * d) + (n / 4 + 64) * 2.0 ** -23)
        small = n * 2.0 ** -25 * (p * v.amax(-1).T[:, None]).amax(-1, keepdim=True)
        whole = torch.einsum("hgn,nhd->hgd", e, v) + e.sum(-1, keepdim=True) * torch.einsum("hgn,nhd->hgd", p, v) + small
        bound[i] = (whole * (1 + half)).reshape(heads, hd) + half * want[i].abs() + torch.finfo(dtype).smallest_normal * half
    return want, bound


def close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound) & ~(torch.isnan(got.double()) & torch.isnan(want))
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst error {float(err[bad].max()):.3e} at {torch.nonzero(bad)[0].tolist()}, "
        f"bound there {float(bound.expand_as(err)[bad].min()):.3e}")


def random_pools(gen, blocks, kv_heads, block, k_head, v_head, bits, std=1.0, device="cuda"):
    """Pools as appends of normal rows leave them, every slot filled."""
    out = empty_pools(blocks, kv_heads, block, k_head, v_head, bits, device)
    for x, head in ((0, k_head), (1, v_head)):
        rows = (torch.randn((blocks, kv_heads, block, head), generator=gen) * std).to(device)
        c, s = quantise(rows.to(torch.bfloat16), bits)
        out[x].copy_(pack(c, bits))
        out[2 + x].copy_(s)
    return out


def tables_for(gen, lens, block, blocks, dtype=torch.int64, device="cuda"):
    """Block tables over distinct blocks in random order; entries behind a sequence's last block are 0."""
    need = [-(-max(0, n) // block) for n in lens]
    order = torch.randperm(blocks, generator=gen)
    assert sum(need) <= blocks
    t = torch.zeros((len(lens), max(1, max(need))), dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t.to(dtype).to(device)
