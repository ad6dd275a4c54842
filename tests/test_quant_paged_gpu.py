"""GPU checks of the operators over quantised pools against plain 64-bit forms: codes and scales bit for bit, values read
back bit for bit, attention within bounds that follow from the roundings of its arithmetic."""
import contextlib
import math
import os

import pytest
import torch

import quant_helpers as qh

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ib():
    import infinicore_b200

    yield infinicore_b200
    torch.cuda.synchronize()
    assert infinicore_b200.kernel_status() == 0


@contextlib.contextmanager
def environment(**values):
    old = {k: os.environ.get(k) for k in values}
    os.environ.update({k: str(v) for k, v in values.items()})
    try:
        yield
    finally:
        for k, v in old.items():
            os.environ.pop(k, None) if v is None else os.environ.__setitem__(k, v)


def same_bits(a, b):
    view = lambda t: t.contiguous().view(torch.int16) if t.element_size() == 2 else t.contiguous()  # noqa: E731
    return bool(torch.equal(view(a.cpu()), view(b.cpu())))


def same_scales(a, b):
    a, b = a.cpu(), b.cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def rows(gen, shape, dtype):
    """Normal rows with a spread of sizes, a loud channel, an all-zero group and signed zeros."""
    x = torch.randn(shape, generator=gen) * torch.exp(torch.randn(shape[:-1] + (1,), generator=gen))
    x[..., 3] *= 20
    if x.numel():
        x[0, :, 32:64 if shape[-1] > 32 else 32] = 0
        x[..., 5] = -0.0
    return x.to(dtype)


# ---- writing ----------------------------------------------------------------------------------------------

WRITE = [  # tokens, kv_heads, k head, v head, block, blocks
    (1, 1, 64, 64, 16, 2), (2, 8, 128, 128, 16, 3), (33, 3, 96, 32, 7, 9), (64, 8, 128, 128, 16, 40), (5, 2, 576, 512, 16, 4),
    (17, 1, 1024, 1024, 1, 20), (130, 5, 256, 256, 32, 6), (9, 2, 192, 160, 64, 1), (4, 2, 288, 320, 3, 4), (1000, 2, 64, 64, 128, 9),
]


@pytest.mark.parametrize("case", WRITE)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_are_written_bit_for_bit_and_nothing_else_is(ib, case, bits, dtype):
    tokens, kvh, kh, vh, bs, blocks = case
    g = torch.Generator().manual_seed(tokens * 7 + kvh)
    k, v = rows(g, (tokens, kvh, kh), dtype), rows(g, (tokens, kvh, vh), dtype)
    slots = torch.randperm(blocks * bs, generator=g)[:tokens]
    slots = torch.cat([slots, torch.full((tokens - slots.numel(),), -1, dtype=torch.int64)])
    slots[::5] = -1 - torch.arange(slots[::5].numel()) if tokens > 4 else slots[::5]
    want = qh.empty_pools(blocks, kvh, bs, kh, vh, bits, fill=0x5A)
    got = [t.cuda() for t in want]
    qh.write(want, k, v, slots, bits)
    res = ib.quant_paged_caching(*got, k.cuda(), v.cuda(), slots.cuda())
    assert all(r is t for r, t in zip(res, got))
    for a, b in zip(got, want):
        assert same_bits(a, b)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_halves_extremes_and_values_that_are_none(ib, bits, dtype):
    """Exact halves (away from zero), the largest and smallest magnitudes, subnormals, infinities and NaN."""
    q = qh.limits(bits)
    fi = torch.finfo(dtype)
    x = torch.zeros((12, 1, 64))
    for c in range(q):
        x[0, 0, c % 32 + 32 * (c // 32 % 2)] = (c + 0.5) * (1 if c % 2 else -1)
    x[0, 0, 31] = x[0, 0, 63] = q          # scale 1: the halves are exact where the type holds them
    x[1] = x[0] * 0.25
    x[2] = x[0] * 3
    x[3, 0, ::2], x[3, 0, 1::2] = fi.max, fi.max / 3
    x[4, 0, 0], x[4, 0, 40] = -fi.max, fi.smallest_normal
    x[5] = fi.smallest_normal * torch.linspace(-2, 2, 64)
    x[6] = fi.smallest_normal * fi.eps * torch.arange(64)
    x[7, 0, 1], x[7, 0, 2] = float("inf"), 1.0
    x[8, 0, 33], x[8, 0, 2] = float("nan"), 1.0
    x[9, 0, 1], x[9, 0, 33] = -float("inf"), float("nan")
    x[10, 0, 0] = fi.smallest_normal * q * 1.01
    x[11] = -0.0
    x = x.to(dtype)
    want = qh.empty_pools(1, 1, 16, 64, 64, bits, fill=0x11)
    got = [t.cuda() for t in want]
    slots = torch.arange(12) + 2
    qh.write(want, x, x.flip(0), slots, bits)
    ib.quant_paged_caching(*got, x.cuda(), x.flip(0).contiguous().cuda(), slots.cuda())
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(got[2:], want[2:]):
        assert same_scales(a, b)
    back = ib.quant_paged_cache_read(*got, slots.cuda(), FP32)
    for a, b in zip(back, qh.read(want, slots, bits)):
        assert bool(((a.cpu().double() == b.float().double()) | (a.cpu().isnan() & b.isnan())).all())
    assert bool(back[0][7].isnan().any()) and bool(back[0][8].isnan().any())


@pytest.mark.parametrize("bits", [4, 8])
def test_slices_odd_addresses_and_other_orders(ib, bits):
    """Rows that are slices of a fused projection (aligned and not), pools with tokens before heads, pools and rows at odd
    addresses, scales in an order of their own."""
    g = torch.Generator().manual_seed(11)
    tokens, kvh, hd, bs, blocks = 21, 3, 96, 8, 5
    for shift in (0, 1, 8):
        fused = torch.randn((tokens, kvh * 2 * hd + 24), generator=g).to(BF16)
        k = fused[:, shift:shift + kvh * hd].unflatten(1, (kvh, hd))
        v = fused[:, shift + kvh * hd:shift + 2 * kvh * hd].unflatten(1, (kvh, hd))
        dev = fused.cuda()
        dk = dev[:, shift:shift + kvh * hd].unflatten(1, (kvh, hd))
        dv = dev[:, shift + kvh * hd:shift + 2 * kvh * hd].unflatten(1, (kvh, hd))
        slots = torch.randperm(blocks * bs, generator=g)[:tokens]
        want = qh.empty_pools(blocks, kvh, bs, hd, hd, bits, fill=3)
        qh.write(want, k, v, slots, bits)
        got = []
        for i, t in enumerate(want):
            n, w = t.numel(), t.shape[-1]
            raw = torch.zeros(n + 16, dtype=t.dtype, device="cuda")[shift:shift + n]
            if i == 1:      # [blocks, block, heads, width]
                p = raw.view(blocks, bs, kvh, w).transpose(1, 2)
            elif i == 2:    # [heads, blocks, block, width]
                p = raw.view(kvh, blocks, bs, w).transpose(0, 1)
            else:
                p = raw.view(blocks, kvh, bs, w)
            p.copy_(qh.empty_pools(blocks, kvh, bs, hd, hd, bits, fill=3)[i])
            got.append(p)
        ib.quant_paged_caching(*got, dk, dv, slots.cuda())
        for a, b in zip(got, want):
            assert same_bits(a, b), shift
        out = torch.full((tokens, 2, kvh, hd + 1 + shift), 7.0, dtype=FP16, device="cuda")
        pair = (out[:, 0, :, :hd], out[:, 1, :, 1:hd + 1])
        ib.quant_paged_cache_read(*got, slots.cuda(), out=pair)
        for a, b in zip(pair, qh.read(want, slots, bits)):
            assert same_bits(a, b.to(FP16))
        assert bool((out[:, 0, :, hd:] == 7).all()) and bool((out[:, 1, :, :1] == 7).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_a_pool_of_more_than_four_gigabytes(ib, bits):
    """Offsets that pass 32 bits, in codes and in the number of slots."""
    kvh, hd, bs = 1, 1024, 64
    width = hd if bits == 8 else hd // 2
    blocks = (1 << 32) // (bs * width) + 70
    codes = [torch.zeros((blocks, kvh, bs, width), dtype=torch.int8 if bits == 8 else torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.zeros((blocks, kvh, bs, qh.groups(bits, hd)), dtype=BF16, device="cuda") for _ in "kv"]
    g = torch.Generator().manual_seed(3)
    k, v = rows(g, (3, kvh, hd), BF16), rows(g, (3, kvh, hd), BF16)
    slots = torch.tensor([blocks * bs - 1, 5, (blocks - 60) * bs + 1])
    pools = (*codes, *scales)
    ib.quant_paged_caching(*pools, k.cuda(), v.cuda(), slots.cuda())
    back = ib.quant_paged_cache_read(*pools, slots.cuda(), BF16)
    for a, x in zip(back, (k, v)):
        c, s = qh.quantise(x, bits)
        assert same_bits(a, qh.values(qh.pack(c, bits), s, bits).to(BF16))
    assert int((codes[0] != 0).any(-1).sum()) == 3


def test_no_tokens_and_no_slots(ib):
    pools = qh.empty_pools(3, 2, 16, 64, 64, 8, "cuda", fill=9)
    before = [t.clone() for t in pools]
    none = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    ib.quant_paged_caching(*pools, none, none, empty)
    k, v = ib.quant_paged_cache_read(*pools, empty)
    assert k.shape == v.shape == (0, 2, 64)
    some = torch.ones((4, 2, 64), dtype=BF16, device="cuda")
    ib.quant_paged_caching(*pools, some, some, torch.full((4,), -1, dtype=torch.int64, device="cuda"))
    for a, b in zip(pools, before):
        assert same_bits(a, b)


# ---- reading ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", [(1, 64, 64, 16), (3, 128, 128, 16), (2, 96, 32, 5), (8, 256, 256, 32), (1, 576, 512, 16)])
def test_reading_is_the_rounded_product(ib, shape, bits, dtype):
    kvh, kh, vh, bs = shape
    g = torch.Generator().manual_seed(kh + bits)
    pools = qh.empty_pools(9, kvh, bs, kh, vh, bits)
    for c in pools[:2]:  # every byte a user's pool may hold, -8 and -128 included
        c.copy_(torch.randint(-128, 128, c.shape, generator=g).to(c.dtype))
    for s in pools[2:]:
        s.copy_(torch.exp(3 * torch.randn(s.shape, generator=g)).to(BF16))
    slots = torch.cat([torch.randint(0, 9 * bs, (37,), generator=g), torch.tensor([-1, 0, 0, -7, 9 * bs - 1])])
    k, v = ib.quant_paged_cache_read(*[t.cuda() for t in pools], slots.cuda(), dtype)
    for a, b in zip((k, v), qh.read(pools, slots, bits)):
        assert torch.equal(a.cpu(), b.to(dtype) if dtype != FP32 else b.float())
    assert bool((k[37] == 0).all()) and bool((v[40] == 0).all())


# ---- attention --------------------------------------------------------------------------------------------

@contextlib.contextmanager
def rows_path():
    """Descriptors made here use the kernel for any layout; none of them is kept."""
    with environment(INFINIOP_QUANT_ATTENTION_PATH="rows"):
        forget()
        yield
    forget()


def forget():
    from infinicore_b200 import _torch_ops

    _torch_ops.clear_cache()


def check_attention(ib, gen, lens, heads, kvh, hd, bs, bits, dtype, scale=None, alibi=False, ix=torch.int64, std=1.0, qstd=1.0, what=""):
    lens_t = torch.tensor(lens)
    blocks = max(1, sum(-(-max(0, n) // bs) for n in lens)) + 2
    pools = qh.random_pools(gen, blocks, kvh, bs, hd, hd, bits, std)
    tables = qh.tables_for(gen, lens, bs, blocks, ix)
    q = (torch.randn((len(lens), heads, hd), generator=gen) * qstd).to(dtype).cuda()
    slopes = torch.exp2(-8.0 * (torch.arange(heads) + 1) / heads).cuda() if alibi else None
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full((len(lens), heads, hd), 3.0, dtype=dtype, device="cuda")
    got = ib.quant_paged_attention(q, *pools, tables, lens_t.to(ix).cuda(), slopes, scale, out=out)
    want, bound = qh.attend_bound(q, pools, tables, lens_t, scale, bits, dtype, slopes, torch.full_like(out, 3.0))
    qh.close(got, want, bound, what)
    with rows_path():
        other = ib.quant_paged_attention(q, *pools, tables, lens_t.to(ix).cuda(), slopes, scale, out=torch.full_like(out, 3.0))
    qh.close(other, want, bound, what + " (rows)")
    for i, n in enumerate(lens):
        if n <= 0:
            assert bool((got[i] == 3).all()) and bool((other[i] == 3).all())
    return q, pools, tables, lens_t, got


LENGTHS = {
    "one": [1], "edges": [1, 2, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65], "ragged": [700, 1, 0, 4096, 129, 2047],
    "many": [3, 250, 77, 0, 16] * 13, "long": [20011],
}


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
@pytest.mark.parametrize("lens", LENGTHS)
def test_attention_over_lengths_and_heads(ib, lens, hd, bits):
    g = torch.Generator().manual_seed(hd + bits)
    dtype = BF16 if hd in (64, 256) else FP16
    check_attention(ib, g, LENGTHS[lens], 8, 2, hd, 16, bits, dtype, what=lens)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (4, 4), (6, 3), (5, 1), (7, 1), (8, 1), (9, 1), (16, 2), (12, 1), (32, 2), (20, 1), (48, 1), (64, 2)])
def test_attention_over_groups(ib, heads, kvh, dtype, bits):
    g = torch.Generator().manual_seed(heads)
    check_attention(ib, g, [300, 1, 0, 45, 16], heads, kvh, 128, 16, bits, dtype, what=f"{heads}/{kvh}")
    check_attention(ib, g, [33, 500], heads, kvh, 64, 32, bits, dtype, alibi=True, what=f"{heads}/{kvh} alibi")
    check_attention(ib, g, [65, 2], heads, kvh, 256, 16, bits, dtype, what=f"{heads}/{kvh} 256")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("bs", [1, 3, 8, 16, 24, 48, 64, 256])
def test_attention_over_block_sizes(ib, bs, bits):
    g = torch.Generator().manual_seed(bs)
    check_attention(ib, g, [1, bs, bs + 1, 5 * bs - 1, 333, 0], 8, 2, 128, bs, bits, BF16, what=f"block {bs}")
    check_attention(ib, g, [2 * bs, 77], 4, 4, 64, bs, bits, FP16, ix=torch.int32, what=f"block {bs} int32")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens", [[40], [1000, 3, 500]])
def test_attention_that_looks_at_few_tokens(ib, lens, bits):
    """Scores far apart: an output is one token's row or two, so a token lost, doubled or out of place shows in full."""
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        check_attention(ib, g, lens, 8, 2, 128, 16, bits, FP16, scale=3.0, what="peaked")
        check_attention(ib, g, lens, 8, 8, 64, 16, bits, BF16, scale=-2.0, alibi=True, what="peaked, negative scale")


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_over_values_of_all_sizes(ib, bits):
    """V rows whose scales differ by 2^40 from token to token, all-zero V rows among them, large and tiny q."""
    g = torch.Generator().manual_seed(5)
    hd, kvh, bs, n = 128, 2, 16, 200
    pools = qh.random_pools(g, 14, kvh, bs, hd, hd, bits)
    pools[3].copy_((pools[3].float() * torch.exp2(torch.randint(-20, 21, pools[3].shape, generator=g).float().cuda())).to(BF16))
    pools[3][2:5] = 0
    tables = qh.tables_for(g, [n], bs, 14)
    lens = torch.tensor([n])
    for qstd, scale in ((1.0, 0.1), (1e-6, 1e5), (3e4, 3e-6), (1e-3, 0.0)):
        q = (torch.randn((1, 8, hd), generator=g) * qstd).to(BF16).cuda()
        got = ib.quant_paged_attention(q, *pools, tables, lens.cuda(), None, scale)
        want, bound = qh.attend_bound(q, pools, tables, lens, scale, bits, BF16)
        qh.close(got, want, bound, f"q {qstd}")
    zero = torch.zeros_like(pools[3])
    got = ib.quant_paged_attention(q, pools[0], pools[1], pools[2], zero, tables, lens.cuda(), None, 0.1)
    assert bool((got == 0).all())
    big = torch.full_like(pools[3], 2.0 ** 60)
    got = ib.quant_paged_attention(q, pools[0], pools[1], pools[2], big, tables, lens.cuda(), None, 0.1)
    want, bound = qh.attend_bound(q, (*pools[:3], big), tables, lens, 0.1, bits, BF16)
    qh.close(got, want, bound, "large V")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 128, 192])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e14])
def test_attention_over_scores_of_any_size(ib, size, hd, bits):
    """Scores of up to `size`: their softmax is one token's row (the largest score stands out by far more than fp32 loses of it), and
    the output is that row rounded to the type."""
    g = torch.Generator().manual_seed(hd)
    lens, bs, kvh, heads = [300, 37, 1], 16, 2, 8
    pools = qh.random_pools(g, 30, kvh, bs, hd, hd, bits)
    pools[2].mul_(1e3)
    pools[3].mul_(1e-3)
    tables = qh.tables_for(g, lens, bs, 30)
    lens_t = torch.tensor(lens)
    q = torch.randn((3, heads, hd), generator=g).to(BF16).cuda()
    for sign in (1.0, -1.0):
        scale = sign * size / 1e3 / hd ** 0.5
        got = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, scale)
        assert bool(torch.isfinite(got).all())
        for i, n in enumerate(lens):
            t = torch.arange(n, device="cuda")
            block, off = tables[i][t // bs], t % bs
            k, v = (qh.values(pools[x][block, :, off], pools[x + 2][block, :, off], bits) for x in (0, 1))
            s = torch.einsum("hgd,nhd->hgn", q[i].double().view(kvh, 4, hd), k) * scale
            best = s.max(-1)
            second = s.scatter(-1, best.indices[..., None], -float("inf")).amax(-1)
            # fp32 loses 2^-18 of sum |q k| at most, the bound of attend_bound; 40 more leave nothing of the second
            lost = torch.einsum("hgd,nhd->hgn", q[i].double().view(kvh, 4, hd).abs(), k.abs()).amax(-1) * abs(scale) * 2.0 ** -17
            clear = best.values - second > lost + 40
            assert int(clear.sum()) >= (4 if size > 1e3 else 1)
            want = torch.stack([v[best.indices[h], h] for h in range(kvh)])  # [kvh, g, hd]
            err = (got[i].double().view(kvh, 4, hd) - want).abs()
            # the weight is rounded to fp16 and the sum divided by p: 2^-11 + 2^-20, and half a step of bf16; the n - 1 other tokens weigh
            # less than e^-40 each
            ok = err <= want.abs() * (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) + n * math.exp(-40) * v.abs().max()
            assert bool(ok[clear].all()), (size, sign, i)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_what_lies_behind_a_sequence_does_not_matter(ib, hd, bits):
    """NaN and infinite scales in every slot that no sequence reaches, in the last page of each too; a NaN or an infinity
    that a sequence does reach makes its rows NaN, and no other's."""
    g = torch.Generator().manual_seed(hd)
    lens, bs, kvh = [5, 40, 17, 64], 16, 2
    pools = qh.random_pools(g, 20, kvh, bs, hd, hd, bits)
    tables = qh.tables_for(g, lens, bs, 20)
    live = torch.zeros((20, bs), dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(n):
            live[int(tables[i, t // bs]), t % bs] = True
    dead = (~live).cuda()[:, None, :, None]
    pools[2].masked_fill_(dead, float("nan"))
    pools[3].copy_(torch.where(dead, torch.tensor(float("inf"), dtype=BF16, device="cuda"), pools[3]))
    q = torch.randn((4, 8, hd), generator=g).to(BF16).cuda()
    lens_t = torch.tensor(lens)
    got = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, 0.1)
    want, bound = qh.attend_bound(q, pools, tables, lens_t, 0.1, bits, BF16)
    assert bool(torch.isfinite(want).all())
    qh.close(got, want, bound)
    for which in (2, 3):
        bad = [t.clone() for t in pools]
        block, off = int(tables[1, 20 // bs]), 20 % bs
        bad[which][block, 1, off, 0] = float("nan")
        got = ib.quant_paged_attention(q, *bad, tables, lens_t.cuda(), None, 0.1)
        hit = torch.zeros((4, 8, hd), dtype=torch.bool, device="cuda")
        hit[1, 4:, :(hd if which == 2 or bits == 8 else qh.GROUP)] = True
        assert torch.equal(got.isnan(), hit)
        qh.close(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, 0.0, want), bound)
    q2 = q.clone()
    q2[2, 3, 7] = float("nan")
    q2[0, 5, 1] = float("inf")
    got = ib.quant_paged_attention(q2, *pools, tables, lens_t.cuda(), None, 0.1)
    hit = torch.zeros((4, 8, 1), dtype=torch.bool, device="cuda")
    hit[2, 3], hit[0, 5] = True, True
    qh.close(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, 0.0, want), bound)
    assert bool(got[2, 3].isnan().all())


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_over_other_layouts(ib, bits):
    """Strided q and out, tokens before heads in the pools, a table that is a slice, odd addresses and strides."""
    g = torch.Generator().manual_seed(9)
    lens, heads, kvh, hd, bs, blocks = [50, 0, 131], 8, 2, 128, 16, 14
    pools = qh.random_pools(g, blocks, kvh, bs, hd, hd, bits)
    tables = qh.tables_for(g, lens, bs, blocks)
    wide = torch.zeros((3, tables.shape[1] + 5), dtype=torch.int64, device="cuda")
    wide[:, :tables.shape[1]] = tables
    tables = wide[:, :tables.shape[1]]
    lens_t = torch.tensor(lens)
    base = torch.randn((3, 2 * heads * hd + 8), generator=g).to(FP16).cuda()
    want, bound = None, None
    for case in ("plain", "token first", "gaps", "odd", "rows of odd length"):
        p = []
        for t in pools:
            w = t.shape[-1]
            if case == "token first":
                n = t.transpose(1, 2).contiguous().transpose(1, 2)
            elif case == "gaps":
                n = torch.zeros((blocks, kvh + 1, bs, 2 * w), dtype=t.dtype, device="cuda")[:, 1:, :, :w]
                n.copy_(t)
            elif case == "odd":
                n = torch.zeros(t.numel() + 3, dtype=t.dtype, device="cuda")[3:].view(t.shape)
                n.copy_(t)
            elif case == "rows of odd length":
                n = torch.zeros((blocks, kvh, bs, w + 1), dtype=t.dtype, device="cuda")[..., :w]
                n.copy_(t)
            else:
                n = t
            p.append(n)
        shift = 1 if case == "odd" else 0
        q = base[:, shift:shift + 2 * heads * hd].unflatten(1, (heads, 2 * hd))[:, :, :hd]
        out = torch.full((3, heads, 3 * hd), 5.0, dtype=FP16, device="cuda")
        got = ib.quant_paged_attention(q, *p, tables, lens_t.cuda(), None, 0.1, out=out[:, :, shift:shift + hd])
        want, bound = qh.attend_bound(q, pools, tables, lens_t, 0.1, bits, FP16, None, torch.full((3, heads, hd), 5.0).cuda())
        qh.close(got, want, bound, case)
        assert bool((out[:, :, hd + shift:] == 5).all()) and bool((out[1] == 5).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_lengths_beyond_the_table_are_cut_and_negative_ones_are_empty(ib, bits):
    g = torch.Generator().manual_seed(2)
    pools = qh.random_pools(g, 8, 1, 16, 64, 64, bits)
    tables = qh.tables_for(g, [64, 64], 16, 8)
    q = torch.randn((2, 4, 64), generator=g).to(BF16).cuda()
    full = ib.quant_paged_attention(q, *pools, tables, torch.tensor([64, 64], device="cuda"), None, 0.125)
    out = torch.full_like(full, 9.0)
    for big in (65, 1 << 31, (1 << 40) + 3):
        ib.quant_paged_attention(q, *pools, tables, torch.tensor([big, -big], device="cuda"), None, 0.125, out=out)
        assert torch.equal(out[0], full[0]) and bool((out[1] == 9).all())
    none = torch.zeros((2, 0), dtype=torch.int64, device="cuda")
    assert bool((ib.quant_paged_attention(q, *pools, none, torch.tensor([3, 0], device="cuda")) == 0).all())
    nobody = ib.quant_paged_attention(q[:0], *pools, tables[:0], torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert nobody.shape == (0, 4, 64)
    alone = ib.quant_paged_attention(q, *pools, tables, torch.tensor([0, -4], device="cuda"))
    assert bool((alone == 0).all())


def test_attention_in_a_pool_of_more_than_four_gigabytes(ib):
    g = torch.Generator().manual_seed(4)
    hd, bs, kvh = 256, 64, 2
    blocks = (1 << 32) // (kvh * bs * hd) + 9
    codes = [torch.zeros((blocks, kvh, bs, hd), dtype=torch.int8, device="cuda") for _ in "kv"]
    scales = [torch.zeros((blocks, kvh, bs, 1), dtype=BF16, device="cuda") for _ in "kv"]
    small = qh.random_pools(g, 5, kvh, bs, hd, hd, 8)
    at = torch.tensor([blocks - 1, 2, blocks - 7, blocks // 2, 0], device="cuda")
    for big, t in zip((*codes, *scales), small):
        big[at] = t
    q = torch.randn((1, 8, hd), generator=g).to(BF16).cuda()
    lens = torch.tensor([5 * bs - 3])
    got = ib.quant_paged_attention(q, *codes, *scales, at[None], lens.cuda(), None, 0.06)
    want, bound = qh.attend_bound(q, small, torch.arange(5, device="cuda")[None], lens, 0.06, 8, BF16)
    qh.close(got, want, bound)


# ---- together, streams, graphs, checks --------------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_prefill_read_back_and_steps_of_decode(ib, bits, dtype):
    """Prompts written, their history read back as dense rows that serve the prefill operator as a pool, then steps of
    append and attend: every stage against the plain forms on pools of its own."""
    g = torch.Generator().manual_seed(21)
    kvh, heads, hd, bs, blocks = 2, 8, 128, 16, 40
    lens = [70, 16, 33]
    pools = qh.empty_pools(blocks, kvh, bs, hd, hd, bits, "cuda")
    plain = qh.empty_pools(blocks, kvh, bs, hd, hd, bits)
    tables = qh.tables_for(g, [n + 20 for n in lens], bs, blocks)

    def slots_of(i, first, last):
        t = torch.arange(first, last)
        return tables[i].cpu()[t // bs] * bs + t % bs

    def append(slots):
        k, v = (torch.randn((slots.numel(), kvh, hd), generator=g).to(dtype) for _ in "kv")
        qh.write(plain, k, v, slots, bits)
        ib.quant_paged_caching(*pools, k.cuda(), v.cuda(), slots.cuda())
        for a, b in zip(pools, plain):
            assert same_bits(a, b)

    append(torch.cat([slots_of(i, 0, n) for i, n in enumerate(lens)]))
    # the history as a paged pool: one page of 16 slots after the other, padding behind each sequence's end
    pages = [-(-n // bs) for n in lens]
    slots = torch.cat([torch.cat([slots_of(i, 0, n), torch.full((p * bs - n,), -1)]) for i, (n, p) in enumerate(zip(lens, pages))])
    rows_k, rows_v = ib.quant_paged_cache_read(*pools, slots.cuda(), dtype)
    paged = [r.view(-1, bs, kvh, hd).transpose(1, 2) for r in (rows_k, rows_v)]
    first = torch.tensor([0, pages[0], pages[0] + pages[1]])
    small = torch.zeros((3, max(pages)), dtype=torch.int64)
    for i, p in enumerate(pages):
        small[i, :p] = first[i] + torch.arange(p)
    new = torch.tensor([10, 16, 1])
    q = torch.randn((int(new.sum()), heads, hd), generator=g).to(dtype).cuda()
    cum = torch.tensor([0, 10, 26, 27])
    got = ib.paged_attention_prefill(q, *paged, small.cuda(), torch.tensor(lens).cuda(), cum.cuda(), None, 0.09)
    tol = 1e-2 if dtype == BF16 else 2e-3  # of the prefill operator itself
    at = 0
    for i, n in enumerate(lens):
        for t in range(int(new[i])):
            upto = n - int(new[i]) + t + 1
            want = qh.attend(q[at:at + 1], pools, tables[i:i + 1], torch.tensor([upto]), 0.09, bits)
            err = (got[at:at + 1].double() - want).abs()
            # the rows read back were rounded to the type, half a step each
            assert bool((err <= tol + tol * want.abs() + 2 * torch.finfo(dtype).eps * 4).all())
            at += 1
    for step in range(3):
        append(torch.cat([slots_of(i, n + step, n + step + 1) for i, n in enumerate(lens)]))
        now = torch.tensor(lens) + step + 1
        q = torch.randn((3, heads, hd), generator=g).to(dtype).cuda()
        got = ib.quant_paged_attention(q, *pools, tables, now.cuda(), None, 0.09)
        want, bound = qh.attend_bound(q, pools, tables, now, 0.09, bits, dtype)
        qh.close(got, want, bound, f"step {step}")


def problem(gen, bits, lens, hd=128, heads=8, kvh=2, bs=16, dtype=BF16):
    blocks = sum(-(-n // bs) for n in lens) + 1
    pools = qh.random_pools(gen, blocks, kvh, bs, hd, hd, bits)
    tables = qh.tables_for(gen, lens, bs, blocks)
    q = torch.randn((len(lens), heads, hd), generator=gen).to(dtype).cuda()
    lens_t = torch.tensor(lens)
    want, bound = qh.attend_bound(q, pools, tables, lens_t, 0.09, bits, dtype)
    return q, pools, tables, lens_t.cuda(), want, bound


@pytest.mark.parametrize("bits", [4, 8])
def test_two_streams_at_once_and_two_graphs_at_once(ib, bits):
    """Calls on two streams, and graphs captured on one stream but replayed on two, at the same time: each has its scratch."""
    g = torch.Generator().manual_seed(31)
    a, b = problem(g, bits, [9000, 700]), problem(g, bits, [5, 8000, 300], heads=16)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()

    def call(p, out):
        ib.quant_paged_attention(p[0], *p[1], p[2], p[3], None, 0.09, out=out)

    outs = [torch.zeros_like(a[0]), torch.zeros_like(b[0])]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, p, o in ((s1, a, outs[0]), (s2, b, outs[1])):
            with torch.cuda.stream(s):
                call(p, o)
    torch.cuda.synchronize()
    qh.close(outs[0], a[4], a[5])
    qh.close(outs[1], b[4], b[5])

    graphs = []
    for p, o in zip((a, b), outs):
        o.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s1):
            call(p, o)
        graphs.append(graph)
    for _ in range(20):
        for s, graph in zip((s1, s2), graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    qh.close(outs[0], a[4], a[5])
    qh.close(outs[1], b[4], b[5])


@pytest.mark.parametrize("bits", [4, 8])
def test_a_captured_step_follows_lengths_and_slots(ib, bits):
    """Append and attend captured once, replayed with other lengths, tables and slots, empty sequences among them."""
    g = torch.Generator().manual_seed(41)
    kvh, heads, hd, bs, blocks, seqs = 2, 8, 64, 16, 64, 4
    pools = qh.empty_pools(blocks, kvh, bs, hd, hd, bits, "cuda")
    order = torch.randperm(blocks, generator=g).view(seqs, -1)
    k, v = (torch.zeros((seqs, kvh, hd), dtype=BF16, device="cuda") for _ in "kv")
    q = torch.zeros((seqs, heads, hd), dtype=BF16, device="cuda")
    slots = torch.full((seqs,), -1, dtype=torch.int64, device="cuda")
    lens = torch.zeros(seqs, dtype=torch.int64, device="cuda")
    tables = order.cuda()
    out = torch.zeros_like(q)

    def step():
        ib.quant_paged_caching(*pools, k, v, slots)
        ib.quant_paged_attention(q, *pools, tables, lens, None, 0.1, out=out)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    plain = [t.cpu() for t in pools]
    now = [0, 0, 0, 0]
    for turn in range(40):
        grow = [i for i in range(seqs) if (turn + i) % (i + 1) == 0]
        at = torch.full((seqs,), -1, dtype=torch.int64)
        for i in grow:
            at[i] = order[i, now[i] // bs] * bs + now[i] % bs
            now[i] += 1
        nk, nv = (torch.randn((seqs, kvh, hd), generator=g).to(BF16) for _ in "kv")
        qh.write(plain, nk, nv, at, bits)
        for t, x in ((k, nk), (v, nv), (q, torch.randn(q.shape, generator=g).to(BF16)), (slots, at), (lens, torch.tensor(now))):
            t.copy_(x)
        out.fill_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(pools, plain):
            assert same_bits(a, b)
        want, bound = qh.attend_bound(q, pools, tables, torch.tensor(now), 0.1, bits, BF16, None, torch.full_like(out, 2.0))
        qh.close(out, want, bound, f"turn {turn}")


@pytest.mark.parametrize("bits", [4, 8])
def test_the_same_call_twice_gives_the_same_bits(ib, bits):
    g = torch.Generator().manual_seed(51)
    q, pools, tables, lens, _, _ = problem(g, bits, [7000, 12, 900, 40, 3000, 1], heads=16, hd=64)
    first = ib.quant_paged_attention(q, *pools, tables, lens, None, 0.09)
    for _ in range(5):
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda").fill_(0xFF)
        assert torch.equal(ib.quant_paged_attention(q, *pools, tables, lens, None, 0.09), first)


def test_checked_indices_raise_flags_and_touch_nothing_foreign(ib):
    """INFINIOP_PAGED_CHECK_INDICES=1 when a descriptor is made: blocks and slots outside the pool are reported; a bad slot's
    row is skipped (zeros when read), a bad block is read as block 0."""
    g = torch.Generator().manual_seed(61)
    ib.kernel_status()
    forget()
    with environment(INFINIOP_PAGED_CHECK_INDICES=1):
        pools = qh.random_pools(g, 6, 2, 16, 64, 64, 8)
        before = [t.clone() for t in pools]
        x = torch.randn((3, 2, 64), generator=g).to(BF16).cuda()
        slots = torch.tensor([6 * 16, -1, 1 << 40], device="cuda")
        ib.quant_paged_caching(*pools, x, x, slots)
        assert ib.kernel_status() == 4
        for a, b in zip(pools, before):
            assert same_bits(a, b)
        k, _ = ib.quant_paged_cache_read(*pools, slots)
        assert ib.kernel_status() == 4 and bool((k == 0).all())
        q = torch.randn((2, 4, 64), generator=g).to(BF16).cuda()
        bad = torch.tensor([[3, 6, 1], [2, 1, -5]], device="cuda")
        mended = torch.tensor([[3, 0, 1], [2, 1, 0]], device="cuda")
        lens = torch.tensor([48, 40], device="cuda")
        got = ib.quant_paged_attention(q, *pools, bad, lens, None, 0.125)
        assert ib.kernel_status() == 2
        assert torch.equal(got, ib.quant_paged_attention(q, *pools, mended, lens, None, 0.125))
        # an entry behind the last page is not read
        ib.quant_paged_attention(q, *pools, bad, torch.tensor([16, 20], device="cuda"), None, 0.125)
        assert ib.kernel_status() == 0
    forget()  # descriptors made here must not serve later tests


def test_refusals_reach_python(ib):
    from infinicore_b200.libinfiniop import InfiniStatusError

    pools = qh.empty_pools(3, 2, 16, 64, 64, 8, "cuda")
    x = torch.zeros((4, 2, 64), dtype=BF16, device="cuda")
    slots = torch.arange(4, device="cuda")
    with pytest.raises(InfiniStatusError) as e:
        ib.quant_paged_caching(*pools, x, x, slots.to(torch.int32))
    assert e.value.status == 10
    with pytest.raises(InfiniStatusError) as e:
        ib.quant_paged_caching(*pools, x[:, :1], x, slots)
    assert e.value.status == 11
    with pytest.raises(InfiniStatusError) as e:
        ib.quant_paged_attention(x.transpose(1, 2).contiguous().transpose(1, 2), *pools, slots[:, None], slots)
    assert e.value.status == 12
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ib.quant_paged_cache_read(*pools, slots.cpu())


# ---- calls that share, repeat or leave out --------------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_sequences_that_share_pages_and_a_page_twice_in_a_table(ib, hd, bits):
    """One table for all sequences, by a stride of zero; and tables that repeat pages within a sequence and between them."""
    g = torch.Generator().manual_seed(hd)
    pools = qh.random_pools(g, 20, 2, 16, hd, hd, bits)
    lens = torch.tensor([300, 1, 0, 257, 32, 299])
    q = torch.randn((6, 8, hd), generator=g).to(BF16).cuda()
    one = torch.randperm(20, generator=g)[:19].cuda()
    shared = one[None].expand(6, 19)
    assert shared.stride(0) == 0
    repeated = torch.randint(0, 3, (6, 19), generator=g).cuda()
    for tables in (shared, repeated):
        got = ib.quant_paged_attention(q, *pools, tables, lens.cuda(), None, hd ** -0.5)
        want, bound = qh.attend_bound(q, pools, tables, lens, hd ** -0.5, bits, BF16)
        qh.close(got, want, bound, "shared" if tables is shared else "repeated")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hd", [64, 128, 192])
def test_a_query_that_is_no_number_spoils_its_own_row_only(ib, hd, dtype, bits):
    """A NaN in q makes its scores NaN; an infinity makes them infinite or NaN, whose softmax is NaN.  Heads that share a pass
    with such a one, and one of subnormal numbers, keep their values."""
    g = torch.Generator().manual_seed(hd + bits)
    lens = torch.tensor([200, 1, 33])
    pools = qh.random_pools(g, 20, 2, 16, hd, hd, bits)
    tables = qh.tables_for(g, lens.tolist(), 16, 20)
    q = torch.randn((3, 8, hd), generator=g).to(dtype).cuda()
    q[:, 3] *= torch.finfo(dtype).smallest_normal / 8
    clean = q.clone()
    q[0, 1, 5], q[1, 2, 0], q[2, 6, hd - 1] = float("nan"), float("inf"), -float("inf")
    got = ib.quant_paged_attention(q, *pools, tables, lens.cuda(), None, hd ** -0.5)
    want, bound = qh.attend_bound(clean, pools, tables, lens, hd ** -0.5, bits, dtype)
    for i, h in ((0, 1), (1, 2), (2, 6)):
        assert bool(got[i, h].isnan().all()), (i, h)
        got[i, h], want[i, h], bound[i, h] = 0, 0, 0
    qh.close(got, want, bound, "beside it")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("width", [1, 64, 900])
def test_a_large_batch_that_is_mostly_empty(ib, width, bits):
    """3001 sequences of which one in 37 has tokens, in tables of one page, of as many as a short table may have, and far wider
    than any sequence: the rows of the empty ones stay as they were."""
    g = torch.Generator().manual_seed(width)
    lens = [int(torch.randint(1, min(16 * width, 200) + 1, (1,), generator=g)) if i % 37 == 5 else 0 for i in range(3001)]
    blocks = sum(-(-n // 16) for n in lens)
    pools = qh.random_pools(g, blocks, 2, 16, 64, 64, bits)
    tables = torch.zeros((3001, width), dtype=torch.int64, device="cuda")
    narrow = qh.tables_for(g, lens, 16, blocks)
    tables[:, :narrow.shape[1]] = narrow
    q = torch.randn((3001, 8, 64), generator=g).to(FP16).cuda()
    out = torch.full_like(q, 3.0)
    got = ib.quant_paged_attention(q, *pools, tables, torch.tensor(lens).cuda(), None, 0.125, out=out)
    live = torch.tensor([i for i, n in enumerate(lens) if n]).cuda()
    want, bound = qh.attend_bound(q[live], pools, tables[live], torch.tensor([n for n in lens if n]), 0.125, bits, FP16)
    qh.close(got[live], want, bound, f"width {width}")
    empty = torch.tensor([n == 0 for n in lens]).cuda()
    assert bool((got[empty] == 3).all())
