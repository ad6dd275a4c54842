"""Decode attention over 4-bit pools whose groups of 32 V channels differ much in size, and over pools of either width whose
tokens do: every group of an output is held to its own size."""
import math

import pytest
import torch

import quant_helpers as qh
from test_quant_paged_gpu import ib, rows_path  # noqa: F401  (a fixture, and descriptors of the kernel for any layout)

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def group_bound(q, pools, tables, lens, scale, bits, dtype, weight=2.0 ** -11):
    """The output in 64 bits and how far a kernel's may be from it, by the sizes of an element's own group.

    An output sum_j p_j v_j / sum_j p_j is off by at most
      sum_j p_j |v_j| (2^-11 + x_j)      one rounding of the weight p_j * scale_jg to fp16 (`weight`), and x_j of the rest
      |out| sum_j p_j x_j                the denominator adds p in fp32
      n 2^-25 max_j p_j s_jg             weights that are subnormal in fp16 are off by 2^-25; the largest of a group (p_j times its scale) has come
                                         to 2^7 times its own factor, and the factor in use is at most 2^6 below that: 2^-26 of it, a token's
                                         scale times a code of at most 2^(bits - 1) is s_jg; twice that
      n 2^-131                           unless the group's factor is at its limit of 2^126, where p s_jg is below 2^-119: then the 2^-25 are
                                         2^-25 2^-126 of p v, times a code of at most 2^3, over a sum of p of 2^-17 at least (the largest
                                         score's p is in 2^-17 to 2^-8): 2^-131 a token
    with x_j = 2 d_j + 2^-19 + (n / 4 + 64) 2^-23: d_j the score's error (2^-18 of sum |q k|: 16 steps that may truncate, 2^-22 each; and 2^-21
    of the largest |q| for elements that are subnormal in fp16), exp2 of an argument of at most 32 that is rounded to 2^-20 of 1 and
    the products around it, and sums over n tokens in fp32, at least four side by side.  The result is rounded once."""
    k_cache, v_cache, k_scales, v_scales = pools
    bs, kvh = k_cache.shape[2], k_cache.shape[1]
    seqs, heads, hd = q.shape
    g = heads // kvh
    size = qh.GROUP if bits == 4 else hd
    half = torch.finfo(dtype).eps / 2
    want, bound = (torch.zeros((seqs, heads, hd), dtype=torch.float64, device=q.device) for _ in range(2))
    for i in range(seqs):
        n = int(lens[i])
        t = torch.arange(n, device=q.device)
        block, off = tables[i].long()[t // bs], t % bs
        k = qh.values(k_cache[block, :, off], k_scales[block, :, off], bits)
        v = qh.values(v_cache[block, :, off], v_scales[block, :, off], bits)
        s_v = v_scales[block, :, off].double() * (2 ** (bits - 1))
        qq = q[i].double().view(kvh, g, hd)
        s = torch.einsum("hgd,nhd->hgn", qq, k) * scale
        d = torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs()) * abs(scale) * 2.0 ** -18
        d = d + qq.abs().amax(-1, keepdim=True) * k.abs().sum(-1).T[:, None] * abs(scale) * 2.0 ** -21
        p = torch.softmax(s, -1)
        x = torch.expm1(2 * d) + 2.0 ** -19 + (n / 4 + 64) * 2.0 ** -23
        o = torch.einsum("hgn,nhd->hgd", p, v)
        few = n * 2.0 ** -25 * torch.einsum("hgn,nhc->hgnc", p, s_v).amax(2).repeat_interleave(size, -1)
        b = torch.einsum("hgn,nhd->hgd", p * (weight + x), v.abs()) + o.abs() * (p * x).sum(-1, keepdim=True) + few
        want[i] = o.reshape(heads, hd)
        bound[i] = ((b + n * 2.0 ** -131) * (1 + half)).reshape(heads, hd) + half * want[i].abs() + torch.finfo(dtype).smallest_normal * half
    return want, bound


def check(ib, q, pools, tables, lens, scale, bits, dtype, what):
    lens_t = torch.tensor(lens)
    want, bound = group_bound(q, pools, tables, lens_t, scale, bits, dtype)
    got = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, scale)
    qh.close(got, want, bound, what)
    with rows_path():
        other = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, scale)
    qh.close(other, want, bound, what + " (rows)")


def case(seed, bits, hd, heads, kvh, lens, dtype, qstd):
    g = torch.Generator().manual_seed(seed)
    blocks = sum(-(-n // 16) for n in lens) + 1
    pools = qh.random_pools(g, blocks, kvh, 16, hd, hd, bits)
    tables = qh.tables_for(g, lens, 16, blocks)
    q = (torch.randn((len(lens), heads, hd), generator=g) * qstd).to(dtype).cuda()
    return g, pools, tables, q


@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 8, 2), (128, 16, 1), (192, 4, 1), (256, 8, 2)])
@pytest.mark.parametrize("step", [6, 14, 20, 26, 40])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_groups_of_very_different_sizes(ib, hd, heads, kvh, step, dtype):  # noqa: F811
    """Each group's scales 2^step below the one before, in either order, at 4 bits; fp16 outputs only as small as fp16 holds."""
    lens = [700, 33, 1]
    for order in (1, -1):
        g, pools, tables, q = case(hd + step, 4, hd, heads, kvh, lens, dtype, 1.0)
        far = torch.arange(hd // 32, dtype=torch.float32).clamp(max=2 if step > 20 else 7)
        if dtype == FP16:
            far = far.clamp(max=max(1, 24 // step))
        factor = torch.exp2(-step * far)
        factor = factor if order == 1 else factor.flip(0)
        pools[3].copy_((pools[3].float() * factor.cuda()).to(BF16))
        check(ib, q, pools, tables, lens, 1.5 * hd ** -0.5, 4, dtype, f"step {step} order {order}")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 8, 2), (128, 16, 1), (256, 4, 1)])
@pytest.mark.parametrize("spread", [4, 20, 40])
def test_groups_whose_sizes_change_from_token_to_token(ib, bits, hd, heads, kvh, spread):  # noqa: F811
    """Every token's group has a size of its own, over 2^spread; with growing sizes and with shrinking ones."""
    lens = [900, 40]
    for how in ("mixed", "growing", "shrinking"):
        g, pools, tables, q = case(hd + spread, bits, hd, heads, kvh, lens, BF16, 1.0)
        e = torch.randint(-spread // 2, spread // 2 + 1, pools[3].shape, generator=g).float()
        if how != "mixed":  # along the table of the first sequence
            pos = torch.zeros(pools[3].shape[0])
            pos[tables[0].cpu()] = torch.arange(tables.shape[1]).float()
            e = e * 0.1 + ((pos / tables.shape[1] - 0.5) * spread * (1 if how == "growing" else -1))[:, None, None, None]
        pools[3].copy_((pools[3].float() * torch.exp2(e.round()).cuda()).to(BF16))
        check(ib, q, pools, tables, lens, 2 * hd ** -0.5, bits, BF16, f"{how} {spread}")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lead", [8, 20, 30])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_a_token_that_leads_by_far_and_has_nothing_in_some_groups(ib, hd, lead, at):  # noqa: F811
    """One token's score is `lead` above the others' and its V is zero in every second group: those groups are the others' alone,
    weighed by e^-lead."""
    lens, heads, kvh = [800, 50], 8, 2
    g, pools, tables, q = case(hd + lead, 4, hd, heads, kvh, lens, BF16, 0.02)
    pools[2].mul_(0.01)
    for i, n in enumerate(lens):
        t = {"first": 0, "middle": n // 2, "last": n - 1}[at]
        block, off = int(tables[i, t // 16]), t % 16
        # K of that token: codes of 7 throughout, scales so that q . k is the lead for a q of ones
        pools[0][block, :, off] = 0x77
        pools[2][block, :, off] = lead / (7 * hd)
        pools[3][block, :, off, ::2] = 0
    q = (1 + q.float()).to(BF16)
    check(ib, q, pools, tables, lens, 1.0, 4, BF16, f"lead {lead} {at}")


def test_the_smallest_and_largest_values_that_a_pool_holds(ib):  # noqa: F811
    """V scales of 2^-90 and 2^110 beside one another, group by group."""
    lens, hd = [300], 128
    g, pools, tables, q = case(3, 4, hd, 8, 2, lens, BF16, 1.0)
    for e in ((-90, 0, 100, -50), (100, 100, -90, -90), (110, -80, 110, 0)):
        scaled = list(pools)
        scaled[3] = (pools[3].float() * torch.exp2(torch.tensor(e).float()).cuda()).to(BF16)
        check(ib, q, scaled, tables, lens, hd ** -0.5, 4, BF16, f"{e}")
        assert math.isfinite(float(scaled[3].float().max()))


@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 8, 2), (128, 16, 1), (192, 4, 1), (256, 8, 2)])
@pytest.mark.parametrize("later", [None, 0, -30, 30])
def test_groups_that_are_zero_for_a_while(ib, hd, heads, kvh, later):  # noqa: F811
    """Groups of zeros, as padded heads have, for all tokens or up to some token, where values of 2^later times the others' size begin."""
    lens = [700, 64, 1]
    for first in (1, 17, 500):
        g, pools, tables, q = case(hd + first, 4, hd, heads, kvh, lens, BF16, 1.0)
        factor = torch.zeros(pools[3].shape)
        if later is not None:
            for i, n in enumerate(lens):
                for t in range(min(first * (i + 1), n), n):
                    factor[int(tables[i, t // 16]), :, t % 16] = 2.0 ** later
        factor[..., 0] = 1.0
        pools[3].copy_((pools[3].float() * factor.cuda()).to(BF16))
        check(ib, q, pools, tables, lens, 1.5 * hd ** -0.5, 4, BF16, f"from token {first}")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (8, 2, 128), (3, 3, 128), (6, 2, 192), (8, 2, 256), (7, 1, 128), (16, 2, 64), (16, 1, 128), (12, 1, 64), (8, 1, 256)])
def test_fp16_outputs_are_as_exact_as_32_bit_arithmetic(ib, bits, heads, kvh, hd):  # noqa: F811
    """Weights for fp16 outputs are exact to 2^-13: p' * scale with the three leading bits of p (3 + 8 bits: exact), and the rest, less than
    a quarter of it, rounded once.  Element by element where a sequence has few tokens, so that the rounding of a weight shows in full;
    over many tokens by the norm of the error: the roundings of n weights add up like independent ones, 2^-13 of sqrt(sum p_j^2 v_j^2)
    at most, which for values of either sign is the size of the outputs, whose own rounding has a norm of at least 2^-12 / sqrt(3) of that
    over 2^-11 / sqrt(3): between 1.4e-4 and 2.8e-4, 2.0e-4 for outputs of all sizes, against 2^-13 = 1.2e-4 at most: 1.17 together."""
    lens = [1, 2, 3, 4, 1, 1, 17, 2]
    for seed in range(3):
        g, pools, tables, q = case(seed, bits, hd, heads, kvh, lens, FP16, 1.0)
        want, bound = group_bound(q, pools, tables, torch.tensor(lens), hd ** -0.5, bits, FP16, 2.0 ** -13)
        got = ib.quant_paged_attention(q, *pools, tables, torch.tensor(lens).cuda(), None, hd ** -0.5)
        qh.close(got, want, bound, f"seed {seed}")
    lens = [3000, 700, 1500]
    g, pools, tables, q = case(9, bits, hd, heads, kvh, lens, FP16, 1.0)
    want, _ = group_bound(q, pools, tables, torch.tensor(lens), hd ** -0.5, bits, FP16)
    got = ib.quant_paged_attention(q, *pools, tables, torch.tensor(lens).cuda(), None, hd ** -0.5)
    err, rounding = ((x.double() - want).norm() / want.norm() for x in (got, want.to(FP16)))
    assert float(err) <= 1.2 * float(rounding), (float(err), float(rounding))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (16, 2, 64), (16, 1, 128), (8, 1, 256)])
@pytest.mark.parametrize("size", [1e4, 1e7, 1e12])
def test_fp16_outputs_over_scores_of_any_size(ib, bits, heads, kvh, hd, size):  # noqa: F811
    """Scores of up to `size`: the output is the row of the token that leads (by more than fp32 loses of the scores, 2^-17 of sum |q k|, and 40), its
    weight off by 2^-11 at most where scores pass 2^20 (one rounding), and the output's own rounding of 2^-11."""
    lens = [300, 37, 1]
    g, pools, tables, q = case(hd, bits, hd, heads, kvh, lens, FP16, 1.0)
    pools[2].mul_(1e3)
    for sign in (1.0, -1.0):
        scale = sign * size / 1e3 / hd ** 0.5
        got = ib.quant_paged_attention(q, *pools, tables, torch.tensor(lens).cuda(), None, scale)
        for i, n in enumerate(lens):
            t = torch.arange(n, device="cuda")
            block, off = tables[i][t // 16], t % 16
            k, v = (qh.values(pools[x][block, :, off], pools[x + 2][block, :, off], bits) for x in (0, 1))
            qq = q[i].double().view(kvh, heads // kvh, hd)
            s = torch.einsum("hgd,nhd->hgn", qq, k) * scale
            best = s.max(-1)
            second = s.scatter(-1, best.indices[..., None], -float("inf")).amax(-1)
            lost = torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs()).amax(-1) * abs(scale) * 2.0 ** -17
            clear = best.values - second > lost + 40
            assert int(clear.sum()) >= 4
            want = torch.stack([v[best.indices[h], h] for h in range(kvh)])
            err = (got[i].double().view(kvh, heads // kvh, hd) - want).abs()
            assert bool((err <= want.abs() * (2.0 ** -10 + 2.0 ** -20) + n * math.exp(-40) * v.abs().max() + 2.0 ** -25)[clear].all()), (sign, i)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kvh", [(16, 2), (16, 1), (6, 2)])
def test_a_head_that_is_no_number_leaves_the_others_of_its_pass(ib, bits, heads, kvh):  # noqa: F811
    """NaN and infinite q in groups of 3, 8 and 16, fp16: the columns of an instruction that other heads share with them stay right."""
    lens = [200, 1, 33]
    g, pools, tables, q = case(heads, bits, 128, heads, kvh, lens, FP16, 1.0)
    want, bound = group_bound(q, pools, tables, torch.tensor(lens), 0.09, bits, FP16)
    bad = q.clone()
    bad[0, 1, 5], bad[1, 2, 0], bad[2, heads - 1, 127] = float("nan"), float("inf"), float("nan")
    got = ib.quant_paged_attention(bad, *pools, tables, torch.tensor(lens).cuda(), None, 0.09)
    for i, h in ((0, 1), (1, 2), (2, heads - 1)):
        assert bool(got[i, h].isnan().all()), (i, h)
        got[i, h], want[i, h], bound[i, h] = 0, 0, 0
    qh.close(got, want, bound, "beside it")
