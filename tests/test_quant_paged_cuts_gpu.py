"""Decode attention over quantised pools at long lengths, looking at two tokens at a time: at tile and page borders, at the ends of
sequences, wherever ranges are cut.  Every key is a row of signs, so that the query that is the sum of two keys scores both alike and all
others far below: a token that is lost leaves the other one's row, one that counts twice shifts the weights from 1 : 1 to 2 : 1."""
import pytest
import torch

import quant_helpers as qh
from test_quant_paged_groups_gpu import group_bound
from test_quant_paged_gpu import ib, rows_path  # noqa: F401  (a fixture, and descriptors of the kernel for any layout)

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def sign_pools(g, blocks, kvh, bs, hd, bits):
    """Keys of 1 and -1 (codes of +-7 or +-127), V as appends of normal rows leave it."""
    pools = qh.random_pools(g, blocks, kvh, bs, hd, hd, bits)
    codes = (torch.randint(0, 2, (blocks, kvh, bs, hd), generator=g) * 2 - 1).to(torch.int8) * qh.limits(bits)
    pools[0].copy_(qh.pack(codes, bits))
    pools[2].fill_(1.0 / qh.limits(bits))
    return pools


def places(g, n, bs, many):
    """Tokens to look at: ends, borders of pages and of 16, 32 and 64 tokens, and anywhere."""
    ends = [0, n - 1, n - 2, n // 2]
    steps = [s * int(torch.randint(0, n // s + 1, (1,), generator=g)) + d for s in (16, 32, 64, 128, bs) for d in (-1, 0) for _ in range(max(1, many // 16))]
    anywhere = torch.randint(0, n, (many,), generator=g).tolist()
    return [min(max(t, 0), n - 1) for t in (ends + steps + anywhere)[:many]]


CASES = [  # bits, heads, kv_heads, head, block, lengths, calls
    (4, 32, 4, 128, 16, [20011, 4096, 700, 129, 1], 6), (8, 32, 4, 128, 16, [20011, 4096, 700, 129, 1], 6),
    (4, 16, 2, 64, 16, [9000, 33, 2049, 64], 6), (8, 16, 2, 64, 32, [9000, 33, 2049, 64], 6),
    (4, 16, 2, 256, 16, [7001, 300], 4), (8, 16, 2, 192, 24, [7001, 300], 4), (4, 16, 2, 192, 8, [5003, 77], 4),
    (4, 32, 2, 128, 64, [12345, 17], 4), (8, 32, 2, 64, 16, [12345, 17], 4), (4, 16, 2, 128, 16, [131072], 4), (8, 8, 1, 128, 16, [100003], 4),
    (4, 8, 2, 128, 16, [500, 17, 256, 31, 1], 4), (8, 8, 2, 64, 16, [500, 17, 256, 31, 1], 4),
]


@pytest.mark.parametrize("case", CASES)
def test_no_token_is_lost_or_counted_twice(ib, case):  # noqa: F811
    bits, heads, kvh, hd, bs, lens, calls = case
    g = torch.Generator().manual_seed(hd + bits + lens[0])
    blocks = sum(-(-n // bs) for n in lens) + 1
    pools = sign_pools(g, blocks, kvh, bs, hd, bits)
    tables = qh.tables_for(g, lens, bs, blocks)
    lens_t = torch.tensor(lens)
    scale = 64.0 / hd
    for turn in range(calls):
        q = torch.zeros((len(lens), heads, hd))
        for i, n in enumerate(lens):
            first = places(g, n, bs, heads)
            for h in range(heads):
                for t in (first[h], int(torch.randint(0, n, (1,), generator=g))):
                    block, off = int(tables[i, t // bs]), t % bs
                    q[i, h] += torch.sign(qh.unpack(pools[0][block, h // (heads // kvh), off], bits).float()).cpu()
        q = q.to(BF16 if turn % 2 else FP16).cuda()
        want, bound = group_bound(q, pools, tables, lens_t, scale, bits, q.dtype)
        got = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, scale)
        qh.close(got, want, bound, f"call {turn}")
    if max(lens) <= 20011:
        with rows_path():
            other = ib.quant_paged_attention(q, *pools, tables, lens_t.cuda(), None, scale)
        qh.close(other, want, bound, "rows")


def test_the_bound_sees_a_lost_and_a_doubled_token(ib):  # noqa: F811
    """What the test above rests on, with the mistakes made in the reference: one token left out, or counted twice, is far outside."""
    g = torch.Generator().manual_seed(5)
    n, hd = 20011, 128
    pools = sign_pools(g, -(-n // 16), 1, 16, hd, 8)
    tables = torch.arange(-(-n // 16), device="cuda")[None]
    for t in (n - 1, 4096, 0):
        q = sum(torch.sign(pools[0][u // 16, 0, u % 16].float()) for u in (t, 777))[None, None].to(BF16)
        want, bound = group_bound(q, pools, tables, torch.tensor([n]), 0.5, 8, BF16)
        rows = [u for u in (t, 777)]
        v = [qh.values(pools[1][u // 16, 0, u % 16], pools[3][u // 16, 0, u % 16], 8) for u in rows]
        assert bool(((want[0, 0] - (v[0] + v[1]) / 2).abs() <= bound[0, 0]).all())
        for wrong in (v[1], (2 * v[0] + v[1]) / 3):
            assert float(((want[0, 0] - wrong).abs() > 4 * bound[0, 0]).float().mean()) > 0.7
