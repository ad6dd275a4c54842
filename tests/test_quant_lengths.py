"""Lengths of the quantised paged attention at the ends of their range: the arithmetic on any machine, the operator on a GPU."""
import subprocess
from pathlib import Path

import pytest
import torch

import quant_helpers as qh

ROOT = Path(__file__).resolve().parent.parent
BF16 = torch.bfloat16


def live_tokens(tmp_path, pairs):
    exe = tmp_path / "quant_lengths_test"
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'infinicore_b200' / 'csrc'}",
                          str(ROOT / "tests" / "cpp" / "quant_lengths_test.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    out = subprocess.run([str(exe), *[str(x) for p in pairs for x in p]], capture_output=True, text=True, check=True).stdout
    return [int(x) for x in out.split()]


BELOW = [-1, -(2 ** 31), -(2 ** 31) - 1, -(2 ** 32) + 5, -(2 ** 32), -(2 ** 40) + 64, -(2 ** 63) + 7, -(2 ** 63)]


def test_a_length_is_never_negative_and_never_beyond_the_table(tmp_path):
    pairs = [(n, most) for n in BELOW + [0] for most in (1, 64, 2 ** 31 - 64)]
    assert live_tokens(tmp_path, pairs) == [0] * len(pairs)
    pairs = [(n, most) for n in (1, 63, 64, 65, 2 ** 31 - 65, 2 ** 31, 2 ** 32 + 3, 2 ** 63 - 1) for most in (1, 64, 2 ** 31 - 64)]
    assert live_tokens(tmp_path, pairs) == [min(p) for p in pairs]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("width", [4, 64])
@pytest.mark.parametrize("path", ["auto", "rows"])
def test_negative_lengths_of_any_size_leave_their_rows(bits, width, path, monkeypatch):
    """Both kernels, with units that are cut between CTAs and with a CTA to each; the entries of an empty sequence say anything."""
    import infinicore_b200 as ib
    from infinicore_b200 import _torch_ops

    _torch_ops.clear_cache()
    monkeypatch.setenv("INFINIOP_QUANT_ATTENTION_PATH", path)
    g = torch.Generator().manual_seed(bits)
    pools = qh.random_pools(g, 9, 2, 16, 64, 64, bits)
    n = len(BELOW)
    tables = torch.zeros((n + 2, width), dtype=torch.int64)
    tables[0, :4] = tables[n + 1, :4] = torch.tensor([3, 1, 8, 2])
    lens = torch.tensor([64, *BELOW, 37])
    q = torch.randn((n + 2, 8, 64), generator=g).to(BF16).cuda()
    out = torch.full_like(q, 5.0)
    ib.quant_paged_attention(q, *pools, tables.cuda(), lens.cuda(), None, 0.125, out=out)
    ends = torch.tensor([0, n + 1])
    want, bound = qh.attend_bound(q[ends.cuda()], pools, tables[ends].cuda(), lens[ends], 0.125, bits, BF16)
    qh.close(out[ends.cuda()], want, bound)
    assert bool((out[1:n + 1] == 5).all())
    _torch_ops.clear_cache()
