"""Lengths of the quantised paged attention at the ends of their range: the arithmetic on any machine, the operator on a GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import quant_helpers as qh

ROOT = Path(__file__).resolve().parent.parent
BF16 = torch.bfloat16


def program(tmp_path, args):
    exe = tmp_path / "quant_lengths_test"
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'infinicore_b200' / 'csrc'}",
                          str(ROOT / "tests" / "cpp" / "quant_lengths_test.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    out = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout
    return [int(x) for x in out.split()]


def live_tokens(tmp_path, pairs):
    return program(tmp_path, [x for p in pairs for x in p])


BELOW = [-1, -(2 ** 31), -(2 ** 31) - 1, -(2 ** 32) + 5, -(2 ** 32), -(2 ** 40) + 64, -(2 ** 63) + 7, -(2 ** 63)]


def test_a_length_is_never_negative_and_never_beyond_the_table(tmp_path):
    pairs = [(n, most) for n in BELOW + [0] for most in (1, 64, 2 ** 31 - 64)]
    assert live_tokens(tmp_path, pairs) == [0] * len(pairs)
    pairs = [(n, most) for n in (1, 63, 64, 65, 2 ** 31 - 65, 2 ** 31, 2 ** 32 + 3, 2 ** 63 - 1) for most in (1, 64, 2 ** 31 - 64)]
    assert live_tokens(tmp_path, pairs) == [min(p) for p in pairs]


def test_a_stored_length_keeps_its_value_whatever_its_type(tmp_path):
    small = [0, 1, 5000, 2 ** 31 - 1]
    assert program(tmp_path, ["i64", *small, *BELOW, 2 ** 40]) == [*small, *BELOW, 2 ** 40]
    assert program(tmp_path, ["i32", *small, -1, -(2 ** 31)]) == [*small, -1, -(2 ** 31)]
    assert program(tmp_path, ["u32", *small, 2 ** 31, 2 ** 32 - 1]) == [*small, 2 ** 31, 2 ** 32 - 1]


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


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("path", ["auto", "rows"])
def test_unsigned_lengths_beyond_the_table_are_cut(bits, path, monkeypatch):
    """U32 lengths and tables, which torch tensors do not reach the operator with: the C calls themselves."""
    from infinicore_b200.libinfiniop import LIBINFINIOP as L
    from infinicore_b200.libinfiniop import CTensor, InfiniDeviceEnum, InfiniDtype, create_handle, destroy_handle, infiniopOperatorDescriptor_t

    monkeypatch.setenv("INFINIOP_QUANT_ATTENTION_PATH", path)
    g = torch.Generator().manual_seed(bits)
    pools = qh.random_pools(g, 9, 2, 16, 64, 64, bits)
    tables = torch.tensor([[3, 1, 8, 2], [0, 4, 5, 6], [7, 7, 7, 7], [6, 2, 1, 0]], dtype=torch.int32).cuda()
    stored = [64, 2 ** 31 + 1, 0, 2 ** 32 - 1]
    lens = torch.tensor([n - (2 ** 32 if n >= 2 ** 31 else 0) for n in stored], dtype=torch.int32).cuda()
    q = torch.randn((4, 8, 64), generator=g).to(BF16).cuda()
    out = torch.full_like(q, 5.0)
    assert L.infinirtSetDevice(InfiniDeviceEnum.NVIDIA, 0) == 0
    handle, desc = create_handle(), infiniopOperatorDescriptor_t()
    D = InfiniDtype
    kinds = [D.BF16, D.BF16] + [D.I8 if bits == 8 else D.U8] * 2 + [D.BF16, D.BF16, D.U32, D.U32]
    tensors = [out, q, *pools, tables, lens]
    made = [CTensor(kind, list(t.shape), list(t.stride())) for kind, t in zip(kinds, tensors)]
    assert L.infiniopCreateQuantPagedAttentionDescriptor(handle, ctypes.byref(desc), *[t.descriptor for t in made], None, 0.125) == 0
    size = ctypes.c_size_t(0)
    assert L.infiniopGetQuantPagedAttentionWorkspaceSize(desc, ctypes.byref(size)) == 0
    scratch = torch.empty(size.value + 256, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.infiniopQuantPagedAttention(desc, scratch.data_ptr(), size.value, *[t.data_ptr() for t in tensors], None, None) == 0
    torch.cuda.synchronize()
    want, bound = qh.attend_bound(q, pools, tables, torch.tensor([64, 64, 0, 64]), 0.125, bits, BF16, None, torch.full_like(out, 5.0))
    qh.close(out, want, bound)
    assert bool((out[2] == 5).all())
    assert L.infiniopDestroyQuantPagedAttentionDescriptor(desc) == 0
    for t in made:
        t.destroy_desc()
    destroy_handle(handle)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_a_table_that_names_more_tokens_than_an_int_holds(bits):
    """32769 pages of 65536 slots in a table whose rows are one row; sequences of a few tokens, and one into the second page."""
    import infinicore_b200 as ib

    g = torch.Generator().manual_seed(bits)
    pools = qh.random_pools(g, 2, 1, 65536, 64, 64, bits)
    row = torch.full((32769,), 1 << 20, dtype=torch.int32)  # behind the sequences' ends: never looked at
    row[:2] = torch.tensor([1, 0])
    lens = torch.tensor([5, 65541, 0, 129], dtype=torch.int32)
    q = torch.randn((4, 2, 64), generator=g).to(BF16).cuda()
    out = torch.full_like(q, 5.0)
    ib.quant_paged_attention(q, *pools, row.cuda()[None].expand(4, -1), lens.cuda(), None, 0.125, out=out)
    want, bound = qh.attend_bound(q, pools, row[:2].cuda()[None].expand(4, -1), lens, 0.125, bits, BF16, None, torch.full_like(out, 5.0))
    qh.close(out, want, bound)
    assert bool((out[2] == 5).all())
