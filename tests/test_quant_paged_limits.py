"""Limits of the quantised operators' plans and calls: tables of any width, pools without a block."""
import ctypes

import pytest
import torch

from infinicore_b200.libinfiniop import LIBINFINIOP, InfiniDtype
from test_quant_lengths import live_tokens
from test_quant_paged_cpu import ROWS, attention, make, pools, with_

D = InfiniDtype


def workspace(bits, hd, block, max_blocks, seqs=3):
    """0 where the plan is the kernel for any layout (it needs none)."""
    tensors = with_(attention(bits, hd=hd, bs=block, seqs=seqs, ix=D.I32), 6, (D.I32, [seqs, max_blocks]))
    st, desc = make("QuantPagedAttention", tensors, 0.1)
    assert st == 0
    size = ctypes.c_size_t(7)
    assert LIBINFINIOP.infiniopGetQuantPagedAttentionWorkspaceSize(desc, ctypes.byref(size)) == 0
    assert LIBINFINIOP.infiniopDestroyQuantPagedAttentionDescriptor(desc) == 0
    return size.value


@pytest.mark.parametrize("bits,hd", [(4, 64), (4, 128), (4, 256), (8, 64), (8, 128), (8, 256)])
@pytest.mark.parametrize("block", [8, 16, 65536])
def test_tables_whose_tokens_do_not_fit_an_int_go_to_the_kernel_that_counts_in_64_bits(bits, hd, block):
    """The tiles kernel counts tokens and tiles in 32 bits, a whole tile behind the last token included."""
    assert workspace(bits, hd, block, (2 ** 31 - 65536) // block) > 0
    for tokens in (2 ** 31, 2 ** 31 + 65536, 2 ** 32, 2 ** 34):
        if tokens // block <= 2 ** 31 - 1:
            assert workspace(bits, hd, block, tokens // block) == 0, tokens


def test_lengths_beyond_an_int_are_kept(tmp_path):
    pairs = [(2 ** 31, 2 ** 32), (2 ** 33 + 5, 2 ** 33), (2 ** 40, 2 ** 40), (2 ** 62, 2 ** 47)]
    assert live_tokens(tmp_path, pairs) == [min(p) for p in pairs]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("checked", ["0", "1"])
def test_no_kernel_looks_into_a_pool_without_blocks(bits, checked, monkeypatch):
    """No sequence can have a token there: the call succeeds before any launch (which would fail here, or read a block that is
    not there); its pools' addresses may be null."""
    monkeypatch.setenv("INFINIOP_PAGED_CHECK_INDICES", checked)
    for block in (16, 3):
        st, desc = make("QuantPagedAttention", attention(bits, blocks=0, bs=block), 0.1)
        assert st == 0
        for p in (64, None):
            assert LIBINFINIOP.infiniopQuantPagedAttention(desc, 256, 1 << 40, 64, 64, p, p, p, p, 64, 64, None, None) == 0
        assert LIBINFINIOP.infiniopQuantPagedAttention(desc, 256, 1 << 40, None, 64, 64, 64, 64, 64, 64, 64, None, None) == 4
        assert LIBINFINIOP.infiniopDestroyQuantPagedAttentionDescriptor(desc) == 0
    # rows and slots are still asked for
    st, write = make("QuantPagedCaching", pools(bits, blocks=0) + ROWS)
    assert st == 0
    assert LIBINFINIOP.infiniopQuantPagedCaching(write, None, 0, None, None, None, None, None, 64, 64, None) == 4
    assert LIBINFINIOP.infiniopDestroyQuantPagedCachingDescriptor(write) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_a_pool_without_blocks_on_a_gpu(bits):
    """Padding is skipped, reads are zeros, attention leaves every row; a slot or length all the same touches nothing."""
    import infinicore_b200 as ib
    import quant_helpers as qh

    empty = qh.empty_pools(0, 2, 16, 64, 64, bits, "cuda")
    x = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    padding = torch.full((3,), -1, dtype=torch.int64, device="cuda")
    ib.kernel_status()
    ib.quant_paged_caching(*empty, x, x, padding)
    k, v = ib.quant_paged_cache_read(*empty, padding, torch.float32)
    assert k.shape == (3, 2, 64) and bool((k == 0).all()) and bool((v == 0).all())
    assert ib.kernel_status() == 0
    out = torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros((3, 4), dtype=torch.int64, device="cuda")
    ib.quant_paged_attention(out.clone(), *empty, tables, torch.tensor([0, -1, 5], device="cuda"), None, 0.1, out=out)
    assert bool((out == 7).all()) and ib.kernel_status() == 0
    bad = torch.tensor([0, -1, 1 << 40], device="cuda")
    ib.quant_paged_caching(*empty, x, x, bad)
    assert ib.kernel_status() == 4
    k, v = ib.quant_paged_cache_read(*empty, bad, torch.float32)
    assert ib.kernel_status() == 4 and bool((k == 0).all()) and bool((v == 0).all())
