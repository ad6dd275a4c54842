"""Which kernel the quantised paged attention plans for tables of any width: no GPU needed."""
import ctypes

import pytest

from infinicore_b200.libinfiniop import LIBINFINIOP, InfiniDtype
from test_quant_lengths import live_tokens
from test_quant_paged_cpu import attention, make, with_

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
