"""What the quantised paged operators refuse, and what their plain forms say about themselves: no GPU needed.

Descriptors are created on a handle made by hand, with the properties of a B200 (the library makes one only where there is a
GPU), so every refusal comes back before anything touches a device."""
import ctypes

import pytest
import torch

import quant_helpers as qh
from infinicore_b200.libinfiniop import (
    LIBINFINIOP, CTensor, InfiniDeviceEnum, InfiniDtype, infiniopHandle_t, infiniopOperatorDescriptor_t,
)

D = InfiniDtype
DTYPE, SHAPE, STRIDES, NULL, BAD, DEVICE = 10, 11, 12, 4, 3, 5


class Props(ctypes.Structure):
    """csrc/common.h, DeviceProps"""
    _fields_ = [("device_id", ctypes.c_int), ("cc_major", ctypes.c_int), ("cc_minor", ctypes.c_int), ("sm_count", ctypes.c_int),
                ("max_threads_per_block", ctypes.c_int), ("warp_size", ctypes.c_int), ("smem_per_block_optin", ctypes.c_size_t),
                ("smem_per_sm", ctypes.c_size_t), ("kernel_flags", ctypes.c_void_p)]


class Handle(ctypes.Structure):
    """{device, device_id} and a shared pointer: an address and no owner"""
    _fields_ = [("device", ctypes.c_int), ("device_id", ctypes.c_int), ("props", ctypes.POINTER(Props)), ("owner", ctypes.c_void_p)]


_PROPS = Props(0, 10, 0, 148, 1024, 32, 232448, 233472, None)


def hand_made(device):
    return ctypes.cast(ctypes.pointer(Handle(device, 0, ctypes.pointer(_PROPS), None)), infiniopHandle_t)


def make(name, tensors, *extra, handle="default"):
    """Status of infiniopCreate<name>Descriptor for [(dtype, shape, strides or None) or None, ...]."""
    made = [CTensor(*t) if t is not None else None for t in tensors]
    desc = infiniopOperatorDescriptor_t()
    h = hand_made(InfiniDeviceEnum.NVIDIA) if handle == "default" else handle
    status = getattr(LIBINFINIOP, f"infiniopCreate{name}Descriptor")(
        h, ctypes.byref(desc), *[t.descriptor if t is not None else None for t in made], *extra)
    for t in made:
        if t is not None:
            t.destroy_desc()
    return status, desc


def pools(bits=8, blocks=6, kvh=2, bs=16, kh=128, vh=128):
    w = (lambda h: h) if bits == 8 else (lambda h: h // 2)
    dt = D.I8 if bits == 8 else D.U8
    return [(dt, [blocks, kvh, bs, w(kh)]), (dt, [blocks, kvh, bs, w(vh)]),
            (D.BF16, [blocks, kvh, bs, qh.groups(bits, kh)]), (D.BF16, [blocks, kvh, bs, qh.groups(bits, vh)])]


def with_(base, at, value):
    return base[:at] + [value] + base[at + 1:]


ROWS = [(D.BF16, [5, 2, 128]), (D.BF16, [5, 2, 128]), (D.I64, [5])]


@pytest.mark.parametrize("bits", [4, 8])
def test_write_accepts_and_refuses(bits):
    def status(tensors):
        st, desc = make("QuantPagedCaching", tensors)
        if st == 0:
            assert LIBINFINIOP.infiniopDestroyQuantPagedCachingDescriptor(desc) == 0
        return st

    good = pools(bits) + ROWS
    assert status(good) == 0
    assert status(pools(bits, kh=576, vh=512) + [(D.F16, [5, 2, 576]), (D.F16, [5, 2, 512]), (D.I64, [5])]) == 0
    assert status(pools(bits) + [(D.F16, [0, 2, 128]), (D.F16, [0, 2, 128]), (D.I64, [0])]) == 0
    # strides: rows that are a slice of a fused projection, pools with tokens before heads
    assert status(pools(bits) + [(D.BF16, [5, 2, 128], [768, 128, 1]), (D.BF16, [5, 2, 128], [768, 128, 1]), (D.I64, [5])]) == 0
    for at, dt in ((4, D.F32), (4, D.F16), (5, D.F16), (6, D.I32), (2, D.F16), (3, D.F32), (0, D.BF16), (1, D.U8 if bits == 8 else D.I8)):
        assert status(with_(good, at, (dt, good[at][1]))) == DTYPE, (at, dt)
    for at, shape in ((4, [5, 3, 128]), (4, [4, 2, 128]), (4, [5, 2, 96]), (4, [10, 128]), (5, [5, 2, 64]), (6, [4]), (6, [5, 1]),
                      (0, [6, 2, 16, 80]), (0, [6, 2, 16 * 128]), (1, [6, 2, 8] + good[1][1][3:]), (2, [6, 2, 16, 3]), (2, [6, 2, 15] + good[2][1][3:]),
                      (3, [5, 2, 16] + good[3][1][3:])):
        assert status(with_(good, at, (good[at][0], shape))) == SHAPE, (at, shape)
    # head sizes: a multiple of 32, at most 1024, not 0; blocks of at least one slot
    for kh in (48, 1056, 0):
        assert status(pools(bits, kh=kh, vh=kh) + [(D.BF16, [5, 2, kh]), (D.BF16, [5, 2, kh]), (D.I64, [5])]) == SHAPE, kh
    assert status(pools(bits, bs=0) + ROWS) == SHAPE
    for at, strides in ((4, [512, 256, 2]), (5, [512, 256, 2]), (6, [2]), (0, None), (2, None)):
        dt, shape = good[at]
        if strides is None:
            strides = [shape[1] * shape[2] * shape[3] * 2, shape[2] * shape[3] * 2, shape[3] * 2, 2]
        want = 0 if at == 2 and bits == 8 else STRIDES  # a single scale has no last stride
        assert status(with_(good, at, (dt, shape, strides))) == want, (at, strides)
    for at in range(7):
        assert status(with_(good, at, None)) == NULL
    assert make("QuantPagedCaching", good, handle=None)[0] == NULL


@pytest.mark.parametrize("bits", [4, 8])
def test_read_accepts_and_refuses(bits):
    def status(tensors):
        st, desc = make("QuantPagedCacheRead", tensors)
        if st == 0:
            assert LIBINFINIOP.infiniopDestroyQuantPagedCacheReadDescriptor(desc) == 0
        return st

    for dt in (D.F16, D.BF16, D.F32):
        assert status([(dt, [5, 2, 128]), (dt, [5, 2, 128])] + pools(bits) + [(D.I64, [5])]) == 0
    good = ROWS[:2] + pools(bits) + ROWS[2:]
    assert status(with_(good, 0, (D.F64, [5, 2, 128]))) == DTYPE
    assert status(with_(good, 1, (D.F32, [5, 2, 128]))) == DTYPE
    assert status(with_(good, 6, (D.I32, [5]))) == DTYPE
    assert status(with_(good, 0, (D.BF16, [5, 2, 64]))) == SHAPE
    assert status(with_(good, 1, (D.BF16, [6, 2, 128]))) == SHAPE
    assert status(with_(good, 0, (D.BF16, [5, 2, 128], [256, 1, 2]))) == STRIDES
    for at in range(7):
        assert status(with_(good, at, None)) == NULL


def attention(bits=8, seqs=3, heads=8, hd=128, ix=D.I64, dt=D.BF16, kvh=2, **kw):
    return ([(dt, [seqs, heads, hd]), (dt, [seqs, heads, hd])] + pools(bits, kvh=kvh, kh=hd, vh=hd, **kw)
            + [(ix, [seqs, 4]), (ix, [seqs]), None])


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_accepts_and_refuses(bits):
    def status(tensors):
        st, desc = make("QuantPagedAttention", tensors, 0.1)
        if st == 0:
            size = ctypes.c_size_t(7)
            assert LIBINFINIOP.infiniopGetQuantPagedAttentionWorkspaceSize(desc, ctypes.byref(size)) == 0
            assert LIBINFINIOP.infiniopDestroyQuantPagedAttentionDescriptor(desc) == 0
        return st

    good = attention(bits)
    for hd in (64, 128, 192, 256):
        for ix in (D.I64, D.I32, D.U32):
            assert status(attention(bits, hd=hd, ix=ix, dt=D.F16)) == 0
    for hd in (32, 96, 160, 288, 576):
        assert status(attention(bits, hd=hd)) == SHAPE, hd
    assert status(good[:8] + [(D.F32, [8])]) == 0
    assert status(good[:8] + [(D.F16, [8])]) == DTYPE
    assert status(good[:8] + [(D.F32, [2])]) == SHAPE
    assert status(good[:8] + [(D.F32, [8], [2])]) == STRIDES
    assert status(attention(bits, seqs=0)) == 0
    for at, dt in ((0, D.F16), (1, D.F32), (2, D.BF16), (4, D.F32), (6, D.I32), (7, D.U32)):
        assert status(with_(good, at, (dt, good[at][1]))) == DTYPE, (at, dt)
    assert status(attention(bits, dt=D.F32)) == DTYPE
    for at, shape in ((0, [3, 8, 64]), (0, [2, 8, 128]), (1, [3, 7, 128]), (1, [24, 128]), (6, [2, 4]), (6, [12]), (7, [4]), (7, [3, 1])):
        assert status(with_(good, at, (good[at][0], shape))) == SHAPE, (at, shape)
    assert status(attention(bits, kvh=0)) == SHAPE
    assert status(attention(bits, heads=7)) == SHAPE
    for at, strides in ((0, [2048, 256, 2]), (1, [2048, 256, 2]), (6, [8, 2]), (7, [2])):
        assert status(with_(good, at, (good[at][0], good[at][1], strides))) == STRIDES, (at, strides)
    for at in range(8):
        assert status(with_(good, at, None)) == NULL


def test_calls_refuse_missing_pointers_wrong_descriptors_and_small_workspaces():
    st, write = make("QuantPagedCaching", pools() + ROWS)
    st2, read = make("QuantPagedCacheRead", ROWS[:2] + pools() + ROWS[2:])
    st3, attend = make("QuantPagedAttention", attention(), 0.1)
    assert st == st2 == st3 == 0
    p = [64] * 9  # addresses that no call gets far enough to use
    L = LIBINFINIOP
    for i in range(7):
        assert L.infiniopQuantPagedCaching(write, None, 0, *with_(p[:7], i, None), None) == NULL
        assert L.infiniopQuantPagedCacheRead(read, None, 0, *with_(p[:7], i, None), None) == NULL
    size = ctypes.c_size_t(0)
    assert L.infiniopGetQuantPagedAttentionWorkspaceSize(attend, ctypes.byref(size)) == 0
    for i in range(8):
        assert L.infiniopQuantPagedAttention(attend, 256, size.value, *with_(p, i, None), None) == NULL
    if size.value:
        assert L.infiniopQuantPagedAttention(attend, 256, size.value - 1, *p, None) == 13
        assert L.infiniopQuantPagedAttention(attend, None, size.value, *p, None) == NULL
    # one operator's descriptor handed to another
    assert L.infiniopQuantPagedCaching(read, None, 0, *p[:7], None) == BAD
    assert L.infiniopQuantPagedCacheRead(attend, None, 0, *p[:7], None) == BAD
    assert L.infiniopQuantPagedAttention(write, None, 0, *p, None) == BAD
    assert L.infiniopDestroyQuantPagedCachingDescriptor(attend) == BAD
    assert L.infiniopDestroyQuantPagedCacheReadDescriptor(write) == BAD
    assert L.infiniopDestroyQuantPagedAttentionDescriptor(read) == BAD
    for f in ("QuantPagedCaching", "QuantPagedCacheRead", "QuantPagedAttention"):
        n = 9 if f == "QuantPagedAttention" else 7
        assert getattr(L, f"infiniop{f}")(None, None, 0, *p[:n], None) == NULL
        assert getattr(L, f"infiniopGet{f}WorkspaceSize")(None, None) == NULL
        assert getattr(L, f"infiniopDestroy{f}Descriptor")(None) == NULL
    assert L.infiniopDestroyQuantPagedCachingDescriptor(write) == 0
    assert L.infiniopDestroyQuantPagedCacheReadDescriptor(read) == 0
    assert L.infiniopDestroyQuantPagedAttentionDescriptor(attend) == 0


def test_only_a_gpu_handle_is_taken():
    h = hand_made(InfiniDeviceEnum.CPU)
    assert make("QuantPagedCaching", pools() + ROWS, handle=h)[0] == DEVICE
    assert make("QuantPagedCacheRead", ROWS[:2] + pools() + ROWS[2:], handle=h)[0] == DEVICE
    assert make("QuantPagedAttention", attention(), 0.1, handle=h)[0] == DEVICE


def test_python_calls_refuse_cpu_tensors():
    import infinicore_b200 as ib

    p = qh.empty_pools(2, 1, 16, 64, 64, 8)
    rows = torch.zeros((3, 1, 64), dtype=torch.float16)
    slots = torch.arange(3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ib.quant_paged_caching(*p, rows, rows, slots)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ib.quant_paged_cache_read(*p, slots)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ib.quant_paged_attention(rows, *p, torch.zeros((3, 1), dtype=torch.int64), torch.ones(3, dtype=torch.int64))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_value_is_half_a_step_from_what_it_stands_for(bits, dtype):
    """|x - code * scale| <= scale / 2 for every element, the largest included (its scale is rounded by at most 2^-9)."""
    g = torch.Generator().manual_seed(bits)
    x = (torch.randn((200, 128), generator=g) * torch.exp(4 * torch.randn((200, 1), generator=g))).to(dtype)
    codes, scales = qh.quantise(x, bits)
    assert int(codes.abs().max()) <= qh.limits(bits)
    stored = qh.pack(codes, bits)
    assert torch.equal(qh.unpack(stored, bits), codes)
    step = scales.double().repeat_interleave(128 // scales.shape[-1], -1)
    fine = torch.isfinite(x).unflatten(-1, (scales.shape[-1], -1)).all(-1)  # some fp16 rows overflow: NaN by definition
    assert torch.equal(fine, ~torch.isnan(scales))
    held = fine.repeat_interleave(128 // scales.shape[-1], -1)
    assert bool(((x.double() - qh.values(stored, scales, bits)).abs() <= step / 2)[held].all()) and int(held.sum()) > 20000


@pytest.mark.parametrize("bits", [4, 8])
def test_the_scale_by_a_product_is_the_definition(bits):
    """The kernel's scale is bf16(fma(fma(-t, Q, A), i, t)) with t = A i, i = fp32(1 / Q): the same bf16 as A / Q for every 11-bit A."""
    q = torch.tensor(float(qh.limits(bits)))
    i = (1.0 / q.double()).float()
    a = torch.arange(1024, 2048).float()
    t = a * i
    residual = (a.double() - t.double() * q.double()).float()     # exact in 53 bits, and one rounding as an fma has
    s = (residual.double() * i.double() + t.double()).float()
    assert torch.equal(s.to(torch.bfloat16), (a / q).to(torch.bfloat16))
    assert torch.equal((a.double() / q.double()).float().to(torch.bfloat16), (a / q).to(torch.bfloat16))


@pytest.mark.parametrize("bits", [4, 8])
def test_the_rounding_by_a_reciprocal_is_the_definition(bits):
    """The kernel rounds fma(x, r, 1.5 * 2^23) with r = fp32(i (1 + 2^-21)), i = 1 / s to 1 ulp, instead of dividing.  Here the
    same arithmetic in fp32 on every bf16 scale significand and every fp16 significand below the limit gives the codes of the
    definition, exact halves included, with i rounded either way."""
    q = qh.limits(bits)
    s = (torch.arange(128, 256).double() / 128).float()                      # every bf16 significand
    x = torch.cat([torch.arange(1024, 2048).double() * 2.0 ** e for e in range(-14, 1)])   # every fp16 significand
    x = x[None].expand(128, -1)
    keep = x <= (q + 0.4) * s[:, None].double()
    exact = torch.floor(x / s[:, None].double() + 0.5)
    nearest = (1.0 / s.double()).float()
    for i in (nearest, torch.nextafter(nearest, torch.zeros(())), torch.nextafter(nearest, torch.full((), 2.0))):
        r = i * torch.tensor(1 + 2.0 ** -21)
        prod = x * r[:, None].double()          # 11 + 24 bits: exact in 53
        rounded = torch.round(prod)             # one rounding of the exact product, to the nearest integer
        assert bool((rounded == exact)[keep].all())
    halves = (2 * x / s[:, None].double()) % 2 == 1
    assert int((halves & keep).sum()) > 100     # there are exact halves among them
