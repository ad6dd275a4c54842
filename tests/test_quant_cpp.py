"""The C++ wrappers of the operators over quantised pools (include/infinicore_b200/ops.hpp): they compile without a warning on any
machine, and on a GPU their results are the plain forms'."""
import subprocess
from pathlib import Path

import pytest
import torch

import quant_helpers as qh

ROOT = Path(__file__).resolve().parent.parent
LIBDIR = ROOT / "infinicore_b200" / "lib"


def build_program(out_dir):
    from infinicore_b200.build import build

    build()
    exe = out_dir / "quant_ops_test"
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'include'}",
                          str(ROOT / "tests" / "cpp" / "quant_ops_test.cpp"), "-o", str(exe), f"-L{LIBDIR}", "-linfiniop", "-linfinirt",
                          f"-Wl,-rpath,{LIBDIR}"], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    return exe


def test_program_compiles_and_says_its_usage(tmp_path):
    res = subprocess.run([str(build_program(tmp_path))], capture_output=True, text=True)
    assert res.returncode == 2 and "usage" in res.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_wrappers_against_the_plain_forms(tmp_path, bits):
    exe = build_program(tmp_path)
    g = torch.Generator().manual_seed(bits)
    kvh, heads, hd, bs = 2, 8, 128, 16
    lens = [100, 17, 700]
    pages = [-(-n // bs) for n in lens]
    blocks = sum(pages)
    tables = qh.tables_for(g, lens, bs, blocks, device="cpu")
    slots = torch.cat([tables[i, torch.arange(n) // bs] * bs + torch.arange(n) % bs for i, n in enumerate(lens)])
    k, v = (torch.randn((slots.numel(), kvh, hd), generator=g).to(torch.bfloat16) for _ in "kv")
    q = torch.randn((3, heads, hd), generator=g).to(torch.bfloat16)
    for name, t in (("k", k), ("v", v), ("q", q), ("slots", slots), ("tables", tables), ("lens", torch.tensor(lens))):
        raw = t.contiguous().view(torch.int16) if t.dtype == torch.bfloat16 else t.contiguous()
        (tmp_path / f"{name}.bin").write_bytes(raw.numpy().tobytes())
    args = [bits, slots.numel(), kvh, hd, blocks, bs, 3, heads, tables.shape[1]]
    res = subprocess.run([str(exe), str(tmp_path), *map(str, args)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    pools = qh.empty_pools(blocks, kvh, bs, hd, hd, bits)
    qh.write(pools, k, v, slots, bits)
    for name, want in zip(("k_back", "v_back"), qh.read(pools, slots, bits)):
        got = torch.frombuffer(bytearray((tmp_path / f"{name}.out.bin").read_bytes()), dtype=torch.float32).view(want.shape)
        assert torch.equal(got, want.float())
    out = torch.frombuffer(bytearray((tmp_path / "out.out.bin").read_bytes()), dtype=torch.bfloat16).view(3, heads, hd)
    want, bound = qh.attend_bound(q, pools, tables, torch.tensor(lens), 0.1, bits, torch.bfloat16)
    qh.close(out, want, bound)
