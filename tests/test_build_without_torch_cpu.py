"""The libraries and the module over the C++ layer are built where torch is not installed: only the operators on its tensors are left out."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

CHILD = """
import sys
sys.modules["torch"] = None  # an import of it raises ImportError
sys.path.insert(0, %r)
from infinicore_b200 import build
paths = build.build()
print(sorted(paths))
build.main()
""" % str(ROOT)


def test_what_needs_no_torch_is_built_without_it():
    from infinicore_b200.build import build

    assert {"infinirt", "infiniop", "infiniccl", "pybind", "torch_ops"} == set(build())
    res = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    assert res.stdout.splitlines()[0] == "['infiniccl', 'infiniop', 'infinirt', 'pybind']"
    assert "torch" in res.stderr and "quant_paged" in res.stderr
