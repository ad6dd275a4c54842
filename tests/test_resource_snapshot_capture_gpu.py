"""Captured collectives are not sampled, however long the capture takes: the one-second window is empty when it begins, so nothing of
before can leave it in the meantime."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

from test_resource_snapshot_gpu import COMM_CHILD

pytestmark = pytest.mark.gpu

BEGIN = COMM_CHILD[:COMM_CHILD.index("out = {")]  # the snapshot call, a communicator, x and y

CHILD = BEGIN + """
g = torch.cuda.CUDAGraph()
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    comm.all_reduce(x, y)
    side.synchronize()
    sampled = snap()["bytes"]
    time.sleep(1.3)                            # out of the window
    empty = snap()["bytes"]
    with torch.cuda.graph(g, stream=side):
        comm.all_reduce(x, y)
    captured = snap()["bytes"]
    for _ in range(3):
        g.replay()
    side.synchronize()
out = {"sampled": sampled, "empty": empty, "captured": captured, "replayed": snap()["bytes"], "ok": bool((y == 1).all())}
torch.cuda.synchronize()
del g
comm.destroy()
print(json.dumps(out))
"""


def test_a_captured_collective_adds_nothing_to_an_empty_window():
    import os

    env = dict(os.environ)
    env.pop("INFINIRT_MANAGEMENT_LIBRARY", None)
    res = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-3000:]
    r = json.loads(res.stdout.strip().splitlines()[-1])
    assert r["ok"] and r["empty"] == r["captured"] == r["replayed"] == 0
    assert r["sampled"] in (0, 64 << 20)  # nothing, if this machine took a second between the collective and the snapshot
