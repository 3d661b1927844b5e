"""The cases of perf/operators.py, without a GPU."""
import subprocess
import sys

from conftest import ROOT

# In a process of its own: torch brings its own HIP runtime.
STREAMS = """
import importlib, sys, types
sys.path.insert(0, {root!r})
import numpy as np
import torch
from perf import operators as ops

current, seen = [0], []
torch.cuda.current_device = lambda: 0
torch.cuda.current_stream = lambda *a: types.SimpleNamespace(cuda_stream=current[0])
torch._C._cuda_getCurrentRawStream = lambda device: current[0]
kept = torch.empty
torch.empty = lambda *a, **k: kept(*a, **dict(k, device="cpu"))

def call(name):
    def f(*args):
        seen.append((name, args[-1].value or 0, args[-3].value if name == "lg_hip_sample" else None))
        return 0
    return f

class Lib:
    lg_hip_paged_write, lg_hip_sample = call("lg_hip_paged_write"), call("lg_hip_sample")
    lg_hip_sample_workspace = staticmethod(lambda rows, vocab: 4096)

real = importlib.import_module("little-gemma_amd").hiplib
ops._own = lambda: types.SimpleNamespace(load_hip=lambda: Lib, Pages=real.Pages, hip_check=real.hip_check)
ops.own = True
ops._i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32))

def state(case):
    s = ops._State()
    s.case, s.call, s.calls, s.device = case, None, {{}}, 0
    return s

w = state(dict(kind="write", n_tok=3, kv=2, hd=64, page=16, fused=0))
w.x = torch.zeros(3, 256); w.k, w.v = w.x[:, :128], w.x[:, 128:]
w.n_pages, w.slots = 2, ops._i32([0, 1, 2])
w.kpool, w.vpool = (torch.zeros(2, 16, 128, dtype=torch.float16) for _ in range(2))
s = state(dict(kind="sample", rows=2, vocab=9000, mode="chat"))
s.logits, s.u, s.prob = torch.zeros(2, 9000), torch.zeros(2), torch.zeros(2)
s.params, s.tok, s.kept = torch.zeros(2, 16, dtype=torch.uint8), ops._i32([0, 0]), ops._i32([0, 0])
order = [0, 4096, 4096, 0, 8192, 4096]
for x in order:
    current[0] = x
    ops.run(w); ops.run(s)
assert [x[1] for x in seen if x[0] == "lg_hip_paged_write"] == order, seen
drawn = [x for x in seen if x[0] == "lg_hip_sample"]
assert [x[1] for x in drawn] == order, seen
memory = {{}}
for _, stream, work in drawn:
    memory.setdefault(stream, set()).add(work)
assert all(len(x) == 1 for x in memory.values()) and len(set.union(*memory.values())) == 3, memory
print("ok")
"""


def test_a_case_runs_on_the_stream_that_is_current_at_each_pass():
    """The framework's calls of a state go to the current stream, as the plain forms do, whichever it was at the first pass, each stream's with working memory of its own
    (calls on two streams can overlap)."""
    r = subprocess.run([sys.executable, "-c", STREAMS.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
