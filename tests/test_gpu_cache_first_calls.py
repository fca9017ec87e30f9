"""GPU: what the first calls of a process prepare, in processes of their own."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import torch
sys.path.insert(0, ".")
from ops_tensor_b200 import native

dim, kind = int(sys.argv[1]), getattr(torch, sys.argv[2])
device = torch.device("cuda:0")
cache = native.PagedCache.empty(80, 2, 16, dim, device)
g = torch.Generator(device=device)
g.manual_seed(1)
def i32(x): return torch.tensor(x, dtype=torch.int32, device=device)
def call(rows, kv, **kw):
    q = torch.randn((rows, 4, dim), generator=g, device=device).to(kind)
    need = native.cache_attention_workspace(cache, q, requests=1, max_q=rows, max_kv=1200, **kw)
    args = (cache, q, i32([0, rows]), i32([kv]), torch.arange(80, dtype=torch.int32, device=device)[None, :75])
    return lambda out: native.cache_attention(*args, max_q=rows, max_kv=1200, out=out, workspace=need, **kw), torch.zeros_like(q)
k, v = (torch.randn((1200, 2, dim), generator=g, device=device).to(kind) for _ in range(2))
native.cache_store(cache, k, v, torch.arange(1200, device=device))
first, out = call(1, 900)                 # one token: the few-rows kernel's smaller form
first(out)
torch.cuda.synchronize()
for rows, kw in ((7, {}), (200, dict(sm_limit=1))):
    launch, out = call(rows, 1100, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):         # nothing that these launch has run before
        launch(out)
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    out.zero_()
    launch(out)
    assert bool((out != 0).any()) and torch.equal(got, out), rows
assert native.device_status() == 0
print("captured")
"""


@pytest.mark.parametrize("dim,kind", [(64, "float16"), (128, "bfloat16")])
def test_one_decode_step_prepares_every_capture(cuda_device, dim, kind):
    """After one call with a head size and type, calls that take its other kernels may be captured at once."""
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(dim), kind], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
