"""GPU tests of where `extend` and `decode_window` report: from a graph that was captured before any of their calls, and through the C entries without
a status word."""
import subprocess
import sys

import pytest
import torch

import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SM_SCALE
from test_extend_gpu import chunk

pytestmark = pytest.mark.gpu

CAPTURED = """
import torch
import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SM_SCALE, SyntheticCache

c = SyntheticCache([700, 300], 64, 16, 0.37, 0.021, seed=0, device="cuda")
cache = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache)
n = {n}
q, qp = torch.zeros(n, 16, 512, device="cuda").bfloat16(), torch.zeros(n, 16, 64, device="cuda").bfloat16()
indptr = torch.tensor([0, n - 1, n], dtype=torch.int32, device="cuda")
mla.decode(q[:2], qp[:2], *cache, c.page_table, c.kv_lens, SM_SCALE, max_kv_len=700)  # (the device's set-up)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    if n == 2:
        mla.decode_window(q, qp, *cache, c.page_table, c.kv_lens, SM_SCALE, 650)
    else:
        mla.extend(q, qp, *cache, c.page_table, c.kv_lens, indptr, SM_SCALE, max_kv_len=700)
graph.replay()
assert mla.workspace_status() == 0
good = c.page_table.clone()
c.page_table[0, 2] = c.ckv_cache.shape[0]
graph.replay()
assert mla.workspace_status() == 3 and mla.workspace_status(clear=True) == 3 and mla.workspace_status() == 0
c.page_table.copy_(good)
graph.replay()
assert mla.workspace_status("cuda:0") == 0
print("fine")
"""


@pytest.mark.parametrize("n", [2, 3, 300])  # windowed decode; a chunk by token; a chunk whose rows share a pass
def test_a_graph_captured_before_any_call_reports(n):
    run = subprocess.run([sys.executable, "-c", CAPTURED.format(n=n)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("q_len", [3, 300])
def test_without_a_status_word_the_workspace_receives_the_codes(q_len):
    lib = mla._lib.load()
    c = chunk([700], [q_len], 16, 64)
    ws = torch.zeros(lib.nvfp4_mla_extend_workspace_bytes(1, q_len, 16, 64, c.page_table.shape[1], 700, 0, 0), dtype=torch.uint8, device="cuda")
    out = torch.empty(q_len, 16, 512, dtype=torch.bfloat16, device="cuda")

    def status():
        assert lib.nvfp4_mla_extend(c.q_nope.data_ptr(), c.q_pe.data_ptr(), *(t.data_ptr() for t in c.cache), c.ckv_cache.shape[0], 64, c.page_table.data_ptr(),
                                    c.page_table.stride(0), c.page_table.shape[1], c.kv_lens.data_ptr(), c.indptr.data_ptr(), 1, q_len, 16, SM_SCALE, c.ckv_scale,
                                    c.kpe_scale, 700, 0, 0, out.data_ptr(), ws.data_ptr(), ws.numel(), None, torch.cuda.current_stream().cuda_stream) == 0
        return lib.nvfp4_mla_workspace_status(ws.data_ptr(), torch.cuda.current_stream().cuda_stream)

    assert status() == 0
    c.page_table[0, 2] = c.ckv_cache.shape[0]
    assert status() == 3
