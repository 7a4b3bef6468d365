"""GPU tests of NaN in the log-sum-exp merge: a partial that is NaN makes its row NaN, output and log-sum-exp alike, so that no later merge takes the
row for an empty one."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SM_SCALE
from test_extend_gpu import chunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 400])  # (few rows: four thread groups share a row)
@pytest.mark.parametrize("parts", [1, 2, 40])
def test_combine_carries_nan_on(rows, parts):
    g = torch.Generator(device="cuda").manual_seed(0)
    o = torch.randn(parts, rows, 512, generator=g, device="cuda")
    lse = torch.randn(parts, rows, generator=g, device="cuda")
    want, want_lse = mla.combine(o, lse, torch.float32, return_lse=True)
    lse[:, 0] = float("nan")   # every partial NaN
    lse[parts - 1, 1] = float("nan")   # one of them
    lse[:, 2] = -torch.inf     # empty
    lse[:, 3] = -torch.inf     # empty but for a NaN
    lse[0, 3] = float("nan")
    out, out_lse = mla.combine(o, lse, torch.float32, return_lse=True)
    nan = [0, 1, 3]
    assert out[nan].isnan().all() and out_lse[nan].isnan().all()
    assert (out[2] == 0).all() and out_lse[2] == -torch.inf
    assert torch.equal(out[4:], want[4:]) and torch.equal(out_lse[4:], want_lse[4:])
    # merged once more with a partial that is not empty: NaN stays
    again, again_lse = mla.combine(torch.stack([out, o[0]]), torch.stack([out_lse, want_lse]), torch.float32, return_lse=True)
    assert again[nan].isnan().all() and again_lse[nan].isnan().all() and torch.equal(again[2], o[0, 2])


@pytest.mark.parametrize("heads,requests", [(16, 3), (128, 64)])
def test_a_windowed_row_that_is_nan_has_a_nan_lse(heads, requests):
    """A NaN block scale in the window of request 1, through the C entry."""
    lib, n, window = mla._lib.load(), 2000, 700
    c = chunk([n] * requests, [1] * requests, heads, 64)
    c.ckv_sf_cache.view(torch.uint8)[int(c.page_table[1, (n - 5) // 64]), (n - 5) % 64, 3] = 0x7F
    out = torch.zeros(requests, heads, 512, device="cuda")
    lse = torch.zeros(requests, heads, device="cuda")
    sizes = (requests, heads, 64, c.page_table.shape[1], n, window, 4)
    ws = torch.empty(lib.nvfp4_mla_decode_window_workspace_bytes(*sizes), dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.nvfp4_mla_decode_window(c.q_nope.data_ptr(), c.q_pe.data_ptr(), *(t.data_ptr() for t in c.cache), c.ckv_cache.shape[0], 64, c.page_table.data_ptr(),
                                       c.page_table.stride(0), c.page_table.shape[1], c.kv_lens.data_ptr(), requests, heads, SM_SCALE, c.ckv_scale, c.kpe_scale, n, window,
                                       4, None, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr(),
                                       torch.cuda.current_stream().cuda_stream) == 0
    assert out[1].isnan().all() and lse[1].isnan().all()
    others = [i for i in range(requests) if i != 1]
    assert not out[others].isnan().any() and lse[others].isfinite().all() and int(status) == 0
