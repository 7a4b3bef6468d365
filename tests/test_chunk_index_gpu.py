"""GPU tests of query indexes that `extend` does not allow (they run backwards, or past the query tokens): the call reports it and gives zeros, whatever its
output held before."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SM_SCALE
from test_extend_gpu import chunk

pytestmark = pytest.mark.gpu


def call(c, indptr, kv_lens, page_table, total, heads, ps, max_kv_len, window):
    lib, batch = mla._lib.load(), len(indptr) - 1
    assert lib.nvfp4_mla_extend_shares(batch, total, heads, max_kv_len, window, 0) == 1
    indptr, kv_lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (indptr, kv_lens))
    ws = torch.full((lib.nvfp4_mla_extend_workspace_bytes(batch, total, heads, ps, page_table.shape[1], max_kv_len, window, 0),), 0x7E, dtype=torch.uint8, device="cuda")
    out = torch.full((total, heads, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.nvfp4_mla_extend(c.q_nope.data_ptr(), c.q_pe.data_ptr(), *(t.data_ptr() for t in c.cache), c.ckv_cache.shape[0], ps, page_table.data_ptr(),
                                page_table.stride(0), page_table.shape[1], kv_lens.data_ptr(), indptr.data_ptr(), batch, total, heads, SM_SCALE, c.ckv_scale, c.kpe_scale,
                                max_kv_len, window, 0, out.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    return out, int(status)


@pytest.mark.parametrize("indptr,window", [([0, 200, 0, 200, 0, 200], 0), ([7, 200000], 64), ([0, 150, 3, 200, 20, 180], 0)])
def test_more_query_tokens_than_there_are(indptr, window):
    c = chunk([5000], [200], 16, 64)
    batch = len(indptr) - 1
    out, status = call(c, indptr, [5000] * batch, c.page_table.expand(batch, -1), 200, 16, 64, 5000, window)
    assert status == 2 and (out == 0).all()


def test_counts_that_pass_32_bits():
    """128 requests that each claim 2^25 - 2 blocks of the cache: their sum is -256 in 32 bits, below any room there is."""
    c = chunk([3000], [200], 24, 1024)
    table = torch.zeros(1, 1 << 21, dtype=torch.int32, device="cuda").expand(256, -1)
    out, status = call(c, [199, 2 ** 31 - 1] * 128 + [199], [2 ** 31 - 64] * 256, table, 200, 24, 1024, 2 ** 31 - 1, 64)
    assert status == 2 and (out == 0).all()
