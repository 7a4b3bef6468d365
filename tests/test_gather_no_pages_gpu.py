"""GPU test of the gather with a page table without columns."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SyntheticCache

pytestmark = pytest.mark.gpu


def test_gather_with_a_page_table_without_columns():
    """Requests without tokens and rows of no request; a token that would need a page is reported and 0."""
    c = SyntheticCache([100, 50], 16, 16, 0.37, 0.021, seed=3, device="cuda")
    args = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.page_table[:, :0])
    out = torch.full((9, 512), 7.0, device="cuda"), torch.full((9, 64), 8.0, device="cuda")
    indptr = torch.zeros(3, dtype=torch.int32, device="cuda")
    mla.gather_paged_mla_kv_cache(*args, indptr, 9, dtype=torch.float32, out=out, check=True)
    assert (out[0] == 7).all() and (out[1] == 8).all()
    indptr[2] = 2
    mla.gather_paged_mla_kv_cache(*args, indptr, 9, dtype=torch.float32, out=out)
    assert (out[0][:2] == 0).all() and (out[1][:2] == 0).all() and (out[0][2:] == 7).all()
    with pytest.raises(RuntimeError, match="page table"):
        mla.gather_paged_mla_kv_cache(*args, indptr, 9, check=True)
