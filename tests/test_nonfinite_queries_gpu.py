"""GPU tests of query rows that are not finite, in every form of `extend` and `decode_window`: such a row is NaN where it sees a token and 0
where it sees none, and no other row changes."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from chunk_reference import ROW_TOL, worst_row
from nvfp4_mla_b200.testing import SM_SCALE
from test_extend_gpu import chunk, run

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
# heads, tokens, query tokens of one request; whether its rows share a pass, whether 16-bit heads-as-M rows are taken by token
FORMS = [(16, 700, 3, 0, 0), (128, 160000, 1, 0, 1), (16, 700, 300, 1, 0), (24, 300, 5, 1, 0)]


@pytest.mark.parametrize("heads,n,m,shares,many", FORMS)
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("part,channel", [("q_nope", 0), ("q_nope", 511), ("q_pe", 7)])
def test_a_row_that_is_not_finite_is_nan(heads, n, m, shares, many, value, part, channel):
    lib = mla._lib.load()
    assert lib.nvfp4_mla_extend_shares(1, m, heads, n, 0, 0) == shares
    if not shares:
        assert lib.nvfp4_mla_decode_multi_folds(m, 2, heads // 2 // 16 * 16, n, 0) == many  # (the same estimate, for as many rows)
    c = chunk([n], [m], heads, 64)
    clean = run(c)
    row = torch.zeros(m, heads, dtype=torch.bool, device="cuda")
    row[m // 2, heads // 3] = row[m - 1, heads - 1] = True
    getattr(c, part)[row, channel] = value
    out = run(c)
    assert out[row].isnan().all()
    assert worst_row(out[~row][:, None], clean[~row][:, None].double()) <= 2 * ROW_TOL  # (each within ROW_TOL of the definition)
    assert mla.workspace_status() == 0


@pytest.mark.parametrize("heads,requests,n,window", [(16, 3, 900, 100), (128, 32, 3000, 2001), (128, 2, 160000, 150000)])
def test_windowed_rows_that_are_not_finite(heads, requests, n, window):
    c = chunk([n] * requests, [1] * requests, heads, 64)

    def call():
        return mla.decode_window(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, SM_SCALE, window, 4, c.ckv_scale, c.kpe_scale, max_kv_len=n)

    clean = call()
    row = torch.zeros(requests, heads, dtype=torch.bool, device="cuda")
    row[0, 5] = row[requests - 1, heads - 1] = row[1, 0] = True
    c.q_nope[0, 5, 100], c.q_nope[requests - 1, heads - 1, 300], c.q_pe[1, 0, 63] = INF, NAN, -INF
    out = call()
    assert out[row].isnan().all()
    assert worst_row(out[~row][:, None], clean[~row][:, None].double()) <= 2 * ROW_TOL


@pytest.mark.parametrize("kv_lens,q_lens", [([3], [5]), ([3, 300], [5, 300])])
def test_a_row_that_is_not_finite_and_sees_nothing_is_zero(kv_lens, q_lens):
    c = chunk(kv_lens, q_lens, 16, 64)
    clean = run(c)
    c.q_nope[0], c.q_pe[1, 3, 2] = NAN, INF  # the first two query tokens are in front of the request's first token
    c.q_nope[2, 1, 7] = INF                  # the third sees one token
    out = run(c)
    assert (out[:2] == 0).all() and out[2, 1].isnan().all()
    assert worst_row(out[3:], clean[3:].double()) <= 2 * ROW_TOL
