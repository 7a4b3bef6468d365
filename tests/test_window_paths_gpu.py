"""GPU tests of the ways through `decode_window`, `extend` and the gather that sizes choose: the unrounded output and the log-sum-exp of the C entry, more requests
than a decode kernel schedules by itself, pages of which whole tiles are not seen, rows that HBM has to bring; and that every form repeats itself
bit for bit."""
import math

import pytest
import torch

import nvfp4_mla_b200 as mla
from chunk_reference import ROW_TOL, rows64, worst_row
from nvfp4_mla_b200.testing import SM_SCALE, SyntheticCache
from test_extend_gpu import chunk, forget, reference, run

pytestmark = pytest.mark.gpu

# The unrounded output is off by the parts of ROW_TOL other than the rounding to BF16, and by fp32 sums. The scores are off by 2^-10 at
# most (nats); the log-sum-exp moves by no more than its largest score does.
OUT_TOL = ROW_TOL - 2.0 ** -8 + 2.0 ** -18
LSE_TOL = 2.0 ** -10 / math.log(2.0) + 2.0 ** -18


def lse64(c, window, sinks):
    """Log-sum-exp of every request's last token, log2 units."""
    out = []
    for b, n in enumerate(c.lens):
        tokens = torch.tensor([t for t in range(n) if t >= n - window or t < sinks], device="cuda")
        ckv, kpe = rows64(c.cache, c.page_table[b], tokens, c.ckv_scale, c.kpe_scale)
        out.append(torch.logsumexp((c.q_nope[b].double() @ ckv.T + c.q_pe[b].double() @ kpe.T) * SM_SCALE, -1) / math.log(2.0))
    return torch.stack(out)


def outputs(c, heads, ps, window, sinks):
    """The C entry's unrounded output and log-sum-exp (asked for these it takes the decode kernels, whatever the sizes)."""
    lib, B, n = mla._lib.load(), len(c.lens), max(c.lens)
    ws = torch.full((lib.nvfp4_mla_decode_window_workspace_bytes(B, heads, ps, c.page_table.shape[1], n, window, sinks),), 0xFF, dtype=torch.uint8, device="cuda")
    out, rounded = torch.zeros(B, heads, 512, device="cuda"), torch.zeros(B, heads, 512, device="cuda", dtype=torch.bfloat16)
    lse, status = torch.zeros(B, heads, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = lib.nvfp4_mla_decode_window(c.q_nope.data_ptr(), c.q_pe.data_ptr(), *(t.data_ptr() for t in c.cache), c.ckv_cache.shape[0], ps, c.page_table.data_ptr(),
                                     c.page_table.stride(0), c.page_table.shape[1], c.kv_lens.data_ptr(), B, heads, SM_SCALE, c.ckv_scale, c.kpe_scale, n, window, sinks,
                                     rounded.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.nvfp4_mla_last_error().decode()
    assert int(status) == 0 and torch.equal(rounded, out.bfloat16())
    return out, lse


# the last four: more requests than the decode kernels schedule by themselves (640, and 896 of the heads-as-M kernel); pages of 256 and more tokens
PATHS = [([1, 5, 64, 65, 300, 1027, 9000], 16, 64, 100, 7), ([3000, 40], 128, 64, 2001, 17), ([2500] * 40, 64, 32, 1500, 4),
         ([1 + 3 * i % 301 for i in range(700)], 16, 16, 100, 3), ([1 + 3 * i % 301 for i in range(1000)], 64, 16, 150, 3),
         ([9000, 20, 1024, 5000], 16, 1024, 16, 3), ([5000 + 7 * i for i in range(64)], 128, 256, 16, 3)]


@pytest.mark.parametrize("kv_lens,heads,ps,window,sinks", PATHS)
def test_window_outputs_of_the_c_entry(kv_lens, heads, ps, window, sinks):
    c = chunk(kv_lens, [1] * len(kv_lens), heads, ps)
    want, want_lse = reference(c, window, sinks), lse64(c, window, sinks)
    forget(c, window, sinks)
    out, lse = outputs(c, heads, ps, window, sinks)
    assert worst_row(out, want) <= OUT_TOL
    assert float((lse - want_lse).abs().max()) <= LSE_TOL


@pytest.mark.parametrize("kv_lens,heads,ps,window,sinks", PATHS[3:])
def test_window_decode_on_these_paths(kv_lens, heads, ps, window, sinks):
    c = chunk(kv_lens, [1] * len(kv_lens), heads, ps)
    want = reference(c, window, sinks)
    forget(c, window, sinks)
    out = mla.decode_window(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, SM_SCALE, window, sinks, c.ckv_scale, c.kpe_scale, max_kv_len=max(kv_lens))
    assert worst_row(out, want) <= ROW_TOL
    assert mla.workspace_status() == 0


@pytest.mark.parametrize("kv_lens,q_lens,heads,window,sinks", [([700, 3000], [3, 2], 16, 0, 0), ([700, 3000, 90, 1500], [600, 300, 90, 1], 32, 0, 0), ([9000] * 3, [130] * 3, 16, 300, 5),
                                                               ([4000] * 32, [1] * 32, 128, 2000, 4), ([20000], [4], 32, 0, 0)])
def test_calls_repeat_themselves(kv_lens, q_lens, heads, window, sinks):
    c = chunk(kv_lens, q_lens, heads, 64)
    want = run(c, window=window, sink_tokens=sinks)
    for i in range(3):
        junk = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 20, 1 << 24, 3 << 22)]  # (what the next call's workspace holds)
        del junk
        assert torch.equal(run(c, window=window, sink_tokens=sinks), want)


def poison(c, tokens):
    """NaN block scales and a NaN rope element at these tokens of every request."""
    ps = c.ckv_cache.shape[1]
    for b in range(len(c.lens)):
        for t in tokens:
            at = int(c.page_table[b, t // ps]), t % ps
            c.ckv_sf_cache.view(torch.uint8)[at] = 0x7F
            c.kpe_cache.view(torch.uint8)[at][5] = 0x7F


@pytest.mark.parametrize("heads,requests", [(16, 2), (64, 40), (128, 64)])
@pytest.mark.parametrize("window,sinks", [(100, 2), (130, 70)])
def test_nan_between_the_first_tokens_and_the_window(heads, requests, window, sinks):
    """Tokens that are not seen, in pages of which other tokens are, may hold anything."""
    c = chunk([700] * requests, [1] * requests, heads, 64)
    out, lse = outputs(c, heads, 64, window, sinks)
    plain = run(c, window=window, sink_tokens=sinks)
    poison(c, [sinks, sinks + 20, 700 - window - 20, 700 - window - 1])
    got, got_lse = outputs(c, heads, 64, window, sinks)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    assert torch.equal(run(c, window=window, sink_tokens=sinks), plain)


@pytest.mark.parametrize("heads,m", [(16, 4), (16, 300), (24, 250)])
def test_a_nan_token_reaches_the_rows_whose_window_holds_it(heads, m):
    window, sinks, n = 100, 3, 700
    c = chunk([n], [m], heads, 64)
    clean = run(c, window=window, sink_tokens=sinks)
    for token in (5, n - m - window + 1, n - 2, n - m // 2):
        d = chunk([n], [m], heads, 64)
        poison(d, [token])
        out = run(d, window=window, sink_tokens=sinks)
        hit = torch.tensor([p - window < token <= p for p in range(n - m, n)], device="cuda")
        assert out[hit].isnan().all() and worst_row(out[~hit], clean[~hit].double()) <= 2 * ROW_TOL


def test_gather_of_many_rows_to_fp32():
    lens = [40000, 90000, 1, 70003]
    c = SyntheticCache(lens, 64, 16, 0.37, 0.021, seed=3, device="cuda")
    indptr = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    got = mla.gather_paged_mla_kv_cache(c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.page_table, indptr, sum(lens), None, c.ckv_scale, c.kpe_scale, torch.float32, check=True)
    whole = mla.dequantize(c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.ckv_scale, c.kpe_scale, torch.float32)
    at = torch.cat([c.page_table[b].long()[torch.arange(n, device="cuda") // 64] * 64 + torch.arange(n, device="cuda") % 64 for b, n in enumerate(lens)])
    for x, y in zip(got, whole):
        assert torch.equal(x, y.flatten(0, 1)[at])
