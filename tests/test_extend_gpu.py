"""GPU tests of the attention of a chunk of new tokens (`extend`) and of the windowed decode (`decode_window`) against their
definitions in 64 bits."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from chunk_reference import ROW_TOL, attention64, worst_row
from nvfp4_mla_b200.testing import SM_SCALE, SyntheticCache

pytestmark = pytest.mark.gpu


def chunk(kv_lens, q_lens, heads, ps, seed=0, ckv_scale=0.37, kpe_scale=0.021, pad=0):
    """A cache of the given lengths (unused slots hold random bytes, NaN scales among them) and queries of the chunks."""
    c = SyntheticCache([max(n, 1) for n in kv_lens], ps, 16, ckv_scale, kpe_scale, seed=seed, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    n = sum(q_lens) + pad
    c.q_nope = torch.randn(n, heads, 512, generator=g, device="cuda").bfloat16()
    c.q_pe = torch.randn(n, heads, 64, generator=g, device="cuda").bfloat16()
    c.lens, c.q_lens = list(kv_lens), list(q_lens)
    c.kv_lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    c.indptr = torch.tensor([0, *torch.tensor(q_lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    c.cache = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache)
    return c


def run(c, **kw):
    kw.setdefault("max_kv_len", max(c.lens))
    return mla.extend(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, c.indptr, SM_SCALE, c.ckv_scale, c.kpe_scale, **kw)


def reference(c, window=0, sinks=0):
    n = sum(c.q_lens)
    return attention64(c.q_nope[:n], c.q_pe[:n], c.cache, c.page_table, c.lens, c.q_lens, SM_SCALE, c.ckv_scale, c.kpe_scale, window, sinks)


def forget(c, window, sinks):
    """Page-table entries of pages that no query sees are made to point outside the cache."""
    ps = c.ckv_cache.shape[1]
    for b, (n, m) in enumerate(zip(c.lens, c.q_lens)):
        first = max(0, n - m - window + 1)
        for p in range(c.page_table.shape[1]):
            if (p * ps >= sinks and (p + 1) * ps <= first) or p * ps >= n:
                c.page_table[b, p] = -1 if p % 2 else 1 << 30


RAGGED = [
    ([1], [1], 16, 64),
    ([200], [16], 16, 64),
    ([300, 2, 129, 1], [7, 2, 129, 1], 16, 64),
    ([1000, 1, 517, 64, 2049], [1, 1, 65, 64, 33], 16, 16),
    ([256, 257, 255], [256, 1, 100], 32, 128),
    ([130, 700], [3, 40], 128, 32),
    ([90, 4000], [20, 5], 64, 1),
    ([3, 300], [5, 300], 16, 256),      # more new tokens than the cache holds: the first ones see nothing
    ([50, 0, 77], [50, 0, 0], 16, 64),  # requests without query tokens, without anything
    ([700, 3000, 90, 1500], [600, 300, 90, 1], 32, 64),  # more row tiles than CTA pairs, of unequal length
    ([20000], [4], 32, 64),             # one row tile for all CTA pairs
    ([900, 5000, 3], [30, 9, 3], 8, 64), ([300], [100], 24, 16), ([2000, 40], [70, 1], 3, 64), ([500], [260], 1, 32),
    ([400] * 70, [1, 5] * 35, 16, 64),  # many requests
]


@pytest.mark.parametrize("kv_lens,q_lens,heads,ps", RAGGED)
def test_extend_matches_the_definition(kv_lens, q_lens, heads, ps):
    c = chunk(kv_lens, q_lens, heads, ps)
    assert worst_row(run(c), reference(c)) <= ROW_TOL
    assert mla.workspace_status() == 0


WINDOWS = [(1, 0), (1, 1), (5, 3), (64, 0), (64, 64), (100, 7), (129, 130), (1000, 1), (100000, 4)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("kv_lens,q_lens,heads,ps", [RAGGED[2], RAGGED[3], RAGGED[5], RAGGED[7]])
def test_extend_with_a_window(kv_lens, q_lens, heads, ps, window, sinks):
    c = chunk(kv_lens, q_lens, heads, ps)
    want = reference(c, window, sinks)
    forget(c, window, sinks)
    assert worst_row(run(c, window=window, sink_tokens=sinks), want) <= ROW_TOL
    assert mla.workspace_status() == 0


@pytest.mark.parametrize("window,sinks", WINDOWS + [(4096, 4), (2001, 17)])
@pytest.mark.parametrize("kv_lens,heads,ps", [([1, 5, 64, 65, 300, 1027, 9000], 16, 64), ([8000] * 40 + [11] * 25, 16, 16),
                                              ([7000, 300, 2], 128, 32), ([5000] * 20, 64, 128), ([600, 3], 32, 1)])
def test_window_decode_matches_the_definition(kv_lens, heads, ps, window, sinks):
    c = chunk(kv_lens, [1] * len(kv_lens), heads, ps)
    want = reference(c, window, sinks)
    forget(c, window, sinks)
    out = mla.decode_window(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, SM_SCALE, window, sinks, c.ckv_scale, c.kpe_scale,
                            max_kv_len=max(kv_lens))
    assert worst_row(out, want) <= ROW_TOL
    assert mla.workspace_status() == 0


def test_a_window_over_everything_is_decode():
    c = chunk([1, 300, 4097], [1] * 3, 32, 64)
    out = mla.decode_window(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, SM_SCALE, 2 ** 31 - 1, 0, c.ckv_scale, c.kpe_scale)
    want = mla.decode(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, SM_SCALE, c.ckv_scale, c.kpe_scale)
    assert torch.equal(out, want)


@pytest.mark.parametrize("q_lens", [[4, 3], [130, 200]])
def test_query_tokens_of_no_request_give_zeros(q_lens):
    c = chunk([200, 300], q_lens, 16, 64, pad=37)
    out = run(c)
    n = sum(q_lens)
    assert worst_row(out[:n], reference(c)) <= ROW_TOL and (out[n:] == 0).all()
    c.indptr += 11  # and in front of the first request
    c.q_nope, c.q_pe = c.q_nope.roll(11, 0), c.q_pe.roll(11, 0)
    moved = run(c)
    assert torch.equal(moved[11:11 + n], out[:n]) and (moved[:11] == 0).all() and (moved[11 + n:] == 0).all()


@pytest.mark.parametrize("q_len", [3, 300])
def test_a_nan_scale_reaches_only_those_who_see_it(q_len):
    c = chunk([700], [q_len], 16, 64)
    want = run(c)
    token = 698  # seen by the last two query tokens
    page, slot = int(c.page_table[0, token // 64]), token % 64
    c.ckv_sf_cache.view(torch.uint8)[page, slot, 3] = 0x7F
    out = run(c)
    assert torch.equal(out[:-2], want[:-2]) and out[-2:].isnan().all()
    out = run(c, window=100, sink_tokens=2)
    assert not out[:-2].isnan().any() and out[-2:].isnan().all()


def test_a_bad_page_is_reported_and_not_read():
    c = chunk([700, 300], [200, 3], 16, 64)
    want = run(c)
    c.page_table[0, 2] = c.ckv_cache.shape[0]
    out = run(c)
    torch.cuda.synchronize()
    assert mla.workspace_status(clear=True) == 3 and mla.workspace_status() == 0
    assert torch.equal(out[200:], want[200:])


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 200, 1]])
def test_captured_and_replayed_with_other_lengths(q_lens):
    """A captured call serves other lengths and chunks below its bounds; two captured graphs and eager calls do not disturb each other."""
    c, d = chunk([900, 700, 800], q_lens, 16, 64, seed=1), chunk([100, 650, 1], [2, sum(q_lens) - 3, 1] if sum(q_lens) > 3 else [1, 1, 1], 16, 64, seed=2)
    run(c), run(d)
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for x in (c, d):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(mla.extend(x.q_nope, x.q_pe, *x.cache, x.page_table, x.kv_lens, x.indptr, SM_SCALE, x.ckv_scale, x.kpe_scale,
                                   max_kv_len=1000, window=300, sink_tokens=5))
        graphs.append(graph)
    c.lens, c.q_lens = [651, 20, 896], q_lens[::-1]
    c.kv_lens.copy_(torch.tensor(c.lens)), c.indptr.copy_(torch.tensor([0, *torch.tensor(c.q_lens).cumsum(0).tolist()]))
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert worst_row(outs[0], reference(c, 300, 5)) <= ROW_TOL
    assert worst_row(outs[1], reference(d, 300, 5)) <= ROW_TOL


@pytest.mark.parametrize("q_lens", [[1, 2], [150, 180]])
def test_on_other_streams_at_once(q_lens):
    cs = [chunk([600 + i, 900], q_lens, 16, 64, seed=i) for i in range(4)]
    torch.cuda.synchronize()
    outs = []
    for c in cs:
        with torch.cuda.stream(torch.cuda.Stream()):
            outs.append(run(c))
    torch.cuda.synchronize()
    for c, out in zip(cs, outs):
        assert worst_row(out, reference(c)) <= ROW_TOL


def test_page_table_may_be_a_slice():
    c = chunk([300, 500], [70, 3], 16, 32)
    want = run(c)
    wide = torch.full((2, c.page_table.shape[1] + 9), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + c.page_table.shape[1]] = c.page_table
    c.page_table = wide[:, 2:2 + c.page_table.shape[1]]
    assert torch.equal(run(c), want)


@pytest.mark.parametrize("scale", [-SM_SCALE, 0.0, 5.0])
@pytest.mark.parametrize("q_len", [2, 140])
def test_other_softmax_scales(scale, q_len):
    c = chunk([400], [q_len], 16, 64)
    c.q_nope *= 0.05 if scale == 5.0 else 1
    c.q_pe *= 0.05 if scale == 5.0 else 1
    out = mla.extend(c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, c.indptr, scale, c.ckv_scale, c.kpe_scale)
    want = attention64(c.q_nope, c.q_pe, c.cache, c.page_table, c.lens, c.q_lens, scale, c.ckv_scale, c.kpe_scale)
    assert worst_row(out, want) <= ROW_TOL * (4 if scale == 5.0 else 1)  # (the scores are 5 * 0.05 / 0.072 times as large)


def test_nothing_to_do():
    c = chunk([5, 6], [0, 0], 16, 64)
    assert run(c).shape == (0, 16, 512)
    c = chunk([5, 6], [2, 0], 16, 64)
    out = mla.extend(c.q_nope, c.q_pe, *c.cache, c.page_table[:, :0], c.kv_lens * 0, c.indptr, SM_SCALE)
    assert (out == 0).all()


def test_refusals():
    c = chunk([100, 200], [5, 6], 16, 64)
    ok = [c.q_nope, c.q_pe, *c.cache, c.page_table, c.kv_lens, c.indptr, SM_SCALE]

    def call(i, value, error=RuntimeError, **kw):
        args = list(ok)
        args[i] = value
        with pytest.raises(error):
            mla.extend(*args, **kw)

    call(0, c.q_nope.float()), call(0, c.q_nope[:, :, :256]), call(1, c.q_pe[:5]), call(0, c.q_nope.transpose(0, 1)), call(0, c.q_nope.cpu())
    call(5, c.page_table.long()), call(5, c.page_table[:1]), call(5, c.page_table.t().contiguous().t()), call(6, c.kv_lens[:1]), call(6, c.kv_lens.long())
    call(7, c.indptr[:2]), call(7, c.indptr.long()), call(7, c.indptr.cpu())
    call(8, SM_SCALE, ckv_scale=0.0), call(8, SM_SCALE, ValueError, window=-1), call(8, SM_SCALE, ValueError, window=5, sink_tokens=-1)
    call(8, SM_SCALE, ValueError, window=2 ** 31)
    args = [c.q_nope[:2], c.q_pe[:2], *c.cache, c.page_table, c.kv_lens, SM_SCALE]
    with pytest.raises(ValueError):
        mla.decode_window(*args, 0)
    with pytest.raises(RuntimeError):
        mla.decode_window(c.q_nope, c.q_pe, *args[2:], 5)
    with pytest.raises(RuntimeError):
        mla.decode_window(c.q_nope[:2, :8].contiguous(), c.q_pe[:2, :8].contiguous(), *args[2:], 5)


@pytest.mark.parametrize("window", [0, 500])
def test_a_loose_bound_takes_the_requests_in_groups(window):
    """The bound of the lengths sizes the workspace (1152 bytes per token and request): far above what a group of requests may take."""
    kv_lens, q_lens = [300, 2, 129, 1, 700, 40], [70, 2, 100, 1, 0, 33]
    c = chunk(kv_lens, q_lens, 24, 64, pad=5)
    table = torch.zeros(6, 100000, dtype=torch.int32, device="cuda")
    table[:, :c.page_table.shape[1]] = c.page_table
    small = run(c, window=window, sink_tokens=3)
    c.page_table = table
    out = run(c, max_kv_len=6_000_000, window=window, sink_tokens=3)
    assert worst_row(out[:-5], reference(c, window, 3)) <= ROW_TOL and (out[-5:] == 0).all()
    assert worst_row(out, small.double()) <= 2 * ROW_TOL


@pytest.mark.parametrize("kv_lens,q_lens,window,sinks", [([300, 65, 1], [90, 2, 1], 0, 0), ([1000, 70], [60, 60], 130, 70), ([64], [64], 0, 0), ([130], [2], 1, 0)])
def test_what_the_workspace_held_before_does_not_matter(kv_lens, q_lens, window, sinks):
    """The C entry with a workspace full of NaN and one just as large as asked for."""
    lib, heads, ps = mla._lib.load(), 24, 64
    c = chunk(kv_lens, q_lens, heads, ps)
    sizes = (len(kv_lens), sum(q_lens), heads, ps, c.page_table.shape[1], max(kv_lens), window, sinks)
    ws = torch.full((lib.nvfp4_mla_extend_workspace_bytes(*sizes),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((sum(q_lens), heads, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(nbytes):
        return lib.nvfp4_mla_extend(c.q_nope.data_ptr(), c.q_pe.data_ptr(), *(t.data_ptr() for t in c.cache), c.ckv_cache.shape[0], ps, c.page_table.data_ptr(),
                                    c.page_table.stride(0), c.page_table.shape[1], c.kv_lens.data_ptr(), c.indptr.data_ptr(), len(kv_lens), sum(q_lens), heads, SM_SCALE,
                                    c.ckv_scale, c.kpe_scale, max(kv_lens), window, sinks, out.data_ptr(), ws.data_ptr(), nbytes, status.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)

    assert call(ws.numel() - 1) != 0 and "workspace" in lib.nvfp4_mla_last_error().decode()
    assert call(ws.numel()) == 0
    assert worst_row(out, reference(c, window, sinks)) <= ROW_TOL and int(status) == 0


def test_more_requests_than_are_scheduled_at_once():
    """2500 requests of one and two new tokens (the schedule takes 2048 at a time)."""
    n = 2500
    kv_lens, q_lens = [1 + i % 90 for i in range(n)], [1 + i % 2 for i in range(n)]
    q_lens = [min(q, k) for q, k in zip(q_lens, kv_lens)]
    c = chunk(kv_lens, q_lens, 8, 16)
    out = run(c)
    for b in (0, 1, 2046, 2047, 2048, 2049, 2499):
        at = int(c.indptr[b])
        want = attention64(c.q_nope[at:at + q_lens[b]], c.q_pe[at:at + q_lens[b]], c.cache, c.page_table[b:b + 1], [kv_lens[b]], [q_lens[b]], SM_SCALE, c.ckv_scale, c.kpe_scale)
        assert worst_row(out[at:at + q_lens[b]], want) <= ROW_TOL
    assert not out.isnan().any() and mla.workspace_status() == 0


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (2 ** 31 - 1, 0), (30, 5000)])
@pytest.mark.parametrize("q_lens", [[2, 1, 3], [200, 1, 130]])
def test_windows_and_first_tokens_beyond_every_length(q_lens, window, sinks):
    c = chunk([700, 64, 150], q_lens, 16, 64)
    assert worst_row(run(c, window=window, sink_tokens=sinks, max_kv_len=None), reference(c, window, sinks)) <= ROW_TOL
    last = c.indptr[1:].long() - 1
    out = mla.decode_window(c.q_nope[last].contiguous(), c.q_pe[last].contiguous(), *c.cache, c.page_table, c.kv_lens, SM_SCALE, window, sinks,
                            c.ckv_scale, c.kpe_scale)
    assert worst_row(out, reference(c, window, sinks)[last]) <= ROW_TOL
    assert mla.workspace_status() == 0


@pytest.mark.parametrize("heads", [16, 64])
def test_single_tokens_of_more_requests_than_a_slice_takes(heads):
    """1100 requests of one new token, and padding behind them."""
    kv_lens = [1 + 7 * i % 2000 for i in range(1100)]
    c = chunk(kv_lens, [1] * 1100, heads, 16, pad=30)
    for kw in (dict(), dict(window=150, sink_tokens=20)):
        out = run(c, **kw)
        assert worst_row(out[:-30], reference(c, kw.get("window", 0), kw.get("sink_tokens", 0))) <= ROW_TOL and (out[-30:] == 0).all()
    assert mla.workspace_status() == 0


def test_window_decode_captured_and_replayed_beside_another_stream():
    """A graph of two windowed decodes that share its pool, replayed with other lengths and pages while the call runs on another stream."""
    c = chunk([3000, 900, 64, 1], [1] * 4, 16, 64)
    d = chunk([500] * 4, [1] * 4, 64, 64, seed=7)
    kv_lens = c.kv_lens.clone()

    def call(x, lens, window, sinks):
        return mla.decode_window(x.q_nope, x.q_pe, *x.cache, x.page_table, lens, SM_SCALE, window, sinks, x.ckv_scale, x.kpe_scale)

    call(c, kv_lens, 100, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = call(c, kv_lens, 100, 4), call(c, kv_lens, 1000, 0)
    other = torch.cuda.Stream()
    for lens in ([3000, 900, 64, 1], [17, 0, 30, 1], [2999, 101, 5, 0]):
        c.lens = lens
        kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            beside = [call(d, d.kv_lens, 200, 9) for _ in range(3)]
        torch.cuda.synchronize()
        c.q_lens = [min(n, 1) for n in lens]
        live = [i for i, n in enumerate(lens) if n]
        for out, window, sinks in ((first, 100, 4), (second, 1000, 0)):
            want = attention64(c.q_nope[live], c.q_pe[live], c.cache, c.page_table[live], [lens[i] for i in live], [1] * len(live), SM_SCALE, c.ckv_scale,
                               c.kpe_scale, window, sinks)
            assert worst_row(out[live], want) <= ROW_TOL
            assert all((out[i] == 0).all() for i, n in enumerate(lens) if not n)
        for out in beside:
            assert worst_row(out, reference(d, 200, 9)) <= ROW_TOL
    assert mla.workspace_status() == 0
