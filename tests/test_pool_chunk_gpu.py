"""The pool's prefill path, run as a serving engine runs it: projected rows appended chunk by chunk, each chunk's attention, windowed and plain
decode steps, rows read back; against the definitions in 64 bits over the pool's own rows."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from chunk_reference import ROW_TOL, attention64, rows64, worst_row
from nvfp4_mla_b200 import serving
from nvfp4_mla_b200.testing import SM_SCALE
from test_cache_io_gpu import normed

pytestmark = pytest.mark.gpu


def angles(n):
    a = torch.arange(n, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, device="cuda").double() / 64)
    return torch.cat([a.cos(), a.sin()], 1).float()


def queries(g, n, heads):
    return (torch.randn(n, heads, 512, generator=g, device="cuda").bfloat16(), torch.randn(n, heads, 64, generator=g, device="cuda").bfloat16())


@pytest.mark.parametrize("heads,page_size,window,sinks", [(16, 64, 0, 0), (128, 16, 0, 0), (16, 64, 150, 4), (32, 1, 70, 100)])
def test_prefill_in_chunks_then_decode(heads, page_size, window, sinks):
    g = torch.Generator(device="cuda").manual_seed(heads)
    pool = serving.PagedLatentCache(2000 if page_size == 1 else 200, page_size, 4, -(-800 // page_size), 0.0031, 0.017)
    weight, cos_sin = (1 + 0.1 * torch.randn(512, generator=g, device="cuda")).bfloat16(), angles(800)
    held = {r: [torch.zeros(0, 576, device="cuda")] for r in range(4)}
    for step in [[(0, 300), (2, 17)], [(2, 200), (0, 1), (3, 64)], [(1, 1)], [(0, 129), (1, 7), (2, 1), (3, 0)]]:
        n = sum(c for _, c in step)
        kv_a = torch.randn(n, 576, generator=g, device="cuda").bfloat16()
        pool.append_projected(step, kv_a, weight, cos_sin)
        q_nope, q_pe = queries(g, n, heads)
        out = pool.extend(step, q_nope, q_pe, SM_SCALE, window=window, sink_tokens=sinks)
        at = 0
        for r, c in step:
            held[r].append(kv_a[at:at + c])
            at += c
        live = [(r, c) for r, c in step if c]
        want = attention64(q_nope, q_pe, (pool.ckv_cache, pool.ckv_sf_cache, pool.kpe_cache), pool.page_table[[r for r, _ in live]], [pool._lens[r] for r, _ in live],
                           [c for _, c in live], SM_SCALE, pool.ckv_scale, pool.kpe_scale, window, sinks)
        assert worst_row(out, want) <= ROW_TOL
    # the pool holds what the plain writer makes of the normalised rows, request by request
    plain = serving.PagedLatentCache(2000 if page_size == 1 else 200, page_size, 4, -(-800 // page_size), 0.0031, 0.017)
    for r in range(4):
        kv_a = torch.cat(held[r]).bfloat16()
        plain.append([(r, len(kv_a))], *normed(kv_a, weight, cos_sin, torch.arange(len(kv_a), device="cuda"), 1e-6, True))
    everything = [(r, 0, pool._lens[r]) for r in range(4)]
    for x, y in zip(pool.gather(everything, torch.float32), plain.gather(everything, torch.float32)):
        assert torch.equal(x, y)
    # a range of rows
    ckv, kpe = pool.gather([(2, 5, 100), (-1, 0, 3), (2, 0, 0)])
    for got, want in ((ckv[:100], 0), (kpe[:100], 1)):
        row = rows64((pool.ckv_cache, pool.ckv_sf_cache, pool.kpe_cache), pool.page_table[2], torch.arange(5, 105, device="cuda"), pool.ckv_scale, pool.kpe_scale)[want]
        assert ((got.double() - row).abs() <= row.abs() * (2.0 ** -8 + 2.0 ** -22)).all()  # one rounding to BF16 behind two to fp32
    # decode steps
    for ids in ([0, 1, 2, 3], [2]):
        q_nope, q_pe = queries(g, len(ids), heads)
        out = pool.decode(ids, q_nope, q_pe, SM_SCALE, window=window, sink_tokens=sinks)
        want = attention64(q_nope, q_pe, (pool.ckv_cache, pool.ckv_sf_cache, pool.kpe_cache), pool.page_table[ids], [pool._lens[r] for r in ids], [1] * len(ids), SM_SCALE,
                           pool.ckv_scale, pool.kpe_scale, window, sinks)
        assert worst_row(out, want) <= ROW_TOL
    w_uv = torch.randn(heads, 512, 24, generator=g, device="cuda").bfloat16()
    n = 129 + 7
    q_nope, q_pe = queries(g, n, heads)
    latent = pool.extend([(0, 129), (1, 7)], q_nope, q_pe, SM_SCALE)
    assert torch.equal(pool.extend([(0, 129), (1, 7)], q_nope, q_pe, SM_SCALE, w_uv=w_uv), torch.einsum("bhc,hcv->bhv", latent, w_uv))
    assert mla.workspace_status() == 0


def test_refusals_leave_the_pool_as_it_was():
    pool = serving.PagedLatentCache(20, 16, 3, 10, 0.5, 2.0)
    weight, cos_sin = torch.ones(512, device="cuda").bfloat16(), angles(100)
    rows = lambda n: torch.ones(n, 576, device="cuda").bfloat16()  # noqa: E731
    pool.append_projected([(0, 40), (1, 5)], rows(45), weight, cos_sin)
    before = [t.clone() for t in (pool._tables, pool.ckv_cache, pool.kpe_cache)], pool.free_pages, list(pool._lens)
    for bad, error in ((lambda: pool.append_projected([(0, 61)], rows(61), weight, cos_sin), RuntimeError),        # past the angles
                       (lambda: pool.append_projected([(0, 3)], rows(4), weight, cos_sin), RuntimeError),
                       (lambda: pool.append_projected([(0, 3)], rows(3)[:, :512], weight, cos_sin), RuntimeError),
                       (lambda: pool.append_projected([(0, 3)], rows(3), weight[:8], cos_sin), RuntimeError),
                       (lambda: pool.append_projected([(0, 3)], rows(3), weight, cos_sin, eps=-1.0), ValueError),
                       (lambda: pool.append_projected([(3, 3)], rows(3), weight, cos_sin), IndexError)):
        with pytest.raises(error):
            bad()
    assert all(torch.equal(x, y) for x, y in zip(before[0], (pool._tables, pool.ckv_cache, pool.kpe_cache)))
    assert before[1:] == (pool.free_pages, pool._lens)
    q = lambda n: (torch.zeros(n, 16, 512, device="cuda").bfloat16(), torch.zeros(n, 16, 64, device="cuda").bfloat16())  # noqa: E731
    for requests, n, error in (([], 0, IndexError), ([(0, 41)], 41, ValueError), ([(0, -1)], 0, ValueError), ([(0, 2), (0, 2)], 4, ValueError),
                               ([(0, 2), (-3, 2)], 4, ValueError), ([(0, 2)], 3, RuntimeError), ([(5, 1)], 1, IndexError)):
        with pytest.raises(error):
            pool.extend(requests, *q(n), SM_SCALE)
    for ranges in ([(0, 39, 2)], [(0, -1, 1)], [(0, 0, -1)], [(2, 0, 1)]):
        with pytest.raises(ValueError):
            pool.gather(ranges)
    with pytest.raises(ValueError):
        pool.decode([0], *q(1), SM_SCALE, precision="fp8", window=5)
