"""What the C entries of the chunk, window, writer and gather operators refuse, without a GPU: every check comes before the first CUDA call."""
import ctypes

import pytest
import torch

import nvfp4_mla_b200 as mla
from chunk_reference import attention64, seen
from nvfp4_mla_b200 import _lib, build

A = 0x10000  # an aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def refused(lib, rc, text):
    assert rc != 0 and text in lib.nvfp4_mla_last_error().decode()


def append(lib, ckv=A, ckv_stride=576, kpe=A, kpe_stride=576, weight=A, cos_sin=A, max_position=10, eps=1e-6, nnz=4, pages=8, ps=16, batch=2, scale=1.0):
    return lib.nvfp4_mla_norm_rope_append(ckv, ckv_stride, kpe, kpe_stride, weight, cos_sin, max_position, eps, 1, A, A, nnz, A, A, A, pages, ps, A, A,
                                          batch, scale, 1.0, None, None)


def gather(lib, ckv=A, pages=8, ps=16, stride=4, width=4, batch=2, total=9, out=A, kpe_out=A):
    return lib.nvfp4_mla_gather(ckv, A, A, pages, ps, A, stride, width, A, None, batch, total, 1.0, 1.0, 1, out, kpe_out, None, None)


@pytest.mark.parametrize("kw,text", [(dict(ckv=A + 8), "aligned"), (dict(ckv_stride=580), "strides"), (dict(ckv_stride=504), "strides"), (dict(kpe_stride=65), "strides"),
                                     (dict(weight=A + 2), "aligned"), (dict(cos_sin=None), "null"), (dict(eps=-1.0), "eps"), (dict(nnz=-1), "nnz"),
                                     (dict(ps=48), "page_size"), (dict(pages=0), "num_pages"), (dict(pages=1 << 40), "num_pages"), (dict(scale=0.0), "positive"),
                                     (dict(max_position=-1), "max_position")])
def test_the_norm_writer_refuses(lib, kw, text):
    refused(lib, append(lib, **kw), text)


@pytest.mark.parametrize("kw,text", [(dict(ckv=A + 2), "aligned"), (dict(out=A + 8), "aligned"), (dict(kpe_out=A + 4), "aligned"), (dict(ckv=None), "null"), (dict(total=-1), "total"),
                                     (dict(total=1 << 31), "total"), (dict(ps=0), "page_size"), (dict(pages=0), "num_pages"), (dict(width=-1), "width"), (dict(batch=-1), "batch")])
def test_the_gather_refuses(lib, kw, text):
    refused(lib, gather(lib, **kw), text)


def test_nothing_to_do_needs_no_gpu(lib):
    assert append(lib, nnz=0) == 0 and gather(lib, total=0) == 0 and gather(lib, batch=0) == 0


@pytest.mark.parametrize("ps,window,sinks,text", [(48, 5, 0, "page_size"), (16, 0, 0, "window"), (16, -3, 0, "window"), (16, 5, -1, "sink")])
def test_the_window_decode_refuses(lib, ps, window, sinks, text):
    assert lib.nvfp4_mla_decode_window_workspace_bytes(2, 16, ps, 4, 64, window, sinks) == -1
    assert text in lib.nvfp4_mla_last_error().decode()
    refused(lib, lib.nvfp4_mla_decode_window(A, A, A, A, A, 8, ps, A, 4, 4, A, 2, 16, 0.1, 1.0, 1.0, 64, window, sinks, A, None, None, A, 1 << 40, None, None), text)


@pytest.mark.parametrize("ps,window,sinks,total,text", [(48, 5, 0, 3, "page_size"), (16, -1, 0, 3, "window"), (16, 5, -1, 3, "sink"), (16, 0, 0, -1, "total_q")])
def test_extend_refuses(lib, ps, window, sinks, total, text):
    refused(lib, lib.nvfp4_mla_extend(A, A, A, A, A, 8, ps, A, 4, 4, A, A, 2, total, 16, 0.1, 1.0, 1.0, 64, window, sinks, A, A, 1 << 40, None, None), text)


def test_python_refuses_host_tensors():
    q, qp = torch.zeros(2, 16, 512, dtype=torch.bfloat16), torch.zeros(2, 16, 64, dtype=torch.bfloat16)
    cache = (torch.zeros(4, 16, 256, dtype=torch.uint8), torch.zeros(4, 16, 32).to(torch.float8_e4m3fn), torch.zeros(4, 16, 64).to(torch.float8_e4m3fn))
    table, lens, ptr = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        mla.extend(q, qp, *cache, table, lens, ptr, 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        mla.decode_window(q, qp, *cache, table, lens, 0.1, 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        mla.gather_paged_mla_kv_cache(*cache, table, ptr, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        mla.norm_rope_append_paged_mla_kv_cache(q[:, 0], qp[:, 0], q[0, 0], torch.zeros(4, 64), lens, lens, *cache, lens, ptr)
    with pytest.raises(ValueError, match="window"):
        mla.decode_window(q, qp, *cache, table, lens, 0.1, 0)
    with pytest.raises(ValueError, match="dtype"):
        mla.gather_paged_mla_kv_cache(*cache, table, ptr, 2, dtype=torch.int8)


def test_the_reference_of_the_gpu_tests():
    """The 64-bit reference against single rows computed by hand: masks, a window, a token that sees nothing."""
    assert seen(4, 2, 0, 0).tolist() == [[True, True, True, False], [True, True, True, True]]
    assert seen(5, 1, 2, 1).tolist() == [[True, False, False, True, True]]
    assert seen(1, 3, 0, 0).tolist() == [[False], [False], [True]]
    g = torch.Generator().manual_seed(0)
    cache = (torch.randint(0, 256, (2, 4, 256), generator=g, dtype=torch.uint8), torch.rand(2, 4, 32, generator=g).to(torch.float8_e4m3fn),
             torch.randn(2, 4, 64, generator=g).to(torch.float8_e4m3fn))
    q, qp = torch.randn(1, 2, 512, generator=g).bfloat16(), torch.randn(1, 2, 64, generator=g).bfloat16()
    table = torch.tensor([[1, 0]])
    out = attention64(q, qp, cache, table, [6], [1], 0.05, 2.0, 0.5, window=2, sinks=1)
    from nvfp4_mla_b200.testing import dequantize
    ckv, kpe = (x.double() for x in dequantize(*cache, 2.0, 0.5))
    k, r = torch.stack([ckv[1, 0], ckv[0, 0], ckv[0, 1]]), torch.stack([kpe[1, 0], kpe[0, 0], kpe[0, 1]])  # tokens 0, 4, 5
    want = torch.softmax((q[0].double() @ k.T + qp[0].double() @ r.T) * 0.05, -1) @ k
    assert torch.allclose(out[0], want, rtol=1e-12)
    assert (attention64(q, qp, cache, table, [0], [1], 0.05, 2.0, 0.5) == 0).all()
