"""GPU tests of the writer behind the latent projection (`norm_rope_append_paged_mla_kv_cache`) and of reading ranges back
(`gather_paged_mla_kv_cache`)."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from nvfp4_mla_b200.testing import SyntheticCache, dequantize

pytestmark = pytest.mark.gpu


def normed(kv_a, weight, cos_sin, positions, eps, interleaved):
    """The BF16 rows that the writer quantises: 64-bit arithmetic, by way of fp32."""
    x = kv_a[:, :512].double()
    ckv = (x * weight.double() / (x.square().mean(-1, keepdim=True) + eps).sqrt()).float().bfloat16()
    cos, sin = cos_sin[positions.long()].double().chunk(2, -1)
    r = kv_a[:, 512:].double()
    a, b = (r[:, 0::2], r[:, 1::2]) if interleaved else (r[:, :32], r[:, 32:])
    a, b = a * cos - b * sin, b * cos + a * sin
    kpe = torch.stack([a, b], -1).flatten(1) if interleaved else torch.cat([a, b], 1)
    return ckv, kpe.float().bfloat16()


def rows(lens, held, ps, seed=0, dev="cuda", size=1.0):
    """Raw rows of ``lens`` new tokens behind ``held`` ones per request, their tables, and an empty pool with a guard page."""
    g = torch.Generator(device=dev).manual_seed(seed)
    B, total = len(lens), sum(lens)
    need = [-(-(n + h) // ps) for n, h in zip(lens, held)]
    pages = sum(need)
    kv_indices = torch.randperm(pages, generator=g, device=dev).int()
    kv_indptr = torch.tensor([0, *torch.tensor(need).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    b = torch.repeat_interleave(torch.arange(B), torch.tensor(lens)).int()
    pos = torch.cat([torch.arange(h, h + n) for n, h in zip(lens, held)]).int()
    kv_a = torch.randn(total, 576, generator=g, device=dev).bfloat16() * size
    weight = (1 + 0.2 * torch.randn(512, generator=g, device=dev)).bfloat16()
    angle = torch.arange(max(n + h for n, h in zip(lens, held)), device=dev).double()[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, device=dev).double() / 64)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    cache = [torch.full((pages + 1, ps, w), 0x5A, dtype=torch.uint8, device=dev) for w in (256, 32, 64)]
    cache = (cache[0], cache[1].view(torch.float8_e4m3fn), cache[2].view(torch.float8_e4m3fn))
    return kv_a, weight, cos_sin, b.to(dev), pos.to(dev), cache, kv_indices, kv_indptr


def raw(cache):
    return [t.view(torch.uint8) for t in cache]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("lens,held,ps,size", [([1], [0], 64, 1.0), ([1] * 24, list(range(0, 240, 10)), 16, 1.0), ([300, 1, 77], [5, 0, 63], 64, 3.0),
                                               ([5000, 3000], [0, 129], 128, 0.01), ([3, 4], [1, 0], 1, 1e4)])
def test_bytes_are_the_writers_on_the_normalised_rows(lens, held, ps, size, interleaved):
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows(lens, held, ps, size=size)
    want = tuple(t.clone() for t in cache)
    ckv, kpe = normed(kv_a, weight, cos_sin, pos, 1e-6, interleaved)
    mla.quantize_append_paged_mla_kv_cache(ckv, kpe, b, pos, *want, kv_indices, kv_indptr, None, 0.0031, 0.017)
    mla.norm_rope_append_paged_mla_kv_cache(kv_a[:, :512], kv_a[:, 512:], weight, cos_sin, b, pos, *cache, kv_indices, kv_indptr,
                                            ckv_scale=0.0031, kpe_scale=0.017, interleaved=interleaved, check=True)
    for got, exp in zip(raw(cache), raw(want)):  # (slots of no token and the guard page among them)
        assert torch.equal(got, exp)


def test_values_of_unequal_size_and_separate_rows():
    """Rows from tiny to huge, zeros, an outlier channel, an eps that matters; latent and rope rows in tensors of their own."""
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([400], [3], 64)
    kv_a *= torch.logspace(-30, 30, 400, device="cuda").bfloat16()[:, None]
    kv_a[7] = 0
    kv_a[9, 100] = 3e38
    kv_a[11, :512] = 1e-40
    weight[5], weight[6] = 0, -3e38
    for eps in (1e-6, 1e3):
        want = tuple(t.clone() for t in cache)
        ckv, kpe = normed(kv_a, weight, cos_sin, pos, eps, True)
        mla.quantize_append_paged_mla_kv_cache(ckv, kpe, b, pos, *want, kv_indices, kv_indptr, None, 0.5, 2.0)
        mla.norm_rope_append_paged_mla_kv_cache(kv_a[:, :512].contiguous(), kv_a[:, 512:].contiguous(), weight, cos_sin, b, pos, *cache,
                                                kv_indices, kv_indptr, eps=eps, ckv_scale=0.5, kpe_scale=2.0)
        for got, exp in zip(raw(cache), raw(want)):
            assert torch.equal(got, exp)


@pytest.mark.parametrize("scale", [1.0, 0.25, 6.5 / 2688, 1 / 448, 3.140625 / 2688, 0.0031, 1e-37, 3e38])
def test_codes_at_every_block_scale(scale):
    """Scales of the cache that make ties everywhere, somewhere and nowhere; rows of sizes that reach every block scale; more tokens than
    a warp looks up at a time."""
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([160000, 3], [0, 5], 64)
    weight[:] = (torch.arange(512, device="cuda") // 16 - 16).float().exp2().bfloat16()  # block j of a row is scaled by 2^(j - 16)
    want = tuple(t.clone() for t in cache)
    ckv, kpe = normed(kv_a, weight, cos_sin, pos, 1e-6, True)
    mla.quantize_append_paged_mla_kv_cache(ckv, kpe, b, pos, *want, kv_indices, kv_indptr, None, scale, 0.02)
    mla.norm_rope_append_paged_mla_kv_cache(kv_a[:, :512], kv_a[:, 512:], weight, cos_sin, b, pos, *cache, kv_indices, kv_indptr, ckv_scale=scale,
                                            kpe_scale=0.02, check=True)
    for got, exp in zip(raw(cache), raw(want)):
        assert torch.equal(got, exp)


def test_products_below_the_range_of_fp32():
    """Channels whose product with the weight is below fp32's normal numbers, the normalised value and the cache's scale above."""
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([200], [0], 64)
    kv_a *= 2.0 ** -27
    g = torch.Generator(device="cuda").manual_seed(3)
    kv_a.view(torch.int16)[:, :256] = torch.randint(1, 64, (200, 256), generator=g, device="cuda").short()  # times 2^-133
    weight[:256] *= 2.0 ** -15
    want = tuple(t.clone() for t in cache)
    ckv, kpe = normed(kv_a, weight, cos_sin, pos, 0.0, True)
    mla.quantize_append_paged_mla_kv_cache(ckv, kpe, b, pos, *want, kv_indices, kv_indptr, None, 2.0 ** -110, 1.0)
    mla.norm_rope_append_paged_mla_kv_cache(kv_a[:, :512], kv_a[:, 512:], weight, cos_sin, b, pos, *cache, kv_indices, kv_indptr, eps=0.0,
                                            ckv_scale=2.0 ** -110)
    assert want[1].float()[:-1].any()
    for got, exp in zip(raw(cache), raw(want)):
        assert torch.equal(got, exp)


def test_tokens_outside_the_tables_are_skipped():
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([40, 3], [0, 0], 16)
    before = [t.clone() for t in raw(cache)]
    args = (kv_a[:, :512], kv_a[:, 512:], weight, cos_sin)
    b[:], pos[:] = -1, 0
    b[1], pos[1] = 2, 0
    b[2], pos[2] = 1, 16          # past its pages
    b[3], pos[3] = 0, -5
    b[4], pos[4] = 0, 47          # in its pages, past the table of angles
    mla.norm_rope_append_paged_mla_kv_cache(*args, b, pos, *cache, kv_indices, kv_indptr)
    assert all(torch.equal(x, y) for x, y in zip(raw(cache), before))
    with pytest.raises(RuntimeError):
        mla.norm_rope_append_paged_mla_kv_cache(*args, b, pos, *cache, kv_indices, kv_indptr, check=True)


def test_writer_refusals():
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([6], [0], 16)
    ok = [kv_a[:, :512], kv_a[:, 512:], weight, cos_sin, b, pos, *cache, kv_indices, kv_indptr]
    wide = torch.zeros(6, 580, device="cuda", dtype=torch.bfloat16)
    for i, value in ((0, kv_a[:, :500]), (0, kv_a[:, :512].float()), (0, wide[:, :512]), (0, wide[:, 1:513]), (1, kv_a[:3, 512:]), (1, kv_a[:, 512:].cpu()), (2, weight[:8]),
                     (2, weight.float()), (3, cos_sin.double()), (3, cos_sin[:, :32]), (4, b[:3]), (5, pos.long()), (9, kv_indices.long())):
        args = list(ok)
        args[i] = value
        with pytest.raises(RuntimeError):
            mla.norm_rope_append_paged_mla_kv_cache(*args)
    with pytest.raises(ValueError):
        mla.norm_rope_append_paged_mla_kv_cache(*ok, eps=-1.0)
    with pytest.raises(RuntimeError):
        mla.norm_rope_append_paged_mla_kv_cache(*ok, ckv_scale=0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,ps", [([1], 64), ([500], 64), ([3, 0, 0, 700, 1], 16), ([257] * 40, 128), ([9, 33], 1), ([40000, 20000], 64)])
def test_gather_is_the_dequantised_rows(lens, ps, dtype):
    c = SyntheticCache([n + 70 for n in lens], ps, 16, 0.37, 0.021, seed=3, device="cuda")
    starts = torch.tensor([(17 * i) % 60 for i in range(len(lens))], dtype=torch.int32, device="cuda")
    indptr = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    # every token's row, straight from the definition, rounded once more to the output's type
    ckv, kpe = dequantize(c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.ckv_scale, c.kpe_scale)
    tokens = [torch.arange(n, device="cuda") + s for n, s in zip(lens, starts.tolist())]
    at = torch.cat([c.page_table[b].long()[t // ps] * ps + t % ps for b, t in enumerate(tokens)])
    want = [x.flatten(0, 1)[at].to(dtype) for x in (ckv, kpe)]
    got = mla.gather_paged_mla_kv_cache(c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.page_table, indptr, sum(lens), starts, c.ckv_scale, c.kpe_scale,
                                        dtype=dtype, check=True)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_gather_leaves_rows_of_no_request():
    c = SyntheticCache([100, 50], 16, 16, 0.37, 0.021, seed=3, device="cuda")
    out = torch.full((200, 512), 7.0, device="cuda"), torch.full((200, 64), 8.0, device="cuda")
    indptr = torch.tensor([5, 105, 155], dtype=torch.int32, device="cuda")
    args = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache, c.page_table)
    mla.gather_paged_mla_kv_cache(*args, indptr, 200, dtype=torch.float32, out=out)
    for x, v in zip(out, (7, 8)):
        assert (x[:5] == v).all() and (x[155:] == v).all()
    want = mla.gather_paged_mla_kv_cache(*args, indptr - 5, 150, dtype=torch.float32)
    assert all(torch.equal(x[5:155], y) for x, y in zip(out, want))
    short = mla.gather_paged_mla_kv_cache(*args, indptr - 5, 77, dtype=torch.float32)  # fewer rows than the indptr names
    assert all(torch.equal(x, y[:77]) for x, y in zip(short, want))


def test_gather_of_bad_pages_gives_zeros():
    c = SyntheticCache([100, 50], 16, 16, 0.37, 0.021, seed=3, device="cuda")
    indptr = torch.tensor([0, 100, 150], dtype=torch.int32, device="cuda")
    c.page_table[0, 1], c.page_table[1, 0] = -1, c.ckv_cache.shape[0]
    args = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache)
    ckv, kpe = mla.gather_paged_mla_kv_cache(*args, c.page_table, indptr, 150)
    for x in (ckv, kpe):
        assert (x[16:32] == 0).all() and (x[100:116] == 0).all() and (x[:16] != 0).any() and (x[116:] != 0).any()
    with pytest.raises(RuntimeError):
        mla.gather_paged_mla_kv_cache(*args, c.page_table, indptr, 150, check=True)
    starts = torch.tensor([10 ** 6, -3], dtype=torch.int32, device="cuda")
    ckv, _ = mla.gather_paged_mla_kv_cache(*args, c.page_table, indptr, 150, starts)
    assert (ckv[:103] == 0).all()


def test_gather_refusals():
    c = SyntheticCache([100, 50], 16, 16, 0.37, 0.021, seed=3, device="cuda")
    indptr = torch.tensor([0, 100, 150], dtype=torch.int32, device="cuda")
    args = (c.ckv_cache, c.ckv_sf_cache, c.kpe_cache)
    call = mla.gather_paged_mla_kv_cache
    for kw in (dict(dtype=torch.float16), dict(total=-1)):
        with pytest.raises(ValueError):
            call(*args, c.page_table, **{"indptr": indptr, "total": 150, **kw})
    for table, ptr, starts, out in ((c.page_table.long(), indptr, None, None), (c.page_table[:1], indptr, None, None), (c.page_table, indptr.long(), None, None),
                                    (c.page_table, indptr, indptr, None), (c.page_table, indptr.cpu(), None, None),
                                    (c.page_table, indptr, None, (torch.empty(150, 512, device="cuda"), torch.empty(150, 64, device="cuda")))):
        with pytest.raises(RuntimeError):
            call(*args, table, ptr, 150, starts, out=out)
    with pytest.raises(RuntimeError):
        call(*args, c.page_table, indptr, 150, kpe_scale=-1.0)
