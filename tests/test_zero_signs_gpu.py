"""GPU test of the signs of zeros that the writer behind the latent projection stores: a code of value 0 keeps the sign of what it stands
for, as in `quantize_append_paged_mla_kv_cache`."""
import pytest
import torch

import nvfp4_mla_b200 as mla
from test_cache_io_gpu import normed, raw, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1.0, 0.5, 2.0 ** -9, 6.5 / 2688])
def test_zeros_keep_their_sign_at_every_block_scale(scale):
    """Channels with a weight of 0 and inputs of -0 in blocks of every scale (with a power of two as the cache's scale a third of the block
    scales settles its codes with two products, whose sum must not turn -0 into +0)."""
    kv_a, weight, cos_sin, b, pos, cache, kv_indices, kv_indptr = rows([60000], [0], 64)
    weight[:] = (torch.arange(512, device="cuda") // 16 - 16).float().exp2().bfloat16()  # block j of a row is scaled by 2^(j - 16)
    weight[1::16] = 0
    weight[2::16] = -0.0
    kv_a[:, 3:512:16] = -0.0
    want = tuple(t.clone() for t in cache)
    ckv, kpe = normed(kv_a, weight, cos_sin, pos, 1e-6, True)
    mla.quantize_append_paged_mla_kv_cache(ckv, kpe, b, pos, *want, kv_indices, kv_indptr, None, scale, 1.0)
    mla.norm_rope_append_paged_mla_kv_cache(kv_a[:, :512], kv_a[:, 512:], weight, cos_sin, b, pos, *cache, kv_indices, kv_indptr, ckv_scale=scale, check=True)
    minus = (raw(want)[0][:-1, :, 1::8] >> 4) == 8  # channel 3 of every block
    scales = raw(want)[1][:-1]
    assert minus[scales > 0].float().mean() > 0.99 and len(scales[minus].unique()) > 100  # -0 is met at nearly every block scale
    for got, exp in zip(raw(cache), raw(want)):
        assert torch.equal(got, exp)
