"""The chunk, windowed and read-back operators from their definitions, in 64 bits, one request at a time."""
import torch

from nvfp4_mla_b200.testing import _E2M1

CKV, KPE = 512, 64


def rows64(cache, page_table_row, tokens, ckv_scale, kpe_scale):
    """fp64 latent ``[n, 512]`` and rope ``[n, 64]`` rows of the tokens (a long tensor) of one request."""
    ckv, sf, kpe = cache
    ps = ckv.shape[1]
    page, slot = page_table_row.long()[tokens // ps], tokens % ps
    byte = ckv[page, slot].long()
    codes = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
    values = torch.tensor(_E2M1, dtype=torch.double, device=ckv.device)[codes]
    scales = sf.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).double()
    rope = kpe.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).double()
    return values * scales.repeat_interleave(16, -1) * ckv_scale, rope * kpe_scale


def seen(n, m, window, sinks):
    """``[m, n]`` bool: which of n tokens the last m of them see (a negative position sees nothing)."""
    t, p = torch.arange(n)[None, :], torch.arange(n - m, n)[:, None]
    mask = t <= p
    if window:
        mask &= (t > p - window) | (t < sinks)
    return mask


def attention64(q_nope, q_pe, cache, page_table, kv_lens, q_lens, sm_scale, ckv_scale, kpe_scale, window=0, sinks=0):
    """``[sum(q_lens), heads, 512]`` fp64. A token that sees nothing gives zeros. Only visible tokens are read."""
    out, at = [], 0
    for b, (n, m) in enumerate(zip(kv_lens, q_lens)):
        mask = seen(n, m, window, sinks).to(q_nope.device)
        tokens = mask.any(0).nonzero()[:, 0]
        ckv, kpe = rows64(cache, page_table[b], tokens, ckv_scale, kpe_scale)
        qn, qp = q_nope[at:at + m].double(), q_pe[at:at + m].double()
        x = (qn @ ckv.T + qp @ kpe.T) * sm_scale
        mask = mask[:, tokens][:, None].expand_as(x)
        x = torch.where(mask, x, -torch.inf)
        w = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300)) if tokens.numel() else x
        w = torch.where(mask, w, 0.0)
        total = w.sum(-1, keepdim=True)
        out.append((w @ ckv) / torch.where(total > 0, total, 1.0))
        at += m
    return torch.cat(out) if out else q_nope.new_zeros(0, *q_nope.shape[1:], dtype=torch.double)


# What a row (512 channels) may be off in the 2-norm. The output's rounding to BF16 is at most 2^-8 of each channel. P is rounded to
# FP16 (2^-11 per weight; a row is a weighted sum of independent rows, so that its 2-norm moves by no more than that share) and
# the scores are off by less than 2^-10 (query terms 2^-12 of a 32-channel maximum, rope rounded to 2^-11, times sm_scale, for N(0, 1)
# queries and rows: 0.072 * sqrt(576) * 2^-11), which moves the weights by as much.
ROW_TOL = 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -10


def worst_row(got, want):
    """Largest relative 2-norm error of a row; rows whose reference is 0 have to be 0."""
    got, want = got.double().flatten(0, -2), want.flatten(0, -2)
    norm = want.norm(dim=-1)
    assert (got[norm == 0] == 0).all()
    if not (norm > 0).any():
        return 0.0
    return float(((got - want).norm(dim=-1)[norm > 0] / norm[norm > 0]).max())
