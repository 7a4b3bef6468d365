"""The operators around the decode path, each in a plain form and as the framework's calls: what they are timed and checked on.

A case is one operator at one size. `listed()` are the fixed ones, `draw()` gives further cases of the same ranges. Four operators:

  extend   `extend`: attention of a chunk of new tokens per request (ragged, causal, their rows already in the cache) over the
           paged NVFP4 cache, with or without a sliding window and visible first tokens: chunked prefill
  window   `decode_window`: one query token per request over the last `window` tokens and the first `sinks` tokens of its cache
  write    `norm_rope_append_paged_mla_kv_cache`: the latent projection's raw rows are normalised, rotated, quantised and written
           into the cache, and read back by `gather_paged_mla_kv_cache`
  gather   `gather_paged_mla_kv_cache`: a range of tokens of every request, out of the pages, in BF16 or FP32

Where `own` is false the same results come from elementary torch operations.
"""
import math
import random

import torch

own = False  # whether run() makes the framework's calls

CKV, KPE = 512, 64
SM_SCALE = (128 + KPE) ** -0.5
# amax / (6 * 448) and amax / 448 of N(0, 1) data, as the fp32 numbers that the cache's rounding steps take
CKV_SCALE, KPE_SCALE = torch.tensor([6.5 / (6 * 448), 6.5 / 448], dtype=torch.float32).tolist()
EPS = 1e-6
MAX_PAIRS = 128 * 1024 * 16384   # heads x queries x tokens of the largest listed chunk (padded to the longest request)
MAX_WINDOW_PAIRS = 128 * 32 * 4100  # heads x requests x visible tokens of the largest listed window case
MAX_TOKENS = 600000              # rows written or gathered
CHUNK = 1 << 17                  # rows generated at a time


def listed():
    return [
        # a short prompt of one user on a tensor-parallel shard, a few tokens at a time: latency and launches
        dict(name="extend_h16_b1_16_of_200", op="extend", heads=16, batch=1, q_lo=16, q_hi=16, lo=184, hi=184, page_size=64, window=0, sinks=0),
        # chunked prefill as a serving engine schedules it: four prompts, 512 tokens each, 8K behind them
        dict(name="extend_h16_b4_512_of_8k", op="extend", heads=16, batch=4, q_lo=512, q_hi=512, lo=7680, hi=7680, page_size=64, window=0, sinks=0),
        # all heads on one GPU, one long prompt: compute-bound
        dict(name="extend_h128_b1_1024_of_16k", op="extend", heads=128, batch=1, q_lo=1024, q_hi=1024, lo=15360, hi=15360, page_size=64, window=0, sinks=0),
        # a mixed batch of an engine step, ragged chunks from a single token up, small pages
        dict(name="extend_h16_b24_ragged", op="extend", heads=16, batch=24, q_lo=1, q_hi=400, lo=0, hi=8000, page_size=16, window=0, sinks=0),
        # the chunk of a long conversation that keeps a window and its first tokens
        dict(name="extend_h32_b8_window4k", op="extend", heads=32, batch=8, q_lo=200, q_hi=256, lo=6000, hi=32000, page_size=64, window=4096, sinks=128),
        # one user's long conversation, windowed: latency
        dict(name="window_h16_b1_1k", op="window", heads=16, batch=1, lo=5000, hi=5000, page_size=64, window=1024, sinks=4),
        # a full batch of long conversations on a tensor-parallel shard
        dict(name="window_h16_b64_4k", op="window", heads=16, batch=64, lo=4096, hi=65536, page_size=64, window=4096, sinks=4),
        # all heads on one GPU, ragged batch, some requests shorter than the window, odd sizes
        dict(name="window_h128_b32_ragged", op="window", heads=128, batch=32, lo=100, hi=50000, page_size=32, window=2001, sinks=17),
        # the newest token of every request of a decode step
        dict(name="write_b24_step", op="write", batch=24, q_lo=1, q_hi=1, lo=1, hi=1000, page_size=16, interleaved=True),
        # prompts of a prefill step
        dict(name="write_b32_prompts", op="write", batch=32, q_lo=1000, q_hi=16384, lo=0, hi=5000, page_size=64, interleaved=True),
        # the context of one short request, for an up-projection
        dict(name="gather_b1_500", op="gather", batch=1, lo=500, hi=500, page_size=64, dtype="bf16"),
        # the contexts of a prefill step's requests
        dict(name="gather_b64_ragged", op="gather", batch=64, lo=1000, hi=16384, page_size=64, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["extend"] * 4 + ["window"] * 3 + ["write", "gather"])
    case = dict(op=op, page_size=rng.choice([16, 32, 64, 64, 64, 128]))
    if op in ("write", "gather"):
        batch = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(32768, MAX_TOKENS // batch))
        lo = max(1, hi // rng.choice([1, 2, 16]))
        if op == "gather":
            return dict(case, batch=batch, lo=lo, hi=hi, dtype=rng.choice(["bf16", "bf16", "fp32"]))
        before = rng.randint(0, 20000 // batch)
        return dict(case, batch=batch, q_lo=lo, q_hi=hi, lo=before // 2, hi=before, interleaved=rng.choice([True, True, False]))
    heads = rng.choice([16, 16, 16, 32, 64, 128])
    case.update(heads=heads)
    if op == "window":
        sinks = rng.choice([0, 1, 4, 64, _log_int(rng, 1, 500)])
        window = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(128, MAX_WINDOW_PAIRS // heads // (window + sinks))))
        hi = _log_int(rng, 1, 65536)
        return dict(case, batch=batch, lo=max(1, hi // rng.choice([1, 2, 16, hi])), hi=hi, window=window, sinks=sinks)
    heads = case["heads"] = rng.choice([heads, heads, heads, 8, 24])
    q_hi = _log_int(rng, 1, 2048)
    batch = _log_int(rng, 1, 32)
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 8192), rng.choice([0, 4, 100]))])
    q_hi = max(1, min(q_hi, MAX_PAIRS // 512 // heads // batch))
    most = MAX_PAIRS // (heads * batch * q_hi)  # visible tokens per query, the chunk among them
    hi = rng.randint(0, 65000) if window and window + sinks + q_hi <= most else _log_int(rng, 1, max(1, min(65000, most) - q_hi + 1)) - 1
    if window and window + sinks + q_hi > most:
        window = sinks = 0
    return dict(case, batch=batch, q_lo=max(1, q_hi // rng.choice([1, 2, q_hi])), q_hi=q_hi, lo=hi // rng.choice([1, 2, hi + 1]), hi=hi,
                window=window, sinks=sinks)


def _lens(case):
    """(query tokens or rows, tokens in the cache with them) per request: part of the case, the same for every seed."""
    r = random.Random(case["batch"] * 1000003 + case["lo"] * 101 + case["hi"] + case.get("q_hi", 0))
    q = [r.randint(case.get("q_lo", 1), case.get("q_hi", 1)) for _ in range(case["batch"])]
    held = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    return q, held if case["op"] in ("window", "gather") else [a + b for a, b in zip(held, q)]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _e2m1(y):
    """Nearest E2M1 code, ties to the even mantissa, magnitudes above 6 saturate."""
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    for above, tie in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= above) if tie else (a > above)
    return code | (torch.signbit(y).to(torch.uint8) << 3)


def _quantise(ckv, kpe):
    """The cache's bytes of BF16 rows: packed E2M1, E4M3 block scales, E4M3 rope; every step one fp32 operation (the divisors
    are tensors: division by a number is a product with its reciprocal, and ties are common)."""
    six, ckv_scale, kpe_scale = torch.tensor([6.0, CKV_SCALE, KPE_SCALE], device="cuda").split(1)
    x = ckv.float().reshape(-1, CKV // 16, 16)
    sf8 = (x.abs().amax(-1) / six / ckv_scale).clamp(max=448.0).to(torch.float8_e4m3fn)
    sf = (sf8.float() * ckv_scale)[..., None]
    codes = _e2m1(torch.where(sf > 0, x / sf, 0.0)).reshape(-1, CKV)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), sf8, (kpe.float() / kpe_scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _fill(cache, g):
    """Every slot of the pool holds a quantised N(0, 1) row."""
    ckv, sf, kpe = (t.view(-1, t.shape[-1]) for t in cache)
    for i in range(0, ckv.shape[0], CHUNK):
        n = min(CHUNK, ckv.shape[0] - i)
        rows = torch.randn(n, CKV + KPE, generator=g, device="cuda", dtype=torch.bfloat16)
        c, s, k = _quantise(rows[:, :CKV], rows[:, CKV:])
        ckv[i:i + n], sf.view(torch.uint8)[i:i + n], kpe.view(torch.uint8)[i:i + n] = c, s.view(torch.uint8), k.view(torch.uint8)


def _pool(case, lens, first, g):
    """An empty cache and a shuffled page table. Pages that no token of a request needs any more (between the first `sinks` tokens and token `first`)
    have gone back to the pool: their entries hold -1."""
    ps, sinks = case["page_size"], case.get("sinks", 0)
    need = [-(-n // ps) for n in lens]
    width = max(max(need), 1)
    live = torch.tensor([[p < n and (p * ps < sinks or (p + 1) * ps > f) for p in range(width)] for n, f in zip(need, first)], device="cuda")
    total = max(1, sum(sum(1 for p in range(n) if p * ps < sinks or (p + 1) * ps > f) for n, f in zip(need, first)))
    page_table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    page_table[live] = torch.randperm(total, generator=g, device="cuda").int()[:int(live.sum())]
    cache = (torch.zeros(total, ps, CKV // 2, dtype=torch.uint8, device="cuda"),
             torch.zeros(total, ps, CKV // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
             torch.zeros(total, ps, KPE, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn))
    return cache, page_table


def _indptr(counts):
    return torch.tensor([0] + [sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, (q, lens) = case["op"], _lens(case)
    W, S = case.get("window", 0), case.get("sinks", 0)
    first = [max(0, n - m - W + 1) if W else 0 for n, m in zip(lens, q)]  # first token that a query of the request sees in its window
    cache, page_table = _pool(case, lens, first, g)
    state = dict(op=op, cache=cache, page_table=page_table, kv_lens=_int32(lens), max_kv_len=max(lens), window=W, sinks=S)
    if op in ("extend", "window"):
        _fill(cache, g)
        n = sum(q)
        state.update(q_nope=torch.randn(n, case["heads"], CKV, generator=g, device="cuda", dtype=torch.bfloat16),
                     q_pe=torch.randn(n, case["heads"], KPE, generator=g, device="cuda", dtype=torch.bfloat16), qo_indptr=_indptr(q),
                     max_q=max(q), span=max(n - max(f, S if W else 0) for n, f in zip(lens, first)))
        return state
    if op == "gather":
        _fill(cache, g)
        state.update(starts=torch.zeros_like(state["kv_lens"]), indptr=_indptr(lens), total=sum(lens), dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        return state
    total, width = sum(q), page_table.shape[1]
    angles = torch.arange(max(lens), device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, KPE, 2, device="cuda").double() / KPE)
    requests = torch.repeat_interleave(torch.arange(len(q), device="cuda"), torch.tensor(q, device="cuda"))
    indptr, starts = _indptr(q), _int32([n - m for n, m in zip(lens, q)])
    positions = torch.arange(total, device="cuda") - indptr[requests] + starts[requests]
    # the raw projection's rows are of unequal size, and the norm's weights are those of a trained model: around 1
    rows = torch.randn(total, CKV + KPE, generator=g, device="cuda", dtype=torch.bfloat16)
    size = torch.randn(total, 1, generator=g, device="cuda", dtype=torch.bfloat16).exp()
    weight = (1 + 0.1 * torch.randn(CKV, generator=g, device="cuda")).bfloat16()
    state.update(kv_a=torch.cat([rows[:, :CKV] * size, rows[:, CKV:]], 1), weight=weight, cos_sin=torch.cat([angles.cos(), angles.sin()], 1).float(),
                 batch_indices=requests.int(), positions=positions.int(), kv_indices=page_table.view(-1),
                 kv_indptr=torch.arange(0, (len(q) + 1) * width, width, dtype=torch.int32, device="cuda"), interleaved=case["interleaved"],
                 starts=starts, indptr=indptr, total=total, dtype=torch.bfloat16)
    return state


# ---- the operators in elementary operations ---------------------------------------------------------------------------
def _read(s, requests, tokens):
    """fp32 rows of the cache: token `tokens` of request `requests` (two arrays of one shape)."""
    ps = s["cache"][0].shape[1]
    row = s["page_table"][requests, tokens // ps].long() * ps + tokens % ps
    ckv, sf, kpe = (t.view(-1, t.shape[-1]) for t in s["cache"])
    packed = ckv[row]
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    sf, kpe = sf.view(torch.uint8)[row].view(torch.float8_e4m3fn).float(), kpe.view(torch.uint8)[row].view(torch.float8_e4m3fn).float()
    return (values[codes].unflatten(-1, (-1, 16)) * sf[..., None]).flatten(-2) * CKV_SCALE, kpe * KPE_SCALE


def _attention(s):
    """All requests at once, padded: token list [B, T] = the first tokens, then everything from the first window on."""
    W, S = s["window"], s["sinks"]
    B, Q, H = s["kv_lens"].numel(), s["max_q"], s["q_nope"].shape[1]
    lens, start = s["kv_lens"].long(), s["qo_indptr"].long()
    counts = start[1:] - start[:-1]
    skip = torch.clamp(lens - counts - W + 1, min=S) if W else torch.zeros_like(lens)
    tokens = skip[:, None] + torch.arange(s["span"], device="cuda")
    if W and S:
        tokens = torch.cat([torch.arange(S, device="cuda").expand(B, S), tokens], 1)
    known = tokens < lens[:, None]
    each = torch.arange(B, device="cuda")[:, None].expand_as(tokens)
    ckv, kpe = _read(s, each, torch.minimum(tokens, (lens - 1).clamp(min=0)[:, None]))  # [B, T, 512], [B, T, 64]
    i = torch.arange(Q, device="cuda")
    row = torch.minimum(start[:-1, None] + i, start[1:, None] - 1)  # query tokens past a request's last repeat it
    q = torch.cat([s["q_nope"], s["q_pe"]], -1).float()[row].reshape(B, Q * H, CKV + KPE)
    x = torch.matmul(q, torch.cat([ckv, kpe], -1).transpose(1, 2)).mul_(SM_SCALE).view(B, Q, H, -1)
    at = (lens - counts)[:, None] + i  # position of a query token
    seen = known[:, None] & (tokens[:, None] <= at[..., None])
    if W:
        seen &= (tokens[:, None] > at[..., None] - W) | (tokens[:, None] < S)
    x.masked_fill_(~seen[:, :, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, Q * H, -1), ckv).view(B, Q, H, CKV) / torch.where(total > 0, total, 1.0)
    return out[i < counts[:, None]].bfloat16()


def _write(s):
    """The norm and the rotation in 64 bits, rounded to BF16 once, then the cache's own rounding steps."""
    x = s["kv_a"][:, :CKV].double()
    ckv = (x * s["weight"].double() * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).bfloat16()
    cos, sin = s["cos_sin"].double()[s["positions"].long()].chunk(2, -1)
    r = s["kv_a"][:, CKV:].double()
    a, b = (r[:, 0::2], r[:, 1::2]) if s["interleaved"] else r.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    kpe = (torch.stack([a, b], -1).flatten(1) if s["interleaved"] else torch.cat([a, b], -1)).bfloat16()
    ps = s["cache"][0].shape[1]
    row = s["page_table"][s["batch_indices"].long(), s["positions"].long() // ps].long() * ps + s["positions"] % ps
    for held, new in zip(s["cache"], _quantise(ckv, kpe)):
        held.view(torch.uint8).view(-1, held.shape[-1])[row] = new.view(torch.uint8)


def _gather(s):
    counts = (s["indptr"][1:] - s["indptr"][:-1]).long()
    each = torch.repeat_interleave(torch.arange(counts.numel(), device="cuda"), counts, output_size=s["total"])
    ckv, kpe = _read(s, each, torch.arange(s["total"], device="cuda") - s["indptr"].long()[each] + s["starts"].long()[each])
    return ckv.to(s["dtype"]), kpe.to(s["dtype"])


def run(s):
    if own:
        import nvfp4_mla_b200 as mla
        scales = dict(ckv_scale=CKV_SCALE, kpe_scale=KPE_SCALE)
        if s["op"] == "extend":
            return mla.extend(s["q_nope"], s["q_pe"], *s["cache"], s["page_table"], s["kv_lens"], s["qo_indptr"], SM_SCALE,
                              max_kv_len=s["max_kv_len"], window=s["window"], sink_tokens=s["sinks"], **scales)
        if s["op"] == "window":
            return mla.decode_window(s["q_nope"], s["q_pe"], *s["cache"], s["page_table"], s["kv_lens"], SM_SCALE, s["window"],
                                     sink_tokens=s["sinks"], max_kv_len=s["max_kv_len"], **scales)
        if s["op"] == "write":
            mla.norm_rope_append_paged_mla_kv_cache(s["kv_a"][:, :CKV], s["kv_a"][:, CKV:], s["weight"], s["cos_sin"], s["batch_indices"],
                                                    s["positions"], *s["cache"], s["kv_indices"], s["kv_indptr"], eps=EPS,
                                                    interleaved=s["interleaved"], **scales)
        return mla.gather_paged_mla_kv_cache(*s["cache"], s["page_table"], s["indptr"], s["total"], starts=s["starts"], dtype=s["dtype"], **scales)
    if s["op"] in ("extend", "window"):
        return _attention(s)
    if s["op"] == "write":
        _write(s)
    return _gather(s)


def work(case):
    """A token of the cache is 352 bytes and read once per request, queries come in and outputs go out in BF16; 2176 operations per
    head, query token and token that it sees: 576 channels in the scores, 512 in the sum."""
    q, lens = _lens(case)
    if case["op"] in ("write", "gather"):
        rows = sum(q) if case["op"] == "write" else sum(lens)
        out = rows * (352 + (CKV + KPE) * (4 if case.get("dtype") == "fp32" else 2))
        return dict(bytes=out + (rows * (2 * (CKV + KPE) + 8 + 352) if case["op"] == "write" else 0), flops=0)
    W, S = case["window"], case["sinks"]
    held = pairs = 0
    for m, n in zip(q, lens):
        # query at position p sees p + 1 tokens, or with a window min(p + 1, W + min(S, p + 1 - W))
        at = range(n - m, n)
        pairs += sum(p + 1 if not W else min(p + 1, W + max(0, min(S, p + 1 - W))) for p in at)
        held += n if not W else min(n, W + m - 1 + max(0, min(S, n - m - W + 1)))
    rows = sum(q) * case["heads"]
    return dict(bytes=held * 352 + rows * 2 * (CKV + KPE + CKV), flops=2176 * pairs * case["heads"])


# ---- the definitions in 64 bits, request by request -------------------------------------------------------------------
def _rows64(s, b, tokens):
    """fp64 latent and rope rows of tokens (an index array) of request b."""
    ckv, sf, kpe = s["cache"]
    ps = ckv.shape[1]
    page, slot = s["page_table"][b].long()[tokens // ps], tokens % ps
    byte = ckv[page, slot].long()
    code = torch.empty(len(tokens), CKV, dtype=torch.long, device="cuda")
    code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
    mantissa, exponent = code % 2, code % 8 // 2
    value = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.pow(2.0, exponent.double() - 1))
    value = torch.where(code >= 8, -value, value)
    scale = sf.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).double()
    return value * scale.repeat_interleave(16, -1) * CKV_SCALE, kpe.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).double() * KPE_SCALE


def exact(case, seed):
    s = prepare(case, seed)
    q, lens = _lens(case)
    if case["op"] in ("extend", "window"):
        out, W, S, at = [], case["window"], case["sinks"], 0
        for b, (m, n) in enumerate(zip(q, lens)):
            tokens = [t for t in range(n) if not W or t < S or t > n - m - W]
            tokens = torch.tensor(tokens, device="cuda")
            ckv, kpe = _rows64(s, b, tokens)
            for i in range(0, m, 128):
                k = min(128, m - i)
                p = torch.arange(n - m + i, n - m + i + k, device="cuda")[:, None]
                seen = (tokens <= p) & ((tokens > p - W) | (tokens < S)) if W else tokens <= p
                x = s["q_nope"][at + i:at + i + k].double() @ ckv.T + s["q_pe"][at + i:at + i + k].double() @ kpe.T
                x = torch.where(seen[:, None], x * SM_SCALE, -math.inf)
                out.append(torch.softmax(x, -1) @ ckv)
            at += m
        return torch.cat(out)
    if case["op"] == "gather":
        rows = [_rows64(s, b, torch.arange(n, device="cuda")) for b, n in enumerate(lens)]
        return torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
    ckv, kpe = [], []
    for i in range(0, sum(q), CHUNK):
        x = s["kv_a"][i:i + CHUNK].double()
        latent, rope = x[:, :CKV], x[:, CKV:]
        latent = (latent / torch.sqrt((latent ** 2).sum(-1, keepdim=True) / CKV + EPS) * s["weight"].double()).bfloat16().double()
        # the cache's format is defined by its rounding steps: each quotient and product is rounded to 24 bits
        block, divisor = latent.unflatten(-1, (32, 16)), torch.tensor([[6.0, CKV_SCALE, KPE_SCALE]], device="cuda", dtype=torch.double)
        stored = (((block.abs().amax(-1, keepdim=True) / divisor[:, 0]).float().double() / divisor[:, 1]).float().clamp(max=448)).to(torch.float8_e4m3fn).double()
        y = (block / (stored * divisor[:, 1]).float().double().clamp(min=1e-300)).float()
        size = y.abs()
        # E2M1 is spaced by 1/2 below 2, by 1 below 4, by 2 up to 6: round to the spacing, ties to even
        grid = torch.where(size < 1.75, torch.round(size * 2) / 2, torch.where(size < 3.5, torch.round(size), torch.round(size / 2) * 2)).clamp(max=6.0)
        ckv.append((torch.copysign(grid, y).double() * stored * CKV_SCALE).flatten(-2))
        angle = s["cos_sin"][s["positions"][i:i + CHUNK].long()].double()
        z = torch.complex(angle[:, :32], angle[:, 32:])
        r = torch.complex(rope[:, 0::2], rope[:, 1::2]) if case["interleaved"] else torch.complex(rope[:, :32], rope[:, 32:])
        r = r * z
        r = torch.view_as_real(r).flatten(1) if case["interleaved"] else torch.cat([r.real, r.imag], 1)
        kpe.append((r.bfloat16().double() / divisor[:, 2]).float().clamp(-448, 448).to(torch.float8_e4m3fn).double() * KPE_SCALE)
    return torch.cat(ckv), torch.cat(kpe)
