"""Performance cases of the quantised paged KV cache.

The cache holds 8-bit codes, ``[blocks, kv_heads, 16, head_dim]`` for K and for V,
and one fp32 scale for each token's row of a KV head, ``[blocks, kv_heads, 2, 16]``
(K's scales, then V's).  A code stands for code * scale:

  e4m3  scale 2^e, the least with amax / 2^e <= 448; code = x / scale, rounded to e4m3
  int8  scale amax / 127; code = x * (127 / amax), rounded to a whole number

(ties to even; amax: the row's largest |x|, at least 2^-100).  Each case is one
pass as a serving program makes it:

  write   new tokens are quantised into the cache's slots
          (``quantized.reshape_and_cache_quantized``), and read back as the values
          that the cache now stands for, which the tokens' own attention takes
          (``quantized.gather_quantized_kv``)
  read    the cached tokens of whole sequences, or of a part of them, are read back
          into contiguous rows of the model's type
          (``quantized.gather_quantized_kv``)
  decode  attention of one new token per sequence over its cached ones
          (``quantized.quantized_decode_attention``)

With ``own`` false a pass computes the same in elementary torch operations in 32
bits.  ``listed()`` are fixed cases, ``draw(rng)`` gives further ones of the same
ranges.  Pages are 16 tokens from a seeded permuted pool; K, V and Q are normal,
the size of K and V rows varies from token to token.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEVICE = "cuda"
TINY = 2.0 ** -100


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The one new token of an interactive request, Mixtral heads.
        dict(name="write_b1_step", kind="write", batch=1, n_lo=1, n_hi=1, past=129, hkv=8,
             dim=128, dtype="bfloat16", codec="e4m3", fused=False, lens_seed=0),
        # A serving step's 64 new tokens, slices of the projection's one output tensor.
        dict(name="write_b64_step", kind="write", batch=64, n_lo=1, n_hi=1, past=4000, hkv=8,
             dim=128, dtype="bfloat16", codec="e4m3", fused=True, lens_seed=1),
        # A step that admits four long prompts.
        dict(name="write_4x4096_prompts", kind="write", batch=4, n_lo=4096, n_hi=4096, past=0,
             hkv=8, dim=128, dtype="bfloat16", codec="e4m3", fused=False, lens_seed=0),
        # Ragged chunks that continue their sequences inside a page; fp16, head_dim 64, int8.
        dict(name="write_b8_d64_int8", kind="write", batch=8, n_lo=17, n_hi=2000, past=300,
             hkv=8, dim=64, dtype="float16", codec="int8", fused=True, lens_seed=2),
        # The histories that a continuation chunk of eight requests attends to.
        dict(name="read_8x4096", kind="read", batch=8, n_lo=4096, n_hi=4096, past=0, hkv=8,
             dim=128, dtype="bfloat16", codec="e4m3", lens_seed=0),
        # Parts of ragged histories, from the middle of a page on; head_dim 256, int8.
        dict(name="read_b5_d256_int8", kind="read", batch=5, n_lo=100, n_hi=3001, past=333,
             hkv=4, dim=256, dtype="bfloat16", codec="int8", lens_seed=3),
        # A decode step of one short request.
        dict(name="decode_b1_129", kind="decode", batch=1, lo=129, hi=129, hkv=8, group=4,
             dim=128, dtype="bfloat16", codec="e4m3", q_std=1.0, lens_seed=0),
        # The serving decode step of the benchmark: Mixtral shape, 64 requests.
        dict(name="decode_b64_mixtral", kind="decode", batch=64, lo=512, hi=4096, hkv=8, group=4,
             dim=128, dtype="bfloat16", codec="e4m3", q_std=1.0, lens_seed=2),
        # The same step over int8 codes.
        dict(name="decode_b64_mixtral_int8", kind="decode", batch=64, lo=512, hi=4096, hkv=8,
             group=4, dim=128, dtype="bfloat16", codec="int8", q_std=1.0, lens_seed=2),
        # Long contexts.
        dict(name="decode_b16_32k", kind="decode", batch=16, lo=32767, hi=32767, hkv=8, group=4,
             dim=128, dtype="bfloat16", codec="e4m3", q_std=2.0, lens_seed=0),
        # Many short requests; fp16, head_dim 64, eight query heads per KV head.
        dict(name="decode_b128_short_d64_fp16", kind="decode", batch=128, lo=1, hi=600, hkv=8,
             group=8, dim=64, dtype="float16", codec="int8", q_std=1.0, lens_seed=5),
        # Few long requests with few heads of head_dim 256.
        dict(name="decode_b3_d256", kind="decode", batch=3, lo=2000, hi=12001, hkv=2, group=3,
             dim=256, dtype="bfloat16", codec="e4m3", q_std=1.0, lens_seed=4),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    hi = max(lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "write", "read", "read", "decode", "decode", "decode",
                       "decode"])
    case = dict(kind=kind, hkv=rng.choice([1, 2, 3, 4, 8, 8, 16]),
                dim=rng.choice([64, 128, 128, 256]),
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]),
                codec=rng.choice(["e4m3", "e4m3", "int8"]), lens_seed=rng.randrange(1 << 20))
    row = case["hkv"] * case["dim"]
    if kind == "decode":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 2, min(60000, (1 << 28) // (batch * row)))
        lo = rng.choice([0, 1, int(hi * rng.uniform(0.1, 1.0)), hi])
        return dict(case, batch=batch, lo=lo if batch > 1 else max(1, lo), hi=hi,
                    group=rng.choice([1, 2, 3, 4, 4, 5, 8, 16]), q_std=rng.choice([1.0, 2.0]))
    batch = _log(rng, 1, 64)
    n_hi = _log(rng, 1, min(16000, (1 << 26) // (batch * row)))
    case.update(batch=batch, n_lo=max(1, int(n_hi * rng.uniform(0.1, 1.0))), n_hi=n_hi,
                past=rng.choice([0, _log(rng, 1, 2000)]))
    return dict(case, fused=rng.random() < 0.5) if kind == "write" else case


# ------------------------------------------------------------------ inputs
def _lens(case, lo, hi, salt=0):
    """The case's ragged lengths (part of the case, not of the inputs)."""
    r = random.Random(case["lens_seed"] * 8 + salt)
    lens = [r.randint(min(lo, hi), hi) for _ in range(case["batch"])]
    lens[-1] = max(lens[-1], 1)
    return lens


def _shape(case):
    """(tokens before, tokens of the pass) of each sequence."""
    if case["kind"] == "decode":
        return [0] * case["batch"], _lens(case, case["lo"], case["hi"])
    past = _lens(case, case["past"] // 2, case["past"], 1) if case["past"] else [0] * case["batch"]
    return past, _lens(case, case["n_lo"], case["n_hi"])


def _randn(shape, g, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _indptr(counts):
    return [0] + np.cumsum(np.asarray(counts, dtype=np.int64)).tolist()


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _codes_type(case):
    return torch.int8 if case["codec"] == "int8" else torch.float8_e4m3fn


def _rows(shape, g, dtype):
    """K or V rows: normal, each token's of its own size."""
    size = _randn((*shape[:-2], 1, 1), g, torch.float32, 0.5).exp_()
    return _randn(shape, g, torch.float32).mul_(size).to(dtype)


def prepare(case, seed):
    dt, codes = getattr(torch, case["dtype"]), _codes_type(case)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    past, new = _shape(case)
    lens = [a + b for a, b in zip(past, new)]
    hkv, d, batch = case["hkv"], case["dim"], case["batch"]
    total, width = sum(_pages(n) for n in lens) + 2, max(_pages(n) for n in lens)
    order = list(range(total))
    random.Random(seed).shuffle(order)
    at = _indptr([_pages(n) for n in lens])
    s = dict(kind=case["kind"], dtype=dt, heads=(hkv * case.get("group", 1), hkv, d),
             indptr=_ints(at), indices=_ints(order[:at[-1]]), lens=_ints(lens), top=max(lens),
             lpl=_ints([(n - 1) % PAGE + 1 if n else 0 for n in lens]),
             table=_ints([order[a:b] + [-1] * (width - b + a) for a, b in zip(at, at[1:])]),
             kc=torch.empty((total, hkv, PAGE, d), dtype=codes, device=DEVICE),
             vc=torch.empty((total, hkv, PAGE, d), dtype=codes, device=DEVICE),
             scales=torch.empty((total, hkv, 2, PAGE), device=DEVICE))
    # What the cache holds already.
    for i, c in enumerate((s["kc"], s["vc"])):
        x = _rows((total, PAGE, hkv, d), g, dt).transpose(1, 2)
        code, scale = _quantised(x, codes)
        c.view(torch.uint8).copy_(code.view(torch.uint8))
        s["scales"][:, :, i] = scale
        del x, code, scale
    if case["kind"] == "decode":
        s["q"] = _randn((batch, s["heads"][0], d), g, dt, case["q_std"])
        if own:
            from gpu_offloading_amd import quantized

            s["workspace"] = quantized.decode_workspace(batch, *s["heads"], device=DEVICE)
        return s
    n = sum(new)
    seq = np.repeat(np.arange(batch), new)
    pos = np.concatenate([np.arange(a, a + m) for a, m in zip(past, new)])
    s.update(first=_ints(_indptr(new)), start=_ints(past), most=max(new),
             seq=_ints(seq, torch.int64), pos=_ints(pos, torch.int64),
             out_k=torch.empty((n, hkv, d), dtype=dt, device=DEVICE),
             out_v=torch.empty((n, hkv, d), dtype=dt, device=DEVICE))
    if case["kind"] == "write":
        if case["fused"]:
            qkv = _rows((n, 6 * hkv, d), g, dt)
            s.update(k=qkv[:, 4 * hkv:5 * hkv], v=qkv[:, 5 * hkv:])
        else:
            s.update(k=_rows((n, hkv, d), g, dt), v=_rows((n, hkv, d), g, dt))
        s["slots"] = s["table"].long()[s["seq"], s["pos"] // PAGE] * PAGE + s["pos"] % PAGE
    return s


# ------------------------------------------------------------- plain forms
def _quantised(x, codes):
    """Codes and fp32 scales of rows ``[..., head_dim]``."""
    x = x.float()
    amax = x.abs().amax(-1).clamp_min(TINY)
    if codes is torch.int8:
        code = (x * (127.0 / amax)[..., None]).round_().to(torch.int8)
        return code, amax / 127.0
    m, e = torch.frexp(amax)                       # amax = m 2^e, 1/2 <= m < 1;  448 = 7/8 2^9
    e = e - 9 + (m > 0.875).to(torch.int32)
    up, down = (((127 + i) << 23).view(torch.float32) for i in (e, -e))          # 2^e, 2^-e
    return (x * down[..., None]).to(torch.float8_e4m3fn), up


def _values(s, blk, off):
    """K and V in 32 bits of the tokens at slots ``off`` of blocks ``blk`` (any shape): [..., heads, dim]."""
    got = []
    for i, c in enumerate((s["kc"], s["vc"])):
        code = c.view(torch.uint8)[blk, :, off].view(c.dtype).float()
        got.append(code.mul_(s["scales"][blk, :, i, off][..., None]))
    return got


def _plain_write(s):
    blk, off = s["slots"] // PAGE, s["slots"] % PAGE
    for i, (x, c) in enumerate(((s["k"], s["kc"]), (s["v"], s["vc"]))):
        code, scale = _quantised(x, c.dtype)
        c.view(torch.uint8)[blk, :, off] = code.view(torch.uint8)
        s["scales"][blk, :, i, off] = scale


def _plain_read(s):
    blk = s["table"].long()[s["seq"], s["pos"] // PAGE]
    k, v = _values(s, blk, s["pos"] % PAGE)
    s["out_k"].copy_(k)
    s["out_v"].copy_(v)
    return s["out_k"], s["out_v"]


def _plain_decode(s):
    hq, hkv, d = s["heads"]
    at = torch.arange(s["top"], device=DEVICE)
    blk = s["table"].long().clamp_min(0)[:, at // PAGE]                          # [batch, top]
    k, v = (x.transpose(1, 2) for x in _values(s, blk, (at % PAGE).expand_as(blk)))
    q = (s["q"].float() / math.sqrt(d)).unflatten(1, (hkv, hq // hkv))
    p = torch.matmul(k, q.transpose(2, 3).contiguous())                          # [batch, hkv, top, group]
    p.masked_fill_((at[None, :] >= s["lens"][:, None])[:, None, :, None], -math.inf)
    top = p.amax(2, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)                                      # a sequence of no tokens
    p.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    out = torch.matmul(p.transpose(2, 3).contiguous(), v) / total.transpose(2, 3).clamp_min(TINY)
    lse = (top + total.log()).flatten(1)
    return out.flatten(1, 2).to(s["dtype"]), lse


# --------------------------------------------------------------------- run
def run(s):
    if not own:
        if s["kind"] == "decode":
            return _plain_decode(s)
        if s["kind"] == "write":
            _plain_write(s)
        return _plain_read(s)
    from gpu_offloading_amd import quantized

    cache = s["kc"], s["vc"], s["scales"]
    if s["kind"] == "decode":
        return quantized.quantized_decode_attention(s["q"], *cache, s["indptr"], s["indices"],
                                                    s["lpl"], return_lse=True,
                                                    workspace=s["workspace"])
    if s["kind"] == "write":
        quantized.reshape_and_cache_quantized(s["k"], s["v"], *cache, s["slots"])
    return quantized.gather_quantized_kv(*cache, s["table"], s["first"], s["most"], s["out_k"],
                                         s["out_v"], s["start"])


# -------------------------------------------------------------------- work
def work(case):
    hkv, d = case["hkv"], case["dim"]
    t = sum(_shape(case)[1])
    codes, values = 2 * t * hkv * (d + 4), 2 * t * hkv * d * 2
    if case["kind"] == "decode":
        hq = hkv * case["group"]
        return dict(bytes=codes + case["batch"] * hq * (4 * d + 4), flops=4 * d * hq * t)
    if case["kind"] == "write":
        return dict(bytes=2 * values + codes + 8 * t, flops=0)
    return dict(bytes=values + codes, flops=0)


# ------------------------------------------------------------------- exact
def _power_of_two(x):
    """The largest power of two that is not above x > 0, in 64 bits."""
    return (x.view(torch.int64) >> 52 << 52).view(torch.float64)


def _exact_rows(x, codec):
    """What the codes of rows ``x`` stand for, in 64 bits."""
    x = x.double()
    amax = x.abs().max(-1, keepdim=True).values.clamp_min(TINY)
    if codec == "int8":
        return torch.round(x / amax * 127.0) * (amax / 127.0)
    scale = _power_of_two(amax / 448.0)
    scale = torch.where(scale * 448.0 < amax, 2.0 * scale, scale)
    y = x / scale
    # e4m3: three bits after the leading one, exponents from -6 on
    step = _power_of_two(y.abs().clamp_min(2.0 ** -6)) / 8.0
    return torch.round(y / step) * step * scale


def _exact_cache(case, s, page, h):
    """K and V ``[tokens, dim]`` of head h of the blocks ``page``, in 64 bits."""
    got = []
    for i, c in enumerate((s["kc"], s["vc"])):
        code = c.view(torch.uint8)[page, h].long()
        if case["codec"] == "int8":
            code = torch.where(code > 127, code - 256, code).double()
        else:
            e, m = (code // 8) % 16, (code % 8).double()
            code = torch.where(code >= 128, -1.0, 1.0).double() * torch.where(
                e > 0, (8 + m) * (e + 1013 << 52).view(torch.float64), m / 512.0)
        got.append((code * s["scales"][page, h, i].double()[..., None]).flatten(0, 1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = s["heads"]
    if case["kind"] == "write":
        return _exact_rows(s["k"], case["codec"]), _exact_rows(s["v"], case["codec"])
    past, new = _shape(case)
    first, at = _indptr(new), s["indptr"].tolist()
    if case["kind"] == "read":
        k, v = (torch.empty((first[-1], hkv, d), dtype=torch.float64, device=DEVICE) for _ in "kv")
    else:
        k = torch.zeros((len(new), hq, d), dtype=torch.float64, device=DEVICE)
        v = torch.full((len(new), hq), -math.inf, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(new):
        page = s["indices"][at[b]:at[b + 1]].long()
        for h in range(hkv if n else 0):
            ck, cv = (x[past[b]:past[b] + n] for x in _exact_cache(case, s, page, h))
            if case["kind"] == "read":
                k[first[b]:first[b + 1], h], v[first[b]:first[b + 1], h] = ck, cv
                continue
            mine = slice(h * hq // hkv, (h + 1) * hq // hkv)
            x = s["q"][b, mine].double() @ ck.t() / math.sqrt(d)
            v[b, mine] = torch.logsumexp(x, 1)
            k[b, mine] = torch.exp(x - v[b, mine, None]) @ cv
    return k, v
