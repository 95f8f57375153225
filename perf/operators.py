"""Performance cases of prompt attention and of eviction by attention weight.

Each case is one pass through an operator as a serving program calls it:

  prompt   attention of whole prompts over their own contiguous K/V, packed
           one after another (``BatchPromptAttentionWrapper.run``), with the
           log-sum-exp that the weights below need
  weights  the attention weight that each cached token of a paged cache
           receives from a chunk's queries, or from the last ones of a
           prompt, accumulated (``BatchAttentionWeightsWrapper.run``)
  token    the same for a decode step, one query token per sequence
           (``ops.decode_attention_weights``)
  evict    the tokens of least weight of every sequence and KV head give
           their slots to later ones that stay (``ops.evict_kv``), after the
           engine put its own (smoothed) scores into the cache's array
  turn     a chat turn in a bounded cache: every sequence is evicted back to
           its bound, the turn's tokens are appended and their attention
           weights accumulated

With ``own`` false a pass computes the same in elementary torch operations
in 32 bits.  ``listed()`` are fixed cases, ``draw(rng)`` gives further ones of
the same ranges.  Pages are 16 tokens from a seeded permuted pool; K, V and Q
are normal, logits have a standard deviation of ``q_std``.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEVICE = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One interactive request: a prompt just past 128 tokens, Mixtral heads.
        dict(name="prompt_b1_129", kind="prompt", batch=1, lo=129, hi=129, hkv=8, group=4,
             dim=128, dtype="bfloat16", causal=True, fused=False, q_std=1.0, lens_seed=0),
        # A step that admits 16 prompts of a chat load, q/k/v being slices of
        # the projection's one output tensor.
        dict(name="prompt_b16_ragged", kind="prompt", batch=16, lo=17, hi=2000, hkv=8, group=4,
             dim=128, dtype="bfloat16", causal=True, fused=True, q_std=1.0, lens_seed=1),
        # One long document.
        dict(name="prompt_b1_16k", kind="prompt", batch=1, lo=16384, hi=16384, hkv=8, group=4,
             dim=128, dtype="bfloat16", causal=True, fused=False, q_std=2.0, lens_seed=0),
        # fp16, head_dim 64, eight query heads per KV head.
        dict(name="prompt_b8_d64_fp16", kind="prompt", batch=8, lo=500, hi=3001, hkv=8, group=8,
             dim=64, dtype="float16", causal=True, fused=False, q_std=1.0, lens_seed=5),
        # head_dim 256 without a causal mask (prefix or encoder tokens).
        dict(name="prompt_b4_d256_full", kind="prompt", batch=4, lo=700, hi=1500, hkv=4, group=2,
             dim=256, dtype="bfloat16", causal=False, fused=False, q_std=1.0, lens_seed=2),
        # The last 32 tokens of 8 prompts vote on the 4096 cached ones.
        dict(name="weights_8x4096_window", kind="weights", batch=8, q_lo=32, q_hi=32, lo=4096,
             hi=4096, fresh="all", hkv=8, group=4, dim=128, dtype="bfloat16", q_std=1.0,
             lens_seed=0),
        # Every token of 4 prompts votes, ragged lengths.
        dict(name="weights_4_prompts", kind="weights", batch=4, q_lo=4096, q_hi=4096, lo=1200,
             hi=2048, fresh="all", hkv=8, group=4, dim=128, dtype="bfloat16", q_std=1.0,
             lens_seed=3),
        # A decode step of one short request.
        dict(name="token_b1_129", kind="token", batch=1, lo=129, hi=129, hkv=8, group=4, dim=128,
             dtype="bfloat16", q_std=1.0, lens_seed=0),
        # The serving decode step of the benchmark: Mixtral shape, 64 requests.
        dict(name="token_b64_mixtral", kind="token", batch=64, lo=512, hi=4096, hkv=8, group=4,
             dim=128, dtype="bfloat16", q_std=1.0, lens_seed=2),
        # Prompts cut to a bound of 1024 tokens after prefill, 64 requests.
        dict(name="evict_b64_to_1024", kind="evict", batch=64, lo=512, hi=4096, keep=1024,
             recent=64, hkv=8, dim=128, dtype="bfloat16", lens_seed=2),
        # Long contexts cut to an eighth.
        dict(name="evict_b16_32k_to_4096", kind="evict", batch=16, lo=32767, hi=32767, keep=4096,
             recent=128, hkv=8, dim=128, dtype="bfloat16", lens_seed=0),
        # A chat turn of up to 200 tokens over 2048 that stay of each cache.
        dict(name="turn_b8_2048", kind="turn", batch=8, q_lo=20, q_hi=200, keep=2048, recent=32,
             hkv=8, group=4, dim=128, dtype="bfloat16", q_std=1.0, lens_seed=4),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    hi = max(lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "weights", "weights", "token", "token",
                       "evict", "turn"])
    ls = rng.randrange(1 << 20)
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    group, dim = rng.choice([1, 2, 3, 4, 4, 8]), rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    batch = _log(rng, 1, 32)
    heads = hkv * group
    if kind == "prompt":
        # at most a quarter of the pairs of 16384 causal tokens with 32 heads
        hi = _log(rng, 2, min(8000, int(math.sqrt((1 << 31) / (batch * heads)))))
        return dict(kind=kind, batch=batch, lo=max(1, int(hi * rng.uniform(0.1, 1.0))), hi=hi,
                    hkv=hkv, group=group, dim=dim, dtype=dtype, causal=rng.random() < 0.8,
                    fused=rng.random() < 0.5, q_std=rng.choice([1.0, 2.0]), lens_seed=ls)
    if kind == "weights":
        q_hi = _log(rng, 2, 2000)
        most = min(16000, (1 << 30) // (batch * heads * q_hi), (1 << 18) * 8 // (batch * hkv))
        hi = _log(rng, min(q_hi, most), most)
        return dict(kind=kind, batch=batch, q_lo=max(1, int(q_hi * rng.uniform(0.3, 1.0))),
                    q_hi=q_hi, lo=max(1, int(hi * rng.uniform(0.2, 1.0))), hi=hi,
                    fresh=rng.choice(["all", "queries"]), hkv=hkv, group=group, dim=dim,
                    dtype=dtype, q_std=1.0, lens_seed=ls)
    if kind == "token":
        batch = _log(rng, 1, 128)
        hi = _log(rng, 2, min(32767, (1 << 30) // (batch * hkv * dim * 4)))
        return dict(kind=kind, batch=batch, lo=max(1, int(hi * rng.uniform(0.1, 1.0))), hi=hi,
                    hkv=hkv, group=group, dim=dim, dtype=dtype, q_std=1.0, lens_seed=ls)
    if kind == "evict":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 40, min(32767, (1 << 30) // (batch * hkv * dim * 4)))
        keep = max(1, int(hi * rng.uniform(0.1, 0.9)))
        return dict(kind=kind, batch=batch, lo=max(1, int(hi * rng.uniform(0.2, 1.0))), hi=hi,
                    keep=keep, recent=min(keep, _log(rng, 1, 200)), hkv=hkv, dim=dim,
                    dtype=dtype, lens_seed=ls)
    q_hi = _log(rng, 2, 400)
    batch = min(batch, 16)
    keep = _log(rng, 50, min(6000, (1 << 29) // (batch * heads * q_hi)))
    return dict(kind=kind, batch=batch, q_lo=max(1, q_hi // 4), q_hi=q_hi, keep=keep,
                recent=min(keep, _log(rng, 1, 100)), hkv=hkv, group=group, dim=dim, dtype=dtype,
                q_std=1.0, lens_seed=ls)


# ------------------------------------------------------------------ inputs
def _lens(case, lo, hi, salt=0):
    """The case's ragged lengths (part of the case, not of the inputs)."""
    r = random.Random(case["lens_seed"] * 8 + salt)
    return [r.randint(min(lo, hi), hi) for _ in range(case["batch"])]


def _shape(case):
    """(tokens cached, query tokens, tokens that get their first score) of each sequence."""
    if case["kind"] == "turn":
        q = _lens(case, case["q_lo"], case["q_hi"], 1)
        return [case["keep"] + n for n in q], q, q
    n = _lens(case, case["lo"], case["hi"])
    if case["kind"] == "weights":
        q = [min(a, b) for a, b in zip(_lens(case, case["q_lo"], case["q_hi"], 1), n)]
        return n, q, (n if case["fresh"] == "all" else q)
    return n, [1] * len(n), [1] * len(n)


def _randn(shape, g, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _indptr(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _table(lens, seed):
    """Block-table rows from a seeded permuted pool, padded with -1, and the pool's size."""
    total = sum(_pages(n) for n in lens) + 2
    order = list(range(total))
    random.Random(seed).shuffle(order)
    at = _indptr([_pages(n) for n in lens])
    width = max(_pages(n) for n in lens)
    return [order[a:b] + [-1] * (width - b + a) for a, b in zip(at, at[1:])], total


def _where(lens, last=None):
    """Of every sequence's last ``last`` tokens (default: all), packed: the sequence and the slot."""
    last = lens if last is None else last
    seq = np.repeat(np.arange(len(lens)), last)
    slot = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, last)])
    return _ints(seq, torch.int64), _ints(slot, torch.int64)


def prepare(case, seed):
    kind, dt = case["kind"], getattr(torch, case["dtype"])
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    lens, qlens, fresh = _shape(case)
    hkv, d = case["hkv"], case["dim"]
    hq = hkv * case.get("group", 1)
    s = dict(kind=kind, heads=(hq, hkv, d), scale=1.0 / math.sqrt(d))
    if kind == "prompt":
        t = sum(lens)
        if case["fused"]:
            qkv = _randn((t, hq + 2 * hkv, d), g, dt)
            qkv[:, :hq] *= case["q_std"]
            s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
        else:
            s.update(q=_randn((t, hq, d), g, dt, case["q_std"]), k=_randn((t, hkv, d), g, dt),
                     v=_randn((t, hkv, d), g, dt))
        seq, slot = _where(lens)
        s.update(lens=_ints(lens), top=max(lens), seq=seq, slot=slot, causal=case["causal"],
                 first=_ints(_indptr(lens), torch.int64))
        if own:
            from gpu_offloading_amd.prompt import BatchPromptAttentionWrapper

            w = BatchPromptAttentionWrapper(torch.empty(1 << 20, dtype=torch.uint8, device=DEVICE))
            w.plan(torch.tensor(_indptr(lens), dtype=torch.int32), num_qo_heads=hq,
                   num_kv_heads=hkv, head_dim=d, causal=case["causal"], q_data_type=dt)
            s["wrapper"] = w
        return s

    rows, total = _table(lens, seed)
    cache = _randn((total, 2, PAGE, hkv, d), g, dt)
    seq, slot = _where(lens)
    s.update(kc=cache[:, 0], vc=cache[:, 1], table=_ints(rows), lens=_ints(lens), top=max(lens),
             seq=seq, slot=slot,
             scores=torch.empty((total, hkv, PAGE), device=DEVICE).exponential_(generator=g))
    if kind in ("evict", "turn"):
        # Smoothed scores that the engine made of the attention weights.
        s.update(pooled=torch.empty((total, hkv, PAGE), device=DEVICE).exponential_(generator=g),
                 keep=_ints([min(n, case["keep"]) for n in lens]),
                 recent=_ints([min(n, case["recent"]) for n in lens]))
    if kind == "evict":
        return s

    s.update(q=_randn((sum(qlens), hq, d), g, dt, case["q_std"]), qlens=_ints(qlens),
             q_first=_ints(_indptr(qlens), torch.int64), q_top=max(qlens),
             fresh=_ints(fresh), positions=torch.zeros((total, hkv, PAGE), dtype=torch.int32,
                                                       device=DEVICE))
    # The log-sum-exp as the attention over these keys returned it: normal logits of variance v
    # over n keys have log(n) + v/2, give or take.
    qseq, qslot = _where(lens, qlens)
    s.update(qseq=qseq, qslot=qslot)
    s["lse"] = ((qslot + 1).float().log() + case["q_std"] ** 2 / 2)[:, None] + \
        0.1 * torch.empty((sum(qlens), hq), device=DEVICE).normal_(generator=g)
    # Tokens evicted from each sequence earlier: slot + offset is a new token's position.
    off = [random.Random(i * 7 + case["lens_seed"]).randrange(1000) if kind == "turn" else 0
           for i in range(len(lens))]
    s["offsets"] = _ints(off)
    if kind == "turn":
        s.update(k=_randn((sum(qlens), hkv, d), g, dt), v=_randn((sum(qlens), hkv, d), g, dt))
        # Positions of a cache that was evicted before: the kept tokens in any order, then the
        # last turn's.
        for b, n in enumerate(lens):
            old = torch.argsort(torch.rand((hkv, case["keep"]), device=DEVICE, generator=g))
            t = torch.arange(n, device=DEVICE)
            place = torch.cat([old, t[case["keep"]:].expand(hkv, -1)], 1) + off[b]
            s["positions"][s["table"][b].long()[t // PAGE], :, t % PAGE] = place.to(torch.int32).t()
        s["slots"] = s["table"].long()[qseq, qslot // PAGE] * PAGE + qslot % PAGE
    pages = [_pages(n) for n in lens]
    s["indptr"] = _ints(_indptr(pages))
    s["indices"] = torch.cat([s["table"][b, :n] for b, n in enumerate(pages)])
    s["lpl"] = _ints([(n - 1) % PAGE + 1 for n in lens])
    if own and kind != "token":
        from gpu_offloading_amd.eviction import BatchAttentionWeightsWrapper

        w = BatchAttentionWeightsWrapper(torch.empty(1 << 20, dtype=torch.uint8, device=DEVICE))
        w.plan(torch.tensor(_indptr(qlens), dtype=torch.int32), s["indptr"].cpu(), s["indices"],
               s["lpl"].cpu(), num_qo_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=PAGE,
               q_data_type=dt, new_tokens=torch.tensor(fresh, dtype=torch.int32))
        s["wrapper"] = w
    return s


# ------------------------------------------------------------- plain forms
def _padded(x, first, lens, top):
    """Packed rows as [batch, heads, top, dim] in 32 bits (rows past a sequence repeat its last)."""
    at = torch.arange(top, device=x.device)[None, :].minimum((lens.long() - 1).clamp_min(0)[:, None])
    return x[(first[:-1, None] + at).clamp_max(x.shape[0] - 1)].float().transpose(1, 2)


def _plain_prompt(s):
    hq, hkv, d = s["heads"]
    q = _padded(s["q"], s["first"], s["lens"], s["top"])
    k = _padded(s["k"], s["first"], s["lens"], s["top"]).repeat_interleave(hq // hkv, 1)
    v = _padded(s["v"], s["first"], s["lens"], s["top"]).repeat_interleave(hq // hkv, 1)
    at = torch.arange(s["top"], device=q.device)
    hidden = (at[None, :] >= s["lens"][:, None])[:, None, None, :]
    if s["causal"]:
        hidden = hidden | (at[None, :] > at[:, None])[None, None]
    p = torch.matmul(q * s["scale"], k.transpose(2, 3).contiguous())
    p.masked_fill_(hidden, -math.inf)
    top = p.amax(3, keepdim=True)
    p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p, v).div_(total)
    lse = (top + total.log())[..., 0]
    return (out[s["seq"], :, s["slot"]].to(s["q"].dtype).contiguous(),
            lse[s["seq"], :, s["slot"]].contiguous())


def _plain_weights(s):
    """Adds each cached token's weight to ``scores``; new tokens start from it."""
    hq, hkv, d = s["heads"]
    group, table, lens = hq // hkv, s["table"].long(), s["lens"].long()
    q = _padded(s["q"], s["q_first"], s["qlens"], s["q_top"])
    k = s["kc"][table.clamp_min(0)].float().flatten(1, 2)[:, :s["top"]].transpose(1, 2)
    x = torch.matmul((q * s["scale"]).unflatten(1, (hkv, group)).flatten(2, 3),
                     k.transpose(2, 3).contiguous())
    lse = _padded(s["lse"][..., None], s["q_first"], s["qlens"], s["q_top"])
    at = torch.arange(s["top"], device=q.device)
    row = torch.arange(s["q_top"], device=q.device)
    sees = lens[:, None] - s["qlens"].long()[:, None] + row[None, :]          # last key that row sees
    seen = (at[None, None, :] <= sees[:, :, None]) & (row[None, :] < s["qlens"][:, None])[:, :, None]
    p = x.unflatten(2, (group, -1)).sub_(lse.unflatten(1, (hkv, group))).exp_()
    w = p.masked_fill_(~seen[:, None, None], 0.0).sum((2, 3))                  # [batch, hkv, top]
    blk, off = table[s["seq"], s["slot"] // PAGE], s["slot"] % PAGE
    new = s["slot"] >= (lens - s["fresh"].long())[s["seq"]]
    w = w[s["seq"], :, s["slot"]]
    s["scores"][blk, :, off] = torch.where(new[:, None], w, s["scores"][blk, :, off] + w)
    place = (s["slot"] + s["offsets"].long()[s["seq"]]).to(torch.int32)
    s["positions"][blk, :, off] = torch.where(new[:, None], place[:, None],
                                              s["positions"][blk, :, off])


def _plain_evict(s, positions):
    """Keeps, per sequence and KV head, the recent tokens and those of the largest scores."""
    hkv = s["heads"][1]
    table, lens, keep = s["table"].long(), s["lens"].long(), s["keep"].long()
    at = torch.arange(s["top"], device=table.device)
    blk, off = table[:, at // PAGE].clamp_min(0), at % PAGE                    # [batch, top], [top]
    score = s["scores"][blk, :, off[None]].transpose(1, 2)                     # [batch, hkv, top]
    place = at.expand_as(score) if positions is None else \
        positions[blk, :, off[None]].transpose(1, 2).long()
    end = lens if positions is None else lens + s["offsets"].long()
    recent = place >= (end - s["recent"].long())[:, None, None]
    inside = (at[None, :] < lens[:, None])[:, None, :].expand_as(score)
    # Rank: tokens of the sequence, recent ones, larger scores, lower slots first.
    order = torch.sort(score, dim=2, descending=True, stable=True).indices
    for flag in (recent, inside):
        pick = torch.sort(flag.gather(2, order).to(torch.uint8), dim=2, descending=True,
                          stable=True).indices
        order = order.gather(2, pick)
    kept = torch.zeros_like(inside).scatter(2, order, (at[None, :] < keep[:, None])[:, None]
                                            .expand_as(inside).contiguous())
    low = (at[None, :] < keep[:, None])[:, None]
    dst, src = (low & ~kept).nonzero(as_tuple=True), (~low & kept).nonzero(as_tuple=True)
    to, frm = ((blk[b, t], off[t], h) for b, h, t in (dst, src))
    for cache in (s["kc"], s["vc"]):
        cache[to] = cache[frm]
    to, frm = ((a, h, o) for a, o, h in (to, frm))
    for x in (s["scores"],) if positions is None else (s["scores"], positions):
        x[to] = x[frm]


# --------------------------------------------------------------------- run
def run(s):
    kind = s["kind"]
    if kind == "prompt":
        if own:
            return s["wrapper"].run(s["q"], s["k"], s["v"], return_lse=True)
        return _plain_prompt(s)
    if own:
        from gpu_offloading_amd import ops
    if kind in ("evict", "turn"):
        s["scores"].copy_(s["pooled"])
        seen = (s["positions"], s["offsets"]) if kind == "turn" else (None, None)
        if own:
            ops.evict_kv(s["kc"], s["vc"], s["scores"], s["table"], s["lens"], s["keep"],
                         s["recent"], s["top"], *seen)
        else:
            _plain_evict(s, seen[0])
    if kind == "evict":
        return s["kc"], s["vc"], s["scores"]
    if kind == "turn":
        s["offsets"].add_(s["lens"] - s["keep"])
        if own:
            ops.reshape_and_cache_flash(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        else:
            s["kc"][s["slots"] // PAGE, s["slots"] % PAGE] = s["k"]
            s["vc"][s["slots"] // PAGE, s["slots"] % PAGE] = s["v"]
    if not own:
        _plain_weights(s)
    elif kind == "token":
        ops.decode_attention_weights(s["q"], s["lse"], s["kc"], s["indptr"], s["indices"],
                                     s["lpl"], s["scores"], s["positions"], s["offsets"])
    else:
        s["wrapper"].run(s["q"], s["lse"], s["kc"], s["scores"], s["positions"], s["offsets"])
    if kind == "turn":
        return s["kc"], s["vc"], s["scores"], s["positions"]
    return s["scores"], s["positions"]


# -------------------------------------------------------------------- work
def _pairs(n, q, causal=True):
    """(query, key) pairs of the last q of n tokens."""
    return q * n - (q * (q - 1) // 2 if causal else 0)


def work(case):
    lens, qlens, _ = _shape(case)
    hkv, d = case["hkv"], case["dim"]
    hq, t = hkv * case.get("group", 1), sum(lens)
    if case["kind"] == "prompt":
        pairs = sum(_pairs(n, n, case["causal"]) for n in lens)
        return dict(bytes=t * (2 * hq + 2 * hkv) * d * 2 + 4 * t * hq, flops=4 * d * hq * pairs)
    moved = 0.0
    if case["kind"] in ("evict", "turn"):
        # Kept tokens above the bound: the recent ones and their share of the others.
        for n in lens:
            k = min(n, case["keep"])
            r = min(case["recent"], k, n - k)
            moved += r + (k - min(case["recent"], k)) * (n - k - r) / max(1, n - r)
    evict = moved * hkv * (4 * d * 2 + 8) + 4 * t * hkv
    if case["kind"] == "evict":
        return dict(bytes=evict + 8 * t * hkv, flops=0)
    q = sum(qlens)
    weights = t * hkv * (d * 2 + 8) + q * hq * (d * 2 + 4)
    flops = 2 * d * hq * sum(_pairs(n, m) for n, m in zip(lens, qlens))
    if case["kind"] == "turn":
        return dict(bytes=weights + evict + 8 * t * hkv + 8 * q * hkv * d, flops=flops)
    return dict(bytes=weights, flops=flops)


# ------------------------------------------------------------------- exact
def _exact_prompt(case, s):
    """Sequence by sequence and KV head by KV head in 64 bits."""
    hq, hkv, d = s["heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=DEVICE)
    at = _indptr(_shape(case)[0])
    for a, b in zip(at, at[1:]):
        i = torch.arange(b - a, device=DEVICE)
        for h in range(hq):
            k, v = (s[x][a:b, h * hkv // hq].double() for x in "kv")
            x = s["q"][a:b, h].double() @ k.t() / math.sqrt(d)
            if case["causal"]:
                x += torch.where(i[None, :] > i[:, None], -math.inf, 0.0)
            m = x.max(1).values
            e = torch.exp_(x.sub_(m[:, None]))
            z = e.sum(1)
            out[a:b, h] = (e @ v) / z[:, None]
            lse[a:b, h] = m + z.log()
    return out, lse


def _exact_weights(case, s):
    hq, hkv, d = s["heads"]
    lens, qlens, fresh = _shape(case)
    scores, positions = s["scores"].double(), s["positions"].clone()
    at = _indptr(qlens)
    for b, (n, m, f) in enumerate(zip(lens, qlens, fresh)):
        t = torch.arange(n, device=DEVICE)
        blk, off = s["table"][b].long()[t // PAGE], t % PAGE
        i = torch.arange(m, device=DEVICE)
        hide = t[None, :] > (n - m + i)[:, None]
        for h in range(hkv):
            k = s["kc"][blk, off, h].double()
            w = torch.zeros(n, dtype=torch.float64, device=DEVICE)
            for j in range(h * hq // hkv, (h + 1) * hq // hkv):
                x = s["q"][at[b]:at[b + 1], j].double() @ k.t() / math.sqrt(d)
                x = torch.exp(x - s["lse"][at[b]:at[b + 1], j].double()[:, None])
                w += torch.where(hide, 0.0, x).sum(0)
            old = scores[blk, h, off]
            scores[blk, h, off] = w + torch.where(t < n - f, old, 0.0)
            positions[blk, h, off] = torch.where(t < n - f, positions[blk, h, off],
                                                 (t + s["offsets"][b]).to(torch.int32))
    return scores, positions


def _exact_evict(case, s, scores, positions):
    """On the host, a sequence and a head at a time: which slot gets which token."""
    table, keep, recent = (s[x].cpu().numpy() for x in ("table", "keep", "recent"))
    lens = _shape(case)[0]
    sc = scores.cpu().numpy()
    ps = None if positions is None else positions.cpu().numpy()
    moves = []
    for b, n in enumerate(lens):
        t = np.arange(n)
        blk, off = table[b, t // PAGE], t % PAGE
        for h in range(s["heads"][1]):
            place = t if ps is None else ps[blk, h, off] - int(s["offsets"][b])
            first = np.lexsort((t, -sc[blk, h, off], place < n - recent[b]))[:keep[b]]
            stays = np.zeros(n, bool)
            stays[first] = True
            to, frm = t[:keep[b]][~stays[:keep[b]]], t[keep[b]:][stays[keep[b]:]]
            moves.append(np.stack([blk[to], off[to], blk[frm], off[frm], np.full(len(to), h)]))
    tb, to, fb, fo, h = torch.from_numpy(np.concatenate(moves, 1).astype(np.int64)).to(DEVICE)
    got = []
    for x in (s["kc"], s["vc"]):
        x = x.clone()
        x[tb, to, h] = x[fb, fo, h]
        got.append(x)
    for x in (scores, positions):
        if x is not None:
            x = x.clone()
            x[tb, h, to] = x[fb, h, fo]
            got.append(x)
    return tuple(got)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "prompt":
        return _exact_prompt(case, s)
    if kind == "evict":
        return _exact_evict(case, s, s["pooled"], None)
    if kind != "turn":
        return _exact_weights(case, s)
    s["kc"], s["vc"], s["scores"], s["positions"] = _exact_evict(case, s, s["pooled"],
                                                                 s["positions"])
    s["offsets"] = s["offsets"] + _ints([n - case["keep"] for n in _shape(case)[0]])
    for cache, new in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        cache[s["slots"] // PAGE, s["slots"] % PAGE] = new
    return s["kc"], s["vc"], *_exact_weights(case, s)
