"""GPU tests of the quantised cache's ops: the write bit for bit against its definition, the
read-back against the same codes rounded once, decode attention against 64 bits within
derived bounds; lengths from none to long ones, pages in any order, slots that hold
garbage, strides, streams, graphs, offsets past 4 GiB."""
import math

import numpy as np
import pytest
import torch

import quant_ref as ref
from gpu_offloading_amd import quantized as qz

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def bits(t):
    return t.detach().cpu().contiguous().view(torch.uint8).numpy()


def rows(shape, seed, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return (torch.randn(*shape, generator=g) * size).to(dtype)


def poisoned(blocks, h, d, codec, device):
    """A cache in which every code and scale is something that must not be used."""
    c = qz.quantized_cache(blocks, h, d, codec, device)
    c.storage.fill_(0x7f)
    c.scales.fill_(float("nan"))
    return c


# ------------------------------------------------------------------- write
def check_written(cache, key, value, slots, codec):
    """The slots hold the rows' codes and scales, all others what ``poisoned`` left."""
    for x, c, i in ((key, cache.key_cache, 0), (value, cache.value_cache, 1)):
        codes, scale = ref.encode(x[:len(slots)], codec)
        got, gots = bits(c), cache.scales[:, :, i].cpu().numpy()
        want, wants = np.full(got.shape, 0x7f, np.uint8), np.full(gots.shape, np.nan, np.float32)
        skip = np.zeros(gots.shape, bool)
        for t, s in enumerate(slots):
            if 0 <= s < c.shape[0] * 16:
                want[s // 16, :, s % 16] = codes[t]
                wants[s // 16, :, s % 16] = scale[t]
                skip[s // 16, :, s % 16] = np.isnan(scale[t])
        assert np.array_equal(gots, wants, equal_nan=True)
        assert np.array_equal(got[~skip], want[~skip])


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,d", [(1, 64), (3, 128), (8, 128), (2, 256)])
@pytest.mark.parametrize("n", [1, 15, 33, 130])
def test_write(gpu, codec, dtype, h, d, n):
    cache = poisoned(12, h, d, codec, gpu)
    k, v = rows((n, h, d), n, dtype, 2.0), rows((n, h, d), n + 1, dtype, 2.0)
    slots = np.random.default_rng(n).permutation(12 * 16)[:n]
    slots[::7] = -1
    qz.reshape_and_cache_quantized(k.to(gpu), v.to(gpu), cache.key_cache, cache.value_cache,
                                   cache.scales, torch.from_numpy(slots).to(gpu))
    check_written(cache, k, v, slots, codec)


@pytest.mark.parametrize("codec", ref.CODECS)
def test_write_special_rows(gpu, codec):
    """Rows of zeros, of the smallest and the largest values, of ties, with infinities and NaN."""
    h, d = 2, 128
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    k = torch.zeros(9, h, d)
    k[1] = tiny
    k[2] = -big
    k[2, :, ::3] = big / 3
    k[3] = torch.arange(d) - 64.0
    k[4] = 2.0 ** -101
    k[4, :, 5] = -2.0 ** -100
    k[5, 0, 7] = math.inf
    k[6, 1, 100] = -math.nan
    k[7] = 448 * 2.0 ** -6
    k[7, 1] = 450                          # above 1.75 * 2^8: the next scale
    k[8] = torch.linspace(-1, 1, d)
    k = k.to(torch.bfloat16)
    v = k.flip(0).contiguous()
    cache = poisoned(2, h, d, codec, gpu)
    slots = torch.arange(9, device=gpu) + 5
    qz.reshape_and_cache_quantized(k.to(gpu), v.to(gpu), *cache[:3], slots)
    check_written(cache, k, v, slots.tolist(), codec)
    # what is not finite reads back as NaN, in its own token and head only
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 9], dtype=torch.int32, device=gpu)
    gk, gv = qz.gather_quantized_kv(*cache[:3], table, cu, 9,
                                    seq_starts=torch.tensor([5], dtype=torch.int32, device=gpu))
    bad = torch.zeros(9, h, dtype=torch.bool)
    bad[5, 0] = bad[6, 1] = True
    assert torch.equal(gk.isnan().all(-1).cpu(), bad) and torch.equal(gk.isnan().any(-1).cpu(), bad)
    assert torch.equal(gv.isnan().any(-1).cpu(), bad.flip(0))


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_largest_values_stay_finite(gpu, codec, dtype):
    """Rows with values up to the type's largest, read back and attended to."""
    h, d, n = 2, 128, 20
    big = torch.finfo(dtype).max
    x = rows((n, h, d), 3, torch.float32, 0.0).clamp(-2, 2) / 2
    x[::2, :, 5], x[1::3, 1, 9] = 1, -1
    x = (x.double() * big).to(dtype)
    assert x.isfinite().all() and x.abs().max() == big
    cache = poisoned(2, h, d, codec, gpu)
    slots = torch.arange(n, device=gpu)
    qz.reshape_and_cache_quantized(x.to(gpu), x.to(gpu), *cache[:3], slots)
    check_written(cache, x, x, slots.tolist(), codec)
    gk, gv = qz.gather_quantized_kv(*cache[:3], ints([[0, 1]], gpu), ints([0, n], gpu), n,
                                    dtype=dtype)
    # Half a step of e4m3 (2^-4; 2^-10 of the scale, at most amax / 224, near zero; 255.9375 as 240 is
    # within it) or of int8 (three fp32 roundings move a code by 127 * 3 * 2^-24 at most), and half a
    # step of the rows' type.
    amax = x.double().abs().amax(-1, keepdim=True)
    step = x.double().abs() / 16 + amax * 2.0 ** -16 if codec is ref.E4M3 else amax / 254 * 1.0002
    for got in (gk, gv):
        err = (got.cpu().double() - x.double()).abs()
        assert (err <= step + torch.finfo(dtype).eps / 2 * amax).all()
    if dtype is torch.float16:         # (sums over bf16's largest values are beyond fp32)
        q = rows((1, h, d), 4, dtype, 0.0).to(gpu) * 1e-4
        out = qz.quantized_decode_attention(q, *cache[:3], ints([0, 2], gpu), ints([0, 1], gpu),
                                            ints([n - 16], gpu))
        assert out.isfinite().all()


def test_write_strided_and_unaligned_sources(gpu):
    """Slices of a fused tensor, rows that are not 16-byte aligned, more rows than slots."""
    h, d, n = 4, 64, 37
    for codec in ref.CODECS:
        for pad in (0, 1, 4):
            fused = rows((n, 6 * h * d + pad), 3, torch.float16, 0.5).to(gpu)
            at = 2 * h * d + pad
            k = fused[:, at:at + h * d].unflatten(1, (h, d))
            v = fused[:, at + h * d:at + 2 * h * d].unflatten(1, (h, d))
            cache = poisoned(3, h, d, codec, gpu)
            slots = np.arange(n - 2)[::-1].copy()
            qz.reshape_and_cache_quantized(k, v, *cache[:3], torch.from_numpy(slots).to(gpu))
            check_written(cache, k, v, slots, codec)


def test_write_skips_and_counts_slots_past_the_end(gpu):
    cache = poisoned(3, 2, 128, ref.E4M3, gpu)
    k = rows((5, 2, 128), 1, torch.bfloat16)
    slots = np.array([48, 0, -1, 10 ** 12, 47])
    oob = torch.zeros(1, dtype=torch.int32, device=gpu)
    qz.reshape_and_cache_quantized(k.to(gpu), k.to(gpu), *cache[:3],
                                   torch.from_numpy(slots).to(gpu), oob_count=oob)
    assert int(oob) == 2
    check_written(cache, k, k, slots, ref.E4M3)
    qz.reshape_and_cache_quantized(k.to(gpu), k.to(gpu), *cache[:3],
                                   torch.empty(0, dtype=torch.int64, device=gpu))


# -------------------------------------------------------------------- read
def random_cache(lens, h, d, codec, device, seed, extra=3):
    """A poisoned cache holding sequences of random codes in permuted pages: (cache, table rows
    padded with -1, code values and scales of each sequence [2][n, H, D] / [2][n, H], on the host)."""
    rng = np.random.default_rng(seed)
    need = [(n + 15) // 16 for n in lens]
    blocks = sum(need) + extra
    c = poisoned(blocks, h, d, codec, device)
    codes = [bits(t).copy() for t in (c.key_cache, c.value_cache)]
    scales = np.full((blocks, h, 2, 16), np.nan, np.float32)
    scales[::2] = np.inf                       # (of slots that hold no token)
    order = rng.permutation(blocks)
    table = np.full((len(lens), max(need + [1]) + 1), -1, np.int32)
    held, at = [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        blk, off = table[b, t // 16], t % 16
        seq = []
        for i in range(2):
            x = rng.integers(0, 256, (n, h, d)).astype(np.uint8)
            if codec is ref.E4M3:
                x[(x & 127) == 127] = 0
                x = np.where(rng.random(x.shape) < 0.5, x & 0xbf, x)     # fewer large codes
            s = np.exp(rng.normal(-4.0, 1.0, (n, h))).astype(np.float32)
            codes[i][blk, :, off] = x
            scales[blk, :, i, off] = s
            seq.append((ref.values(x, codec), s))
        held.append(seq)
    for t, x in zip((c.key_cache, c.value_cache), codes):
        t.copy_(torch.from_numpy(x).view(t.dtype).to(device))
    c.scales.copy_(torch.from_numpy(scales))
    return c, table, held


def ints(x, device):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,d", [(1, 128), (8, 128), (3, 64), (2, 256)])
def test_read(gpu, codec, dtype, h, d):
    lens, starts = [40, 1, 0, 16, 333, 31], [7, 0, 0, 16, 160, 15]
    part = [33, 1, 0, 0, 100, 16]
    cache, table, held = random_cache(lens, h, d, codec, gpu, 1)
    cu = np.concatenate([[2], 2 + np.cumsum(part)])
    outs = [torch.full((cu[-1] + 3, h, d), 7.0, dtype=dtype, device=gpu) for _ in "kv"]
    got = qz.gather_quantized_kv(*cache[:3], ints(table, gpu), ints(cu, gpu), 100, *outs,
                                 ints(starts, gpu))
    for i, t in enumerate(got):
        assert t is outs[i]
        want = torch.full(t.shape, 7.0, dtype=dtype)
        for b, (n, s) in enumerate(zip(part, starts)):
            x, scale = (y[s:s + n] for y in held[b][i])
            want[cu[b]:cu[b + 1]] = (torch.from_numpy(x).float() *
                                     torch.from_numpy(scale)[..., None]).to(dtype)
        assert np.array_equal(bits(t), bits(want))


def test_read_whole_sequences_and_odd_outputs(gpu):
    """Outputs made by the call, and outputs whose rows are not 16-byte aligned."""
    h, d = 4, 64
    cache, table, held = random_cache([100, 17], h, d, ref.INT8, gpu, 2)
    cu = ints([0, 100, 117], gpu)
    gk, gv = qz.gather_quantized_kv(*cache[:3], ints(table, gpu), cu, 100, dtype=torch.float16)
    assert gk.dtype is gv.dtype is torch.float16 and gk.shape == (117, h, d)
    for i, t in enumerate((gk, gv)):
        want = torch.cat([torch.from_numpy(x).float() * torch.from_numpy(s)[..., None]
                          for x, s in (held[0][i], held[1][i])]).to(torch.float16)
        assert torch.equal(t.cpu(), want)
        room = torch.zeros(117 * (h * d + 3) + 1, dtype=torch.float16, device=gpu)
    wide = [room.clone()[1:].unflatten(0, (117, h * d + 3))[:, :h * d].unflatten(1, (h, d))
            for _ in "kv"]
    qz.gather_quantized_kv(*cache[:3], ints(table, gpu), cu, 100, *wide)
    assert torch.equal(wide[0], gk) and torch.equal(wide[1], gv)


def test_read_bad_places(gpu):
    """Missing pages read as zeros and are counted; rows past the outputs or past max_seq_len
    are left alone."""
    h, d = 2, 128
    cache, table, held = random_cache([64, 64], h, d, ref.E4M3, gpu, 3)
    table[0, 1], table[1, 2] = -1, 10 ** 6
    oob = torch.zeros(1, dtype=torch.int32, device=gpu)
    outs = [torch.full((120, h, d), 7.0, dtype=torch.bfloat16, device=gpu) for _ in "kv"]
    qz.gather_quantized_kv(*cache[:3], ints(table, gpu), ints([0, 64, 128], gpu), 60, *outs,
                           oob_count=oob)
    for i, t in enumerate(outs):
        want = torch.full(t.shape, 7.0, dtype=torch.bfloat16)
        for b in range(2):
            x, s = held[b][i]
            y = (torch.from_numpy(x).float() * torch.from_numpy(s)[..., None]).to(torch.bfloat16)
            y[16 * (b + 1):16 * (b + 2)] = 0
            m = min(60, 120 - 64 * b)
            want[64 * b:64 * b + m] = y[:m]
        assert torch.equal(t.cpu(), want)
    assert int(oob) == 32 + 4                  # two pages; rows 120 .. 123 of the second sequence
    # a range that begins before its sequence
    oob.zero_()
    qz.gather_quantized_kv(*cache[:3], ints(table[1:], gpu), ints([0, 20], gpu), 20, *outs,
                           ints([-5], gpu), oob_count=oob)
    assert int(oob) == 5 and not outs[0][:5].any()
    x, s = held[1][0]
    assert torch.equal(outs[0][5:20].cpu(), (torch.from_numpy(x).float() *
                                             torch.from_numpy(s)[..., None]).to(torch.bfloat16)[:15])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_e4m3_values_are_fixed_points(gpu, dtype, d):
    """What is read back and written again gives the same codes and scales."""
    h, n = 3, 50
    a, b = (poisoned(4, h, d, ref.E4M3, gpu) for _ in "ab")
    k, v = rows((n, h, d), 1, dtype).to(gpu), rows((n, h, d), 2, dtype).to(gpu)
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:n].to(gpu)
    table, cu = ints([[0, 1, 2, 3]], gpu), ints([0, 64], gpu)
    qz.reshape_and_cache_quantized(k, v, *a[:3], slots)
    gk, gv = qz.gather_quantized_kv(*a[:3], table, cu, 64, dtype=dtype)
    qz.reshape_and_cache_quantized(gk[slots], gv[slots], *b[:3], slots)
    rk, rv = qz.gather_quantized_kv(*b[:3], table, cu, 64, dtype=dtype)
    assert torch.equal(gk[slots], rk[slots]) and torch.equal(gv[slots], rv[slots])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_e4m3_rows_written_again_may_change_codes_but_not_values(gpu, dtype, d):
    """A row whose largest value is rounded down to 1.75 * 2^k is held with half the scale when what
    was read back is written again: other codes, as the definition has them, and the same values."""
    tops = torch.tensor([225.0, 231.0, 232.0, 233.0, 1.78125, 0.2197265625, 500.0, 300.0, 224.0])
    x = torch.rand(len(tops), 1, d, generator=torch.Generator().manual_seed(d)) * 2 - 1
    x = (x * 0.9 * tops[:, None, None]).to(dtype)
    x[:, 0, 5] = tops.to(dtype)
    halved = [True, True, True, False, True, True, False, False, False]   # (232 is a tie: 224 is even)
    n = len(tops)
    a, b = (poisoned(1, 1, d, ref.E4M3, gpu) for _ in "ab")
    table, cu, slots = ints([[0]], gpu), ints([0, n], gpu), torch.arange(n, device=gpu)
    qz.reshape_and_cache_quantized(x.to(gpu), x.to(gpu), *a[:3], slots)
    once, _ = qz.gather_quantized_kv(*a[:3], table, cu, n, dtype=dtype)
    qz.reshape_and_cache_quantized(once, once, *b[:3], slots)
    twice, _ = qz.gather_quantized_kv(*b[:3], table, cu, n, dtype=dtype)
    assert torch.equal(once, twice)
    held = []
    for c, rows_ in ((a, x), (b, once)):
        codes, scale = ref.encode(rows_[:, 0], ref.E4M3)
        assert np.array_equal(bits(c.key_cache)[0, 0, :n], codes)
        assert np.array_equal(c.scales[0, 0, 0, :n].cpu().numpy(), scale)
        held.append((codes, scale))
    (c0, s0), (c1, s1) = held
    assert (s1 == np.where(halved, s0 / 2, s0)).all()
    assert [(i != j).any() for i, j in zip(c0, c1)] == halved


# ------------------------------------------------------------------ decode
def pages(table, lens, first=0):
    need = [(n + 15) // 16 for n in lens]
    ip = np.concatenate([[0], np.cumsum(need)]) + first
    idx = np.concatenate([np.full(first, 10 ** 6, np.int32)] +
                         [table[b, :m] for b, m in enumerate(need)] + [np.zeros(0, np.int32)])
    return ip, idx, [(n - 1) % 16 + 1 if n else 0 for n in lens]


def check_decode(out, lse, q, held, lens, scale, dtype):
    hkv = held[0][0][0].shape[1]
    group = q.shape[1] // hkv
    for b, n in enumerate(lens):
        for h in range(hkv):
            g = slice(h * group, (h + 1) * group)
            (k, ks), (v, vs) = ((torch.from_numpy(x[:n, h]), torch.from_numpy(s[:n, h]))
                                for x, s in held[b])
            o, l, ot, lt = ref.attention(q[b, g].cpu(), k, ks, v, vs, scale, dtype)
            err, lerr = (out[b, g].cpu().double() - o).abs(), (lse[b, g].cpu().double() - l).abs()
            assert (err <= ot).all(), (b, h, n, (err / ot).max())
            if n:
                assert (lerr <= lt).all(), (b, h, n, (lerr / lt).max())
            else:
                assert (lse[b, g] == -math.inf).all() and not out[b, g].any()


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,group", [(1, 1), (2, 3), (8, 4), (1, 16), (3, 8)])
def test_decode(gpu, codec, dtype, d, hkv, group):
    lens = [1, 16, 17, 0, 33, 300, 15, 64, 0, 700]
    cache, table, held = random_cache(lens, hkv, d, codec, gpu, d + group)
    ip, idx, lpl = pages(table, lens)
    q = rows((len(lens), hkv * group, d), 5, dtype, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, dtype)


@pytest.mark.parametrize("dtype,hkv,group,d", [(torch.bfloat16, 8, 4, 128), (torch.float16, 4, 3, 64),
                                               (torch.bfloat16, 4, 2, 256)])
@pytest.mark.parametrize("longest", [320, 321, 800, 1100])
def test_decode_of_many_short_requests(gpu, dtype, hkv, group, d, longest):
    """Requests that a wave or a workgroup takes whole, and just too long for that."""
    rng = np.random.default_rng(longest)
    lens = rng.integers(0, 100, 200).tolist()
    lens[150] = longest
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, longest)
    ip, idx, lpl = pages(table, lens)
    q = rows((200, hkv * group, d), 5, dtype, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, dtype)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 5, 0], [129], [4096], [20000], [16] * 70,
                                  [513] * 9 + [0] * 80 + [31], [2000, 1, 3000, 17]])
@pytest.mark.parametrize("codec", ref.CODECS)
def test_decode_lengths(gpu, lens, codec):
    """One request to many, cut into few segments and many; a scale of its own."""
    hkv, group, d = 2, 4, 128
    cache, table, held = random_cache(lens, hkv, d, codec, gpu, sum(lens))
    ip, idx, lpl = pages(table, lens)
    q = rows((len(lens), hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True, sm_scale=0.03)
    check_decode(*got, q, held, lens, 0.03, torch.bfloat16)


@pytest.mark.parametrize("long", [[], [3000, 1500]])
@pytest.mark.parametrize("batch", [65, 300, 5000])
def test_decode_of_large_batches(gpu, batch, long):
    """Whole requests and cut ones, runs of empty requests between them, more than 4096 of them."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 40, batch) * (rng.random(batch) < 0.7)
    lens[batch // 2:batch // 2 + 50] = 0
    lens[[7, batch - 2][:len(long)]] = long
    lens = lens.tolist()
    hkv, group, d = 1, 2, 64
    cache, table, held = random_cache(lens, hkv, d, ref.INT8, gpu, batch)
    ip, idx, lpl = pages(table, lens)
    q = rows((batch, group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("batch,hkv,group,d", [(3, 2, 4, 128), (6, 8, 4, 128), (12, 8, 4, 128),
                                               (30, 8, 4, 128), (64, 8, 4, 128), (40, 8, 16, 256)])
def test_decode_joins(gpu, batch, hkv, group, d):
    """Few requests to many with cut ones among them: 64 lanes to one per column of the join."""
    lens = np.random.default_rng(batch).integers(0, 100, batch)
    lens[1], lens[-1] = 3000, 1100
    lens = lens.tolist()
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, batch)
    ip, idx, lpl = pages(table, lens)
    q = rows((batch, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("short,most,long", [(300, 16, [1100]), (60, 40, [3000] * 4), (90, 100, [1500, 0, 5000]),
                                             (1000, 16, [40000]), (20, 64, [1030] * 20)])
@pytest.mark.parametrize("hkv,group,d", [(2, 4, 128), (1, 2, 64)])
def test_decode_of_few_long_requests_among_short_ones(gpu, short, most, long, hkv, group, d):
    """Very short requests are a wave's; long ones begin in front of, between and behind them."""
    rng = np.random.default_rng(short)
    lens = rng.integers(0, most + 1, short).tolist()
    for i, n in enumerate(long):
        lens.insert([0, len(lens), len(lens) // 2, 7][i % 4], n)
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, short)
    ip, idx, lpl = pages(table, lens, first=3)
    q = rows((len(lens), hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    args = q, *cache[:3], ints(ip, gpu), ints(idx, gpu), ints(lpl, gpu)
    got = qz.quantized_decode_attention(*args, return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, torch.bfloat16)
    again = qz.quantized_decode_attention(*args, return_lse=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("hkv,group,d", [(8, 4, 128), (3, 1, 128), (8, 2, 64), (2, 2, 256), (300, 1, 64)])
@pytest.mark.parametrize("n", [800, 5000, 18000])
def test_decode_of_one_long_request(gpu, hkv, group, d, n):
    """A segment per CU, or two, or (more KV heads than CUs) one for all."""
    n = n if hkv < 300 else n // 10
    cache, table, held = random_cache([n], hkv, d, ref.INT8, gpu, n)
    ip, idx, lpl = pages(table, [n])
    q = rows((1, hkv * group, d), 5, torch.float16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, [n], d ** -0.5, torch.float16)


def test_decode_of_queries_that_are_not_finite(gpu):
    """A NaN or an infinity in a query head's row stays in that head."""
    lens, hkv, group, d = [40, 2000], 2, 4, 128
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, 6)
    ip, idx, lpl = pages(table, lens)
    q = rows((2, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    args = ints(ip, gpu), ints(idx, gpu), ints(lpl, gpu)
    base, blse = qz.quantized_decode_attention(q, *cache[:3], *args, return_lse=True)
    bad = torch.zeros(2, hkv * group, dtype=torch.bool)
    for b, h, x in ((0, 1, math.nan), (1, 3, math.inf), (1, 6, -math.inf)):
        q[b, h, 9] = x
        bad[b, h] = True
    out, lse = qz.quantized_decode_attention(q, *cache[:3], *args, return_lse=True)
    assert out[bad].isnan().all()
    assert torch.equal(out[~bad], base[~bad]) and torch.equal(lse[~bad], blse[~bad])


def test_decode_of_shared_pages(gpu):
    """Requests that share pages, and one that holds a page twice."""
    hkv, group, d = 2, 4, 128
    cache, table, held = random_cache([160], hkv, d, ref.E4M3, gpu, 6)
    t = table[0]
    idx = np.concatenate([t[:10], t[:4], [t[3], t[3], t[0]]])
    q = rows((3, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints([0, 10, 14, 17], gpu), ints(idx, gpu),
                                        ints([16, 5, 16], gpu), return_lse=True)
    at = [np.arange(160), np.arange(53), np.r_[48:64, 48:64, 0:16]]
    kept = [[(x[i], s[i]) for x, s in held[0]] for i in at]
    check_decode(*got, q, kept, [160, 53, 48], d ** -0.5, torch.bfloat16)


def test_decode_outputs_strides_and_page_offsets(gpu):
    """q and out as slices, given outputs with more rows, an indptr that begins above 0, a
    workspace used again and again."""
    lens, hkv, group, d = [50, 3, 900, 0], 4, 2, 128
    hq = hkv * group
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, 9)
    ip, idx, lpl = pages(table, lens, first=5)
    fused = rows((4, hq + 2 * hkv, d), 2, torch.bfloat16, 0.3).to(gpu)
    q = fused[:, :hq]
    room = torch.full((6, hq + 1, d), 7.0, dtype=torch.bfloat16, device=gpu)
    lse = torch.full((6, hq), 7.0, device=gpu)
    ws = qz.decode_workspace(4, hq, hkv, d, gpu)
    first = None
    for _ in range(3):
        out, l = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                               ints(lpl, gpu), out=room[:, :hq], lse=lse,
                                               return_lse=True, workspace=ws)
        assert l is lse and out.data_ptr() == room.data_ptr()
        check_decode(out, lse, q, held, lens, d ** -0.5, torch.bfloat16)
        if first is not None:
            assert torch.equal(room, first)        # bit for bit, call after call
        first = room.clone()
    assert (room[:, hq] == 7).all() and (room[4:] == 7).all() and (lse[4:] == 7).all()
    only = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                         ints(lpl, gpu))
    assert torch.equal(only, room[:4, :hq])


def test_decode_pages_that_are_missing(gpu):
    """Page ids outside the cache, and pages past the index list, hold no tokens; a last
    page length outside 0..16 counts as the nearest."""
    lens, hkv, group, d = [100, 64, 40], 2, 4, 128
    cache, table, held = random_cache(lens, hkv, d, ref.INT8, gpu, 4)
    ip, idx, lpl = pages(table, lens)
    idx = idx.copy()
    idx[1], idx[4], idx[7:11] = -7, 10 ** 9, [-1, -2, 10 ** 7, -1]
    q = rows((3, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx[:-1], gpu),
                                        ints([lpl[0], 99, lpl[2]], gpu), return_lse=True)
    left = [np.r_[0:16, 32:64, 80:100], np.arange(0), np.arange(32)]
    kept = [[(x[t], s[t]) for x, s in seq] for t, seq in zip(left, held)]
    check_decode(*got, q, kept, [len(t) for t in left], d ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("batch", [6, 200])
def test_decode_ends_whatever_indptr_holds(gpu, batch):
    """An indptr that goes down or below zero: the call ends, what it gives means nothing, and the next
    call is right."""
    hkv, group, d = 2, 4, 128
    cache, table, held = random_cache([3000] * 2, hkv, d, ref.E4M3, gpu, 4)
    idx = ints(np.concatenate([table[0, :188], table[1, :188]]), gpu)
    q = rows((batch, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    lpl = ints([16] * batch, gpu)
    rng = np.random.default_rng(batch)
    bad = [np.resize([0, 300, 100, 50, 60, 55, 70], batch + 1), np.arange(batch + 1)[::-1] * 2,
           rng.integers(-400, 400, batch + 1), np.resize([5, 0, 3, -9, 376], batch + 1)]
    for ip in bad:
        for n in (376, 40, 0):
            qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), idx[:n], lpl)
            torch.cuda.synchronize()
    ip = np.minimum(np.arange(batch + 1), 2) * 188
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), idx,
                                        ints([8, 8] + [0] * (batch - 2), gpu), return_lse=True)
    lens = [3000] * 2 + [0] * (batch - 2)
    check_decode(*got, q, held + [held[0]] * (batch - 2), lens, d ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("batch,span,have", [(1, 100, 20), (2, 70, 30), (3, 70, 0), (4097, 70, 30),
                                             (4097, 70, 0), (2, 300, 100)])
def test_decode_of_requests_past_the_index_list(gpu, batch, span, have):
    """indptr reaches past the ``have`` indices: what they do not name holds no tokens."""
    hkv, group, d = 2, 4, 128
    cache, table, held = random_cache([have * 16 + 16], hkv, d, ref.E4M3, gpu, 4)
    q = rows((batch, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    ip = np.minimum(np.arange(batch + 1) * span, 4 * span)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(table[0, :have], gpu),
                                        ints([16] * batch, gpu), return_lse=True)
    lens = [16 * max(min(span, have - b * span), 0) for b in range(batch)]
    kept = [[(x[span * 16 * b:][:n], s[span * 16 * b:][:n]) for x, s in held[0]]
            for b, n in enumerate(lens)]
    check_decode(*got, q, kept, lens, d ** -0.5, torch.bfloat16)


@pytest.mark.parametrize("lens", [[600, 100], [900], [17, 17, 17]])
def test_decode_of_a_large_batch_with_few_pages(gpu, lens):
    """More than 4096 requests, almost all of them without tokens."""
    hkv, group, d, batch = 2, 4, 128, 4500
    every = np.zeros(batch, np.int64)
    every[[9, 4200, 4400][:len(lens)]] = lens
    cache, table, held = random_cache(every.tolist(), hkv, d, ref.INT8, gpu, 4)
    ip, idx, lpl = pages(table, every.tolist())
    q = rows((batch, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                        ints(lpl, gpu), return_lse=True)
    check_decode(*got, q, held, every.tolist(), d ** -0.5, torch.bfloat16)


def test_decode_of_rows_that_are_not_finite(gpu):
    """A NaN row of K makes its head's outputs NaN, one of V its values; other heads and
    requests, and tokens past the end, are as before."""
    lens, hkv, group, d = [40, 40, 40], 2, 4, 128
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, 6)
    ip, idx, lpl = pages(table, lens)
    q = rows((3, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    args = ints(ip, gpu), ints(idx, gpu), ints(lpl, gpu)
    base, blse = qz.quantized_decode_attention(q, *cache[:3], *args, return_lse=True)
    cache.scales[table[1, 1], 0, 0, 3] = math.nan          # K of request 1, head 0
    cache.scales[table[2, 2], 1, 1, 7] = math.nan          # V of request 2, head 1
    out, lse = qz.quantized_decode_attention(q, *cache[:3], *args, return_lse=True)
    bad = torch.zeros(3, hkv * group, dtype=torch.bool)
    bad[1, :group] = bad[2, group:] = True
    assert out[bad].isnan().all() and torch.equal(out[~bad], base[~bad])
    bad[2] = False
    assert lse[bad].isnan().all() and torch.equal(lse[~bad], blse[~bad])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_large_and_small_scales(gpu, dtype):
    """V rows of very different sizes, scores far apart, logits beyond 2^20."""
    lens, hkv, group, d = [200, 77], 1, 4, 128
    cache, table, held = random_cache(lens, hkv, d, ref.INT8, gpu, 8)
    for b, n in enumerate(lens):
        t = np.arange(n)
        for i in range(2):
            e = 2.0 ** ((t * 7) % 25 - (20 if i else 4)).astype(np.float32)
            held[b][i][1][:] *= e[:, None]
            blk = torch.from_numpy(table[b, t // 16]).long().to(gpu)
            off = torch.from_numpy(t % 16).to(gpu)
            cache.scales[blk, :, i, off] = torch.from_numpy(held[b][i][1]).to(gpu)
    if dtype is torch.float16:          # outputs within its range
        cache.scales[:, :, 1] *= 2.0 ** -6
        for b in range(2):
            held[b][1][1][:] *= 2.0 ** -6
    ip, idx, lpl = pages(table, lens)
    q = rows((2, group, d), 5, dtype, 1.0).to(gpu)
    for scale in (1e-4, 1.0, 64.0):
        got = qz.quantized_decode_attention(q, *cache[:3], ints(ip, gpu), ints(idx, gpu),
                                            ints(lpl, gpu), return_lse=True, sm_scale=scale)
        assert got[0].isfinite().all()
        check_decode(*got, q, held, lens, scale, dtype)


# ------------------------------------------------- streams, graphs, offsets
def test_step_captured_and_replayed(gpu):
    """Write, read back and decode in one graph, replayed with new tokens, lengths and pages,
    eager work between the replays; every replay equals the eager calls bit for bit."""
    hkv, group, d, batch = 2, 4, 128, 5
    cache = poisoned(90, hkv, d, ref.E4M3, gpu)
    rng = np.random.default_rng(0)
    table = rng.permutation(90)[:batch * 16].reshape(batch, 16).astype(np.int32)
    k, v = (torch.empty(batch, hkv, d, dtype=torch.bfloat16, device=gpu) for _ in "kv")
    q = torch.empty(batch, hkv * group, d, dtype=torch.bfloat16, device=gpu)
    slots = torch.empty(batch, dtype=torch.int64, device=gpu)
    ip, idx = ints(np.zeros(batch + 1), gpu), ints(np.zeros(batch * 16), gpu)
    lpl, start = ints(np.zeros(batch), gpu), ints(np.zeros(batch), gpu)
    tab, cu = ints(table, gpu), ints(np.arange(batch + 1), gpu)
    ok, ov, out = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    lse = torch.empty(batch, hkv * group, device=gpu)
    ws = qz.decode_workspace(batch, hkv * group, hkv, d, gpu)

    def fill(step):
        lens = [(step * 37 + 60 * b) % 250 + 1 for b in range(batch)]
        for i, t in enumerate((k, v, q)):
            t.copy_(rows(tuple(t.shape), step * 3 + i, torch.bfloat16, 0.3))
        pos = np.array(lens) - 1
        slots.copy_(torch.from_numpy(table[np.arange(batch), pos // 16].astype(np.int64) * 16 + pos % 16))
        p, x, l = pages(table, lens)
        ip.copy_(torch.from_numpy(p))
        idx[:len(x)].copy_(torch.from_numpy(x))
        lpl.copy_(ints(l, gpu))
        start.copy_(torch.from_numpy(pos))

    def step():
        qz.reshape_and_cache_quantized(k, v, *cache[:3], slots)
        qz.gather_quantized_kv(*cache[:3], tab, cu, 1, ok, ov, start)
        qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, out=out, lse=lse, workspace=ws)

    # every slot that a step may attend to holds a token
    full = torch.arange(90 * 16, device=gpu)
    qz.reshape_and_cache_quantized(rows((1440, hkv, d), 1, torch.bfloat16).to(gpu),
                                   rows((1440, hkv, d), 2, torch.bfloat16).to(gpu), *cache[:3], full)
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(6):
        fill(n)
        for t in (ok, ov, out, lse):
            t.fill_(7.0)
        graph.replay()
        got = [t.clone() for t in (ok, ov, out, lse)]
        before = cache.storage.clone()
        for t in (ok, ov, out, lse):
            t.fill_(7.0)
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, (ok, ov, out, lse)))
        assert torch.equal(before, cache.storage)


def test_two_graphs_at_a_time(gpu):
    """Decodes captured before any other call of their kind (16 query heads of 256 per KV head: the most
    LDS), each with its workspace, replayed beside each other on two streams."""
    lens, hkv, group, d = [1500, 40, 0, 2600], 2, 16, 256
    cache, table, _ = random_cache(lens, hkv, d, ref.INT8, gpu, 9)
    ip, idx, lpl = (ints(x, gpu) for x in pages(table, lens))
    made = []
    for i in range(2):
        q = rows((4, hkv * group, d), 7 + i, torch.float16, 0.3).to(gpu)
        ws, stream, graph = qz.decode_workspace(4, hkv * group, hkv, d, gpu), torch.cuda.Stream(), \
            torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, return_lse=True,
                                                workspace=ws)
        made.append((q, ws, stream, graph, got))
    wants = [qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, return_lse=True)
             for q, *_ in made]
    for _ in range(3):
        for *_, got in made:
            for t in got:
                t.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(4):
            for _, _, stream, graph, _ in made:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (*_, got), want in zip(made, wants):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_ops_on_a_given_stream(gpu):
    """Each op on a stream that is not the current one, its outputs from that stream."""
    lens, hkv, group, d = [700, 90], 2, 4, 128
    cache, table, held = random_cache(lens, hkv, d, ref.E4M3, gpu, 3)
    ip, idx, lpl = (ints(x, gpu) for x in pages(table, lens))
    q = rows((2, hkv * group, d), 5, torch.bfloat16, 0.3).to(gpu)
    want = qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, return_lse=True)
    tab, cu = ints(table, gpu), ints([0, 700, 790], gpu)
    wk, wv = qz.gather_quantized_kv(*cache[:3], tab, cu, 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, return_lse=True,
                                            stream=side)
        outs = [torch.empty_like(wk) for _ in "kv"]
        side.wait_stream(torch.cuda.current_stream())
        gk, gv = qz.gather_quantized_kv(*cache[:3], tab, cu, 700, *outs, stream=side)
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(gk, wk) and torch.equal(gv, wv)
    k = rows((1, hkv, d), 1, torch.bfloat16).to(gpu)
    slot = torch.tensor([int(table[0, 0]) * 16 + 3], device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    qz.reshape_and_cache_quantized(k, k, *cache[:3], slot, stream=side)
    side.synchronize()
    codes, scale = ref.encode(k, ref.E4M3)
    assert np.array_equal(bits(cache.key_cache)[table[0, 0], :, 3], codes[0])


def test_offsets_past_4_gib(gpu):
    """Blocks whose codes and scales lie beyond 4 GiB, in one storage of blocks."""
    h, d, blocks = 8, 128, 140_000
    c = qz.quantized_cache(blocks, h, d, ref.E4M3, gpu)
    assert c.storage.numel() > 1 << 32
    lens = [300, 40]
    rng = np.random.default_rng(1)
    table = np.concatenate([[blocks - 1, 0], rng.choice(np.arange(130_000, blocks - 1), 20,
                                                        replace=False)]).astype(np.int32)
    table = np.stack([table[:19], np.r_[table[19:22], [-1] * 16]]).astype(np.int32)
    n = sum(lens)
    slots = np.concatenate([table[b, np.arange(m) // 16].astype(np.int64) * 16 + np.arange(m) % 16
                            for b, m in enumerate(lens)])
    k, v = rows((n, h, d), 1, torch.bfloat16), rows((n, h, d), 2, torch.bfloat16)
    qz.reshape_and_cache_quantized(k.to(gpu), v.to(gpu), *c[:3], torch.from_numpy(slots).to(gpu))
    held = []
    enc = [ref.encode(x, ref.E4M3) for x in (k, v)]
    for a, m in ((0, 300), (300, 40)):
        held.append([(ref.values(x[a:a + m], ref.E4M3), s[a:a + m]) for x, s in enc])
    gk, gv = qz.gather_quantized_kv(*c[:3], ints(table, gpu), ints([0, 300, 340], gpu), 300)
    for t, (x, s) in zip((gk, gv), enc):
        assert torch.equal(t.cpu(), (torch.from_numpy(ref.values(x, ref.E4M3)).float() *
                                     torch.from_numpy(s)[..., None]).to(torch.bfloat16))
    q = rows((2, 32, d), 3, torch.bfloat16, 0.3).to(gpu)
    ip, idx, lpl = (ints(x, gpu) for x in pages(table, lens))
    got = qz.quantized_decode_attention(q, *c[:3], ip, idx, lpl, return_lse=True)
    check_decode(*got, q, held, lens, d ** -0.5, torch.bfloat16)


# ------------------------------------------------- the two ways to the C entries
def test_binding_and_python_agree(gpu, monkeypatch):
    """An ordinary call by way of the binding and the same call without it: the same bits;
    what the binding does not take is refused or done in Python."""
    lens, hkv, group, d = [700, 90, 0, 5], 2, 4, 128
    hq = hkv * group
    cache, table, _ = random_cache(lens, hkv, d, ref.E4M3, gpu, 3)
    ip, idx, lpl = (ints(x, gpu) for x in pages(table, lens))
    q = rows((4, hq, d), 5, torch.bfloat16, 0.3).to(gpu)
    k = rows((9, hkv, d), 6, torch.bfloat16).to(gpu)
    slots = torch.arange(9, device=gpu) * 7
    ws = qz.decode_workspace(4, hq, hkv, d, gpu)
    tab, cu = ints(table, gpu), ints([0, 700, 790, 790, 795], gpu)
    took = []

    class Counted:
        def __init__(self, inner):
            self.inner = inner

        def __getattr__(self, name):
            def f(*args):
                got = getattr(self.inner, name)(*args)
                took.append((name, got is not None))
                return got
            return f

    class Nothing:
        def __getattr__(self, name):
            return lambda *args: None

    def all_ops():
        c = [t.clone() for t in cache[:3]]
        qz.reshape_and_cache_quantized(k, k, *c, slots)
        outs = [torch.zeros(795, hkv, d, dtype=torch.bfloat16, device=gpu) for _ in "kv"]
        qz.gather_quantized_kv(*c, tab, cu, 700, *outs)
        got = qz.quantized_decode_attention(q, *c, ip, idx, lpl, return_lse=True, workspace=ws,
                                            sm_scale=0.1)
        return [c[0].view(torch.uint8), c[1].view(torch.uint8), c[2].nan_to_num(3.0), *outs, *got]

    from gpu_offloading_amd import _lib
    inner = _lib.binding()
    monkeypatch.setattr(_lib, "_bind", Counted(inner))
    short = all_ops()
    assert took == [("write", True), ("read", True), ("decode", True)]
    monkeypatch.setattr(_lib, "_bind", Nothing())
    assert all(torch.equal(a, b) for a, b in zip(short, all_ops()))
    # Unusual and wrong arguments, one at a time: None from the binding, and then either a result or
    # RuntimeError from Python.
    monkeypatch.setattr(_lib, "_bind", Counted(inner))
    c = cache[:3]
    out = torch.empty_like(q)
    good = dict(q=q, key_cache=c[0], value_cache=c[1], scales=c[2], indptr=ip, indices=idx,
                last_page_len=lpl)
    for name, bad in (("q", q.float()), ("q", q[:, :3]), ("q", q.transpose(0, 1)), ("q", q.cpu()),
                      ("key_cache", c[0].view(torch.uint8)), ("value_cache", c[1].view(torch.int8)),
                      ("value_cache", c[1][:2]), ("scales", c[2].half()), ("scales", c[2][:, :1]),
                      ("indptr", ip[:3]), ("indptr", ip.long()), ("indices", idx.float()),
                      ("last_page_len", lpl[:3]), ("last_page_len", lpl.cpu())):
        took.clear()
        with pytest.raises(RuntimeError):
            qz.quantized_decode_attention(**{**good, name: bad}, workspace=ws)
        assert took == [("decode", False)], name
    for name, bad in (("out", out.half()), ("out", out[:2]), ("lse", torch.empty(2, device=gpu)),
                      ("workspace", ws[::2])):
        took.clear()
        with pytest.raises(RuntimeError):
            qz.quantized_decode_attention(**{**good, "workspace": ws, name: bad})
        assert took == [("decode", False)], name
    with pytest.raises(RuntimeError, match="WORKSPACE"):
        qz.quantized_decode_attention(**good, workspace=ws[:64])
    with pytest.raises(RuntimeError, match="sm_scale"):
        qz.quantized_decode_attention(**good, workspace=ws, sm_scale=-1.0)
    for args in ((k.float(), k), (k, k.half()), (k[:8], k), (k[:, :1], k), (k, k.cpu())):
        with pytest.raises(RuntimeError):
            qz.reshape_and_cache_quantized(*args, *c, slots)
    for bad in (slots.int(), slots.cpu(), slots[::2], slots[None]):
        with pytest.raises(RuntimeError):
            qz.reshape_and_cache_quantized(k, k, *c, bad)
    outs = [torch.zeros(795, hkv, d, dtype=torch.bfloat16, device=gpu) for _ in "kv"]
    for args in ((tab.long(), cu, 700), (tab[:2], cu, 700), (tab, cu.long(), 700), (tab, cu, -1),
                 (tab, cu, 1 << 31), (tab.t(), cu, 700)):
        with pytest.raises(RuntimeError):
            qz.gather_quantized_kv(*c, *args, *outs)
    for pair in ((outs[0], outs[1].half()), (outs[0][:, :1], outs[1]), (outs[0].float(),) * 2,
                 (outs[0], outs[1].cpu())):
        with pytest.raises(RuntimeError):
            qz.gather_quantized_kv(*c, tab, cu, 700, *pair)
    with pytest.raises(RuntimeError):
        qz.gather_quantized_kv(*c, tab, cu, 700, *outs, ints([0, 0], gpu))


# ------------------------------------------------------------------ threads
WAITS_FOR_A_THREAD = r"""
#include <unistd.h>
volatile int entered, seen;
// 0 once another thread has set `seen`, 1 if none does in two seconds
extern "C" int entry(...) {
  entered = 1;
  for (int i = 0; i < 2000; ++i) {
    if (seen) return 0;
    usleep(1000);
  }
  return 1;
}
"""


def test_python_threads_run_while_a_launch_waits(gpu, tmp_path):
    """A C entry that waits (as a launch into a full queue does) holds up no other Python thread.
    (The binding, over entries that wait until a thread sets a flag.)"""
    import ctypes
    import importlib.util
    import subprocess
    import threading
    import time

    from gpu_offloading_amd.build import BIND_PATH

    src, lib = tmp_path / "entry.cpp", str(tmp_path / "entry.so")
    src.write_text(WAITS_FOR_A_THREAD)
    subprocess.run(["g++", "-shared", "-fPIC", str(src), "-o", lib], check=True)
    waits = ctypes.CDLL(lib)
    entered, seen = (ctypes.c_int.in_dll(waits, name) for name in ("entered", "seen"))
    # (a module of its own, from a copy: the loaded one stays bound to the library)
    copy = tmp_path / "kvc_bind.so"
    copy.write_bytes(open(BIND_PATH, "rb").read())
    spec = importlib.util.spec_from_file_location("kvc_bind", copy)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    at = ctypes.cast(waits.entry, ctypes.c_void_p).value
    m.bind(at, at, at, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream)
    c = qz.quantized_cache(4, 2, 64, ref.INT8, gpu)[:3]
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    ip = ints([0, 1, 2, 3], gpu)
    calls = {m.write: [k, k, *c, torch.arange(3, device=gpu), None, None],
             m.read: [*c, ip.view(1, 4), ip[:2], 3, k, k, None, None, None],
             m.decode: [q, *c, ip, ip, ip[:3], None, None, None, True, ip, None]}
    for f, args in calls.items():
        entered.value = seen.value = 0

        def other():
            while not entered.value:
                time.sleep(1e-3)
            seen.value = 1

        t = threading.Thread(target=other)
        t.start()
        got = f(*args)
        t.join()
        assert got.__class__ is tuple if f is m.decode else got == 0, f.__name__


# --------------------------------------- one captured launch, every way of sharing out requests
def lengths_of(way, batch, rng):
    """Lengths for which the kernels take each request with a wave, with a workgroup, or cut."""
    if way == "wave":
        return rng.integers(1, 300, batch)
    if way == "workgroup":
        return np.r_[rng.integers(330, 500, 1), rng.integers(0, 500, batch - 1)]
    if way == "cut":
        n = rng.integers(0, 60, batch)
        n[::3] = rng.integers(700, 1400, len(n[::3]))
        n[batch // 2] = 2400
        return n
    return np.zeros(batch, np.int64)


@pytest.mark.parametrize("dtype,codec,batch,hkv,group,d", [
    (torch.bfloat16, ref.E4M3, 48, 16, 2, 64), (torch.float16, ref.INT8, 100, 8, 4, 128),
    (torch.bfloat16, ref.INT8, 3, 2, 3, 256), (torch.float16, ref.E4M3, 1, 8, 4, 128)])
@pytest.mark.parametrize("first", ["wave", "cut", "none"])
def test_a_captured_decode_serves_every_length(gpu, dtype, codec, batch, hkv, group, d, first):
    """One launch, captured over lengths of one kind, replayed over all kinds and back, with eager
    work between: bit for bit the eager call's result, within the bounds of 64 bits."""
    pool = 157
    cache, where, seq = random_cache([pool * 16], hkv, d, codec, gpu, 7)
    rng = np.random.default_rng(batch)
    room = batch * 90 + 150
    ip, lpl, idx = (ints(np.zeros(n), gpu) for n in (batch + 1, batch, room))
    q = torch.empty(batch, hkv * group, d, dtype=dtype, device=gpu)
    out = torch.empty_like(q)
    lse = torch.empty(batch, hkv * group, device=gpu)
    ws = qz.decode_workspace(batch, hkv * group, hkv, d, gpu)

    def decode():
        qz.quantized_decode_attention(q, *cache[:3], ip, idx, lpl, out=out, lse=lse, workspace=ws)

    def plan(way, seed):
        lens = lengths_of(way, batch, rng)
        need = (lens + 15) // 16
        places = [rng.integers(0, pool, m) for m in need]      # (pages may be shared)
        ip.copy_(ints(np.r_[0, np.cumsum(need)], gpu))
        lpl.copy_(ints((lens - 1) % 16 + (lens > 0), gpu))
        idx.fill_(1 << 20)
        if need.sum():
            idx[:need.sum()] = ints(where[0][np.concatenate(places)], gpu)
        q.copy_(rows(tuple(q.shape), seed, dtype, 0.3))
        return lens, places

    def check(lens, places):
        held = []
        for n, p in zip(lens, places):
            t = (p[:, None] * 16 + np.arange(16)).reshape(-1)[:n]
            held.append([(x[t], s[t]) for x, s in seq[0]])
        check_decode(out, lse, q, held, lens.tolist(), d ** -0.5, dtype)

    plan(first, 1)
    decode()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode()
    for i, way in enumerate(["cut", "wave", "cut", "workgroup", "none", "cut", "wave", "wave"]):
        lens, places = plan(way, 10 + i)
        out.fill_(math.nan)
        lse.fill_(math.nan)
        ws.fill_(0xff)                     # (nothing that an earlier launch left is used)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        out.fill_(math.nan)
        lse.fill_(math.nan)
        decode()
        assert torch.equal(out, got[0]) and torch.equal(lse, got[1]), (i, way)
        check(lens, places)
