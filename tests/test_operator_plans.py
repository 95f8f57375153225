"""CPU tests of the prompt attention's, the attention weights' and the eviction's
C entries: plan images cover every (query or key tile, KV head) exactly once, and
what the documentation does not allow is refused before any launch."""
import ctypes

import numpy as np
import pytest

from gpu_offloading_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _i32(x):
    return np.ascontiguousarray(x, dtype=np.int32)


def _cum(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]))


def _prompt(lib, qo, kv, hq, hkv, d, causal=1, cap=None):
    s = _lib.KvcPromptSchedule()
    qo, kv = _i32(qo), _i32(kv)
    img = np.zeros(1 << 16 if cap is None else max(cap, 1), np.int32)
    st = lib.kvc_prompt_plan(qo.ctypes.data, kv.ctypes.data, len(qo) - 1, hq, hkv, d, causal,
                             ctypes.byref(s), img.ctypes.data, len(img) if cap is None else cap)
    return st, s, img


def _units(s, img):
    """The unit records, after checking that the workgroups' table partitions them."""
    w = s.num_workgroups
    table = img[:2 * w].reshape(-1, 2)
    at = 0
    for first, n in table.tolist():
        assert first == at and n > 0
        at += n
    assert at == s.num_units
    base = (2 * w + 3) // 4 * 4
    assert s.plan_ints == base + 8 * s.num_units + 8 * s.num_joins
    return img[base:base + 8 * s.num_units].reshape(-1, 8)


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (6, 2, 64), (7, 1, 256), (128, 1, 128)])
@pytest.mark.parametrize("causal", [0, 1])
def test_prompt_units_cover_every_query_once(lib, hq, hkv, d, causal):
    qlens, kvlens = [1, 0, 300, 64, 5, 129], [1, 7, 300, 200, 0, 100]
    qo, kv = _cum(qlens), _cum(kvlens)
    st, s, img = _prompt(lib, qo, kv, hq, hkv, d, causal)
    assert st == 0 and s.total_q == qo[-1] and s.total_kv == kv[-1]
    seen = set()
    for h, t0, m, n, q0, k0, tiles, _ in _units(s, img).tolist():
        assert m > 0 and t0 % s.tile_tokens == 0
        seen.add((h, q0 + t0))
        last = min(t0 + s.tile_tokens, m) - 1
        keys = max(0, min(n, last + n - m + 1)) if causal else n
        assert tiles == -(-keys // (128 if d == 64 else 64))
        b = [i for i in range(6) if qo[i] == q0 and qlens[i] == m][0]
        assert kv[b] == k0 and kvlens[b] == n
    want = {(h, int(qo[b]) + t) for h in range(hkv) for b in range(6)
            for t in range(0, qlens[b], s.tile_tokens)}
    assert seen == want and s.num_units == len(want)


@pytest.mark.parametrize("lens,hq,hkv,d,causal", [
    ([4000], 4, 1, 128, 1), ([2300], 8, 1, 64, 1), ([5000], 2, 2, 256, 1),
    ([2900, 200], 6, 2, 64, 0), ([1070, 1180, 1192, 991], 8, 4, 256, 0), ([2900, 1], 7, 1, 128, 0)])
def test_prompt_pieces_cover_every_key_once(lib, lens, hq, hkv, d, causal):
    """Few units: they are cut along their keys, and a join lists the pieces in order."""
    qo, kv = _cum(lens), _cum([n + 100 for n in lens])
    st, s, img = _prompt(lib, qo, kv, hq, hkv, d, causal)
    assert st == 0 and s.num_joins > 0 and s.num_parts > 0
    per, rows = 128 if d == 64 else 64, 128 if d == 256 else 256
    assert s.tile_tokens == rows // (hq // hkv)
    assert s.workspace_bytes == s.num_parts * rows * (d + 1) * 4
    runs, part_of = {}, {}
    for h, t0, m, n, q0, k0, tiles, part in _units(s, img).tolist():
        b = [i for i in range(len(lens)) if qo[i] == q0 and lens[i] == m][0]
        first = (k0 - int(kv[b])) // per
        assert k0 - kv[b] == first * per and n == lens[b] + 100 - first * per and tiles > 0
        runs.setdefault((h, b, t0), []).append((first, tiles, part))
        if part:
            assert part not in part_of
            part_of[part] = (h, b, t0, first)
    assert sorted(part_of) == list(range(1, s.num_parts + 1))
    assert set(runs) == {(h, b, t) for h in range(hkv) for b in range(len(lens))
                         for t in range(0, lens[b], s.tile_tokens)}
    for (h, b, t0), pieces in runs.items():
        last = min(t0 + s.tile_tokens, lens[b]) - 1
        keys = min(lens[b] + 100, last + 101) if causal else lens[b] + 100
        at = 0
        for first, tiles, part in sorted(pieces):
            assert first == at and (part > 0) == (len(pieces) > 1)
            at += tiles
        assert at == -(-keys // per)
    joins = img[s.plan_ints - 8 * s.num_joins:s.plan_ints].reshape(-1, 8).tolist()
    assert len(joins) == sum(len(p) > 1 for p in runs.values())
    for h, t0, m, q0, part, n, *_ in joins:
        b = [i for i in range(len(lens)) if qo[i] == q0][0]
        assert m == lens[b] and n == len(runs[h, b, t0])
        assert [p for _, _, p in sorted(runs[h, b, t0])] == list(range(part + 1, part + n + 1))


def test_prompt_plan_asks_for_its_capacity(lib):
    qo = _cum([1000])
    st, s, _ = _prompt(lib, qo, qo, 8, 8, 128, cap=10)
    assert st == _lib.KVC_ERR_WORKSPACE and s.plan_ints > 10
    st, t, _ = _prompt(lib, qo, qo, 8, 8, 128, cap=int(s.plan_ints))
    assert st == 0 and t.plan_ints == s.plan_ints
    st, s, _ = _prompt(lib, [0], [0], 8, 8, 128)
    assert st == 0 and s.num_units == 0 and s.plan_ints == 0


@pytest.mark.parametrize("qo,kv,hq,hkv,d,want", [
    ([0, 5, 4], [0, 5, 9], 8, 8, 128, 1),          # decreasing
    ([-1, 5], [0, 5], 8, 8, 128, 1),               # negative
    ([0, 5], [0, 5], 9, 8, 128, 1),                # heads
    ([0, 5], [0, 5], 0, 8, 128, 1),
    ([0, 5], [0, 5], 8, 8, 96, 2),                 # head_dim
    ([0, 5], [0, 5], 129, 1, 128, 2),              # group
    ([0, 2**31 - 1], [0, 5], 128, 1, 64, 1),       # too long
    ([0, 2**29], [0, 5], 128, 1, 64, 1),           # too many units
])
def test_prompt_plan_refuses(lib, qo, kv, hq, hkv, d, want):
    st, *_ = _prompt(lib, qo, kv, hq, hkv, d)
    assert st == want and lib.kvc_last_error()


def test_prompt_run_refuses(lib):
    qo = _cum([40])
    _, s, _ = _prompt(lib, qo, qo, 8, 2, 128)
    ok = dict(plan=64, q=64, qs=1024, k=64, ks=256, v=64, vs=256, dt=1, scale=0.1, out=64, os=1024)

    def run(**kw):
        a = {**ok, **kw}
        return lib.kvc_prompt_run(ctypes.byref(s), a["plan"], a.get("ws"), a.get("wb", 0), a["q"],
                                  a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["dt"],
                                  ctypes.c_float(a["scale"]), a["out"], a["os"], None, None)
    for bad, want in ((dict(plan=None), 1), (dict(q=None), 1), (dict(v=None), 1),
                      (dict(out=None), 1), (dict(qs=1016), 1), (dict(ks=248), 1),
                      (dict(os=8), 1), (dict(vs=1 << 22), 1),
                      (dict(ks=1 << 22), 1), (dict(os=1 << 22), 1), (dict(qs=1 << 22), 1), (dict(q=72), 3), (dict(k=66), 3),
                      (dict(out=68), 3), (dict(plan=68), 3), (dict(qs=1028), 3),
                      (dict(vs=260), 3), (dict(dt=2), 2), (dict(scale=0.0), 1),
                      (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1),
                      (dict(scale=float("inf")), 1)):
        assert run(**bad) == want, bad
    s.num_units += 1
    assert run() == 1
    _, s, _ = _prompt(lib, _cum([4000]), _cum([4000]), 4, 1, 128)
    assert s.num_parts > 0 and s.workspace_bytes == s.num_parts * 256 * 129 * 4
    assert run(qs=512, os=512, ks=128, vs=128) == 4                        # no workspace
    need = s.workspace_bytes
    assert run(qs=512, os=512, ks=128, vs=128, ws=64, wb=need - 1) == 4
    assert run(qs=512, os=512, ks=128, vs=128, ws=72, wb=need) == 3
    assert lib.kvc_prompt_run(None, 64, None, 0, 64, 1024, 64, 256, 64, 256, 1, ctypes.c_float(1.0), 64,
                              1024, None, None) == 1


def _weights(lib, qlens, lens, hq, hkv, d, new=None, causal=1, page=16, lpl=None, qo=None):
    s = _lib.KvcWeightsSchedule()
    lens = np.asarray(lens)
    qo = _cum(qlens) if qo is None else _i32(qo)
    kv = _cum((lens + 15) // 16)
    lpl = _i32(np.where(lens > 0, (lens - 1) % 16 + 1, 0)) if lpl is None else _i32(lpl)
    nw = None if new is None else _i32(new)
    img = np.zeros(1 << 16, np.int32)
    st = lib.kvc_weights_plan(qo.ctypes.data, kv.ctypes.data, lpl.ctypes.data,
                              None if nw is None else nw.ctypes.data, len(lens), hq, hkv, d, page,
                              causal, ctypes.byref(s), img.ctypes.data, len(img))
    return st, s, img, qo, kv


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (6, 2, 64), (7, 1, 256), (128, 1, 64)])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("qlens,new", [([1, 0, 300, 64, 0, 0, 17], None),
                                       ([1, 0, 900, 3, 0, 0, 1], [1, 0, 1000, 0, 33, 0, 17]),
                                       ([1, 0, 2, 3, 0, 0, 1], [1, 0, 300, 0, 33, 0, 17])])
def test_weights_units_cover_every_key_and_row_once(lib, hq, hkv, d, causal, qlens, new):
    """Key tiles of 256, their row blocks of 32 in one run or in several, whose
    partials a join record lists in order."""
    lens = [1, 0, 1000, 64, 200, 0, 17]
    st, s, img, qo, kv = _weights(lib, qlens, lens, hq, hkv, d, new, causal)
    assert st == 0
    n = s.num_units
    assert s.plan_ints == 12 * n + 8 * s.num_joins
    walked = []
    for u in range(s.num_workgroups):
        walked.append(u)
        while img[12 * walked[-1] + 11]:
            walked.append(int(img[12 * walked[-1] + 11]))
    assert sorted(walked) == list(range(n))
    assert s.workspace_bytes == s.num_parts * 256 * 4
    runs, part_of = {}, {}
    for h, k0, m, ln, q0, p0, b, fresh, first, blocks, part, _ in img[:12 * n].reshape(-1, 12).tolist():
        assert (m, ln, q0, p0) == (qlens[b], lens[b], qo[b], kv[b])
        assert fresh == ln - (qlens[b] if new is None else new[b])
        runs.setdefault((h, b, k0), []).append((first, blocks, part))
        if part >= 0:
            assert part not in part_of
            part_of[part] = (h, b, k0, first)
    assert sorted(part_of) == list(range(s.num_parts))
    want = {}
    for h in range(hkv):
        for b, ln in enumerate(lens):
            f = qlens[b] if new is None else new[b]
            if qlens[b] or f:
                for k in range(0, ln, 256):
                    if qlens[b] or k + 256 > ln - f:
                        t = max(0, k - (ln - qlens[b])) if causal else 0
                        want[h, b, k] = -(-(qlens[b] - t) * (hq // hkv) // 32) if qlens[b] else 0
    assert set(runs) == set(want)
    for key, pieces in runs.items():
        pieces.sort()
        at = 0
        for first, blocks, part in pieces:
            assert first == at and (part >= 0) == (len(pieces) > 1)
            assert blocks > 0 or len(pieces) == 1
            at += blocks
        assert at == want[key]
    joins = img[12 * n:12 * n + 8 * s.num_joins].reshape(-1, 8).tolist()
    assert len(joins) == sum(len(p) > 1 for p in runs.values())
    for h, k0, k, ln, first, p0, b, fresh in joins:
        pieces = runs[h, b, k0]
        assert k == len(pieces) and [p[2] for p in pieces] == list(range(first, first + k))
        assert ln == lens[b] and p0 == kv[b]
        assert fresh == ln - (qlens[b] if new is None else new[b])


@pytest.mark.parametrize("kw,want", [
    (dict(qlens=[5], lens=[4]), 1),                       # more queries than tokens
    (dict(qlens=[1], lens=[4], new=[5]), 1),
    (dict(qlens=[1], lens=[4], new=[-1]), 1),
    (dict(qlens=[1], lens=[4], lpl=[17]), 1),
    (dict(qlens=[1], lens=[4], lpl=[0]), 1),
    (dict(qlens=[1], lens=[4], qo=[3, 1]), 1),
    (dict(qlens=[1], lens=[4], hq=3), 1),
    (dict(qlens=[1], lens=[4], page=32), 2),
    (dict(qlens=[1], lens=[4], d=80), 2),
    (dict(qlens=[1], lens=[4], hq=258), 2),
])
def test_weights_plan_refuses(lib, kw, want):
    args = dict(hq=4, hkv=2, d=128)
    args.update(kw)
    st, *_ = _weights(lib, **args)
    assert st == want and lib.kvc_last_error()


def test_weights_run_refuses(lib):
    _, s, *_ = _weights(lib, [5], [40], 4, 2, 128)
    ok = dict(plan=64, q=64, qs=512, lse=64, k=64, bs=4096, ts=256, nb=4, idx=64, ni=3, dt=1,
              scale=0.1, sc=64)

    def chunk(**kw):
        a = {**ok, **kw}
        return lib.kvc_batch_attention_weights_run(
            ctypes.byref(s), a["plan"], None, 0, a["q"], a["qs"], a["lse"], a["k"], a["bs"],
            a["ts"], a["nb"], a["idx"], a["ni"], a["dt"], ctypes.c_float(a["scale"]), a["sc"], None,
            a.get("off"), a.get("no", 0), None, None)

    def decode(**kw):
        a = dict(ok, ip=64, lpl=64, b=2, hq=4, hkv=2, d=128, page=16)
        a.update(kw)
        return lib.kvc_decode_attention_weights(
            a["q"], a["qs"], a["lse"], a["k"], a["bs"], a["ts"], a["nb"], a["ip"], a["idx"],
            a["ni"], a["lpl"], a["b"], a["hq"], a["hkv"], a["d"], a["page"], a["dt"],
            ctypes.c_float(a["scale"]), a["sc"], None, a.get("off"), a.get("no", 0), None, None)
    both = [(dict(q=None), 1), (dict(lse=None), 1), (dict(k=None), 1), (dict(sc=None), 1),
            (dict(idx=None), 1), (dict(nb=0), 1), (dict(ts=248), 1), (dict(bs=256), 1),
            (dict(qs=504), 1), (dict(q=72), 3), (dict(k=66), 3), (dict(qs=516), 3),
            (dict(bs=4100), 3), (dict(ts=260, bs=8192), 3), (dict(dt=7), 2),
            (dict(scale=float("nan")), 1), (dict(qs=1 << 25), 2), (dict(off=64, no=-1), 1)]
    for bad, want in both + [(dict(plan=None), 1), (dict(plan=68), 3), (dict(ni=0), 1)]:
        assert chunk(**bad) == want, bad
    for bad, want in both + [(dict(ip=None), 1), (dict(lpl=None), 1), (dict(b=-1), 1),
                             (dict(hq=3), 1), (dict(d=100), 2), (dict(page=8), 2),
                             (dict(hq=400), 2)]:
        assert decode(**bad) == want, bad
    assert decode(b=0) == 0 and decode(ni=0) == 0     # nothing to do
    s.plan_ints += 8
    assert chunk() == 1
    _, s, *_ = _weights(lib, [900], [900], 128, 1, 64)
    assert s.num_parts > 0 and s.workspace_bytes > 0
    assert chunk(qs=8192, bs=1024, ts=64) == 4        # no workspace


def test_evict_refuses(lib):
    need = lib.kvc_evict_workspace_bytes(2, 3, 100)
    assert need >= 2 * 3 * 50 * 8 and lib.kvc_evict_workspace_bytes(0, 3, 100) == 0
    ok = dict(k=64, v=64, nb=4, h=3, d=64, page=16, e=2, bs=4096, ts=256, sc=64, bt=64,
              rs=7, w=7, rows=2, lens=64, keep=64, rec=64, b=2, top=100, ws=64, wb=need)

    def run(**kw):
        a = {**ok, **kw}
        return lib.kvc_evict_kv(a["k"], a["v"], a["nb"], a["h"], a["d"], a["page"], a["e"],
                                a["bs"], a["ts"], a["sc"], None, a["bt"], a["rs"], a["w"],
                                a["rows"], None, a["lens"], a["keep"], a["rec"], None, a["b"],
                                a["top"], a["ws"], a["wb"], None)
    for bad, want in ((dict(k=None), 1), (dict(v=None), 1), (dict(sc=None), 1), (dict(bt=None), 1),
                      (dict(lens=None), 1), (dict(keep=None), 1), (dict(rec=None), 1),
                      (dict(b=-1), 1), (dict(top=-1), 1), (dict(h=0), 1), (dict(d=0), 1),
                      (dict(e=0), 1), (dict(nb=0), 1), (dict(rs=6), 1), (dict(rows=0), 1),
                      (dict(ts=100), 1), (dict(bs=4000), 1), (dict(page=32), 2), (dict(d=60), 2),
                      (dict(b=30000), 2), (dict(k=72), 3), (dict(bs=4100), 3), (dict(ws=None), 4),
                      (dict(wb=need - 1), 4), (dict(ws=66), 3), (dict(sc=72), 3),
                      (dict(nb=1 << 27), 2)):
        assert run(**bad) == want, bad
    assert run(b=0) == 0 and run(top=0) == 0
