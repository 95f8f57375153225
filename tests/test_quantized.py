"""CPU tests of the quantised cache: the layout of its storage, the reference codes against
torch's own e4m3 rounding, refusals of the ops and of the C entries (nothing is launched)."""
import ctypes

import numpy as np
import pytest
import torch

import quant_ref as ref
from gpu_offloading_amd import _lib
from gpu_offloading_amd import quantized as qz


@pytest.mark.parametrize("codec", ref.CODECS)
@pytest.mark.parametrize("h,d", [(1, 64), (3, 128), (8, 256)])
def test_storage_holds_each_block_in_one_piece(codec, h, d):
    c = qz.quantized_cache(5, h, d, codec, "cpu")
    per = h * 16 * d
    assert c.storage.shape == (5, 2 * per + h * 128) and c.storage.dtype is torch.uint8
    assert c.key_cache.dtype is c.value_cache.dtype is codec
    assert c.key_cache.shape == c.value_cache.shape == (5, h, 16, d)
    assert c.scales.shape == (5, h, 2, 16) and c.scales.dtype is torch.float32
    c.key_cache.view(torch.uint8).fill_(1)
    c.value_cache.view(torch.uint8).fill_(2)
    c.scales.fill_(1.0)
    want = np.r_[np.full(per, 1), np.full(per, 2), np.tile([0, 0, 128, 63], h * 32)]
    assert (c.storage.numpy() == want).all()
    checked = qz._check_quantized(*c[:3])
    assert checked == (5, h, d, qz.CODES[codec], 2 * per + h * 128, (2 * per + h * 128) // 4)


def test_reference_codes():
    """The tests' e4m3 rounding is torch's; an int8 row's largest value gets 127."""
    x = torch.randn(200, 64, generator=torch.Generator().manual_seed(1))
    x[1] = torch.linspace(-448, 448, 64)
    x[2] *= 1e-30
    x[3] = 0
    codes, scale = ref.encode(x, ref.E4M3)
    want = (x / torch.from_numpy(scale)[:, None]).to(torch.float8_e4m3fn)
    assert np.array_equal(codes, want.view(torch.uint8).numpy())
    mant = np.frexp(scale)[0]
    assert (mant == 0.5).all()
    top = np.abs(ref.values(codes, ref.E4M3)).max(1)
    assert (top[x.abs().amax(1) > 1e-29] >= 224).all() and (top <= 448).all()
    assert np.array_equal(ref.e4m3_table()[:127], np.sort(ref.e4m3_table()[:127]))
    codes, scale = ref.encode(x, ref.INT8)
    v = codes.view(np.int8)
    assert (np.abs(v).max(1)[x.abs().amax(1).numpy() > 1e-29] == 127).all() and v.min() >= -127


def test_ops_refuse_what_they_cannot_do():
    c = qz.quantized_cache(4, 2, 64, ref.INT8, "cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    ip = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        qz.reshape_and_cache_quantized(k, k, *c[:3], torch.arange(3))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        qz.gather_quantized_kv(*c[:3], torch.zeros(1, 4, dtype=torch.int32), ip[:2], 3)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        qz.quantized_decode_attention(k, *c[:3], ip, ip, ip)
    for bad in (torch.float8_e5m2, torch.bfloat16, torch.uint8):
        with pytest.raises(RuntimeError, match="kv_dtype"):
            qz.quantized_cache(4, 2, 64, bad, "cpu")
    for shape in ((0, 2, 64), (4, 0, 64), (4, 2, 96), (4, 2, 0)):
        with pytest.raises(RuntimeError):
            qz.quantized_cache(*shape, ref.INT8, "cpu")


def test_cache_checks():
    c = qz.quantized_cache(4, 2, 64, ref.E4M3, "cpu")
    k, v, s = c[:3]
    other = qz.quantized_cache(4, 2, 64, ref.INT8, "cpu")
    for bad in ((k, other.value_cache, s), (k.view(torch.uint8), v.view(torch.uint8), s),
                (k[:3], v, s), (k[0], v[0], s), (k[..., :32], v[..., :32], s),
                (k.transpose(1, 2), v.transpose(1, 2), s), (k, v, s.half()), (k, v, s[:, :1]),
                (k, v, s.transpose(2, 3)), (k, v, s[:3]), (k, v.contiguous(), s)):
        with pytest.raises(RuntimeError):
            qz._check_quantized(*bad)
    # blocks of their own strides are fine, and so is one block
    qz._check_quantized(k[::2], v[::2], s[::2])
    assert qz._check_quantized(k[:1], v[:1], s[:1])[0] == 1
    for bad in (torch.zeros(3, 2, 64), torch.zeros(3, 1, 64, dtype=torch.half),
                torch.zeros(3, 2, 32, dtype=torch.half), torch.zeros(2, 64, dtype=torch.half),
                torch.zeros(3, 64, 2, dtype=torch.half).transpose(1, 2)):
        with pytest.raises(RuntimeError):
            qz._check_tokens("key", bad, 2, 64)


# ---------------------------------------------------------------- C entries
A = 1 << 20          # an aligned address that nothing reads: every call below is refused


def write(**kw):
    a = dict(key=A, value=A, key_cache=A, value_cache=A, scales=A, slots=A, n=3, h=2, d=128, bs=16,
             nb=4, dtype=1, code=0, ks=256, vs=256, cs=4096, ss=64, oob=None, stream=None)
    a.update(kw)
    return _lib.load().kvc_reshape_and_cache_quantized(*a.values())


def read(**kw):
    a = dict(key_cache=A, value_cache=A, scales=A, table=A, row=8, width=8, cu=A, starts=None,
             batch=2, top=50, h=2, d=128, bs=16, nb=4, dtype=1, code=0, cs=4096, ss=64, ok=A, ov=A,
             os=256, rows=100, oob=None, stream=None)
    a.update(kw)
    return _lib.load().kvc_gather_quantized_kv(*a.values())


def decode(**kw):
    a = dict(q=A, qs=1024, key_cache=A, value_cache=A, scales=A, cs=4096, ss=64, nb=4, indptr=A,
             indices=A, ni=8, lpl=A, batch=2, hq=8, hkv=2, d=128, bs=16, dtype=1, code=0,
             scale=ctypes.c_float(0.1), ws=A, wsb=1 << 40, out=A, os=1024, lse=None, stream=None)
    a.update(kw)
    return _lib.load().kvc_quantized_decode(*a.values())


INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = 1, 2, 3, 4


@pytest.mark.parametrize("call,want,kw", [
    (write, INVALID, dict(n=-1)), (write, INVALID, dict(key=None)), (write, INVALID, dict(scales=None)),
    (write, INVALID, dict(slots=None)), (write, INVALID, dict(h=0)), (write, INVALID, dict(nb=0)),
    (write, INVALID, dict(ks=255)), (write, INVALID, dict(vs=0)), (write, INVALID, dict(cs=4080)),
    (write, INVALID, dict(ss=60)), (write, INVALID, dict(n=1 << 31)), (write, INVALID, dict(n=1 << 29)),
    (write, UNSUPPORTED, dict(d=96)), (write, UNSUPPORTED, dict(bs=32)),
    (write, UNSUPPORTED, dict(dtype=2)), (write, UNSUPPORTED, dict(code=2)),
    (write, ALIGNMENT, dict(key=A + 1)), (write, ALIGNMENT, dict(key_cache=A + 8)),
    (write, ALIGNMENT, dict(scales=A + 4)), (write, ALIGNMENT, dict(cs=4104)),
    (write, ALIGNMENT, dict(ss=66)),
    (read, INVALID, dict(batch=-1)), (read, INVALID, dict(top=-1)), (read, INVALID, dict(rows=-1)),
    (read, INVALID, dict(table=None)), (read, INVALID, dict(cu=None)), (read, INVALID, dict(ok=None)),
    (read, INVALID, dict(batch=65536)), (read, INVALID, dict(width=0)), (read, INVALID, dict(os=255)),
    (read, INVALID, dict(cs=0)), (read, UNSUPPORTED, dict(d=32)), (read, UNSUPPORTED, dict(code=-1)),
    (read, ALIGNMENT, dict(value_cache=A + 8)), (read, ALIGNMENT, dict(ov=A + 1)),
    (decode, INVALID, dict(batch=-1)), (decode, INVALID, dict(ni=-1)), (decode, INVALID, dict(ni=(1 << 31) - 1)), (decode, INVALID, dict(q=None)),
    (decode, INVALID, dict(indices=None)), (decode, INVALID, dict(lpl=None)),
    (decode, INVALID, dict(batch=65536)), (decode, INVALID, dict(hq=9)), (decode, INVALID, dict(hkv=0)),
    (decode, INVALID, dict(nb=0)), (decode, INVALID, dict(qs=1023)), (decode, INVALID, dict(os=0)),
    (decode, INVALID, dict(cs=4095)), (decode, INVALID, dict(scale=ctypes.c_float(0.0))),
    (decode, INVALID, dict(scale=ctypes.c_float(-1.0))),
    (decode, INVALID, dict(scale=ctypes.c_float(float("nan")))),
    (decode, INVALID, dict(scale=ctypes.c_float(float("inf")))),
    (decode, UNSUPPORTED, dict(hq=34)), (decode, UNSUPPORTED, dict(d=80)),
    (decode, UNSUPPORTED, dict(bs=8)), (decode, UNSUPPORTED, dict(dtype=5)),
    (decode, UNSUPPORTED, dict(code=7)),
    (decode, ALIGNMENT, dict(q=A + 8)), (decode, ALIGNMENT, dict(qs=1028)),
    (decode, ALIGNMENT, dict(out=A + 4)), (decode, ALIGNMENT, dict(os=1026)),
    (decode, ALIGNMENT, dict(scales=A + 8)),
    (decode, WORKSPACE, dict(ws=None)), (decode, WORKSPACE, dict(wsb=1000)),
    (decode, WORKSPACE, dict(ws=A + 4)),
])
def test_c_entries_refuse(call, want, kw):
    assert call(**kw) == want, _lib.load().kvc_last_error()
    assert _lib.load().kvc_last_error()


@pytest.mark.parametrize("call,kw", [
    (write, dict(n=1 << 26)), (write, dict(n=1 << 25, d=256, ks=512, vs=512, cs=8192)),
    (write, dict(n=1 << 27, d=64)), (read, dict(top=(1 << 31) - 1)), (read, dict(top=1 << 28)),
    (read, dict(h=40000, cs=1 << 30, ss=1 << 30, os=1 << 30))])
def test_c_entries_refuse_more_threads_than_a_launch_has(call, kw):
    assert call(**kw) == INVALID
    assert b"one call" in _lib.load().kvc_last_error()


def test_nothing_to_do_is_no_error():
    assert write(n=0, key=None) == 0
    assert read(batch=0, cu=None) == 0 and read(top=0) == 0
    assert decode(batch=0, q=None) == 0
    ws = _lib.load().kvc_quantized_decode_workspace_bytes
    assert ws(1, 32, 8, 128) > 0 and ws(-1, 32, 8, 128) == 0 and ws(1, 0, 8, 128) == 0


# ------------------------------------------------------------------ binding
def test_binding_leaves_what_is_not_ordinary_to_python():
    """The short way takes nothing that is not on a GPU, whatever it is handed, and raises nothing."""
    m = _lib.binding()
    c = qz.quantized_cache(4, 2, 64, ref.INT8, "cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    ip = torch.zeros(4, dtype=torch.int32)
    calls = {m.write: [k, k, *c[:3], torch.arange(3), None, None],
             m.read: [*c[:3], ip.view(1, 4), ip[:2], 3, k, k, None, None, None],
             m.decode: [k, *c[:3], ip, ip, ip, None, None, None, True, ip, None]}
    for f, args in calls.items():
        assert f(*args) is None
        assert f(*args[:-1]) is None and f() is None
        for i in range(len(args)):
            for odd in (None, 7, "x", 1.5, torch.empty(0)):
                assert f(*args[:i], odd, *args[i + 1:]) is None
    with pytest.raises(TypeError):
        m.bind()
