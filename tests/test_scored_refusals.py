"""What the entry points around attention refuse is refused before a device is touched (runs without one)."""
import ctypes as C

import pytest

from tract_amd import _lib

I4, I3, I2 = C.c_int64 * 4, C.c_int64 * 3, C.c_int64 * 2
A, B_, C_, D_, E_ = (1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20)   # addresses that nothing reads
NAN = float("nan")


def _refused(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    return lib.trocm_last_error().decode()


def _norm(**kw):
    a = dict(q=A, k=B_, wq=None, wk=None, eps=1e-6, cos=C_, sin=C_ + 65536, cs=0, dtype=1, batch=1, hq=4, hkv=2, n=3, d=64, qs=None, ks=None, qo=D_, ko=E_, stream=None)
    a.update(kw)
    return _refused("trocm_qk_norm_rope", *a.values())


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=2), "F32 or F16"), (dict(d=63), "must be even"), (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps"), (dict(q=None), "null pointer"), (dict(cos=None), "cos"),
    (dict(n=-1), "negative"), (dict(qs=I4(1, 1, -1, 1)), "negative strides"), (dict(ks=I4(384, 192, 64, 2)), "contiguous"), (dict(cs=100), "overlap"),
    (dict(qo=A + 64), "overlap"), (dict(qo=B_), "overlap"), (dict(ko=D_), "overlap"), (dict(ko=C_), "cos or sin"), (dict(qo=None), "q_out"),
    (dict(qo=A, qs=I4(768, 64, 256, 1)), "overlap"), (dict(wq=D_), "weight"), (dict(batch=1 << 13, n=1 << 13), "too large")])
def test_norm_rope(kw, says):
    assert says in _norm(**kw)


def _shared(**kw):
    a = dict(q=A, dtype=1, n=2, hq=4, hkv=2, sq=1, d=64, pk=B_, pv=B_ + 65536, p=10, ps=None, k=C_, v=C_ + 65536, kv=I3(2 * 8 * 64, 8 * 64, 64), lens=I2(8, 3), out=D_,
             scale=NAN, causal=1, ws=None, wsb=0, stream=None)
    a.update(kw)
    return _refused("trocm_sdpa_shared_prefix", *a.values())


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=3), "F32 or F16"), (dict(hq=5), "multiple"), (dict(p=-1), "negative"), (dict(lens=None), "lens"), (dict(lens=I2(8, -1)), "length -1"), (dict(pk=None), "prefix_k"),
    (dict(k=None), "null pointer"), (dict(kv=None), "kv_strides"), (dict(kv=I3(1, -1, 1)), "negative K/V"), (dict(ps=I2(-1, 64)), "negative K/V"), (dict(out=A), "out overlaps q"),
    (dict(out=B_), "overlaps the prefix"), (dict(out=C_ + 128), "overlaps k or v"), (dict(sq=1 << 25), "too large"), (dict(hkv=0), "negative")])
def test_shared_prefix(kw, says):
    assert says in _shared(**kw)


def _scored(**kw):
    a = dict(q=A, k=B_, v=C_, out=D_, dtype=1, b=1, hq=4, hkv=2, sq=3, sk=9, d=64, st=None, scale=NAN, cap=0.0, slopes=None, docs=None, pre=None, causal=1, ws=None, wsb=0, stream=None)
    a.update(kw)
    return _refused("trocm_sdpa_scored", *a.values())


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=7), "F32 or F16"), (dict(hkv=3), "multiple"), (dict(cap=-2.0), "softcap"), (dict(cap=NAN), "softcap"), (dict(cap=float("inf")), "softcap"), (dict(k=None), "null pointer"),
    (dict(out=B_ + 2), "out overlaps k"), (dict(out=A), "out overlaps q"), (dict(docs=E_, sk=2), "documents need"), (dict(st=I3(1, 1, -64)), "negative K/V"), (dict(sq=-1), "negative")])
def test_scored(kw, says):
    assert says in _scored(**kw)


def test_workspace_of_a_shared_prefix():
    lib, n = _lib.load(), C.c_size_t()
    assert lib.trocm_sdpa_shared_workspace_bytes(64, 32, 1, 128, C.byref(n)) == 0 and 0 < n.value < 1 << 28
    assert lib.trocm_sdpa_shared_workspace_bytes(-1, 32, 1, 128, C.byref(n)) == 1
    assert lib.trocm_sdpa_shared_workspace_bytes(1, 32, 1, 128, None) == 1
