"""What the entry points over pages and beam search's choice refuse is refused before a device is touched (runs without one)."""
import ctypes as C

import pytest

from tract_amd import _lib

I2, I3 = C.c_int64 * 2, C.c_int64 * 3
M = 1 << 20


def at(i):   # addresses that nothing reads
    return M * i


def _refused(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    return lib.trocm_last_error().decode()


def _with(defaults, kw):
    assert set(kw) <= set(defaults), kw
    return {**defaults, **kw}.values()


def _plan(**kw):
    return _refused("trocm_paged_plan", *_with(dict(
        lens=at(1), new=at(2), n=5, page=16, table=at(3), width=8, free=at(4), count=at(5), pages=40, refs=at(6), tokens=9, lens_out=at(7), starts=at(8), slots=at(9),
        positions=at(10), count_out=at(11), refused=at(12), stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(lens=None), "null pointer"), (dict(new=None), "n_new"), (dict(table=None), "table"), (dict(free=None), "free_pages"), (dict(count=None), "free_count"),
    (dict(slots=None), "slots"), (dict(refused=None), "refused"), (dict(count_out=None), "free_count_out"), (dict(lens_out=None), "lens_out"), (dict(n=-1), "negative"),
    (dict(width=-1), "negative"), (dict(tokens=-1), "negative"), (dict(pages=-1), "negative"), (dict(page=0), "page_size"), (dict(page=1 << 21), "page_size"),
    (dict(n=4097), "sequences"), (dict(pages=(1 << 26) + 1), "2^30"), (dict(width=(1 << 26) + 1), "2^30"), (dict(tokens=(1 << 30) + 1), "2^30"),
    (dict(lens_out=at(1)), "lens_out overlaps lens"), (dict(lens_out=at(2) + 16), "overlaps n_new"), (dict(count_out=at(5)), "overlaps free_count"), (dict(slots=at(3) + 8), "overlaps table"),
    (dict(positions=at(9) + 32), "overlaps slots"), (dict(refs=at(4)), "refs overlaps free_pages"), (dict(starts=at(8) + 2), "aligned"), (dict(lens=at(1) + 1), "aligned")])
def test_plan(kw, says):
    assert says in _plan(**kw)


def _append(**kw):
    return _refused("trocm_paged_append", *_with(dict(
        k=at(1), v=at(2), dtype=1, tokens=7, heads=2, d=64, ks=None, vs=None, slots=at(3), kp=at(4), vp=at(5), pages=8, page=16, ps=None, stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=2), "F32 or F16"), (dict(k=None), "k_new"), (dict(v=None), "v_new"), (dict(slots=None), "slots"), (dict(kp=None), "k_pages"), (dict(tokens=-1), "negative"),
    (dict(heads=-1), "negative"), (dict(d=1 << 24), "too large"), (dict(ks=I2(-1, 64)), "negative strides"), (dict(vs=I2(1, 1 << 30)), "strides too large"), (dict(ps=I3(1, -1, 64)), "negative page strides"),
    (dict(ps=I3(1 << 40, 1, 64)), "page strides too large"), (dict(kp=at(1)), "k_pages overlaps k_new"), (dict(vp=at(4) + 64), "overlaps k_pages"), (dict(kp=at(3)), "overlaps slots"),
    (dict(k=at(1) + 1), "aligned"), (dict(slots=at(3) + 2), "aligned"), (dict(page=0), "page_size"), (dict(pages=(1 << 26) + 1), "2^30"), (dict(page=1 << 20, d=1 << 10), "too large")])
def test_append(kw, says):
    assert says in _append(**kw)


def _sdpa(**kw):
    return _refused("trocm_sdpa_paged", *_with(dict(
        q=at(1), dtype=1, n=3, hq=8, hkv=2, sq=1, d=64, kp=at(2), vp=at(3), pages=8, page=16, ps=None, table=at(4), width=4, lens=at(5), out=at(6), scale=float("nan"), causal=1,
        ws=None, wsb=0, stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=5), "F32 or F16"), (dict(hq=7), "multiple"), (dict(hkv=0), "negative"), (dict(sq=-1), "negative"), (dict(d=-1), "negative"), (dict(q=None), "null pointer"), (dict(out=None), "out"),
    (dict(lens=None), "lens"), (dict(table=None), "table"), (dict(kp=None), "k_pages"), (dict(vp=None), "v_pages"), (dict(out=at(1)), "out overlaps q"), (dict(out=at(2)), "out overlaps k_pages"),
    (dict(out=at(4)), "out overlaps table"), (dict(ps=I3(0, 0, -1)), "negative page strides"), (dict(sq=1 << 24), "too large"), (dict(n=1 << 24), "sequences"), (dict(page=0), "page_size"),
    (dict(out=at(6) + 1), "aligned"), (dict(table=at(4) + 2), "aligned"), (dict(width=-2), "negative")])
def test_sdpa(kw, says):
    assert says in _sdpa(**kw)


def test_sdpa_workspace():
    n = C.c_size_t()
    assert "multiple" in _refused("trocm_sdpa_paged_workspace_bytes", 3, 7, 2, 1, 64, C.byref(n))
    assert "negative" in _refused("trocm_sdpa_paged_workspace_bytes", 3, 8, 0, 1, 64, C.byref(n))
    assert "null pointer" in _refused("trocm_sdpa_paged_workspace_bytes", 3, 8, 2, 1, 64, None)


def _reorder(**kw):
    return _refused("trocm_paged_reorder", *_with(dict(
        parents=at(1), n=4, page=16, table=at(2), width=6, lens=at(3), refs=at(4), free=at(5), count=at(6), pages=30, table_out=at(7), lens_out=at(8), refs_out=at(9), free_out=at(10),
        count_out=at(11), copies=at(12), missing=at(13), stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(parents=None), "parents"), (dict(table=None), "table"), (dict(table_out=None), "table_out"), (dict(refs=None), "refs"), (dict(free=None), "free_pages"), (dict(copies=None), "copies"),
    (dict(missing=None), "missing"), (dict(n=5000), "sequences"), (dict(n=-1), "negative"), (dict(page=0), "page_size"), (dict(table_out=at(2)), "table_out overlaps table"),
    (dict(lens_out=at(3)), "overlaps lens"), (dict(refs_out=at(4) + 8), "overlaps refs"), (dict(free_out=at(5)), "overlaps free_pages"), (dict(count_out=at(6)), "overlaps free_count"),
    (dict(copies=at(1)), "overlaps parents"), (dict(missing=at(12) + 4), "overlaps copies"), (dict(parents=at(1) + 2), "aligned")])
def test_reorder(kw, says):
    assert says in _reorder(**kw)


def _copy(**kw):
    return _refused("trocm_paged_copy", *_with(dict(copies=at(1), n=3, pools=(C.c_void_p * 2)(at(2), at(3)), pn=2, dtype=0, heads=2, d=64, pages=9, page=16, ps=None, stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(copies=None), "copies"), (dict(pools=None), "pools"), (dict(pools=(C.c_void_p * 2)(at(2), None)), "pool 1 is null"), (dict(n=-1), "negative"), (dict(pn=-1), "negative"), (dict(dtype=9), "F32 or F16"),
    (dict(pools=(C.c_void_p * 2)(at(1), at(3))), "overlaps copies"), (dict(pools=(C.c_void_p * 2)(at(2) + 2, at(3))), "aligned"), (dict(ps=I3(-5, 1, 1)), "negative page strides")])
def test_copy(kw, says):
    assert says in _copy(**kw)


def _select(**kw):
    return _refused("trocm_beam_select", *_with(dict(
        logits=at(1), dtype=1, batch=2, beams=4, vocab=1000, stride=0, scores=at(2), ended=None, eos=2, keep=8, so=at(3), parents=at(4), tokens=at(5), eo=at(6), ws=at(7), wsb=1 << 20, stream=None), kw))


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=2), "F32 or F16"), (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(keep=0), "keep"), (dict(keep=65), "keep"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 30), "vocab"),
    (dict(vocab=2, keep=9, eos=1), "continuations"), (dict(stride=999), "row_stride"), (dict(eos=1000), "eos"), (dict(eos=-2), "eos"), (dict(eos=-1, ended=at(8)), "need eos"), (dict(batch=-1), "negative"),
    (dict(logits=None), "logits"), (dict(scores=None), "scores"), (dict(so=None), "scores_out"), (dict(tokens=None), "tokens"), (dict(ws=None), "workspace"), (dict(so=at(2)), "overlaps scores"),
    (dict(tokens=at(4) + 8), "overlaps parents"), (dict(ws=at(1)), "workspace overlaps logits"), (dict(logits=at(1) + 1), "aligned"), (dict(batch=1 << 24), "too large")])
def test_select(kw, says):
    assert says in _select(**kw)


@pytest.mark.parametrize("ps", [I3(1 << 39, 64, 64), I3(1, 1 << 39, 64), I3(1, 64, 1 << 39)])
def test_strides_that_no_memory_has_room_for(ps):
    """(each below 2^40, but products with pages, heads or tokens that would leave 64 bits or any address space)"""
    assert "page strides too large" in _append(ps=ps, pages=1 << 10, page=1 << 12, heads=1 << 12)
    assert "page strides too large" in _sdpa(ps=ps, pages=1 << 10, page=1 << 12, hkv=1 << 12, hq=1 << 12)
    assert "page strides too large" in _copy(ps=ps, pages=1 << 10, page=1 << 12, heads=1 << 12)
    assert "row_stride" in _select(stride=1 << 40, batch=1 << 8)


@pytest.mark.parametrize("call,kw,says", [
    (_sdpa, dict(ws=at(7) + 8, wsb=1 << 16), "16-byte aligned"), (_sdpa, dict(ws=at(6), wsb=1 << 16), "workspace overlaps out"), (_sdpa, dict(ws=at(2), wsb=1 << 16), "workspace overlaps k_pages"),
    (_select, dict(ws=at(7) + 8), "16-byte aligned"), (_reorder, dict(pages=(1 << 24) + 1, page=1), "2^24"), (_copy, dict(n=(1 << 22) + 1), "2^22")])
def test_workspaces_and_what_would_take_too_long(call, kw, says):
    assert says in call(**kw)
