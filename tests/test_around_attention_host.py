"""Host side of the operators around attention: what Python passes on and refuses, with the library's calls recorded (no device)."""
import types

import numpy as np
import pytest

from tract_amd import TractRocmError, scored
from tract_amd.runtime import DeviceTensor

F16 = np.dtype(np.float16)
AT = 1 << 20   # an address that nothing reads



def _tensor(*shape, dtype=F16):
    return DeviceTensor(shape, dtype, ptr=AT)


def _cache(shape):
    return types.SimpleNamespace(_h=1, handle=1, _shape=shape)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(scored, "call", lambda name, *args: made.append(name))
    return made


@pytest.fixture
def sizes(monkeypatch):
    """The sizes that a call passes on, by position: (name, [its whole numbers])."""
    made = []
    monkeypatch.setattr(scored, "call", lambda name, *args: made.append((name, [a for a in args if type(a) is int])))
    monkeypatch.setattr(scored, "Workspace", _Workspace)
    return made


class _Workspace:
    """Takes the place of a workspace; `before` is called once as one is made: what another thread does meanwhile."""
    before = None

    def __init__(self, *args, nbytes=None):
        _Workspace.before, then = None, _Workspace.before
        if then:
            then()
        self.nbytes = self.bytes_for() if nbytes is None else nbytes
        self.buf = types.SimpleNamespace(ptr=AT)

    @staticmethod
    def bytes_for(*_):
        return 1000

    shared_bytes_for = bytes_for


def _interrupt(monkeypatch, then):
    """`then` runs once, as a call has no output yet and is about to make one (the allocation lets other threads run)."""
    output = scored._output

    def interrupted(*args):
        monkeypatch.setattr(scored, "_output", output)
        then()
        return output(*args)

    monkeypatch.setattr(scored, "_output", interrupted)


@pytest.mark.parametrize("d", [64, 256])
def test_a_shared_step_refuses_queries_of_another_head_size_than_the_caches(calls, d):
    """The library sizes q, the new rows and the output by the caches' head size: smaller tensors would be read and written past their ends."""
    caches = [_cache((1, 2, 0, 128)) for _ in range(4)]
    prefix = [_cache((1, 2, 9, 128)) for _ in range(2)]
    q, new = _tensor(2, 4, 1, d), _tensor(2, 2, 1, d)
    ws = types.SimpleNamespace(ptr=AT, nbytes=0)
    for rows in (new, None):
        with pytest.raises(TractRocmError, match="head size"):
            scored.inplace_kv_sdpa_eval_shared(q, rows, rows, *prefix, caches[:2], caches[2:], workspace=ws, out=_tensor(2, 4, 1, d))
    with pytest.raises(TractRocmError, match="rank 4"):
        scored.inplace_kv_sdpa_eval_shared(_tensor(2, 1, 128), None, None, *prefix, caches[:2], caches[2:], workspace=ws)
    assert not calls
    q, new = _tensor(2, 4, 1, 128), _tensor(2, 2, 1, 128)
    scored.inplace_kv_sdpa_eval_shared(q, new, new, *prefix, caches[:2], caches[2:], workspace=ws, out=_tensor(2, 4, 1, 128))
    assert calls == ["trocm_inplace_kv_sdpa_eval_shared"]


def _out(*shape):
    """An output of a shape that is right and a type that is equal but not the same object: looked at by `_output`, and allocates nothing."""
    t = _tensor(*shape)
    t.dtype = np.dtype(F16, copy=True)
    assert t.dtype is not F16
    return t


def test_norms_of_two_threads_keep_their_own_sizes(sizes, monkeypatch):
    op = scored.QkNormRope()

    def norm(n):
        q, k, c = _tensor(1, 4, n, 64), _tensor(1, 2, n, 64), _tensor(1, 1, n, 64)
        op.eval(q, k, None, None, c, c, q_out=_out(1, 4, n, 64), k_out=_tensor(1, 2, n, 64))

    norm(3)
    _interrupt(monkeypatch, lambda: norm(7000))
    norm(3)
    _interrupt(monkeypatch, lambda: norm(9))
    norm(5)
    assert [s[s.index(64) - 1] for _, s in sizes] == [3, 7000, 3, 9, 5]


def test_shared_prefixes_of_two_threads_keep_their_own_sizes(sizes, monkeypatch):
    op = scored.SharedPrefixSdpa()

    def attend(n):
        q, p, k = _tensor(n, 4, 1, 64), _tensor(1, 2, 11, 64), _tensor(n, 2, 5, 64)
        op.eval(q, p, p, k, k, [1] * n, out=_out(n, 4, 1, 64))

    attend(2)
    _interrupt(monkeypatch, lambda: attend(300))
    attend(2)
    assert [s[1] for _, s in sizes] == [2, 300, 2]
    other = scored.SharedPrefixSdpa()      # a first workspace that cannot be had leaves nothing behind
    _Workspace.before = lambda: (_ for _ in ()).throw(TractRocmError("no memory"))
    q, p, k = _tensor(2, 4, 1, 64), _tensor(1, 2, 11, 64), _tensor(2, 2, 5, 64)
    with pytest.raises(TractRocmError, match="no memory"):
        other.eval(q, p, p, k, k, [1, 1], out=_tensor(2, 4, 1, 64))
    other.eval(q, p, p, k, k, [1, 1], out=_tensor(2, 4, 1, 64))
    assert sizes[-1][1][1] == 2


def test_scored_attention_of_two_threads_keeps_its_own_sizes(sizes, monkeypatch):
    op = scored.ScoredSdpa(softcap=5.0)

    def attend(n):
        q, k = _tensor(1, 4, n, 64), _tensor(1, 2, n, 64)
        op.eval(q, k, k, out=_out(1, 4, n, 64))

    attend(2)
    _interrupt(monkeypatch, lambda: attend(300))
    attend(2)
    assert [s[s.index(64) - 1] for _, s in sizes] == [2, 300, 2]


@pytest.mark.parametrize("make", [scored.SharedPrefixSdpa, scored.ScoredSdpa])
def test_a_workspace_that_was_outgrown_stays(sizes, monkeypatch, make):
    """A recorded graph goes on using the workspace of the call that it recorded, by address; a call's share is that of its shape."""
    op, made, alive = make(), [], set()

    class Counted(_Workspace):
        bytes_for = shared_bytes_for = staticmethod(lambda b, hq, sq, d: 100 * b * sq)

        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            made.append(self.nbytes)
            alive.add(self.nbytes)

        def __del__(self):
            alive.discard(getattr(self, "nbytes", None))

    monkeypatch.setattr(scored, "Workspace", Counted)
    for n in (2, 40, 2, 30, 41, 7, 500, 3):
        q, p, k = _tensor(n, 4, 1, 64), _tensor(1, 2, 11, 64), _tensor(n, 2, 5, 64)
        if make is scored.ScoredSdpa:
            op.eval(q, k, k, out=_tensor(n, 4, 1, 64))
        else:
            op.eval(q, p, p, k, k, [1] * n, out=_tensor(n, 4, 1, 64))
        assert sizes[-1][1][-1] == 100 * n
    assert alive == set(made) and len(made) <= 4 and sum(made) <= 2 * made[-1]
