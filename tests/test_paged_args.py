"""Refusals of the paged KV cache's launchers: sizes, types, alignment and null pointers are turned
into a status and a message before any device work (CPU: no device is needed for them)."""
import ctypes as C

import pytest

from tl_amd import BackendError, PagedKV, _lib

F32, F16 = 0, 1
P = 1 << 20  # an aligned address that no refused call follows


def _copy(**kw):
    a = dict(k=P, v=P, layers=1, pages=8, page_bytes=1024, src=(0,), dst=(1,), n=None)
    a.update(kw)
    n = len(a["src"]) if a["n"] is None else a["n"]
    src, dst = ((C.c_int32 * max(1, len(a[i])))(*a[i]) for i in ("src", "dst"))
    return _lib.load().tl_hip_launch_kv_copy_pages(a["k"], a["v"], a["layers"], a["pages"], a["page_bytes"], src, dst, n, None)


def _append(**kw):
    a = dict(kn=P, vn=P, nt=F32, ks=1024, vs=1024, k=P, v=P, kt=F16, pages=8, ps=16, hkv=8, d=128, table=P, stride=4, cu=P,
             lens=P, batch=2, rows=5)
    a.update(kw)
    return _lib.load().tl_hip_launch_kv_append(*a.values(), None)


def _attend(decode, **kw):
    a = dict(q=P, qt=F32, qs=4096, k=P, v=P, kt=F16, pages=8, ps=16, hq=32, hkv=8, d=128, table=P, stride=4, cu=P, lens=P,
             batch=2, rows=5, out=P, scale=0.1, ws=None, wsb=0)
    a.update(kw)
    if decode:
        del a["cu"], a["rows"]
        return _lib.load().tl_hip_launch_paged_attention_decode(*a.values(), None)
    return _lib.load().tl_hip_launch_paged_attention_prefill(*a.values(), None)


def _refused(rc, status):
    lib = _lib.load()
    assert rc == status == lib.tl_hip_last_status() and lib.tl_hip_last_error()


CACHE = [(dict(kt=2), 7), (dict(ps=8), 8), (dict(ps=48), 8), (dict(ps=65536), 8), (dict(d=12), 8), (dict(d=0), 8),
         (dict(d=264), 8), (dict(pages=0), 8), (dict(pages=1 << 31), 8), (dict(batch=-1), 8), (dict(batch=65537), 8),
         (dict(stride=0), 8), (dict(stride=(1 << 26) + 1), 8)]


@pytest.mark.parametrize("kw,status", CACHE + [
    (dict(nt=3), 7), (dict(kn=None), 4), (dict(v=None), 4), (dict(table=None), 4), (dict(cu=None), 4), (dict(lens=None), 4),
    (dict(kn=P + 4), 8), (dict(v=P + 8), 8), (dict(ks=1023), 8), (dict(vs=1020), 8), (dict(nt=F16, ks=1028), 8),
    (dict(hkv=0), 8), (dict(rows=-1), 8), (dict(rows=(1 << 24) + 1), 8)])
def test_append_refuses(kw, status):
    _refused(_append(**kw), status)


@pytest.mark.parametrize("kw,status", [
    (dict(layers=0), 8), (dict(layers=32768), 8), (dict(pages=0), 8), (dict(page_bytes=24), 8), (dict(page_bytes=0), 8),
    (dict(k=None), 4), (dict(v=P + 4), 8), (dict(n=-1), 8), (dict(src=(0,) * 9, dst=tuple(range(9))), 8),
    (dict(src=(8,)), 6), (dict(src=(-1,)), 6), (dict(dst=(8,)), 6), (dict(dst=(-1,)), 6),
    (dict(src=(0, 1), dst=(2, 2)), 8), (dict(src=(0, 1), dst=(1, 2)), 8), (dict(src=(3,), dst=(3,)), 8)])
def test_copy_refuses(kw, status):
    _refused(_copy(**kw), status)


def test_copy_refuses_missing_pairs():
    _refused(_lib.load().tl_hip_launch_kv_copy_pages(P, P, 1, 8, 1024, None, None, 1, None), 4)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kw,status", CACHE + [
    (dict(qt=F16, kt=F32), 7), (dict(qt=5), 7), (dict(hq=30), 8), (dict(hq=0), 8), (dict(hkv=0), 8), (dict(hkv=64), 8),
    (dict(q=None), 4), (dict(k=None), 4), (dict(lens=None), 4), (dict(out=None), 4), (dict(table=None), 4),
    (dict(q=P + 4), 8), (dict(k=P + 8), 8), (dict(out=P + 2), 8), (dict(qs=4095), 8), (dict(qs=4092), 8), (dict(qs=4098), 8),
    (dict(qt=F16, qs=4100), 8), (dict(scale=float("nan")), 8), (dict(scale=float("inf")), 8),
    (dict(ws=P, wsb=8), 8), (dict(ws=P + 8, wsb=1 << 40), 8)])
def test_attention_refuses(decode, kw, status):
    _refused(_attend(decode, **kw), status)


def test_prefill_refuses_a_missing_cu_seqlens():
    _refused(_attend(False, cu=None), 4)
    _refused(_attend(False, rows=-1), 8)


def test_empty_calls_do_nothing():
    assert _append(batch=0) == 0 and _append(rows=0) == 0 and _copy(src=(), dst=()) == 0
    for decode in (True, False):
        assert _attend(decode, batch=0, q=None, out=None) == 0
    assert _attend(False, rows=0) == 0


def test_workspace_sizes():
    ws = _lib.load().tl_hip_paged_attention_workspace
    assert ws(32, 32, 32, 8, 128) > 0 and ws(1, 8192, 32, 8, 256) > 0
    for bad in ((-1, 1, 32, 8, 128), (1, 1, 30, 8, 128), (1, 1, 32, 8, 100), (1, 1 << 25, 32, 8, 128)):
        assert ws(*bad) == 0 and _lib.load().tl_hip_last_status() == 8


@pytest.mark.parametrize("name", ["table", "cu", "lens"])
def test_integer_arrays_off_their_alignment(name):
    _refused(_append(**{name: P + 2}), 8)
    _refused(_attend(False, **{name: P + 2}), 8)
    if name != "cu":
        _refused(_attend(True, **{name: P + 2}), 8)


class _NoDevice:
    """What PagedKV asks of a device, without one: its launches end in an error."""

    class Tensor:
        def __init__(self, shape, dtype):
            self.shape, self.dtype, self.data_ptr = tuple(shape), dtype, P

    def __init__(self):
        self.lib = _lib.load()

    def tensor_zeros(self, shape, dtype=F32):
        return self.Tensor(shape, dtype)

    def tensor_new(self, a):
        return self.Tensor(a.shape, F32)


def _kv():
    kv = PagedKV(_NoDevice(), 8, 16, 2, 64)
    return kv, kv.open(), kv.open()


@pytest.mark.parametrize("counts", [[1], [1, 1, 1], [3, -1]])
def test_prefill_wants_a_row_count_per_sequence(counts):
    kv, a, b = _kv()
    with pytest.raises(BackendError):
        kv.prefill([a, b], counts, _NoDevice.Tensor((sum(counts), 4, 64), F32), 0.1)


def test_an_append_that_fails_leaves_the_lengths():
    kv, a, b = _kv()
    kv.book.grow(a, 5)
    rows = _NoDevice.Tensor((16 * 8, 2, 64), F32)
    with pytest.raises(BackendError):   # a's 100 fit, b's 28 do not
        kv.append([a, b], [100, 28], rows, rows)
    assert (kv.length(a), kv.length(b), kv.book.free_pages) == (5, 0, 7)
    rows = _NoDevice.Tensor((9, 2, 64), 5)   # a type that the launcher refuses
    with pytest.raises(BackendError):
        kv.append([a, b], [4, 5], rows, rows)
    assert (kv.length(a), kv.length(b), kv.book.free_pages) == (5, 0, 7)
    with pytest.raises(BackendError):
        kv.append([a, a], [4, 5], rows, rows)
    assert kv.length(a) == 5
