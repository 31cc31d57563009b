"""The paged KV cache on the GPU: append, page copies, decode and prefill attention against
tests/paged_f64.py at the sizes, types and contents where they can go wrong, and all of them
together through PagedKV."""
import ctypes as C

import numpy as np
import pytest

from paged_f64 import attention
from tl_amd import BackendError, HipDevice, PagedKV, _lib

pytestmark = pytest.mark.gpu
F32, F16 = 0, 1
NP = {F32: np.float32, F16: np.float16}


def put(dev, a):
    """A device tensor with the bytes of `a` (int32 and f32 as f32 words)."""
    a = np.ascontiguousarray(a)
    if a.dtype == np.float16:
        return dev.tensor_new_f16(a)
    return dev.tensor_new(a.view(np.float32))


def get(t, dtype, shape):
    lib = _lib.load()
    a = np.empty(shape, dtype)
    assert lib.tl_hip_synchronize() == 0
    assert lib.tl_hip_memcpy_d2h(a.ctypes.data, t.data_ptr, a.nbytes) == 0
    return a


class Setup:
    """A pool with garbage in every slot that no sequence holds, and scrambled page tables."""

    def __init__(self, dev, seed, lens, ps, hkv, D, kt, width=None, junk=np.nan):
        r = np.random.default_rng(seed)
        self.dev, self.lens, self.ps, self.hkv, self.D, self.kt = dev, list(lens), ps, hkv, D, kt
        need = [-(-n // ps) for n in lens]
        self.n_pages = sum(need) + 3
        self.width = width or max(need + [1])
        order = r.permutation(self.n_pages)
        self.table = np.full((len(lens), self.width), -7, np.int32)   # entries past the length: never read
        self.k = np.full((self.n_pages, hkv, ps, D), junk, NP[kt])
        self.v = np.full((self.n_pages, hkv, ps, D), junk, NP[kt])
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
            j = np.arange(lens[b])
            for x in (self.k, self.v):
                x[self.table[b, j // ps], :, j % ps] = r.standard_normal((lens[b], hkv, D)).astype(NP[kt])
        self.rng = r

    def upload(self):
        self.tk, self.tv, self.tt = put(self.dev, self.k), put(self.dev, self.v), put(self.dev, self.table)
        self.tl = put(self.dev, np.asarray(self.lens, np.int32))


def run_attention(s, q, scale, cu=None, stride=None, ws=None, stream=None, out=None, upload=True):
    """q [rows, heads, D] at a row stride; decode where cu is None."""
    lib, dev = _lib.load(), s.dev
    rows, heads, D = q.shape
    if upload:
        s.upload()
    stride = stride or heads * D
    wide = np.zeros((rows, stride), q.dtype)
    wide[:, : heads * D] = q.reshape(rows, -1)
    tq = put(dev, wide)
    to = out if out is not None else put(dev, np.full(q.shape, 7, q.dtype))
    qt = F16 if q.dtype == np.float16 else F32
    wp, wb = (ws.data_ptr, ws.numel * 4) if ws is not None else (None, 0)
    if cu is None:
        rc = lib.tl_hip_launch_paged_attention_decode(
            tq.data_ptr, qt, stride, s.tk.data_ptr, s.tv.data_ptr, s.kt, s.n_pages, s.ps, heads, s.hkv, D, s.tt.data_ptr,
            s.width, s.tl.data_ptr, len(s.lens), to.data_ptr, scale, wp, wb, stream)
    else:
        tc = put(dev, np.asarray(cu, np.int32))
        rc = lib.tl_hip_launch_paged_attention_prefill(
            tq.data_ptr, qt, stride, s.tk.data_ptr, s.tv.data_ptr, s.kt, s.n_pages, s.ps, heads, s.hkv, D, s.tt.data_ptr,
            s.width, tc.data_ptr, s.tl.data_ptr, len(s.lens), rows, to.data_ptr, scale, wp, wb, stream)
    assert rc == 0, lib.tl_hip_last_error()
    return get(to, q.dtype, q.shape)


def check(got, want, tol):
    """Rows of no sequence (NaN in `want`) still hold what the buffer held."""
    none = np.isnan(want)
    assert np.all(got[none] == 7)
    err = np.abs(got.astype(np.float64) - want)[~none]
    assert np.isfinite(err).all()
    worst = np.max(err - tol[~none]) if err.size else -1
    assert worst <= 0, f"{(err > tol[~none]).sum()} of {err.size} off, the worst by {worst:.3e} beyond the bound"


TYPES = [(np.float32, F32), (np.float32, F16), (np.float16, F16)]


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,G,D,ps,lens", [
    (8, 4, 128, 64, [512]),
    (4, 8, 64, 16, [1, 15, 16, 17, 0, 33, 64, 257]),
    (2, 7, 80, 32, [129, 1000, 31]),
    (1, 16, 256, 128, [300, 1]),
    (3, 1, 96, 64, [65, 127, 128, 700]),
    (1, 33, 128, 16, [70, 200]),
    (2, 3, 8, 16, [40]),
    (2, 4, 200, 256, [513, 0, 0, 255]),
    (5, 2, 40, 64, [2300]),
])
def test_decode(dev, qt, kt, hkv, G, D, ps, lens):
    s = Setup(dev, 11 + D, lens, ps, hkv, D, kt)
    q = s.rng.standard_normal((len(lens), hkv * G, D)).astype(qt)
    scale = D ** -0.5
    got = run_attention(s, q, scale)
    want, tol = attention(q, s.k, s.v, s.table, s.lens, np.arange(len(lens) + 1), ps, scale, qt == np.float16)
    check(got, want, tol)


def test_decode_many_ragged_sequences(dev):
    """More sequences than a wavefront has lanes, most of them short, some empty, one long."""
    r = np.random.default_rng(3)
    lens = r.integers(0, 60, 150).tolist()
    lens[77], lens[149], lens[0] = 5000, 1, 0
    s = Setup(dev, 5, lens, 16, 2, 64, F16)
    q = s.rng.standard_normal((150, 8, 64)).astype(np.float32)
    got = run_attention(s, q, 0.125)
    want, tol = attention(q, s.k, s.v, s.table, lens, np.arange(151), 16, 0.125, False)
    check(got, want, tol)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,G,D,ps,new,past,extra", [
    (2, 4, 64, 16, [1], [0], 0),
    (2, 4, 128, 64, [70, 1, 33], [0, 200, 64], 3),
    (1, 8, 64, 32, [129, 0, 5], [0, 17, 300], 0),
    (2, 1, 96, 128, [100, 64], [13, 0], 1),
    (1, 7, 80, 16, [40, 3], [100, 0], 2),
    (2, 3, 256, 64, [67], [190], 0),
    (1, 16, 40, 256, [19, 2], [500, 254], 0),
    (1, 33, 64, 16, [9], [30], 0),
    (1, 2, 200, 64, [150], [0], 0),
    (4, 8, 64, 64, [300, 280], [0, 40], 5),
    (1, 130, 64, 16, [3], [20], 0),
])
def test_prefill(dev, qt, kt, hkv, G, D, ps, new, past, extra):
    lens = [n + p for n, p in zip(new, past)]
    s = Setup(dev, 17 + D, lens, ps, hkv, D, kt)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = s.rng.standard_normal((cu[-1] + extra, hkv * G, D)).astype(qt)
    scale = D ** -0.5
    got = run_attention(s, q, scale, cu=cu)
    want, tol = attention(q, s.k, s.v, s.table, lens, cu, ps, scale, qt == np.float16)
    check(got, want, tol)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,G,D,ps,new,past,extra,room", [
    (4, 4, 64, 16, [150, 1], [0, 700], 2, 16384),        # few tiles under a wide table: positions cut
    (2, 4, 128, 64, [130, 0, 31], [900, 50, 0], 0, 32768),
    (2, 7, 96, 32, [64], [1500], 1, 32768),
    (1, 3, 256, 128, [200, 70], [333, 0], 0, 65536),
    (1, 5, 136, 16, [90], [400], 0, 65536),
    (1, 1, 40, 256, [300], [2000], 0, 65536),
    (40, 4, 64, 16, [150, 10], [100, 0], 1, 0),          # fewer tiles than CUs, whole
    (50, 4, 128, 64, [128], [300], 0, 0),
    (9, 33, 72, 32, [31, 1, 60], [0, 64, 3], 2, 0),
    (64, 4, 64, 64, [135], [60], 0, 0),                  # enough tiles to stay whole
    (64, 4, 128, 16, [129, 2], [0, 33], 3, 0),
    (66, 4, 80, 64, [128], [0], 0, 0),
    (64, 2, 256, 32, [257], [20], 0, 0),
])
def test_prefill_of_long_prompts(dev, qt, kt, hkv, G, D, ps, new, past, extra, room):
    lens = [n + p for n, p in zip(new, past)]
    s = Setup(dev, 27 + D, lens, ps, hkv, D, kt, width=room // ps or None)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = s.rng.standard_normal((cu[-1] + extra, hkv * G, D)).astype(qt)
    scale = D ** -0.5
    got = run_attention(s, q, scale, cu=cu)
    check(got, *attention(q, s.k, s.v, s.table, lens, cu, ps, scale, qt == np.float16))
    # what only later rows see, on whichever tile's edge it falls
    b = int(np.argmax(new))
    j = lens[b] - new[b] // 2
    s.v[s.table[b, j // ps], :, j % ps, D // 2] = np.inf
    s.k[s.table[b, (lens[b] - 1) // ps], :, (lens[b] - 1) % ps] = np.nan
    again = run_attention(s, q, scale, cu=cu)
    first = cu[b] + new[b] - new[b] // 2
    assert not np.isfinite(again[first:cu[b + 1], :, D // 2]).any() and np.isnan(again[cu[b + 1] - 1]).all()
    same = np.ones(got.shape, bool)
    same[first:cu[b + 1], :, D // 2] = False
    same[cu[b + 1] - 1] = False
    assert np.array_equal(again[same], got[same])


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,G,D,room", [(64, 2, 64, 0), (1, 3, 64, 65536), (1, 2, 128, 65536)])
def test_prefill_of_many_short_prompts(dev, qt, kt, hkv, G, D, room):
    """More sequences than lanes, empty ones and ones with more rows than positions among them."""
    r = np.random.default_rng(33)
    new = r.integers(0, 30, 83)
    lens = [int(n + p) for n, p in zip(new, r.integers(-4, 40, 83))]
    lens = [max(n, 0) for n in lens]
    s = Setup(dev, 34, lens, 16, hkv, D, kt, width=room // 16 or None)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = s.rng.standard_normal((cu[-1] + 1, hkv * G, D)).astype(qt)
    check(run_attention(s, q, 0.2, cu=cu), *attention(q, s.k, s.v, s.table, lens, cu, 16, 0.2, qt == np.float16))


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,room", [(2, 16384), (64, 512)])   # positions cut, and whole
def test_prompts_over_bad_pages_lengths_and_offsets(dev, qt, kt, hkv, room):
    new, past, G, D = [170, 40], [90, 0], 4, 64
    lens = [n + p for n, p in zip(new, past)]
    s = Setup(dev, 35, lens, 16, hkv, D, kt, width=room // 16)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = s.rng.standard_normal((210, hkv * G, D)).astype(qt)
    want = run_attention(s, q, 0.2, cu=cu)
    check(want, *attention(q, s.k, s.v, s.table, lens, cu, 16, 0.2, qt == np.float16))
    good = s.table.copy()
    for entry in (-1, 1 << 30, -(1 << 31)):
        s.table[0, 9] = entry   # positions 144 .. 159
        got = run_attention(s, q, 0.2, cu=cu)
        first = 144 - past[0]
        assert np.isnan(got[first:170]).all()
        assert np.array_equal(got[:first], want[:first]) and np.array_equal(got[170:], want[170:])
    s.table = good
    # a length past the table: rows at positions past its end are NaN, those before see what it holds
    s.width = 16
    s.table = np.ascontiguousarray(good[:, :16])
    s.lens = [260, 40]
    if hkv == 64:
        got = run_attention(s, q, 0.2, cu=cu)
        assert np.isnan(got[166:170]).all() and np.isfinite(got[:166]).all() and np.array_equal(got[170:], want[170:])
        assert np.array_equal(got[:166], want[:166])
    s.table, s.width = good, room // 16
    # offsets that fall or leave the rows: the first to claim a row has it
    got = run_attention(s, q, 0.2, cu=[0, 170, 1 << 30])
    assert np.array_equal(got, want)
    got = run_attention(s, q, 0.2, cu=[-5, 170, 90])
    assert np.array_equal(got[:170], want[:170]) and np.all(got[170:] == 7)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("hkv,G,D", [(2, 5, 64), (1, 8, 40), (1, 4, 80), (2, 16, 128)])
def test_decode_of_few_long_sequences(dev, qt, kt, hkv, G, D):
    lens = [5000, 0, 1, 4097]
    s = Setup(dev, 28, lens, 32, hkv, D, kt)
    q = s.rng.standard_normal((4, hkv * G, D)).astype(qt)
    check(run_attention(s, q, 0.1), *attention(q, s.k, s.v, s.table, lens, range(5), 32, 0.1, qt == np.float16))


@pytest.mark.parametrize("qt,kt", TYPES)
def test_prefill_more_rows_than_positions(dev, qt, kt):
    """kv_lens below the number of rows: the first rows sit before position 0 and are zeros."""
    s = Setup(dev, 8, [20, 0], 16, 2, 64, kt)
    q = s.rng.standard_normal((38, 8, 64)).astype(qt)
    cu = [0, 33, 38]
    got = run_attention(s, q, 0.125, cu=cu)
    want, tol = attention(q, s.k, s.v, s.table, s.lens, cu, 16, 0.125, qt == np.float16)
    assert np.all(want[:13] == 0) and np.all(want[33:] == 0)
    check(got, want, tol)
    assert np.all(got[:13] == 0) and np.all(got[33:] == 0)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(dev, qt, kt, scale):
    s = Setup(dev, 9, [150, 40], 16, 2, 64, kt)
    q = s.rng.standard_normal((12, 8, 64)).astype(qt)
    cu = [0, 9, 12]
    check(run_attention(s, q, scale, cu=cu), *attention(q, s.k, s.v, s.table, s.lens, cu, 16, scale, qt == np.float16))
    q = q[:2]
    check(run_attention(s, q, scale), *attention(q, s.k, s.v, s.table, s.lens, [0, 1, 2], 16, scale, qt == np.float16))


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e25])
def test_queries_far_from_one(dev, size):
    """f32 queries over an f16 cache reach the f16 matrix units in two parts: tiny and huge rows
    keep their digits.  The scale takes the size out again."""
    s = Setup(dev, 10, [190, 33], 16, 2, 128, F16)
    q = (s.rng.standard_normal((2, 8, 128)) * size).astype(np.float32)
    q[:, ::2, :64] *= np.float32(2.0 ** -11)   # small entries beside large ones of the same row
    scale = float(np.float32(0.09 / size))
    check(run_attention(s, q, scale), *attention(q, s.k, s.v, s.table, s.lens, [0, 1, 2], 16, scale, False))
    cu = [0, 1, 2]
    check(run_attention(s, q, scale, cu=cu), *attention(q, s.k, s.v, s.table, s.lens, cu, 16, scale, False))


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_only(dev, qt, kt, bad):
    new, past, ps = [90], [30], 16
    s = Setup(dev, 12, [120], ps, 2, 64, kt)
    for j, d in ((75, 3), (100, 17), (119, 60)):   # dims 3, 17, 60 from positions 75, 100, 119 on
        s.v[s.table[0, j // ps], :, j % ps, d] = bad
    q = s.rng.standard_normal((90, 8, 64)).astype(qt)
    cu = [0, 90]
    got = run_attention(s, q, 0.125, cu=cu).astype(np.float64)
    clean_v = np.where(np.isfinite(s.v), s.v, 0)
    want, tol = attention(q, s.k, clean_v, s.table, [120], cu, ps, 0.125, qt == np.float16)
    sees = np.zeros((90, 64), bool)
    for j, d in ((75, 3), (100, 17), (119, 60)):
        sees[j - 30:, d] = True
    sees = np.broadcast_to(sees[:, None], got.shape)
    assert not np.isfinite(got[sees]).any()
    assert (np.abs(got - want) <= tol)[~sees].all()


@pytest.mark.parametrize("qt,kt", TYPES)
def test_keys_that_are_not_finite_behind_a_row_are_not_seen(dev, qt, kt):
    s = Setup(dev, 13, [60], 16, 1, 64, kt)
    s.k[s.table[0, 3], 0, 2] = np.nan   # position 50
    q = s.rng.standard_normal((40, 4, 64)).astype(qt)
    got = run_attention(s, q, 0.125, cu=[0, 40])
    clean = np.where(np.isnan(s.k), 0, s.k)
    want, tol = attention(q, clean, s.v, s.table, [60], [0, 40], 16, 0.125, qt == np.float16)
    assert np.isnan(got[30:]).all()
    assert (np.abs(got.astype(np.float64) - want) <= tol)[:30].all()


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31)])
def test_bad_pages_make_their_rows_nan_and_nothing_else(dev, qt, kt, entry):
    s = Setup(dev, 14, [100, 64, 100], 16, 2, 64, kt)
    want, tol = attention(np.zeros((3, 8, 64)), s.k, s.v, s.table, s.lens, range(4), 16, 0.125, False)
    q = s.rng.standard_normal((3, 8, 64)).astype(qt)
    want, tol = attention(q, s.k, s.v, s.table, s.lens, range(4), 16, 0.125, qt == np.float16)
    qp = s.rng.standard_normal((30, 8, 64)).astype(qt)
    cu = [0, 10, 20, 30]
    wp, tp = attention(qp, s.k, s.v, s.table, s.lens, cu, 16, 0.125, qt == np.float16)
    s.table[1, 3] = entry   # positions 48 .. 63 of sequence 1
    got = run_attention(s, q, 0.125)
    assert np.isnan(got[1]).all()
    check(got[[0, 2]], want[[0, 2]], tol[[0, 2]])
    got = run_attention(s, qp, 0.125, cu=cu)
    assert np.isnan(got[10:20]).all()       # positions 54 .. 63
    check(np.delete(got, range(10, 20), 0), np.delete(wp, range(10, 20), 0), np.delete(tp, range(10, 20), 0))


def test_lengths_past_the_table(dev):
    """kv_lens past the table's positions: rows at positions past them are NaN, others exact."""
    s = Setup(dev, 15, [64, 30], 16, 1, 64, F16)
    s.lens = [1 << 30, 30]
    q = s.rng.standard_normal((2, 4, 64)).astype(np.float32)
    got = run_attention(s, q, 0.125)
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()
    s.lens = [70, 30]
    q = s.rng.standard_normal((20, 4, 64)).astype(np.float32)   # positions 55 .. 69 and 25 .. 29
    got = run_attention(s, q, 0.125, cu=[0, 15, 20])
    assert np.isnan(got[9:15]).all()
    want, tol = attention(q[6:], s.k, s.v, s.table, [64, 30], [0, 9, 14], 16, 0.125, False)
    q2 = np.concatenate([q[:9], q[15:]])
    want, tol = attention(q2, s.k, s.v, s.table, [64, 30], [0, 9, 14], 16, 0.125, False)
    check(np.concatenate([got[:9], got[15:]]), want, tol)
    s.lens = [-5, 30]
    got = run_attention(s, q2[:2], 0.125)
    assert np.all(got[0] == 0) and np.isfinite(got[1]).all()


def test_cu_seqlens_out_of_range_stay_in_range(dev):
    s = Setup(dev, 16, [40, 40], 16, 1, 64, F16)
    q = s.rng.standard_normal((10, 4, 64)).astype(np.float32)
    got = run_attention(s, q, 0.125, cu=[-3, 4, 1 << 20])       # as 0, 4, 10
    want, tol = attention(q, s.k, s.v, s.table, [40, 40], [0, 4, 10], 16, 0.125, False)
    check(got, want, tol)
    got = run_attention(s, q, 0.125, cu=[4, 2, 6])              # sequence 0 holds no rows
    want, tol = attention(q, s.k, s.v, s.table, [40, 40], [2, 2, 6], 16, 0.125, False)
    check(got, want, tol)


@pytest.mark.parametrize("qt,kt", TYPES)
def test_row_strides_workspaces_and_streams(dev, qt, kt):
    lib = _lib.load()
    lens, new, cu = [200, 900, 17], [3, 40, 2], [0, 3, 43, 45]
    s = Setup(dev, 18, lens, 64, 2, 128, kt, width=40)
    scale = 128 ** -0.5
    q = s.rng.standard_normal((45, 8, 128)).astype(qt)
    need = lib.tl_hip_paged_attention_workspace(3, 45, 8, 2, 128)
    ws = put(dev, np.full(-(-need // 4), np.nan, np.float32))
    plain = run_attention(s, q, scale, cu=cu)
    check(plain, *attention(q, s.k, s.v, s.table, lens, cu, 64, scale, qt == np.float16))
    assert np.array_equal(run_attention(s, q, scale, cu=cu, stride=3 * 8 * 128 + 16, ws=ws), plain)
    first = run_attention(s, q[:3], scale)
    assert np.array_equal(run_attention(s, q[:3], scale, ws=ws, stride=2048), first)


def test_lens_and_splits_repeat_themselves(dev):
    """The same call gives the same bits each time, split over the length or not."""
    s = Setup(dev, 19, [30000, 5], 256, 2, 128, F16)
    q = s.rng.standard_normal((2, 16, 128)).astype(np.float32)
    first = run_attention(s, q, 0.09)
    check(first, *attention(q, s.k, s.v, s.table, s.lens, range(3), 256, 0.09, False))
    for _ in range(3):
        assert np.array_equal(run_attention(s, q, 0.09, upload=False), first)
    qp = s.rng.standard_normal((6, 16, 128)).astype(np.float32)
    first = run_attention(s, qp, 0.09, cu=[0, 4, 6])
    check(first, *attention(qp, s.k, s.v, s.table, s.lens, [0, 4, 6], 256, 0.09, False))
    assert np.array_equal(run_attention(s, qp, 0.09, cu=[0, 4, 6], upload=False), first)


@pytest.mark.parametrize("qt,kt", TYPES)
def test_parts_joined_in_the_same_launch_or_after_it(dev, qt, kt):
    """The two forms give the same bits: long and short sequences, empty ones, more rows than one
    tile holds."""
    lib = _lib.load()
    lens = [9000, 0, 3, 700, 1, 0, 2500]
    s = Setup(dev, 25, lens, 64, 2, 128, kt)
    q = s.rng.standard_normal((len(lens), 40, 128)).astype(qt)
    new = [5, 0, 3, 40, 1, 7, 2]
    cu = np.concatenate([[0], np.cumsum(new)])
    qp = s.rng.standard_normal((cu[-1], 40, 128)).astype(qt)
    got = {}
    was = lib.tl_hip_debug_one_launch_merge(-1)
    for form in (0, 1):
        before = lib.tl_hip_debug_one_launch_merge(form)
        try:
            got[form] = run_attention(s, q, 0.09), run_attention(s, qp, 0.09, cu=cu)
        finally:
            lib.tl_hip_debug_one_launch_merge(before)
    check(got[0][0], *attention(q, s.k, s.v, s.table, lens, range(8), 64, 0.09, qt == np.float16))
    check(got[0][1], *attention(qp, s.k, s.v, s.table, lens, cu, 64, 0.09, qt == np.float16))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    assert lib.tl_hip_debug_one_launch_merge(-1) == was


def test_offsets_past_32_bits(dev):
    """Pools past 4 GiB each: the pages in use lie at their far end."""
    lib = _lib.load()
    ps, hkv, D, lens = 256, 8, 128, [700]
    page = hkv * ps * D
    n_pages = (5 << 30) // (page * 2)
    s = Setup(dev, 20, lens, ps, hkv, D, F16)
    q = s.rng.standard_normal((1, 32, D)).astype(np.float32)
    small = run_attention(s, q, 0.09)
    big = [lib.tl_hip_malloc(n_pages * page * 2) for _ in range(2)]
    try:
        assert all(big)
        far = n_pages - s.n_pages
        for p, a in zip(big, (s.k, s.v)):
            assert lib.tl_hip_memcpy_h2d(p + far * page * 2, np.ascontiguousarray(a).ctypes.data, a.nbytes) == 0
        tt, tq = put(dev, s.table + far), put(dev, q)
        to = put(dev, np.zeros_like(q))
        rc = lib.tl_hip_launch_paged_attention_decode(tq.data_ptr, F32, 32 * D, big[0], big[1], F16, n_pages, ps, 32, hkv, D,
                                                      tt.data_ptr, s.width, s.tl.data_ptr, 1, to.data_ptr, 0.09, None, 0, None)
        assert rc == 0, lib.tl_hip_last_error()
        assert np.array_equal(get(to, np.float32, q.shape), small)
        qp = s.rng.standard_normal((50, 32, D)).astype(np.float32)
        want = run_attention(s, qp, 0.09, cu=[0, 50])
        tq, to, tc = put(dev, qp), put(dev, np.zeros_like(qp)), put(dev, np.asarray([0, 50], np.int32))
        rc = lib.tl_hip_launch_paged_attention_prefill(tq.data_ptr, F32, 32 * D, big[0], big[1], F16, n_pages, ps, 32, hkv, D,
                                                       tt.data_ptr, s.width, tc.data_ptr, s.tl.data_ptr, 1, 50, to.data_ptr,
                                                       0.09, None, 0, None)
        assert rc == 0, lib.tl_hip_last_error()
        assert np.array_equal(get(to, np.float32, qp.shape), want)
        # append and copy at the far end
        rows = s.rng.standard_normal((700, 2, hkv * D)).astype(np.float32)
        tr, tc = put(dev, rows), put(dev, np.asarray([0, 700], np.int32))
        rc = lib.tl_hip_launch_kv_append(tr.data_ptr, tr.data_ptr + 4 * hkv * D, F32, 2 * hkv * D, 2 * hkv * D, big[0], big[1], F16,
                                         n_pages, ps, hkv, D, tt.data_ptr, s.width, tc.data_ptr, s.tl.data_ptr, 1, 700, None)
        assert rc == 0, lib.tl_hip_last_error()
        src, dst = (C.c_int32 * 1)(int(s.table[0, 0]) + far), (C.c_int32 * 1)(0)
        assert lib.tl_hip_launch_kv_copy_pages(big[0], big[1], 1, n_pages, 2 * page, src, dst, 1, None) == 0
        for i, p in enumerate(big):
            got = np.empty((hkv, ps, D), np.float16)
            assert lib.tl_hip_memcpy_d2h(got.ctypes.data, p, got.nbytes) == 0
            want = rows[:ps, i].reshape(ps, hkv, D).transpose(1, 0, 2).astype(np.float16)
            assert np.array_equal(got, want)
    finally:
        lib.tl_hip_synchronize()
        for p in big:
            lib.tl_hip_free(p)


# ------------------------------------------------------------------- append, copy ----
@pytest.mark.parametrize("nt,kt", [(F32, F16), (F32, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("hkv,D,ps,new,past,extra", [
    (8, 128, 64, [1] * 5, [0, 63, 64, 65, 300], 0),
    (4, 64, 16, [33, 0, 100, 1], [5, 7, 0, 15], 3),
    (1, 8, 16, [40], [0], 0),
    (3, 200, 256, [300, 2], [250, 0], 1),
    (2, 256, 32, [31] * 70, [1] * 70, 0),
])
def test_append(dev, nt, kt, hkv, D, ps, new, past, extra):
    lib = _lib.load()
    lens = [n + p for n, p in zip(new, past)]
    s = Setup(dev, 21, lens, ps, hkv, D, kt, junk=3.0)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = s.rng.standard_normal((cu[-1] + extra, 2 * hkv * D + 16)).astype(NP[nt])
    with np.errstate(over="ignore"):
        rows[0, :4] = [65520.0, -1e-8, np.inf, 6e-5]   # past f16's range, below its steps, infinite, subnormal
    s.upload()
    tr, tc = put(dev, rows), put(dev, cu)
    es = 4 if nt == F32 else 2
    rc = lib.tl_hip_launch_kv_append(tr.data_ptr, tr.data_ptr + es * hkv * D, nt, rows.shape[1], rows.shape[1], s.tk.data_ptr,
                                     s.tv.data_ptr, kt, s.n_pages, ps, hkv, D, s.tt.data_ptr, s.width, tc.data_ptr,
                                     s.tl.data_ptr, len(lens), rows.shape[0], None)
    assert rc == 0, lib.tl_hip_last_error()
    with np.errstate(over="ignore"):   # (65520 rounds to infinity)
        for i, (t, want) in enumerate(((s.tk, s.k.copy()), (s.tv, s.v.copy()))):
            for b, n in enumerate(lens):
                j = np.arange(past[b], n)
                x = rows[cu[b]:cu[b + 1], i * hkv * D:(i + 1) * hkv * D].reshape(-1, hkv, D)
                want[s.table[b, j // ps], :, j % ps] = x.astype(NP[kt])
            got = get(t, NP[kt], want.shape)
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8))


def test_append_leaves_out_what_has_no_slot(dev):
    """Rows before position 0, past the table, on bad pages and behind the last sequence."""
    lib = _lib.load()
    s = Setup(dev, 22, [32, 32, 32], 16, 1, 64, F32, junk=3.0)
    s.table[1, 1] = -1
    s.table[2, 0] = s.n_pages
    s.lens = [3, 33, 32]
    cu = np.asarray([0, 5, 25, 57], np.int32)
    rows = s.rng.standard_normal((60, 2, 64)).astype(np.float32)
    s.upload()
    tr, tc = put(dev, rows), put(dev, cu)
    assert 0 == lib.tl_hip_launch_kv_append(tr.data_ptr, tr.data_ptr + 256, F32, 128, 128, s.tk.data_ptr, s.tv.data_ptr, F32,
                                            s.n_pages, 16, 1, 64, s.tt.data_ptr, s.width, tc.data_ptr, s.tl.data_ptr, 3, 60, None)
    for i, (t, want) in enumerate(((s.tk, s.k), (s.tv, s.v))):
        want[s.table[0, 0], 0, :3] = rows[2:5, i]        # positions 0 .. 2
        want[s.table[1, 0], 0, 13:] = rows[5:8, i]       # 13 .. 15; 16 .. 31 on a bad page, 32 past the table
        want[s.table[2, 1], 0] = rows[41:57, i]          # 16 .. 31; 0 .. 15 on a bad page
        assert np.array_equal(get(t, np.float32, want.shape), want)


@pytest.mark.parametrize("layers,n_pages,page,pairs", [(1, 4, 16, 1), (3, 50, 1040, 25), (2, 2000, 256, 1000), (22, 20, 32768, 7)])
def test_copy_pages(dev, layers, n_pages, page, pairs):
    lib = _lib.load()
    r = np.random.default_rng(23)
    pools = [r.integers(0, 1 << 30, (layers, n_pages, page // 4)).astype(np.int32) for _ in range(2)]
    order = r.permutation(n_pages)
    src, dst = order[:pairs].astype(np.int32), order[n_pages - pairs:].astype(np.int32)
    if pairs > 2:
        src[1] = src[0]   # one page to two places
    t = [put(dev, p) for p in pools]
    rc = lib.tl_hip_launch_kv_copy_pages(t[0].data_ptr, t[1].data_ptr, layers, n_pages, page, src.ctypes.data_as(_lib.i32p),
                                         dst.ctypes.data_as(_lib.i32p), pairs, None)
    src[:] = 0   # the call has read them
    assert rc == 0, lib.tl_hip_last_error()
    src = order[:pairs].copy()
    if pairs > 2:
        src[1] = src[0]
    for x, p in zip(t, pools):
        p[:, dst] = p[:, src]
        assert np.array_equal(get(x, np.int32, p.shape), p)


# --------------------------------------------------------------------- all of them ----
@pytest.mark.parametrize("qt,kt", TYPES)
def test_a_cache_through_prompts_forks_decode_and_compaction(dev, qt, kt):
    """Prompts packed, a fork, ragged decode steps, a cut, an end and a compaction, through
    PagedKV; every attention against the positions' plain history."""
    hkv, G, D, ps, scale = 2, 4, 64, 16, 0.125
    r = np.random.default_rng(24)
    kv = PagedKV(dev, 40, ps, hkv, D, dtype=kt)
    hist = {}   # sequence -> rows of (k, v) as the cache holds them

    def new(seqs, counts):
        rows = [r.standard_normal((sum(counts), hkv, D)).astype(np.float32) for _ in range(2)]
        kv.append(seqs, counts, dev.tensor_new(rows[0]), dev.tensor_new(rows[1]))
        at = 0
        for s, n in zip(seqs, counts):
            hist[s] = hist.get(s, []) + [(rows[0][t].astype(NP[kt]), rows[1][t].astype(NP[kt])) for t in range(at, at + n)]
            at += n

    def attend(seqs, counts=None):
        c = counts or [1] * len(seqs)
        q = r.standard_normal((sum(c), hkv * G, D)).astype(qt)
        got = kv.prefill(seqs, c, put(dev, q), scale) if counts else kv.decode(seqs, put(dev, q), scale)
        k, v = (np.zeros((len(seqs), hkv, max(len(hist[s]) for s in seqs) or 1, D), NP[kt]) for _ in range(2))
        for i, s in enumerate(seqs):
            for j, (a, b) in enumerate(hist[s]):
                k[i, :, j], v[i, :, j] = a, b
        table = np.arange(len(seqs))[:, None]
        cu = np.concatenate([[0], np.cumsum(c)])
        check(get(got, qt, q.shape), *attention(q, k, v, table, [len(hist[s]) for s in seqs], cu, k.shape[2], scale, qt == np.float16))

    a, b = kv.open(), kv.open()
    new([a, b], [37, 18])
    attend([a, b], [37, 18])
    c = kv.fork(a)
    hist[c] = list(hist[a])
    new([a, c, b], [1, 1, 1])
    attend([a, b, c])
    new([c, b], [30, 5])
    attend([b, c], [5, 30])
    kv.cut(c, 40)
    hist[c] = hist[c][:40]
    kv.close(b)
    kv.compact()
    for _ in range(3):
        new([c, a], [1, 1])
        attend([a, c])
    assert kv.length(a) == 41 and kv.length(c) == 43
    with pytest.raises(BackendError) as e:
        kv.append([a, c], [10, 1000], *(dev.tensor_zeros((1010, hkv, D), 0) for _ in range(2)))
    assert e.value.variant == "AllocationError" and kv.length(a) == 41 and kv.length(c) == 43
    attend([a, c])
