"""The paged KV cache on caller streams and in graphs (after the tests that want the library's stream
to be the only one): captures replayed over changing lengths, and calls at the same time."""
import ctypes as C

import numpy as np
import pytest

from paged_f64 import attention
from test_gpu_paged import F16, F32, NP, TYPES, Setup, check, get, put, run_attention
from test_gpu_runtime import _hip
from tl_amd import _lib

pytestmark = pytest.mark.gpu


def _stream(hip):
    st = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0   # hipStreamNonBlocking
    return st


@pytest.mark.parametrize("qt,kt", [(np.float32, F16), (np.float16, F16), (np.float32, F32)])
def test_graphs_follow_the_lengths_and_repeat_the_eager_call(dev, qt, kt):
    """Append, decode and a packed prefill captured on a caller stream with the caller's workspaces:
    replays with eager work between them, the integer arrays changed under the graph."""
    hip, lib = _hip(), _lib.load()
    hkv, G, D, ps, lens = 2, 4, 128, 16, [700, 33, 1]
    s = Setup(dev, 29, lens, ps, hkv, D, kt, junk=0.5)
    s.upload()
    q, qp = s.rng.standard_normal((3, hkv * G, D)).astype(qt), s.rng.standard_normal((40, hkv * G, D)).astype(qt)
    tq, tp, to, tpo = put(dev, q), put(dev, qp), put(dev, np.zeros_like(q)), put(dev, np.zeros_like(qp))
    cu1, cu2 = put(dev, np.arange(4, dtype=np.int32)), put(dev, np.asarray([0, 30, 40, 40], np.int32))
    rows = put(dev, s.rng.standard_normal((3, 2, hkv * D)).astype(NP[kt]))
    need = max(lib.tl_hip_paged_attention_workspace(3, n, hkv * G, hkv, D) for n in (3, 40))
    ws = dev.tensor_zeros((need // 4,), F32)
    dev.synchronize()
    cache = (s.tk.data_ptr, s.tv.data_ptr, kt, s.n_pages, ps)
    qd = F16 if qt == np.float16 else F32
    row, head = hkv * D, hkv * G * D
    es = 2 if kt == F16 else 4

    def step(stream):
        rc = lib.tl_hip_launch_kv_append(rows.data_ptr, rows.data_ptr + row * es, kt, 2 * row, 2 * row, *cache, hkv, D,
                                         s.tt.data_ptr, s.width, cu1.data_ptr, s.tl.data_ptr, 3, 3, stream)
        rc = rc or lib.tl_hip_launch_paged_attention_decode(tq.data_ptr, qd, head, *cache, hkv * G, hkv, D, s.tt.data_ptr, s.width,
                                                            s.tl.data_ptr, 3, to.data_ptr, 0.09, ws.data_ptr, need, stream)
        rc = rc or lib.tl_hip_launch_paged_attention_prefill(tp.data_ptr, qd, head, *cache, hkv * G, hkv, D, s.tt.data_ptr, s.width,
                                                             cu2.data_ptr, s.tl.data_ptr, 3, 40, tpo.data_ptr, 0.09, ws.data_ptr,
                                                             need, stream)
        assert rc == 0, lib.tl_hip_last_error()

    st, graph, run = _stream(hip), C.c_void_p(), C.c_void_p()
    try:
        step(st)   # the first call on a stream is not captured
        assert hip.hipStreamSynchronize(st) == 0
        assert hip.hipStreamBeginCapture(st, 2) == 0   # relaxed
        step(st)
        # without the caller's workspace a captured call is refused
        assert lib.tl_hip_launch_paged_attention_decode(tq.data_ptr, qd, head, *cache, hkv * G, hkv, D, s.tt.data_ptr, s.width,
                                                        s.tl.data_ptr, 3, to.data_ptr, 0.09, None, 0, st) == 8
        assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
        for lens in ([700, 33, 1], [650, 1, 0], [16, 30, 1], [700, 33, 1]):
            new = np.asarray(lens, np.int32)
            assert lib.tl_hip_memcpy_h2d(s.tl.data_ptr, new.ctypes.data, new.nbytes) == 0
            step(None)
            want = get(to, qt, q.shape), get(tpo, qt, qp.shape)
            for t, a in ((to, q), (tpo, qp)):
                z = np.zeros_like(a)
                assert lib.tl_hip_memcpy_h2d(t.data_ptr, z.ctypes.data, z.nbytes) == 0
            assert hip.hipGraphLaunch(run, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            assert np.array_equal(get(to, qt, q.shape), want[0])
            assert np.array_equal(get(tpo, qt, qp.shape), want[1])
    finally:
        hip.hipStreamSynchronize(st)
        if run:
            hip.hipGraphExecDestroy(run)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)


@pytest.mark.parametrize("qt,kt", TYPES)
def test_captured_prompts_and_page_copies(dev, qt, kt):
    """A fork's page copies and a prompt whose positions are cut, in one graph: the pairs are the
    graph's own, the rows follow the pages."""
    hip, lib = _hip(), _lib.load()
    hkv, G, D, ps = 2, 4, 128, 64
    s = Setup(dev, 36, [400, 130], ps, hkv, D, kt, width=512, junk=0.25)
    s.upload()
    cu = np.asarray([0, 200, 330], np.int32)
    q = s.rng.standard_normal((330, hkv * G, D)).astype(qt)
    tq, tc, to = put(dev, q), put(dev, cu), put(dev, np.zeros_like(q))
    need = lib.tl_hip_paged_attention_workspace(2, 330, hkv * G, hkv, D)
    ws = dev.tensor_zeros((need // 4,), F32)
    es = 2 if kt == F16 else 4
    spare = [p for p in range(s.n_pages) if p not in s.table]
    src, dst = np.asarray([s.table[0, 0]], np.int32), np.asarray(spare[:1], np.int32)   # sequence 0's first page to a spare one
    s.table[0, 0] = spare[0]
    assert lib.tl_hip_synchronize() == 0
    assert lib.tl_hip_memcpy_h2d(s.tt.data_ptr, s.table.ctypes.data, s.table.nbytes) == 0

    def step(stream):
        rc = lib.tl_hip_launch_kv_copy_pages(s.tk.data_ptr, s.tv.data_ptr, 1, s.n_pages, hkv * ps * D * es,
                                             src.ctypes.data_as(_lib.i32p), dst.ctypes.data_as(_lib.i32p), 1, stream)
        rc = rc or lib.tl_hip_launch_paged_attention_prefill(
            tq.data_ptr, F16 if qt == np.float16 else F32, hkv * G * D, s.tk.data_ptr, s.tv.data_ptr, kt, s.n_pages, ps, hkv * G,
            hkv, D, s.tt.data_ptr, s.width, tc.data_ptr, s.tl.data_ptr, 2, 330, to.data_ptr, 0.09, ws.data_ptr, need, stream)
        assert rc == 0, lib.tl_hip_last_error()

    k = s.k.copy()
    for x in (s.k, s.v):
        x[spare[0]] = x[src[0]]
    st, graph, run = _stream(hip), C.c_void_p(), C.c_void_p()
    try:
        step(st)
        assert hip.hipStreamSynchronize(st) == 0
        assert hip.hipStreamBeginCapture(st, 2) == 0
        step(st)
        assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
        src[0], dst[0] = dst[0], src[0]   # the graph has its pairs
        assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
        for lens in ([400, 130], [300, 100], [400, 130]):
            new = np.asarray(lens, np.int32)
            assert lib.tl_hip_memcpy_h2d(s.tl.data_ptr, new.ctypes.data, new.nbytes) == 0
            junk = np.full(k[0].shape, 9, NP[kt])
            at = int(spare[0]) * junk.nbytes
            assert lib.tl_hip_memcpy_h2d(s.tk.data_ptr + at, junk.ctypes.data, junk.nbytes) == 0
            z = np.full_like(q, 7)
            assert lib.tl_hip_memcpy_h2d(to.data_ptr, z.ctypes.data, z.nbytes) == 0
            assert hip.hipGraphLaunch(run, st) == 0
            assert hip.hipStreamSynchronize(st) == 0
            check(get(to, qt, q.shape), *attention(q, s.k, s.v, s.table, lens, cu, ps, 0.09, qt == np.float16))
    finally:
        hip.hipStreamSynchronize(st)
        if run:
            hip.hipGraphExecDestroy(run)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(st)


def test_calls_that_overlap_on_two_streams(dev):
    """Two streams at once, each its own sequences, one with the library's workspaces and one with its
    own: every result is the one alone."""
    hip, lib = _hip(), _lib.load()
    st = [_stream(hip) for _ in range(2)]
    try:
        sets = []
        for i, lens in enumerate(([9000, 100], [40, 6000, 7])):
            s = Setup(dev, 30 + i, lens, 64, 2, 128, F16)
            q = s.rng.standard_normal((len(lens), 16, 128)).astype(np.float32)
            want = run_attention(s, q, 0.09)
            check(want, *attention(q, s.k, s.v, s.table, lens, range(len(lens) + 1), 64, 0.09, False))
            need = lib.tl_hip_paged_attention_workspace(len(lens), len(lens), 16, 2, 128)
            ws = dev.tensor_zeros((need // 4,), F32) if i else None
            sets.append((s, put(dev, q), [put(dev, np.zeros_like(q)) for _ in range(8)], ws, need, want))
        dev.synchronize()
        for k in range(8):
            for (s, tq, outs, ws, need, _), stream in zip(sets, st):
                rc = lib.tl_hip_launch_paged_attention_decode(
                    tq.data_ptr, F32, 16 * 128, s.tk.data_ptr, s.tv.data_ptr, F16, s.n_pages, 64, 16, 2, 128, s.tt.data_ptr, s.width,
                    s.tl.data_ptr, len(s.lens), outs[k].data_ptr, 0.09, ws.data_ptr if ws else None, need if ws else 0, stream)
                assert rc == 0, lib.tl_hip_last_error()
        for stream in st:
            assert hip.hipStreamSynchronize(stream) == 0
        for s, tq, outs, ws, need, want in sets:
            for o in outs:
                assert np.array_equal(get(o, np.float32, want.shape), want)
    finally:
        for stream in st:
            hip.hipStreamSynchronize(stream)
            hip.hipStreamDestroy(stream)
