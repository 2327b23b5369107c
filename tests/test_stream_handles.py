"""Stream handles that are no objects: the default stream's other name and the thread's own default stream."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qwenasr.cpp_amd")

HANDLES = r"""
#include "common.hpp"
#include <cstdio>
int main() {
    for (size_t h : {size_t(0), size_t(1), size_t(2), size_t(4096)}) std::printf("%zu ", reinterpret_cast<size_t>(qa::as_stream(reinterpret_cast<void *>(h))));
    return 0;
}
"""


def test_default_stream_by_either_name(tmp_path):
    """hipStreamLegacy (1) never reaches the runtime."""
    src, exe = tmp_path / "handles.cpp", tmp_path / "handles"
    src.write_text(HANDLES)
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{ROOT}/include", f"-I{PKG}/csrc", str(src),
                    "-o", str(exe), f"-L{PKG}", "-lqwenasr_amd", "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{PKG}:/opt/rocm/lib",
                    "-Wl,--unresolved-symbols=ignore-all"], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(v) for v in out.split()] == [0, 0, 2, 4096]


@pytest.mark.gpu
@pytest.mark.parametrize("handle", [None, 1, 2])
def test_a_layer_on_the_default_streams(qa, handle):
    """Append, attention, 4-bit products, page bookkeeping and a copy on the default stream by either name, and on the thread's."""
    from test_gpu_pages import Pool, counted
    from test_gpu_paged_serving import Layer

    stream = C.c_void_p(handle)
    layer = Layer(qa, [200, 13, 0], [1, 20, 1], True, 3)
    layer.clear()
    qa.synchronize()
    layer.enqueue(stream)
    qa.synchronize()
    layer.check()
    tables = np.array([[0, 1, -1], [0, 1, -1]], np.int32)
    pool = Pool(qa, counted(tables, 6), tables)
    assert pool.extend([1], [20], [20], stream) == 0
    refs, t, _ = pool.state()
    assert t.tolist() == [[0, 1, -1], [0, 2, 3]] and refs.tolist() == [2, 1, 1, 1, 0, 0]
    a, b = qa.DeviceArray.from_numpy(np.arange(64, dtype=np.int32)), qa.DeviceArray((64,), np.int32)
    qa.check(qa.lib.qa_copy_device(b.ptr, a.ptr, 256, stream))
    qa.check(qa.lib.qa_stream_synchronize(stream))
    np.testing.assert_array_equal(b.numpy(), np.arange(64))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_capture_in_every_mode(qa, mode):
    """No call of a step is one that a global or thread-local capture forbids: attention by both launches, an LM head, bookkeeping."""
    import paged_ref as ref
    from test_gpu_gemv_q4 import packed, weights
    from test_gpu_paged_serving import Hip, Layer

    hip = Hip()
    layers = [Layer(qa, *batch, True, 7) for batch in (([200, 13, 0], [1, 1, 1]), ([3500, 40], [260, 1]))]   # the second on shared tiles
    q, d = weights(np.random.default_rng(0), 16400, 128, 32)
    dw = [qa.DeviceArray.from_numpy(a) for a in packed(q, d)]
    x, y = qa.DeviceArray.from_numpy(np.ones((20, 128), np.float32)), qa.DeviceArray((20, 16400))
    lay = ref.layout(qa, 2, 12, 2, 16, True)
    pool, refs, tables = qa.DeviceArray((2, 2, 12, 2, 16, 128), np.float16), qa.DeviceArray((12,), np.int32), qa.DeviceArray((4, 3), np.int32)
    ints = [qa.DeviceArray.from_numpy(np.array(v, np.int32)) for v in ([0, 1], [0, 0], [20, 9], [2, 3])]
    missing, live = qa.DeviceArray((1,), np.int32), qa.DeviceArray((1,), np.int32)
    need = qa.lib.qa_pages_workspace_bytes(C.byref(lay))
    ws = qa.DeviceArray((need,), np.uint8)
    rows, zero, new, dst = (v.ptr for v in ints)

    def enqueue(stream):
        for layer in layers:
            layer.enqueue(stream)
        qa.check(qa.lib.qa_gemv_q4(dw[0].ptr, dw[1].ptr, 32, 16400, 128, x.ptr, 20, y.ptr, 0, None, 1e-6, stream))
        t = (refs.ptr, 12, tables.ptr, 4, 3, 16)
        qa.check(qa.lib.qa_pages_extend(pool.ptr, C.byref(lay), refs.ptr, tables.ptr, 4, 3, rows, zero, new, 2, missing.ptr, ws.ptr, need, stream))
        qa.check(qa.lib.qa_pages_fork(*t, rows, dst, new, 2, stream))
        qa.check(qa.lib.qa_pages_free(*t, rows, None, 1, stream))
        qa.check(qa.lib.qa_pages_copy(pool.ptr, C.byref(lay), rows, dst, 2, stream))
        qa.check(qa.lib.qa_pages_compact(pool.ptr, C.byref(lay), refs.ptr, tables.ptr, 4, 3, refs.ptr, tables.ptr, live.ptr, ws.ptr, need, stream))

    stream = hip.stream()
    graph, run = C.c_void_p(), C.c_void_p()
    hip.hipStreamBeginCapture(stream, mode)
    try:
        enqueue(stream)
    finally:
        hip.hipStreamEndCapture(stream, C.byref(graph))
    hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0))

    def reset():
        for layer in layers:
            layer.clear()
        refs.upload(np.zeros(12, np.int32))
        tables.upload(np.full((4, 3), -1, np.int32))
        y.upload(np.full((20, 16400), np.nan, np.float32))
        qa.synchronize()

    for _ in range(3):
        reset()
        enqueue(None)
        qa.synchronize()
        eager = refs.numpy(), tables.numpy(), y.numpy(), *(layer.y.numpy() for layer in layers)
        assert np.isfinite(eager[2]).all() and int(live.numpy()[0]) == 3
        reset()
        hip.hipGraphLaunch(run, stream)
        qa.synchronize()
        for a, b in zip(eager, (refs.numpy(), tables.numpy(), y.numpy(), *(layer.y.numpy() for layer in layers))):
            np.testing.assert_array_equal(a, b)
    if mode == 0:
        for layer in layers:
            layer.check()
    hip.drop(graph, run)
    hip.hipStreamDestroy(stream)
