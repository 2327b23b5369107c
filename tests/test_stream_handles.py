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
