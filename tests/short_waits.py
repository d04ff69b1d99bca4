"""A build of the library in which every bounded wait gives up at once, to test the kernels' way out."""
import contextlib
import ctypes
import subprocess

from qwen_tailor_b200 import _lib, build


def compile_library(folder):
    """Compiles all sources with waits of no polls into ``folder``; returns the loaded library."""
    nvcc, objs, procs = build.nvcc_path(), [], []
    for src in build.sources():
        objs.append(str(folder / (src.stem + ".o")))
        procs.append(subprocess.Popen([nvcc, *build.NVCC_FLAGS, "-DGDN_WAIT_POLLS=0", "-c", str(src), "-o", objs[-1]]))
    assert all([p.wait() == 0 for p in procs])
    out = folder / "libgdn_short_waits.so"
    subprocess.run([nvcc, "-shared", "-o", str(out), *objs, "-gencode", "arch=compute_100a,code=sm_100a"], check=True)
    lib = ctypes.CDLL(str(out))
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


@contextlib.contextmanager
def operators_use(lib):
    """The operators (and ``_lib.device_status``) go to ``lib`` inside."""
    normal = _lib.load()
    _lib._lib = lib
    try:
        yield
    finally:
        _lib._lib = normal
