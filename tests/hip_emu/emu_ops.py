"""TEST INFRASTRUCTURE: `HipOps` over the CPU execution model of the kernels (hip_emu.hpp), for the `not gpu` tests.

`emulated(sources)` is a context manager that yields a `beyond_deep_ensembles_amd.ops.HipOps` whose `lib` is the
emulation build of `sources` (tests/hip_emu/build.py) and, while it is open, lets that object take CPU tensors: every
tensor handed to the C ABI is copied into a buffer fenced by guard pages (one per underlying storage, so views alias as
they do on the device), the call runs on those, and the buffers are copied back when the call returns.  The product's
`HipOps` is otherwise unchanged -- same argument checks, same ctypes prototypes, same call sequences."""
import contextlib
import ctypes

import torch

from beyond_deep_ensembles_amd import _lib
from beyond_deep_ensembles_amd import ops as ops_mod

from . import build as B


ALL = ["version.hip", "swag.hip", "swag_batched.hip", "svgd.hip", "svgd_small.hip", "svgd_fused.hip", "gauss.hip", "ivon.hip",
       "lrt.hip", "lrt_bwd.hip", "conv_lrt.hip", "conv_lrt_bwd.hip", "embedding.hip", "topk.hip", "distill.hip"]


class _Shadows:
    def __init__(self, lib):
        self.lib = lib
        self.live = {}                                    # storage data_ptr -> (shadow ptr, nbytes, tensor kept alive)
        self.per_storage = None                           # Traffic: storage data_ptr -> (bytes read, bytes written) by the kernels

    def ptr(self, t):
        st = t.untyped_storage()
        base, nbytes = st.data_ptr(), st.nbytes()
        if nbytes == 0:
            return t.data_ptr()
        hit = self.live.get(base)
        if hit is None:
            sh = self.lib.hip_emu_alloc(nbytes)
            if not sh:
                raise MemoryError("hip_emu_alloc")
            ctypes.memmove(sh, base, nbytes)
            hit = self.live[base] = (sh, nbytes, t)
        return hit[0] + (t.data_ptr() - base)

    def land(self):
        out = (ctypes.c_uint64 * 2)()
        for base, (sh, nbytes, _keep) in self.live.items():
            ctypes.memmove(base, sh, nbytes)
            if self.per_storage is not None:
                self.lib.hip_emu_buffer_traffic(sh, out)
                r, w = self.per_storage.get(base, (0, 0))
                self.per_storage[base] = (r + int(out[0]), w + int(out[1]))
            self.lib.hip_emu_free(sh, nbytes)
        self.live.clear()


LOADED = B.LOADED      # path -> library handle of every CPU-model build this process has loaded (launched_kernels)


def launched_kernels() -> dict:
    """{kernel name (the __global__ function, without template arguments): launches so far} over every CPU-model build this
    process has loaded -- what tests/conftest.py's reach guard compares before and after a test."""
    import re
    import tempfile
    total = {}
    for lib in LOADED.values():
        with tempfile.NamedTemporaryFile("r", suffix=".txt") as fh:
            lib.hip_emu_launch_report(fh.name.encode())
            for line in fh.read().splitlines():
                sym, _, count = line.rpartition(" ")
                m = re.match(r"_ZN3bde(\d+)", sym)                # bde::<name><...>: Itanium length-prefixed identifier
                if m:
                    n = int(m.group(1))
                    sym = sym[m.end():m.end() + n]
                total[sym] = total.get(sym, 0) + int(count)
    return total


def load(sources, defines=()):
    path = B.build(sources, defines)
    lib = ctypes.CDLL(path)
    LOADED[path] = lib
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(lib, name, None)
        if fn is not None:
            fn.restype, fn.argtypes = res, args
    lib.hip_emu_count_traffic.restype, lib.hip_emu_count_traffic.argtypes = None, [ctypes.c_int]
    lib.hip_emu_traffic.restype, lib.hip_emu_traffic.argtypes = None, [ctypes.POINTER(ctypes.c_uint64)]
    lib.hip_emu_buffer_traffic.restype, lib.hip_emu_buffer_traffic.argtypes = None, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint64)]
    lib.hip_emu_alloc.restype, lib.hip_emu_alloc.argtypes = ctypes.c_void_p, [ctypes.c_size_t]
    lib.hip_emu_free.restype, lib.hip_emu_free.argtypes = None, [ctypes.c_void_p, ctypes.c_size_t]
    return lib


class Traffic:
    """``with Traffic(ops) as t: ops.kernel(...)`` -> t.read / t.written (bytes the kernels requested from / sent to the tensors
    handed through HipOps), t.lds_read / t.lds_written, t.mfma32 / t.mfma16 (v_mfma_f32_32x32x2 / 16x16x4 wave-instructions)."""

    def __init__(self, ops):
        self.lib, self.shadows = ops.lib, ops._emu_shadows

    def __enter__(self):
        self.lib.hip_emu_count_traffic(1)
        self.lib.hip_emu_traffic((ctypes.c_uint64 * 6)())
        self.shadows.per_storage = {}
        return self

    def __exit__(self, *exc):
        out = (ctypes.c_uint64 * 6)()
        self.lib.hip_emu_traffic(out)
        self.lib.hip_emu_count_traffic(0)
        self.read, self.written, self.lds_read, self.lds_written, self.mfma32, self.mfma16 = (int(v) for v in out)
        self.per_storage, self.shadows.per_storage = self.shadows.per_storage, None
        return False

    def of(self, tensor):
        """(bytes read, bytes written) by the kernels in the storage of ``tensor`` (its coefficient tables and other
        wave-uniform operands live in other tensors: on the device those are scalar loads, not streams)."""
        return self.per_storage.get(tensor.untyped_storage().data_ptr(), (0, 0))


@contextlib.contextmanager
def emulated(sources, defines=()):
    lib = load(sources, defines)
    ops = ops_mod.HipOps.__new__(ops_mod.HipOps)
    ops.lib = lib
    ops.name = "hip_emu"                                  # the shells' "HIP kernels need CUDA parameters" guard is for the device library
    ops.load_code_objects = lambda device: None            # bde_init() uploads code objects: nothing to upload here
    shadows = _Shadows(lib)
    ops._emu_shadows = shadows
    real_ptr, real_check, real_stream, real_ptr64 = ops_mod._ptr, ops_mod._check, ops_mod._stream, ops_mod._ptr64

    def ptr(t, name="tensor"):
        if t is None:
            return None
        if t.is_cuda:
            raise AssertionError("emulated HipOps takes CPU tensors")
        if t.dtype != torch.float32:
            raise ops_mod.BdeKernelError(f"{name}: expected float32, got {t.dtype}")
        if t.dim() > 0 and t.stride(-1) != 1:
            raise ops_mod.BdeKernelError(f"{name}: last dimension must be contiguous")
        return shadows.ptr(t)

    def check(rc, what):
        shadows.land()
        real_check(rc, what)

    def ptr64(t, name):
        if t.is_cuda or t.dtype != torch.float64:
            raise ops_mod.BdeKernelError(f"{name}: expected a float64 CPU tensor on the model, got {t.dtype} on {t.device}")
        return shadows.ptr(t)

    real_typed = ops_mod._ptr_typed

    def ptr_typed(t, name, dtypes):
        if t is None:
            return None
        if t.is_cuda:
            raise AssertionError("emulated HipOps takes CPU tensors")
        ops_mod._check_typed(t, name, dtypes)
        return shadows.ptr(t)

    ops_mod._ptr, ops_mod._check, ops_mod._stream, ops_mod._ptr64 = ptr, check, lambda: None, ptr64
    ops_mod._ptr_typed = ptr_typed
    real_device, real_sync = torch.cuda.device, torch.cuda.synchronize
    torch.cuda.device = lambda dev: contextlib.nullcontext()          # "the output's device is current": nothing to do
    torch.cuda.synchronize = lambda *a, **k: None                     # every emulated launch has finished when it returns
    try:
        yield ops
    finally:
        shadows.land()
        torch.cuda.device, torch.cuda.synchronize = real_device, real_sync
        ops_mod._ptr, ops_mod._check, ops_mod._stream, ops_mod._ptr64 = real_ptr, real_check, real_stream, real_ptr64
        ops_mod._ptr_typed = real_typed
