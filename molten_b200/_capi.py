"""ctypes binding of libmolten_rt.so (declarations in include/molten_rt.h)."""

from __future__ import annotations

import ctypes
import os
from pathlib import Path

LIB_DIR = Path(__file__).resolve().parent / "lib"
LIB_PATH = LIB_DIR / "libmolten_rt.so"

MOLTEN_OK = 0
MAX_IO = 8
DT_BF16, DT_F16, DT_F32 = 0, 1, 2

# every function of the C ABI: name -> (restype, argtypes)
_c = ctypes
SIGNATURES = {
    "molten_version": (_c.c_int, []),
    "molten_last_error": (_c.c_char_p, []),
    "molten_device_count": (_c.c_int, [_c.POINTER(_c.c_int)]),
    "molten_sync": (_c.c_int, [_c.c_int]),
    "molten_module_load": (_c.c_int, [_c.c_char_p, _c.c_int, _c.POINTER(_c.c_void_p)]),
    "molten_module_load_data": (_c.c_int, [_c.c_void_p, _c.c_size_t, _c.c_int,
                                           _c.POINTER(_c.c_void_p)]),
    "molten_module_unload": (_c.c_int, [_c.c_void_p]),
    "molten_kernel_info": (_c.c_int, [_c.c_void_p, _c.c_char_p, _c.POINTER(_c.c_int),
                                      _c.POINTER(_c.c_int), _c.POINTER(_c.c_int)]),
    "molten_max_resident": (_c.c_int, [_c.c_void_p, _c.c_char_p, _c.c_void_p,
                                       _c.POINTER(_c.c_int), _c.POINTER(_c.c_int)]),
    "molten_launch": (_c.c_int, [_c.c_void_p, _c.c_char_p, _c.c_void_p, _c.c_void_p,
                                 _c.c_size_t, _c.c_void_p]),
    "molten_encode_tma_2d": (_c.c_int, [_c.c_void_p, _c.c_int, _c.c_void_p, _c.c_uint64,
                                        _c.c_uint64, _c.c_uint64, _c.c_uint32, _c.c_uint32,
                                        _c.c_int]),
    "molten_encode_tma_4d": (_c.c_int, [_c.c_void_p, _c.c_int, _c.c_void_p, _c.c_void_p,
                                        _c.c_void_p, _c.c_void_p]),
    "molten_status_word": (_c.c_int, [_c.c_int, _c.POINTER(_c.c_void_p)]),
    "molten_read_status": (_c.c_int, [_c.c_int, _c.POINTER(_c.c_int), _c.c_int]),
    "molten_scores_softmax_bf16_noalloc": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p,
                                                      _c.c_longlong, _c.c_longlong,
                                                      _c.c_longlong, _c.c_void_p]),
}


LAUNCH_PDL = 1          # MOLTEN_LAUNCH_PDL
STATUS_POSITION = 4096  # molten::kRopePositionRange: not a wait, a position past its table


class LaunchCfg(ctypes.Structure):
    _fields_ = [("grid", ctypes.c_uint32 * 3), ("block", ctypes.c_uint32 * 3),
                ("cluster", ctypes.c_uint32 * 3), ("smem_bytes", ctypes.c_uint32),
                ("flags", ctypes.c_uint32)]


class RowArgs(ctypes.Structure):
    """molten_row_args / molten::RowArgs (160 bytes)."""
    _fields_ = [("inp", ctypes.c_void_p * MAX_IO), ("out", ctypes.c_void_p * MAX_IO),
                ("rows", ctypes.c_longlong), ("row_offset", ctypes.c_longlong),
                ("cols", ctypes.c_longlong), ("status", ctypes.c_void_p)]


class GemmArgs(ctypes.Structure):
    """molten_gemm_args / molten::GemmArgs (448 bytes, 64-byte aligned on
    the device side; the explicit tail keeps the host copy the same size)."""
    _fields_ = [("tmap_a", ctypes.c_ubyte * 128), ("tmap_b", ctypes.c_ubyte * 128),
                ("inp", ctypes.c_void_p * MAX_IO), ("out", ctypes.c_void_p * MAX_IO),
                ("m", ctypes.c_longlong), ("n", ctypes.c_longlong), ("k", ctypes.c_longlong),
                ("row_offset", ctypes.c_longlong), ("status", ctypes.c_void_p),
                ("batch", ctypes.c_int), ("pad_", ctypes.c_int), ("work", ctypes.c_void_p),
                ("tile_count", ctypes.c_void_p)]


class AttnArgs(ctypes.Structure):
    """molten_attn_args / molten::AttnArgs (448 bytes, 64-byte aligned on the
    device side)."""
    _fields_ = [("tmap_q", ctypes.c_ubyte * 128), ("tmap_k", ctypes.c_ubyte * 128),
                ("tmap_p", ctypes.c_ubyte * 128), ("out", ctypes.c_void_p),
                ("m", ctypes.c_longlong), ("n", ctypes.c_longlong), ("d", ctypes.c_longlong),
                ("row_offset", ctypes.c_longlong), ("status", ctypes.c_void_p),
                ("batch", ctypes.c_int), ("tail_", ctypes.c_ubyte * 12)]


class RopePosArgs(ctypes.Structure):
    """molten_rope_pos_args / molten::RopePosArgs."""
    _fields_ = [("x", ctypes.c_void_p), ("cos_t", ctypes.c_void_p), ("sin_t", ctypes.c_void_p),
                ("pos", ctypes.c_void_p), ("out", ctypes.c_void_p), ("status", ctypes.c_void_p),
                ("tokens", ctypes.c_longlong), ("x_token", ctypes.c_longlong),
                ("x_head", ctypes.c_longlong), ("table_rows", ctypes.c_longlong),
                ("heads", ctypes.c_int), ("dim", ctypes.c_int), ("axes", ctypes.c_int),
                ("head_lanes", ctypes.c_int), ("bound", ctypes.c_int * 4),
                ("tokens_per_cta", ctypes.c_int), ("reserved", ctypes.c_int)]


class Q4Args(ctypes.Structure):
    """molten_q4_args / molten::Q4Args."""
    _fields_ = [("x", ctypes.c_void_p), ("q", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("zeros", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("x_stride", ctypes.c_longlong), ("n", ctypes.c_longlong), ("m", ctypes.c_int),
                ("k", ctypes.c_int), ("warps_n_log", ctypes.c_int), ("ksplit_log", ctypes.c_int),
                ("chunk", ctypes.c_int), ("tiles", ctypes.c_int),
                ("teams", ctypes.c_int), ("reserved", ctypes.c_int)]


class WindowArgs(ctypes.Structure):
    """molten_window_args / molten::WindowArgs."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "lengths", "out", "part")]
                + [(n, ctypes.c_longlong) for n in ("q_b", "q_s", "q_h", "k_b", "k_s", "k_h",
                                                     "v_b", "v_s", "v_h")]
                + [(n, ctypes.c_int) for n in ("batch", "nq", "cache", "kv_heads", "per", "dim",
                                               "window", "sinks")]
                + [("scale_log2", ctypes.c_float), ("ranks", ctypes.c_int),
                   ("parts", ctypes.c_int), ("reserved", ctypes.c_int)])


class WindowTcArgs(ctypes.Structure):
    """molten_window_tc_args / molten::WindowTcArgs (512 bytes, 64-byte aligned
    on the device side)."""
    _fields_ = ([(n, ctypes.c_ubyte * 128) for n in ("tmap_q", "tmap_k", "tmap_v")]
                + [(n, ctypes.c_void_p) for n in ("v", "lengths", "out", "status")]
                + [(n, ctypes.c_longlong) for n in ("v_b", "v_s", "v_h")]
                + [(n, ctypes.c_int) for n in ("batch", "nq", "cache", "kv_heads", "per", "dim",
                                               "window", "sinks")]
                + [("scale_log2", ctypes.c_float)]
                + [(n, ctypes.c_int) for n in ("positions", "blocks", "parts")]
                + [("part", ctypes.c_void_p), ("tail_", ctypes.c_ubyte * 16)])


class SampleArgs(ctypes.Structure):
    """molten_sample_args / molten::SampleArgs."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "u", "temperature", "top_k", "top_p",
                                                "min_p", "out")]
                + [("row_stride", ctypes.c_longlong)]
                + [(n, ctypes.c_int) for n in ("rows", "vocab", "run", "ranks")]
                + [(n, ctypes.c_float) for n in ("temperature_all", "top_p_all", "min_p_all")]
                + [("top_k_all", ctypes.c_int)])


assert ctypes.sizeof(SampleArgs) == 96
assert ctypes.sizeof(WindowTcArgs) == 512
assert ctypes.sizeof(WindowArgs) == 168
assert ctypes.sizeof(RopePosArgs) == 120
assert ctypes.sizeof(Q4Args) == 88
assert ctypes.sizeof(RowArgs) == 160
assert ctypes.sizeof(AttnArgs) == 448
assert ctypes.sizeof(GemmArgs) == 448


class MoltenError(RuntimeError):
    """A call into libmolten_rt.so failed."""


_lib = None


def load_library(path: os.PathLike = None):
    """Load (once) and return the runtime library; raises if it is missing."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise MoltenError(
            f"{p} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "(molten_b200.build.build_runtime)")
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if path is None:
        _lib = lib
    return lib


def last_error() -> str:
    return load_library().molten_last_error().decode(errors="replace")


def check(rc: int, what: str) -> None:
    if rc != MOLTEN_OK:
        raise MoltenError(f"{what} failed (code {rc}): {last_error()}")


def device_count() -> int:
    n = ctypes.c_int(0)
    check(load_library().molten_device_count(ctypes.byref(n)), "molten_device_count")
    return n.value


class Module:
    """A cubin loaded on one device."""

    def __init__(self, cubin_path: str, device: int):
        self.lib = load_library()
        self.handle = ctypes.c_void_p()
        self.device = device
        self.path = cubin_path
        check(self.lib.molten_module_load(str(cubin_path).encode(), device,
                                          ctypes.byref(self.handle)),
              f"loading {cubin_path}")

    def kernel_info(self, name: str) -> dict:
        regs, thr, smem = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        check(self.lib.molten_kernel_info(self.handle, name.encode(), ctypes.byref(regs),
                                          ctypes.byref(thr), ctypes.byref(smem)),
              f"kernel info of {name}")
        return {"registers": regs.value, "max_threads": thr.value, "static_smem": smem.value}

    def max_resident(self, name: bytes, cfg: LaunchCfg) -> tuple:
        """(CTAs per SM, clusters on the device) that fit at once with cfg."""
        per_sm, clusters = ctypes.c_int(), ctypes.c_int()
        check(self.lib.molten_max_resident(self.handle, name, ctypes.byref(cfg),
                                           ctypes.byref(per_sm), ctypes.byref(clusters)),
              f"occupancy of {name.decode()}")
        return per_sm.value, clusters.value

    def launch(self, name: bytes, cfg: LaunchCfg, params, stream: int) -> None:
        rc = self.lib.molten_launch(self.handle, name, ctypes.byref(cfg), ctypes.byref(params),
                                    ctypes.sizeof(params), ctypes.c_void_p(stream))
        if rc != MOLTEN_OK:
            raise MoltenError(f"launching {name.decode()} failed (code {rc}): {last_error()}")

    def unload(self) -> None:
        if self.handle:
            check(self.lib.molten_module_unload(self.handle), "unloading module")
            self.handle = ctypes.c_void_p()


def encode_tma_2d(dtype_code: int, base: int, inner: int, outer: int, row_stride_bytes: int,
                  box_inner: int, box_outer: int, swizzle: int = 128) -> bytes:
    """128-byte TMA descriptor for a row-major 2-D matrix; ``swizzle`` is the
    span in bytes (0 none, 32, 64, 128)."""
    lib = load_library()
    buf = ctypes.create_string_buffer(128 + 64)
    addr = ctypes.addressof(buf)
    aligned = (addr + 63) & ~63
    check(lib.molten_encode_tma_2d(ctypes.c_void_p(aligned), dtype_code, ctypes.c_void_p(base),
                                   inner, outer, row_stride_bytes, box_inner, box_outer,
                                   int(swizzle)),
          "encoding a TMA descriptor")
    return ctypes.string_at(aligned, 128)


def status_word(device: int) -> int:
    p = ctypes.c_void_p()
    check(load_library().molten_status_word(device, ctypes.byref(p)), "status word")
    return p.value


def read_status(device: int, reset: bool = True) -> int:
    v = ctypes.c_int(0)
    check(load_library().molten_read_status(device, ctypes.byref(v), 1 if reset else 0),
          "reading the status word")
    return v.value
