"""ctypes binding of libhortihip.so -- the only way the Python host reaches the GPU kernels.

There is deliberately NO fallback: if the shared library is missing or fails to load, importing any
compute entry point raises (the product path must fail loudly without its HIP extension)."""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
# HORTIHIP_LIB: development aid for same-box A/B timing of kernel variants (scripts/build_variant.sh builds them under
# build/); unset = the in-tree library.  Either way a missing file is an error, never a fallback.
LIB_PATH = os.environ.get("HORTIHIP_LIB") or os.path.join(_HERE, "libhortihip.so")
_lib = None

c_float_p = ctypes.POINTER(ctypes.c_float)
c_void_p = ctypes.c_void_p
c_int = ctypes.c_int


class HortiHipError(RuntimeError):
    pass


class HmAdapterArgs(ctypes.Structure):
    """ctypes mirror of `hm_adapter_args` (include/hortimapping_amd.h)."""
    _fields_ = [("type", c_int), ("k", c_int), ("n", c_int), ("rank", c_int), ("adapters", c_int), ("segments", c_int),
                ("tag", ctypes.c_uint), ("rows", ctypes.c_longlong), ("d_x", c_void_p), ("ld_x", ctypes.c_longlong),
                ("d_w", c_void_p), ("ld_w", ctypes.c_longlong), ("d_bias", c_void_p), ("d_a", c_void_p), ("d_b", c_void_p),
                ("d_scale", c_void_p), ("d_row_start", c_void_p), ("d_adapter", c_void_p), ("p", ctypes.c_double),
                ("seed", ctypes.c_ulonglong), ("d_seed", c_void_p), ("row0", ctypes.c_ulonglong)]


def _declare(lib):
    lib.hm_last_error.restype = ctypes.c_char_p
    lib.hm_last_error.argtypes = []
    lib.hm_decoder_create.restype = c_int
    lib.hm_decoder_create.argtypes = [c_int, ctypes.POINTER(c_float_p), ctypes.POINTER(c_float_p),
                                      ctypes.POINTER(c_void_p)]
    lib.hm_decoder_create_arch.restype = c_int
    lib.hm_decoder_create_arch.argtypes = [c_void_p, ctypes.POINTER(c_float_p), ctypes.POINTER(c_float_p),
                                           ctypes.POINTER(c_float_p), ctypes.POINTER(c_float_p),
                                           ctypes.POINTER(c_void_p)]
    lib.hm_decoder_destroy.restype = c_int
    lib.hm_decoder_destroy.argtypes = [c_void_p]
    lib.hm_decoder_latent_dim.restype = c_int
    lib.hm_decoder_latent_dim.argtypes = [c_void_p]
    lib.hm_decoder_set_precision.restype = c_int
    lib.hm_decoder_set_precision.argtypes = [c_void_p, c_int]
    lib.hm_decoder_get_precision.restype = c_int
    lib.hm_decoder_get_precision.argtypes = [c_void_p]
    lib.hm_decode_batch.restype = c_int
    lib.hm_decode_batch.argtypes = [c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p,
                                    c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]
    ll, ull, dbl = ctypes.c_longlong, ctypes.c_ulonglong, ctypes.c_double
    lib.hm_dropout.restype = c_int
    lib.hm_dropout.argtypes = [c_void_p, ll, c_void_p, ll, ll, c_int, c_int, c_int, dbl, ull, c_void_p, ctypes.c_uint, ull,
                               c_void_p]
    lib.hm_dropout_backward.restype = c_int
    lib.hm_dropout_backward.argtypes = [c_void_p, ll, c_void_p, ll, c_void_p, ll, ll, c_int, c_int, c_int, dbl, ull, c_void_p,
                                        ctypes.c_uint, ull, c_void_p]
    args_p = ctypes.POINTER(HmAdapterArgs)
    lib.hm_adapter_linear.restype = c_int
    lib.hm_adapter_linear.argtypes = [args_p, c_void_p, ll, c_void_p, c_void_p]
    lib.hm_adapter_linear_backward_bytes.restype = ll
    lib.hm_adapter_linear_backward_bytes.argtypes = [args_p]
    lib.hm_adapter_linear_backward.restype = c_int
    lib.hm_adapter_linear_backward.argtypes = [args_p, c_void_p, ll, c_void_p, c_void_p, ll, c_void_p, c_void_p, c_void_p, ll,
                                               c_void_p]


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise HortiHipError(
                f"{LIB_PATH} not found: build it with `python -m hortimapping_amd.build` "
                "(hipcc --offload-arch=gfx950).  There is no CPU fallback.")
        # torch bundles its own libamdhip64.so.7 / libhsa-runtime64; load it FIRST so that libhortihip.so binds to the
        # same HIP runtime instance (two runtimes in one process cannot share device pointers or streams)
        import torch  # noqa: F401
        _lib = ctypes.CDLL(LIB_PATH)
        _declare(_lib)
    return _lib


def check(rc: int, what: str):
    if rc != 0:
        msg = lib().hm_last_error().decode("utf-8", "replace")
        raise HortiHipError(f"{what} failed (rc={rc}): {msg}")
