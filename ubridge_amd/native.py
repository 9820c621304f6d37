"""The compiled host side of the attention block's calls (binding/native.cpp):
argument checks, results and argument blocks, without a Python line per tensor.
Loaded by attention.py, rope.py, kvcache.py and int8.py."""
import ctypes

import torch

from ._lib import check, lib, register

try:
    from . import _native
except ImportError as e:
    raise ImportError(f"ubridge_amd/_native.so cannot be loaded ({e}); build it with "
                      "`python ubridge_amd/build.py`") from e

_vp, _i = ctypes.c_void_p, ctypes.c_int
_ENTRIES = (register("ubridge_paged_decode", _i, [_vp, _vp]), register("ubridge_rope", _i, [_vp, _vp]),
            register("ubridge_rope_append", _i, [_vp, _vp]),
            register("ubridge_int8_linear", _i, [_vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp]),
            register("ubridge_kv_free", _i, [_vp, _vp, _i, _vp]),
            register("ubridge_kv_fork", _i, [_vp, _vp, _vp, _i, _vp, _vp]),
            register("ubridge_kv_compact", _i, [_vp, _vp, _vp]))
_native.bind(*(ctypes.cast(f, _vp).value for f in _ENTRIES))

_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


def call(fn, stream, *args):
    """fn(*args, stream handle).  With a stream given the results are made on it, so
    that their memory is not handed out again while the call may write it."""
    if not args[0].is_cuda:
        raise ValueError("ubridge_amd ops take device tensors")
    if stream is None:
        r = fn(*args, _raw_stream(_device()))
    else:
        with torch.cuda.stream(stream):
            r = fn(*args, stream.cuda_stream)
    if r.__class__ is int:
        check(r)
    return r
