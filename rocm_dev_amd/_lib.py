"""Loads libsgemm.so and declares the C ABI of include/sgemm.h (and the profiling aids of include/sgemm_debug.h) to ctypes.

`lib` is the library through ctypes; `host` is the extension module (csrc/sg_torch.cpp) that takes the common calls to the
same library without ctypes.  There is no fallback: if either has not been built the import fails loudly.
"""
import ctypes as C
import os

import torch  # (the extension module links against its libraries)

from .build import HOST_PATH, LIB_PATH

for _path in (LIB_PATH, HOST_PATH):
    if not os.path.exists(_path):
        raise ImportError(
            "%s is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "or `make -C rocm_dev_amd/csrc`" % _path)

lib = C.CDLL(LIB_PATH)

from . import _torch_host as host  # noqa: E402

if host.torch_version != torch.__version__:    # it reads torch's own structures
    raise ImportError("%s was built against torch %s, this is %s: build it again" % (HOST_PATH, host.torch_version, torch.__version__))
host.bind(lib._handle)

_vp, _i, _sz = C.c_void_p, C.c_int, C.c_size_t

SIGNATURES = {
    "sg_strerror": (C.c_char_p, [_i]),
    "sg_init": (_i, []),
    "sg_init_stream": (_i, [_vp, _sz]),
    "sg_workspace_bytes": (_sz, []),
    "sg_release_stream": (_i, [_vp]),
    "sg_release_workspaces": (_i, []),
    "sg_workspace_query": (_i, [_i, _i, _i, C.POINTER(_sz)]),
    "sg_workspace_init": (_i, [_vp, _sz, _vp]),
    "sg_skinny_gemm_auto_ws": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _sz, _vp]),
    "sg_debug_stamps": (_i, [_vp, _sz]),
    "sg_debug_wide_gemm": (_i, [_vp] * 6 + [_i] * 7 + [_vp]),
    "sg_debug_line_gemm": (_i, [_vp] * 6 + [_i] * 8 + [_vp]),
    "sg_debug_skinny_line_gemm": (_i, [_vp] * 6 + [_i] * 9 + [_vp]),
    "sg_debug_skinny_line_choice": (_i, [_i, _i, _i, _i, C.POINTER(_i * 5)]),
    "sg_debug_line_choice": (_i, [_i, _i, _i, _i, _i, C.POINTER(_i * 4)]),
    "sg_debug_wide_choice": (_i, [_i, _i, _i, _i, _i, C.POINTER(_i * 3)]),
    "sg_debug_read_stream": (_i, [_vp, _i, _i, _i, _i, _vp]),
    "sg_debug_mxfp4_choice": (_i, [_i] * 5),
    "sg_debug_mxfp4_searches": (_i, []),
    "sg_debug_mxfp4_gemm": (_i, [_vp] * 6 + [_i] * 4 + [_vp]),
    "sg_debug_cu_ingest": (_i, [_vp, _sz, _vp, _sz, _i, _i, _i, _i, _i, _i, _vp, _vp]),
    "sg_skinny_gemm": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _i, _vp]),
    "sg_skinny_gemm_fastpath": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i]),
    "sg_skinny_gemm_auto": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "sg_skinny_gemm_rowcol": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "sg_skinny_gemm_bf16act": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "sg_skinny_gemm_bf16act_tuned": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp]),
    "sg_skinny_gemm_bf16act_choice": (_i, [_i, _i, _i, _vp, C.POINTER(_i)]),
    "sg_skinny_gemm_tuned": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp]),
    "sg_skinny_gemm_tuned_noalloc": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp]),
    "sg_skinny_gemm_pick": (_i, [_i, _i, _i, C.POINTER(_i * 8)]),
    "sg_skinny_gemm_choice": (_i, [_i, _i, _i, _vp, C.POINTER(_i)]),
    "sg_tuning_set": (_i, [_i, _i, _i, _vp]),
    "sg_tuning_get": (_i, [_i, _i, _i, _vp]),
    "sg_tuning_count": (_i, []),
    "sg_tuning_clear": (_i, []),
    "sg_tuning_load": (_i, [C.c_char_p]),
    "sg_tuning_save": (_i, [C.c_char_p]),
    "sg_async_gemm_f32": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "sg_async_gemm_bf16": (_i, [_vp, _vp, _vp, _i, _i, _i]),
    "sg_sparse24_gemm": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_sparse24_gemm_tuned": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp]),
    "sg_sparse24_compress": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_tiled_sum_reduce": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_tiled_sum_reduce_async": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_fp8_encode_rows": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "sg_fp8_decode_rows": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "sg_fp8_reduce_rows": (_i, [_vp, _vp, _vp, _i, _sz, _i, _i, _vp]),
    "sg_mxfp4_encode_rows": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "sg_mxfp4_decode_rows": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "sg_mxfp4_packed_bytes": (_sz, [_i, _i]),
    "sg_mxfp4_pack": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_mxfp4_gemm": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "sg_mxfp4_gemm_fp8act": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
}

for _name, (_res, _args) in SIGNATURES.items():
    _fn = getattr(lib, _name)
    _fn.restype = _res
    _fn.argtypes = _args
