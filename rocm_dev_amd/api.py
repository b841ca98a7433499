"""Host-side mirror of the reference's launcher and torch-binding surface.

Reference interfaces mirrored (paths below the reference's projects/ directory):
  skinny_gemm(...)            skinny_gemm/skinny_gemm_caller.cu:20-43
  skinny_gemm_fastpath(...)   skinny_gemm/skinny_gemm_caller.cu:343-346
  HFRK_skinny_gemm            skinny_gemm/skinny_gemm_binding.cu:64-100
  async_gemm(...)             async_gemm_sparse/sparse_k.cu:45-69
  tiled_sum_reduce(...)       tiled_sum_reduce/src.cu:52-73, tiled_sum_reduce_async/src.cu:179-200 (lds_queue=True)
Every function returns the integer return code of the C ABI (0 = success), as the
reference's launchers do; ``check=True`` raises SgError instead.  Tensors are torch CUDA
tensors used purely as device buffers: fp8 operands are uint8 or float8_e4m3fn, outputs
bfloat16 (or float32 for async_gemm), and everything is enqueued on torch's current stream.
"""
import ctypes as C
import enum

import torch

from ._lib import host, lib


class SgReturnCode(enum.IntEnum):
    SUCCESS = 0
    M_ABOVE_WARPTILE_M = 1
    N_NOT_EVEN = 2
    K_NOT_DIVISIBLE_BY_WARPTILE_K = 3
    TOO_MANY_WARPS = 4
    QSIZE_TOO_SMALL = 5
    INVALID_CONFIG = 6
    LAUNCH_FAILED = 7
    BAD_ALIGNMENT = 8
    BAD_ARGUMENT = 9
    WORKSPACE_TOO_SMALL = 10
    NO_DEVICE = 11


class SgError(RuntimeError):
    def __init__(self, code):
        self.code = int(code)
        super().__init__("libsgemm: %s (code %d)" % (strerror(code), code))


def strerror(code):
    return lib.sg_strerror(int(code)).decode()


def _done(rc, check):
    if check and rc != 0:
        raise SgError(rc)
    return rc


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dev(t, *dtypes):
    if not t.is_cuda:
        raise ValueError("expected a CUDA (HIP) tensor")
    if dtypes and t.dtype not in dtypes:
        raise ValueError("expected dtype in %s, got %s" % (dtypes, t.dtype))
    return t.data_ptr()


_FP8 = (torch.uint8, torch.float8_e4m3fn)

# The entry points that programs call per layer first offer their operands to the extension module (`host`), which
# launches plain ones in a few hundred nanoseconds and returns None for everything else - other devices, layouts the
# kernels would misread, tensor subclasses.  What follows the offer is the complete rule, and the error message.

# The C ABI takes raw pointers with the shapes it is told: everything it will assume about a tensor is checked here,
# before the call - a transposed or sliced operand would otherwise be read with the wrong strides, and a weight matrix
# with fewer columns than k past its allocation.
def _same_device(*tensors):
    live = [t for t in tensors if t is not None]
    for t in live:
        if not t.is_cuda:
            raise ValueError("expected CUDA (HIP) tensors")
        if t.device != live[0].device:
            raise ValueError("operands on different devices: %s and %s" % (live[0].device, t.device))


def _row_major(t, name):
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous (row-major), got strides %s for shape %s"
                         % (name, tuple(t.stride()), tuple(t.shape)))


def _weights(B, cols, name="B"):
    """[n, cols] with the columns contiguous; rows may be further apart than cols (a row stride)."""
    if B.dim() != 2 or B.shape[1] != cols:
        raise ValueError("%s must be [n, %d], got %s" % (name, cols, tuple(B.shape)))
    if B.shape[1] > 1 and B.stride(1) != 1:
        raise ValueError("%s must have contiguous columns, got strides %s" % (name, tuple(B.stride())))
    if B.shape[0] > 1 and B.stride(0) < cols:
        raise ValueError("%s: row stride %d below its %d columns" % (name, B.stride(0), cols))
    return B.stride(0) if B.shape[0] > 1 else max(B.stride(0), cols)


def _gemm_operands(A, B, D, scale_tensor=None, weight_cols=None, extra=()):
    """(m, n, k, b_stride) of D[m, n] = A[m, k] x B[n, weight_cols or k]^T after checking every layout assumption."""
    if A.dim() != 2 or D.dim() != 2:
        raise ValueError("A and D must be 2-D, got %s and %s" % (tuple(A.shape), tuple(D.shape)))
    m, k = A.shape
    b_stride = _weights(B, k if weight_cols is None else weight_cols)
    n = B.shape[0]
    if tuple(D.shape) != (m, n):
        raise ValueError("D must be [%d, %d], got %s" % (m, n, tuple(D.shape)))
    _row_major(A, "A")
    _row_major(D, "D")
    if scale_tensor is not None and (scale_tensor.numel() < 1 or not scale_tensor.is_contiguous()):
        raise ValueError("scale_tensor must hold at least one float")
    _same_device(A, B, D, scale_tensor, *extra)
    return m, n, k, b_stride


def _vector(t, length, name):
    if t is not None and (tuple(t.shape) != (length,) or not t.is_contiguous()):
        raise ValueError("%s must be a contiguous vector of %d floats, got shape %s strides %s"
                         % (name, length, tuple(t.shape), tuple(t.stride())))


def skinny_gemm(A, B, D, scale_tensor, split_k, A_producers, B_producers, consumers, b_lanes, qsize, op_m, ops,
                b_stride=None, check=False):
    """D[m,n] = bf16(scale * A[m,k] @ B[n,k]^T) with explicit tunables.  B is [n, k] with row stride b_stride."""
    m, n, k, row_stride = _gemm_operands(A, B, D, scale_tensor)
    if b_stride is None:
        b_stride = row_stride
    elif n > 1 and b_stride != row_stride:
        raise ValueError("b_stride %d is not the row stride of B (%d)" % (b_stride, row_stride))
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                _dev(scale_tensor, torch.float32), m, n, k, b_stride, split_k, A_producers,
                                B_producers, consumers, b_lanes, qsize, op_m, ops, _stream())
    return _done(rc, check)


def skinny_gemm_fastpath(A, B, D, scale_tensor, check=False):
    """Library-chosen configuration; B is [n, k] (row stride taken from the tensor)."""
    rc = host.skinny_gemm_fastpath(A, B, D, scale_tensor)
    if rc is not None:
        return _done(rc, check)
    m, n, k, b_stride = _gemm_operands(A, B, D, scale_tensor)
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm_auto(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                     _dev(scale_tensor, torch.float32), m, n, k, b_stride, _stream())
    return _done(rc, check)


class SgTuning(C.Structure):
    """Mirror of the C struct SgTuning (include/sgemm.h)."""
    _fields_ = [(name, C.c_int) for name in
                ("engine", "split_k", "waves", "row_tiles", "m_blocks", "depth", "k_chunks", "non_temporal",
                 "persistent_wgs_per_cu", "wave_tiles")]


ENGINE_AUTO, ENGINE_DIRECT, ENGINE_LDS, ENGINE_MID = 0, 1, 2, 4
TUNING_FIELDS = tuple(name for name, _ in SgTuning._fields_)


def tuning_as_dict(t):
    return {name: getattr(t, name) for name in TUNING_FIELDS}


def skinny_gemm_rowcol(A, B, D, scale_tensor=None, row_scales=None, col_scales=None, check=False):
    """D = bf16(((A @ B^T) * scale) * row_scales[:, None] * col_scales[None, :]); any factor may be None."""
    rc = host.skinny_gemm_rowcol(A, B, D, scale_tensor, row_scales, col_scales)
    if rc is not None:
        return _done(rc, check)
    m, n, k, b_stride = _gemm_operands(A, B, D, scale_tensor, extra=(row_scales, col_scales))
    _vector(row_scales, m, "row_scales")
    _vector(col_scales, n, "col_scales")
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm_rowcol(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                       None if scale_tensor is None else _dev(scale_tensor, torch.float32),
                                       None if row_scales is None else _dev(row_scales, torch.float32),
                                       None if col_scales is None else _dev(col_scales, torch.float32),
                                       m, n, k, b_stride, _stream())
    return _done(rc, check)


def skinny_gemm_bf16act(X, B, D, scale_tensor=None, col_scales=None, row_scales_out=None, tuning=None, check=False):
    """The rowcol GEMM on bf16 activations X [m, k]: rows quantised to E4M3 inside the GEMM (as fp8_encode_rows would),
    D = bf16(((q(X) @ B^T) * scale) * row_scale[:, None] * col_scales[None, :]); row_scales_out, if given, receives the
    row scales.  One launch where the fused kernel pays (skinny_gemm_bf16act_choice), two inside the library otherwise;
    with `tuning` (an SgTuning; engine 0 = the library's record for the shape) always the fused kernel."""
    if tuning is None:
        rc = host.skinny_gemm_bf16act(X, B, D, scale_tensor, col_scales, row_scales_out)
        if rc is not None:
            return _done(rc, check)
    m, n, k, b_stride = _gemm_operands(X, B, D, scale_tensor, extra=(col_scales, row_scales_out))
    _vector(col_scales, n, "col_scales")
    _vector(row_scales_out, m, "row_scales_out")
    args = (_dev(X, torch.bfloat16), _dev(B, *_FP8), _dev(D, torch.bfloat16),
            None if scale_tensor is None else _dev(scale_tensor, torch.float32),
            None if col_scales is None else _dev(col_scales, torch.float32),
            None if row_scales_out is None else _dev(row_scales_out, torch.float32), m, n, k, b_stride)
    with torch.cuda.device(X.device):
        if tuning is None:
            rc = lib.sg_skinny_gemm_bf16act(*args, _stream())
        else:
            rc = lib.sg_skinny_gemm_bf16act_tuned(*args, C.byref(tuning), _stream())
    return _done(rc, check)


def skinny_gemm_bf16act_choice(m, n, k):
    """(record, fused): the SgTuning skinny_gemm_bf16act launches for the shape and whether it is the fused kernel."""
    t, fused = SgTuning(), C.c_int(0)
    rc = lib.sg_skinny_gemm_bf16act_choice(m, n, k, C.byref(t), C.byref(fused))
    if rc != 0:
        raise SgError(rc)
    return t, bool(fused.value)


def skinny_gemm_tuned(A, B, D, scale_tensor, engine=ENGINE_AUTO, split_k=1, waves=4, row_tiles=1, m_blocks=None,
                      depth=2, k_chunks=4, non_temporal=1, persistent_wgs_per_cu=0, wave_tiles=0, check=False):
    """The library-native tuning entry (no reference counterpart): pick the engine and its shape."""
    m, n, k, b_stride = _gemm_operands(A, B, D, scale_tensor)
    if m_blocks is None:
        m_blocks = 1 if m <= 16 else 2
    t = SgTuning(engine, split_k, waves, row_tiles, m_blocks, depth, k_chunks, non_temporal, persistent_wgs_per_cu, wave_tiles)
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm_tuned(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                      _dev(scale_tensor, torch.float32), m, n, k, b_stride, C.byref(t), _stream())
    return _done(rc, check)


def skinny_gemm_tuned_noalloc(A, B, D, scale_tensor, engine=ENGINE_AUTO, split_k=1, waves=4, row_tiles=1, m_blocks=None,
                              depth=2, k_chunks=4, non_temporal=1, persistent_wgs_per_cu=0, wave_tiles=0, check=False):
    """skinny_gemm_tuned with the split-K partials in the library's fixed device array: allocates nothing, refuses
    configurations whose partials exceed 8 MB or 4096 tiles with WORKSPACE_TOO_SMALL (no reference counterpart)."""
    m, n, k, b_stride = _gemm_operands(A, B, D, scale_tensor)
    if m_blocks is None:
        m_blocks = 1 if m <= 16 else 2
    t = SgTuning(engine, split_k, waves, row_tiles, m_blocks, depth, k_chunks, non_temporal, persistent_wgs_per_cu, wave_tiles)
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm_tuned_noalloc(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                              _dev(scale_tensor, torch.float32), m, n, k, b_stride, C.byref(t),
                                              _stream())
    return _done(rc, check)


def init_stream(stream=None, partial_bytes=64 << 20, check=True):
    """Create the split-K workspace of `stream` (torch stream; None = torch's current stream) ahead of time."""
    handle = _stream() if stream is None else stream.cuda_stream
    return _done(lib.sg_init_stream(handle, partial_bytes), check)


def workspace_bytes():
    return lib.sg_workspace_bytes()


def release_stream(stream=None, check=True):
    """Wait for `stream` (torch stream; None = torch's current stream) and free what the library holds for it."""
    handle = _stream() if stream is None else stream.cuda_stream
    return _done(lib.sg_release_stream(handle), check)


def release_workspaces(check=True):
    """Wait for the device and free every buffer the library owns on it; workspace_bytes() is 0 afterwards."""
    return _done(lib.sg_release_workspaces(), check)


def workspace_query(m, n, k):
    """Bytes of caller-owned workspace skinny_gemm_auto_ws needs for the shape (0: the launch has no K split)."""
    need = C.c_size_t(0)
    rc = lib.sg_workspace_query(m, n, k, C.byref(need))
    if rc != 0:
        raise SgError(rc)
    return need.value


def workspace_init(workspace, check=True):
    """Clear the counter region of a caller-owned workspace (a uint8 CUDA tensor) in stream order: once per buffer."""
    return _done(lib.sg_workspace_init(_dev(workspace, torch.uint8), workspace.numel(), _stream()), check)


def skinny_gemm_auto_ws(A, B, D, scale_tensor, workspace=None, check=False):
    """skinny_gemm_fastpath on caller-owned memory: `workspace` (uint8 CUDA tensor, 256-byte aligned, prepared once with
    workspace_init; None where workspace_query says 0) holds the split-K partials and counters, nothing is allocated."""
    m, n, k, b_stride = _gemm_operands(A, B, D, scale_tensor, extra=(workspace,))
    if workspace is not None:
        _row_major(workspace, "workspace")
    with torch.cuda.device(A.device):
        rc = lib.sg_skinny_gemm_auto_ws(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                        _dev(scale_tensor, torch.float32), m, n, k, b_stride,
                                        None if workspace is None else _dev(workspace, torch.uint8),
                                        0 if workspace is None else workspace.numel(), _stream())
    return _done(rc, check)


def skinny_gemm_pick(m, n, k):
    """The tunables the fastpath would use: dict with the reference's parameter names."""
    out = (C.c_int * 8)()
    rc = lib.sg_skinny_gemm_pick(m, n, k, C.byref(out))
    if rc != 0:
        raise SgError(rc)
    names = ("split_k", "A_producers", "B_producers", "consumers", "b_lanes", "qsize", "op_m", "ops")
    return dict(zip(names, list(out)))


def skinny_gemm_choice(m, n, k):
    """(record, from_table): the complete SgTuning the fastpath would launch for the shape, and whether it comes
    from the tuning table rather than the built-in heuristics.  Kernels that no record describes may run in the place of the
    heuristics' record: those for rows off their 128-byte lines (skinny_gemm_line_choice; up to 32 rows
    skinny_gemm_skinny_line_choice) and, above 128 rows, a wide tile (skinny_gemm_wide_choice)."""
    t, from_table = SgTuning(), C.c_int(0)
    rc = lib.sg_skinny_gemm_choice(m, n, k, C.byref(t), C.byref(from_table))
    if rc != 0:
        raise SgError(rc)
    return t, bool(from_table.value)


def skinny_gemm_wide_choice(m, n, k, b_stride=None, factors=False):
    """(row_tiles, m_blocks, split_k) of the wide tile the fastpath (with factors: skinny_gemm_rowcol with row or column
    factors) launches for the shape, or None where it launches something else."""
    out = (C.c_int * 3)()
    rc = lib.sg_debug_wide_choice(m, n, k, k if b_stride is None else b_stride, 1 if factors else 0, C.byref(out))
    if rc != 0:
        raise SgError(rc)
    return tuple(out) if out[0] else None


def skinny_gemm_line_choice(m, n, k, b_stride=None, factors=False):
    """(waves, row_tiles, m_blocks, split_k) of the kernel for rows off their 128-byte lines where the fastpath (with factors:
    skinny_gemm_rowcol with row or column factors) launches it for the shape, or None where it launches something else.  Its
    tile is 8 * waves * row_tiles weight rows by 32 * m_blocks activation rows."""
    out = (C.c_int * 4)()
    rc = lib.sg_debug_line_choice(m, n, k, k if b_stride is None else b_stride, 1 if factors else 0, C.byref(out))
    if rc != 0:
        raise SgError(rc)
    return tuple(out) if out[0] else None


def skinny_gemm_skinny_line_choice(m, n, k, b_stride=None):
    """(waves, row_tiles, depth, split_k, resident) of the skinny kernel for rows off their 128-byte lines where the fastpath
    launches it for the shape (up to 32 rows), or None where it launches something else."""
    out = (C.c_int * 5)()
    rc = lib.sg_debug_skinny_line_choice(m, n, k, k if b_stride is None else b_stride, C.byref(out))
    if rc != 0:
        raise SgError(rc)
    return tuple(out) if out[0] else None


def tuning_set(m, n, k, tuning):
    """Store `tuning` (an SgTuning, or None to remove the entry) as the record the fastpath uses for the shape."""
    return _done(lib.sg_tuning_set(m, n, k, None if tuning is None else C.byref(tuning)), True)


def tuning_get(m, n, k):
    """The table's SgTuning for the shape, or None."""
    t = SgTuning()
    return t if lib.sg_tuning_get(m, n, k, C.byref(t)) == 0 else None


def tuning_count():
    return lib.sg_tuning_count()


def tuning_clear():
    return _done(lib.sg_tuning_clear(), True)


def tuning_load(path):
    """Merge a tuning file (written by tuning_save or rocm_dev_amd.autotune) into the table."""
    return _done(lib.sg_tuning_load(str(path).encode()), True)


def tuning_save(path):
    return _done(lib.sg_tuning_save(str(path).encode()), True)


class HFRK_skinny_gemm:
    """Same constructor and method as the reference's torch extension class.

    ``B`` is passed as the reference passes it: a (k, n) *view* of an n x k, K-contiguous
    weight, so n = B.size(1) and b_stride = B.stride(1) (skinny_gemm_binding.cu:36-39).
    op_m follows m: 8, 16 or 32 (skinny_gemm_binding.cu:42-45).  D is bfloat16 and is
    overwritten.
    """

    def __init__(self, world_size):
        self.world_size = world_size  # unused, as in the reference

    def skinny_gemm_torch_binding(self, A, B, D, scale_tensor, split_k, A_producers, B_producers, consumers,
                                  b_lanes, qsize, ops):
        # B arrives as the (K, N) view of an N x K, K-contiguous weight matrix (skinny_gemm_binding.cu:36-41)
        if A.dim() != 2 or B.dim() != 2 or B.size(0) != A.size(1) or tuple(D.shape) != (A.size(0), B.size(1)):
            raise ValueError("A [m, k], B [k, n] (a view of n x k weights) and D [m, n] disagree: %s %s %s"
                             % (tuple(A.shape), tuple(B.shape), tuple(D.shape)))
        if (B.size(0) > 1 and B.stride(0) != 1) or (B.size(1) > 1 and B.stride(1) < B.size(0)):
            raise ValueError("B must be the transposed view of K-contiguous weights, got strides %s" % (tuple(B.stride()),))
        _row_major(A, "A")
        _row_major(D, "D")
        _same_device(A, B, D, scale_tensor)
        m, k = A.size(0), A.size(1)
        n = B.size(1)
        b_stride = B.stride(1) if n > 1 else max(B.stride(1), k)
        op_m = 8 if m <= 8 else (16 if m <= 16 else 32)
        with torch.cuda.device(A.device):
            return lib.sg_skinny_gemm(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16),
                                      _dev(scale_tensor, torch.float32), m, n, k, b_stride, split_k, A_producers,
                                      B_producers, consumers, b_lanes, qsize, op_m, ops, _stream())


def sparse24_gemm(A, B_vals, B_meta, D, scale_tensor, tuning=None, check=False):
    """2:4 sparse weights: B_vals [n, k/2] kept codes, B_meta [n, k/8] position nibbles (include/sgemm.h)."""
    if tuning is None:
        rc = host.sparse24_gemm(A, B_vals, B_meta, D, scale_tensor)
        if rc is not None:
            return _done(rc, check)
    if A.dim() != 2 or A.shape[1] % 8:
        raise ValueError("A must be [m, k] with k a multiple of 8, got %s" % (tuple(A.shape),))
    m, n, k, _ = _gemm_operands(A, B_vals, D, scale_tensor, weight_cols=A.shape[1] // 2, extra=(B_meta,))
    _row_major(B_vals, "B_vals")
    if tuple(B_meta.shape) != (n, k // 8) or not B_meta.is_contiguous():
        raise ValueError("B_meta must be a contiguous [%d, %d], got %s" % (n, k // 8, tuple(B_meta.shape)))
    with torch.cuda.device(A.device):
        if tuning is None:
            rc = lib.sg_sparse24_gemm(_dev(A, *_FP8), _dev(B_vals, *_FP8), _dev(B_meta, torch.uint8),
                                      _dev(D, torch.bfloat16), _dev(scale_tensor, torch.float32), m, n, k, _stream())
        else:
            rc = lib.sg_sparse24_gemm_tuned(_dev(A, *_FP8), _dev(B_vals, *_FP8), _dev(B_meta, torch.uint8),
                                            _dev(D, torch.bfloat16), _dev(scale_tensor, torch.float32), m, n, k,
                                            C.byref(tuning), _stream())
    return _done(rc, check)


def sparse24_compress(B, B_vals, B_meta, check=False):
    """Prune dense E4M3 weights B [n, k] to 2:4 (two largest magnitudes per group of four) and compress them
    into B_vals [n, k/2] and B_meta [n, k/8] (format of include/sgemm.h)."""
    rc = host.sparse24_compress(B, B_vals, B_meta)
    if rc is not None:
        return _done(rc, check)
    if B.dim() != 2 or B.shape[1] % 8:
        raise ValueError("B must be [n, k] with k a multiple of 8, got %s" % (tuple(B.shape),))
    n, k = B.shape
    b_stride = _weights(B, k)
    if tuple(B_vals.shape) != (n, k // 2) or tuple(B_meta.shape) != (n, k // 8):
        raise ValueError("B_vals must be [%d, %d] and B_meta [%d, %d]" % (n, k // 2, n, k // 8))
    _row_major(B_vals, "B_vals")
    _row_major(B_meta, "B_meta")
    _same_device(B, B_vals, B_meta)
    with torch.cuda.device(B.device):
        rc = lib.sg_sparse24_compress(_dev(B, *_FP8), _dev(B_vals, *_FP8), _dev(B_meta, torch.uint8), n, k, b_stride,
                                      _stream())
    return _done(rc, check)


def async_gemm(A, B, D, check=False):
    """D = A @ B^T without a scale on the default stream; D is float32 or bfloat16."""
    m, n, k, _ = _gemm_operands(A, B, D)
    _row_major(B, "B")
    with torch.cuda.device(A.device):
        if D.dtype == torch.float32:
            rc = lib.sg_async_gemm_f32(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D), m, n, k)
        else:
            rc = lib.sg_async_gemm_bf16(_dev(A, *_FP8), _dev(B, *_FP8), _dev(D, torch.bfloat16), m, n, k)
    return _done(rc, check)


def tiled_sum_reduce(A, B, D, check=False, lds_queue=False):
    """D[m,n] = sum_b (A[b,m,n] + B[b,m,n]) in fp32, batch order.  lds_queue=True runs the variant that stages the
    batches through a queue in LDS (tiled_sum_reduce_async/src.cu:179-200); the result bits are the same."""
    if not lds_queue:
        rc = host.tiled_sum_reduce(A, B, D)
        if rc is not None:
            return _done(rc, check)
    if A.dim() != 3 or B.shape != A.shape or tuple(D.shape) != tuple(A.shape[1:]):
        raise ValueError("A and B must be [b, m, n] and D [m, n], got %s, %s, %s" % (tuple(A.shape), tuple(B.shape), tuple(D.shape)))
    for t, name in ((A, "A"), (B, "B"), (D, "D")):
        _row_major(t, name)
    _same_device(A, B, D)
    b, m, n = A.shape
    fn = lib.sg_tiled_sum_reduce_async if lds_queue else lib.sg_tiled_sum_reduce
    with torch.cuda.device(A.device):
        rc = fn(_dev(A, torch.float32), _dev(B, torch.float32), _dev(D, torch.float32), b, m, n, _stream())
    return _done(rc, check)


def _codec_operands(X, Q, scales, nbuf=None):
    if X.dim() != 2 or tuple(Q.shape) != ((tuple(X.shape) if nbuf is None else (nbuf,) + tuple(X.shape))):
        raise ValueError("row-codec operands must agree in shape, got %s and %s" % (tuple(X.shape), tuple(Q.shape)))
    want = (X.shape[0],) if nbuf is None else (nbuf, X.shape[0])
    if tuple(scales.shape) != want:
        raise ValueError("scales must have shape %s, got %s" % (want, tuple(scales.shape)))
    for t, name in ((X, "the bf16 matrix"), (Q, "Q"), (scales, "scales")):
        _row_major(t, name)
    _same_device(X, Q, scales)


def fp8_encode_rows(X, Q, scales, check=False):
    rc = host.fp8_encode_rows(X, Q, scales)
    if rc is not None:
        return _done(rc, check)
    _codec_operands(X, Q, scales)
    rows, cols = X.shape
    with torch.cuda.device(X.device):
        rc = lib.sg_fp8_encode_rows(_dev(X, torch.bfloat16), _dev(Q, *_FP8), _dev(scales, torch.float32),
                                    rows, cols, _stream())
    return _done(rc, check)


def fp8_decode_rows(Q, scales, Y, check=False):
    rc = host.fp8_decode_rows(Q, scales, Y)
    if rc is not None:
        return _done(rc, check)
    _codec_operands(Y, Q, scales)
    rows, cols = Q.shape
    with torch.cuda.device(Q.device):
        rc = lib.sg_fp8_decode_rows(_dev(Q, *_FP8), _dev(scales, torch.float32), _dev(Y, torch.bfloat16),
                                    rows, cols, _stream())
    return _done(rc, check)


def fp8_reduce_rows(Q, scales, Y, check=False):
    """Q [nbuf, rows, cols], scales [nbuf, rows] -> Y [rows, cols] bfloat16."""
    rc = host.fp8_reduce_rows(Q, scales, Y)
    if rc is not None:
        return _done(rc, check)
    if Q.dim() != 3:
        raise ValueError("Q must be [nbuf, rows, cols], got %s" % (tuple(Q.shape),))
    _codec_operands(Y, Q, scales, nbuf=Q.shape[0])
    nbuf, rows, cols = Q.shape
    with torch.cuda.device(Q.device):
        rc = lib.sg_fp8_reduce_rows(_dev(Q, *_FP8), _dev(scales, torch.float32), _dev(Y, torch.bfloat16),
                                    nbuf, Q.stride(0), rows, cols, _stream())
    return _done(rc, check)


# MXFP4 (include/sgemm.h): codes two a byte, one scale byte per 32 columns.
def _mx_operands(X, Q, scales):
    if X.dim() != 2 or X.shape[1] % 32:
        raise ValueError("the bf16 matrix must be [rows, cols] with cols a multiple of 32, got %s" % (tuple(X.shape),))
    rows, cols = X.shape
    _mx_codes(Q, scales, rows, cols, ("Q", "scales"))
    _row_major(X, "the bf16 matrix")
    _same_device(X, Q, scales)
    return rows, cols


def _mx_codes(Q, scales, rows, cols, names):
    if tuple(Q.shape) != (rows, cols // 2) or tuple(scales.shape) != (rows, cols // 32):
        raise ValueError("%s must be [%d, %d] and %s [%d, %d], got %s and %s"
                         % (names[0], rows, cols // 2, names[1], rows, cols // 32, tuple(Q.shape), tuple(scales.shape)))
    _row_major(Q, names[0])
    _row_major(scales, names[1])


def mxfp4_encode_rows(X, Q, scales, check=False):
    """X [rows, cols] bfloat16 -> Q [rows, cols/2] codes and scales [rows, cols/32], both uint8."""
    rc = host.mxfp4_encode_rows(X, Q, scales)
    if rc is not None:
        return _done(rc, check)
    rows, cols = _mx_operands(X, Q, scales)
    with torch.cuda.device(X.device):
        rc = lib.sg_mxfp4_encode_rows(_dev(X, torch.bfloat16), _dev(Q, torch.uint8), _dev(scales, torch.uint8), rows, cols, _stream())
    return _done(rc, check)


def mxfp4_decode_rows(Q, scales, Y, check=False):
    """Q [rows, cols/2] codes and scales [rows, cols/32] -> Y [rows, cols] bfloat16."""
    rc = host.mxfp4_decode_rows(Q, scales, Y)
    if rc is not None:
        return _done(rc, check)
    rows, cols = _mx_operands(Y, Q, scales)
    with torch.cuda.device(Q.device):
        rc = lib.sg_mxfp4_decode_rows(_dev(Q, torch.uint8), _dev(scales, torch.uint8), _dev(Y, torch.bfloat16), rows, cols, _stream())
    return _done(rc, check)


def mxfp4_packed_bytes(n, k):
    """Bytes of the packed form of an n x k weight matrix (k a multiple of 32)."""
    need = lib.sg_mxfp4_packed_bytes(n, k)
    if need == 0:
        raise ValueError("packed weights need n > 0 and k a positive multiple of 32, got n = %d, k = %d" % (n, k))
    return need


def mxfp4_pack(B, B_scales, P, check=False):
    """Weights B [n, k/2] codes (rows at any stride that 16 divides) with scales [n, k/32] -> P, a contiguous uint8 vector of
    mxfp4_packed_bytes(n, k) that the GEMMs read.  Once per weight matrix."""
    if B.dim() != 2 or B.shape[1] % 16:
        raise ValueError("B must be [n, k/2] with k a multiple of 32, got %s" % (tuple(B.shape),))
    n, k = B.shape[0], 2 * B.shape[1]
    b_stride = _weights(B, k // 2)
    if tuple(B_scales.shape) != (n, k // 32):
        raise ValueError("B_scales must be [%d, %d], got %s" % (n, k // 32, tuple(B_scales.shape)))
    _row_major(B_scales, "B_scales")
    _packed(P, n, k)
    _same_device(B, B_scales, P)
    with torch.cuda.device(B.device):
        rc = lib.sg_mxfp4_pack(_dev(B, torch.uint8), _dev(B_scales, torch.uint8), _dev(P, torch.uint8), n, k, b_stride, _stream())
    return _done(rc, check)


def _packed(P, n, k):
    need = mxfp4_packed_bytes(n, k)
    if P.dim() != 1 or P.numel() != need or not P.is_contiguous():
        raise ValueError("P must be a contiguous vector of %d bytes (%d x %d weights packed), got shape %s strides %s"
                         % (need, n, k, tuple(P.shape), tuple(P.stride())))


def _mx_gemm(A, k, P, D, scale_tensor, extra):
    if A.dim() != 2 or D.dim() != 2 or D.shape[0] != A.shape[0]:
        raise ValueError("A and D must be matrices of as many rows, got %s and %s" % (tuple(A.shape), tuple(D.shape)))
    m, n = D.shape
    _packed(P, n, k)
    _row_major(A, "A")
    _row_major(D, "D")
    if scale_tensor is not None and (scale_tensor.numel() < 1 or not scale_tensor.is_contiguous()):
        raise ValueError("scale_tensor must hold at least one float")
    _same_device(A, P, D, scale_tensor, *extra)
    return m, n


def mxfp4_gemm(A, A_scales, P, D, scale_tensor=None, check=False):
    """D[m,n] = bf16(scale * A @ B^T), A [m, k/2] codes with A_scales [m, k/32] (mxfp4_encode_rows), B packed into P
    (mxfp4_pack)."""
    rc = host.mxfp4_gemm(A, A_scales, P, D, scale_tensor)
    if rc is not None:
        return _done(rc, check)
    if A.dim() != 2 or A.shape[1] % 16:
        raise ValueError("A must be [m, k/2] with k a multiple of 32, got %s" % (tuple(A.shape),))
    k = 2 * A.shape[1]
    _mx_codes(A, A_scales, A.shape[0], k, ("A", "A_scales"))
    m, n = _mx_gemm(A, k, P, D, scale_tensor, (A_scales,))
    with torch.cuda.device(A.device):
        rc = lib.sg_mxfp4_gemm(_dev(A, torch.uint8), _dev(A_scales, torch.uint8), _dev(P, torch.uint8), _dev(D, torch.bfloat16),
                               None if scale_tensor is None else _dev(scale_tensor, torch.float32), m, n, k, _stream())
    return _done(rc, check)


def mxfp4_gemm_fp8act(A, P, D, scale_tensor=None, row_scales=None, check=False):
    """D[m,n] = bf16((scale * A @ B^T) * row_scales[:, None]), A [m, k] E4M3 (fp8_encode_rows), B packed into P (mxfp4_pack)."""
    rc = host.mxfp4_gemm_fp8act(A, P, D, scale_tensor, row_scales)
    if rc is not None:
        return _done(rc, check)
    if A.dim() != 2 or A.shape[1] % 32:
        raise ValueError("A must be [m, k] with k a multiple of 32, got %s" % (tuple(A.shape),))
    k = A.shape[1]
    m, n = _mx_gemm(A, k, P, D, scale_tensor, (row_scales,))
    _vector(row_scales, m, "row_scales")
    with torch.cuda.device(A.device):
        rc = lib.sg_mxfp4_gemm_fp8act(_dev(A, *_FP8), _dev(P, torch.uint8), _dev(D, torch.bfloat16),
                                      None if scale_tensor is None else _dev(scale_tensor, torch.float32),
                                      None if row_scales is None else _dev(row_scales, torch.float32), m, n, k, _stream())
    return _done(rc, check)


def _matrix(t, rows, cols, name):
    if tuple(t.shape) != (rows, cols):
        raise ValueError("%s must be [%d, %d], got %s" % (name, rows, cols, tuple(t.shape)))
    _row_major(t, name)


def _ptr(t, *dtypes):
    return None if t is None else _dev(t, *dtypes)


def rmsnorm_fp8_rows(X, Q, scales, weight=None, residual=None, sum_out=None, Y=None, eps=1e-6, check=False):
    """Root-mean-square norm of X (+ residual) [rows, cols] bfloat16, times weight [cols], into E4M3 rows Q with scales [rows]
    (float32): what fp8_encode_rows gives of the norm in 32 bits.  sum_out, if given, receives X + residual (it may be X or
    residual itself), Y the norm in bfloat16."""
    rc = host.rmsnorm_fp8_rows(X, Q, scales, weight, residual, sum_out, Y, eps)
    if rc is not None:
        return _done(rc, check)
    if X.dim() != 2 or X.shape[1] % 16:
        raise ValueError("X must be [rows, cols] with cols a multiple of 16, got %s" % (tuple(X.shape),))
    rows, cols = X.shape
    for t, name in ((X, "X"), (Q, "Q"), (residual, "residual"), (sum_out, "sum_out"), (Y, "Y")):
        if t is not None:
            _matrix(t, rows, cols, name)
    _vector(scales, rows, "scales")
    if weight is not None and (tuple(weight.shape) != (cols,) or not weight.is_contiguous()):
        raise ValueError("weight must be a contiguous vector of %d values, got shape %s strides %s"
                         % (cols, tuple(weight.shape), tuple(weight.stride())))
    _same_device(X, Q, scales, weight, residual, sum_out, Y)
    with torch.cuda.device(X.device):
        rc = lib.sg_rmsnorm_fp8_rows(_dev(X, torch.bfloat16), _ptr(residual, torch.bfloat16), _ptr(weight, torch.bfloat16),
                                     _ptr(sum_out, torch.bfloat16), _ptr(Y, torch.bfloat16), _dev(Q, *_FP8), _dev(scales, torch.float32),
                                     eps, rows, cols, _stream())
    return _done(rc, check)


# 4-bit integers with group scales (include/sgemm.h): codes two a byte, a scale and on request a zero for each group of a row's columns.
_INT4_ZEROS, _INT4_F16_SCALES = 1, 2


def _int4_flags(zeros, scale_dtype):
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("scales must be bfloat16 or float16, got %s" % scale_dtype)
    return (_INT4_ZEROS if zeros else 0) | (_INT4_F16_SCALES if scale_dtype == torch.float16 else 0)


def int4_packed_bytes(n, k, group=128, zeros=False):
    """Bytes of the packed form of n x k weights in groups of 32, 64 or 128 columns (k a multiple of the group), with zeros or without."""
    need = lib.sg_int4_packed_bytes(n, k, group, _INT4_ZEROS if zeros else 0)
    if need == 0:
        raise ValueError("packed weights need n > 0, a group of 32, 64 or 128 and k a positive multiple of it, got n = %d, k = %d, group = %d"
                         % (n, k, group))
    return need


def _int4_packed(P, n, k, group, zeros):
    need = int4_packed_bytes(n, k, group, zeros)
    if P.dim() != 1 or P.numel() != need or not P.is_contiguous():
        raise ValueError("P must be a contiguous vector of %d bytes (%d x %d weights packed in groups of %d%s), got shape %s strides %s"
                         % (need, n, k, group, " with zeros" if zeros else "", tuple(P.shape), tuple(P.stride())))


def int4_pack(B, scales, P, zeros=None, check=False):
    """Weights B [n, k/2] (codes two a byte, the even column in the low nibble; rows at any stride that 16 divides) with scales
    [n, k/group] in bfloat16 or float16 and zeros [n, k/group] in uint8 (None: 8) -> P, a contiguous uint8 vector of
    int4_packed_bytes(n, k, group, zeros is not None) that int4_gemm reads.  Once per weight matrix; the group is what the scales'
    shape says."""
    if B.dim() != 2 or scales.dim() != 2 or scales.shape[1] == 0 or (2 * B.shape[1]) % scales.shape[1]:
        raise ValueError("B must be [n, k/2] and scales [n, k/group], got %s and %s" % (tuple(B.shape), tuple(scales.shape)))
    n, k = B.shape[0], 2 * B.shape[1]
    group = k // scales.shape[1]
    b_stride = _weights(B, k // 2)
    _matrix(scales, n, k // group, "scales")
    if zeros is not None:
        _matrix(zeros, n, k // group, "zeros")
    _int4_packed(P, n, k, group, zeros is not None)
    flags = _int4_flags(zeros is not None, scales.dtype)
    _same_device(B, scales, zeros, P)
    with torch.cuda.device(B.device):
        rc = lib.sg_int4_pack(_dev(B, torch.uint8), _dev(scales), _ptr(zeros, torch.uint8), _dev(P, torch.uint8), n, k, group, flags, b_stride,
                              _stream())
    return _done(rc, check)


def int4_gemm(A, P, D, group=128, zeros=False, scale_dtype=torch.bfloat16, check=False):
    """D[m,n] = bf16(A @ B^T), A [m, k] bfloat16, B packed into P (int4_pack) in groups of `group` columns, with zeros or without, its
    scales in scale_dtype.  P does not record these: its size is checked, but that is the same for both types of scales, and with the
    other one the results are wrong."""
    flags = _int4_flags(zeros, scale_dtype)
    rc = host.int4_gemm(A, P, D, group, flags)
    if rc is not None:
        return _done(rc, check)
    if A.dim() != 2 or D.dim() != 2 or D.shape[0] != A.shape[0]:
        raise ValueError("A and D must be matrices of as many rows, got %s and %s" % (tuple(A.shape), tuple(D.shape)))
    (m, k), n = A.shape, D.shape[1]
    _int4_packed(P, n, k, group, zeros)
    _row_major(A, "A")
    _row_major(D, "D")
    _same_device(A, P, D)
    with torch.cuda.device(A.device):
        rc = lib.sg_int4_gemm(_dev(A, torch.bfloat16), _dev(P, torch.uint8), _dev(D, torch.bfloat16), m, n, k, group, flags, _stream())
    return _done(rc, check)


# A mixture-of-experts layer for up to 64 tokens (include/sgemm.h).
def moe_workspace_bytes(m, hidden, inner, experts, top_k):
    """Bytes of workspace that moe_layer and moe_experts take for these sizes."""
    need = lib.sg_moe_workspace_bytes(m, hidden, inner, experts, top_k)
    if need == 0:
        raise ValueError("1 <= m <= 64 tokens, hidden and inner multiples of 16 up to 2^20, up to 512 experts and top_k <= 16 of them are taken, got m = %d, "
                         "hidden = %d, inner = %d, experts = %d, top_k = %d" % (m, hidden, inner, experts, top_k))
    return need


def _moe_workspace(workspace, need, device):
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.dim() != 1 or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 vector, got %s %s" % (workspace.dtype, tuple(workspace.shape)))
    return workspace


def _moe_choice(X, ids, weights):
    if X.dim() != 2 or ids.dim() != 2 or ids.shape[0] != X.shape[0]:
        raise ValueError("X must be [m, hidden] and ids [m, top_k], got %s and %s" % (tuple(X.shape), tuple(ids.shape)))
    _row_major(X, "X")
    _matrix(ids, *ids.shape, "ids")
    _matrix(weights, *ids.shape, "weights")
    return (*X.shape, ids.shape[1])


def _moe_experts(X, W1, W2, D, S1, S2):
    m, hidden = X.shape
    if W1.dim() != 3 or W1.shape[1] % 2 or W1.shape[2] != hidden:
        raise ValueError("W_gate_up must be [experts, 2 * inner, %d], got %s" % (hidden, tuple(W1.shape)))
    experts, inner = W1.shape[0], W1.shape[1] // 2
    if tuple(W2.shape) != (experts, hidden, inner):
        raise ValueError("W_down must be [%d, %d, %d], got %s" % (experts, hidden, inner, tuple(W2.shape)))
    _row_major(W1, "W_gate_up")
    _row_major(W2, "W_down")
    _matrix(D, m, hidden, "D")
    if S1 is not None:
        _matrix(S1, experts, 2 * inner, "gate_up_scales")
    if S2 is not None:
        _matrix(S2, experts, hidden, "down_scales")
    return experts, inner


def moe_route(X, router, ids, weights, renormalize=True, workspace=None, check=False):
    """The router of a mixture-of-experts layer: X [m, hidden] and router [experts, hidden] bfloat16 -> ids [m, top_k] int32, the experts
    of the largest logits in their order (ties: the lower index), and weights [m, top_k] float32, their softmax (renormalize=False:
    their part of the softmax over all experts)."""
    m, hidden, top_k = _moe_choice(X, ids, weights)
    if router.dim() != 2 or router.shape[1] != hidden:
        raise ValueError("router must be [experts, %d], got %s" % (hidden, tuple(router.shape)))
    _row_major(router, "router")
    experts = router.shape[0]
    moe_workspace_bytes(m, hidden, 16, experts, top_k)
    _same_device(X, router, ids, weights, workspace)
    with torch.cuda.device(X.device):
        ws = _moe_workspace(workspace, 4 * m * experts, X.device)
        rc = lib.sg_moe_route(_dev(X, torch.bfloat16), _dev(router, torch.bfloat16), _dev(ids, torch.int32), _dev(weights, torch.float32), m, hidden,
                              experts, top_k, int(bool(renormalize)), _dev(ws), ws.numel(), _stream())
    return _done(rc, check)


def moe_experts(X, ids, weights, W_gate_up, W_down, D, gate_up_scales=None, down_scales=None, workspace=None, check=False):
    """D [m, hidden] = sum over a token's experts of weight * down(silu(gate(x)) * up(x)): X [m, hidden] bfloat16, ids [m, top_k] int32
    (outside 0..experts-1: none), weights [m, top_k] float32, W_gate_up [experts, 2 * inner, hidden] (the gate's rows first) and W_down
    [experts, hidden, inner] E4M3 with a scale a row ([experts, 2 * inner], [experts, hidden] float32, or None)."""
    m, hidden, top_k = _moe_choice(X, ids, weights)
    experts, inner = _moe_experts(X, W_gate_up, W_down, D, gate_up_scales, down_scales)
    need = moe_workspace_bytes(m, hidden, inner, experts, top_k)
    _same_device(X, ids, weights, W_gate_up, W_down, D, gate_up_scales, down_scales, workspace)
    with torch.cuda.device(X.device):
        ws = _moe_workspace(workspace, need, X.device)
        rc = lib.sg_moe_experts(_dev(X, torch.bfloat16), _dev(ids, torch.int32), _dev(weights, torch.float32), _dev(W_gate_up, *_FP8),
                                _ptr(gate_up_scales, torch.float32), _dev(W_down, *_FP8), _ptr(down_scales, torch.float32),
                                _dev(D, torch.bfloat16), m, hidden, inner, experts, top_k, _dev(ws), ws.numel(), _stream())
    return _done(rc, check)


def moe_layer(X, router, W_gate_up, W_down, D, ids, weights, gate_up_scales=None, down_scales=None, renormalize=True, workspace=None,
              check=False):
    """moe_route and moe_experts in one call; ids [m, top_k] int32 and weights [m, top_k] float32 are outputs.  workspace: a uint8
    vector of moe_workspace_bytes(m, hidden, inner, experts, top_k), allocated for the call if it is None; calls that may overlap need
    one each."""
    rc = host.moe_layer(X, router, W_gate_up, W_down, D, ids, weights, gate_up_scales, down_scales, renormalize, workspace)
    if rc is not None:
        return _done(rc, check)
    m, hidden, top_k = _moe_choice(X, ids, weights)
    experts, inner = _moe_experts(X, W_gate_up, W_down, D, gate_up_scales, down_scales)
    _matrix(router, experts, hidden, "router")
    need = moe_workspace_bytes(m, hidden, inner, experts, top_k)
    _same_device(X, router, W_gate_up, W_down, D, ids, weights, gate_up_scales, down_scales, workspace)
    with torch.cuda.device(X.device):
        ws = _moe_workspace(workspace, need, X.device)
        rc = lib.sg_moe_layer(_dev(X, torch.bfloat16), _dev(router, torch.bfloat16), _dev(W_gate_up, *_FP8), _ptr(gate_up_scales, torch.float32),
                              _dev(W_down, *_FP8), _ptr(down_scales, torch.float32), _dev(D, torch.bfloat16), _dev(ids, torch.int32),
                              _dev(weights, torch.float32), m, hidden, inner, experts, top_k, int(bool(renormalize)), _dev(ws), ws.numel(),
                              _stream())
    return _done(rc, check)
