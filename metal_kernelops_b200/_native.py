"""ctypes binding of the in-tree C-ABI library ``libssm_b200.so``.

The structs mirror ``include/ssm_b200.h`` field for field.  There is no
fallback: if the library is missing or a CUDA tensor reaches an op without it,
the op raises.  The library itself loads without a GPU (it links only the CUDA
runtime), so the CPU test suite can check its exported symbols.
"""

from __future__ import annotations

import ctypes
import pathlib
import threading

import torch

LIB_PATH = pathlib.Path(__file__).resolve().parent / "libssm_b200.so"

SSM_OK, SSM_ERR_INVALID, SSM_ERR_UNSUPPORTED, SSM_ERR_CUDA, SSM_ERR_WORKSPACE = range(5)
SSM_F32, SSM_BF16, SSM_F16 = 0, 1, 2

HAS_D = 0x01
HAS_Z = 0x02
HAS_BIAS = 0x04
SOFTPLUS = 0x08
D_PER_HEAD = 0x10
DT_PER_ROW = 0x20
HAS_INIT = 0x40
HAS_DY = 0x80
HAS_DSTATE = 0x100
CUDA_CORES = 0x200
CONV_SILU = 0x400
IO_DTYPE = 0x800
CHANNEL_LAST = 0x1000
SCAN_PLAIN = 0x2000
SCAN_LEAN = 0x4000

EXPORTS = (
    "ssm_status_string", "ssm_last_error",
    "ssm_selective_scan_sizes", "ssm_selective_scan_fwd", "ssm_selective_scan_bwd",
    "ssm_selective_scan_fwd_workspace",
    "ssm_state_update_sizes", "ssm_state_update_fwd", "ssm_state_update_bwd",
    "ssm_state_update_bwd_noalloc",
    "ssm_chunk_scan_sizes", "ssm_chunk_scan_fwd", "ssm_chunk_scan_bwd",
    "ssm_take_kernel_error", "ssm_selftest_bounded_wait",
    "ssm_ss2d_scan_sizes", "ssm_ss2d_scan_fwd", "ssm_ss2d_scan_bwd",
    "ssm_causal_conv1d_sizes", "ssm_causal_conv1d_fwd", "ssm_causal_conv1d_bwd",
    "ssm_causal_conv1d_update",
    "ssm_gated_rmsnorm_sizes", "ssm_gated_rmsnorm_fwd", "ssm_gated_rmsnorm_bwd",
    "ssm_add_rmsnorm_sizes", "ssm_add_rmsnorm_fwd", "ssm_add_rmsnorm_bwd", "ssm_quantize_int8",
    "ssm_gated_recurrence_sizes", "ssm_gated_recurrence_fwd", "ssm_gated_recurrence_bwd",
    "ssm_gated_recurrence_step", "ssm_int8_linear_sizes", "ssm_int8_linear_fwd",
)

_I64, _I32, _U32, _P, _SZ = ctypes.c_int64, ctypes.c_int32, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_size_t


class SelectiveScanParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("dim", _I64), ("length", _I64), ("groups", _I64), ("dstate", _I64),
        ("act_dtype", _I32), ("bc_dtype", _I32), ("flags", _U32),
        ("u", _P), ("delta", _P), ("A", _P), ("B", _P), ("C", _P),
        ("D", _P), ("z", _P), ("delta_bias", _P),
        ("y", _P), ("checkpoints", _P),
        ("dout", _P), ("du", _P), ("ddelta", _P), ("dz", _P),
        ("dA", _P), ("dB", _P), ("dC", _P), ("dD", _P), ("ddelta_bias", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("status", _P),
    ]


class StateUpdateParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("nheads", _I64), ("headdim", _I64), ("dstate", _I64), ("ngroups", _I64),
        ("dtype", _I32), ("flags", _U32),
        ("state", _P), ("x", _P), ("dt", _P), ("A", _P), ("B", _P), ("C", _P),
        ("D", _P), ("z", _P), ("dt_bias", _P),
        ("new_state", _P), ("y", _P),
        ("dy", _P), ("dnew", _P),
        ("grad_state", _P), ("dx", _P), ("ddt", _P), ("dA", _P), ("dB", _P), ("dC", _P),
        ("dD", _P), ("dz", _P), ("ddt_bias", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("io_dtype", _I32),
        ("status", _P),
    ]


class ChunkScanParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("length", _I64), ("nheads", _I64), ("headdim", _I64),
        ("ngroups", _I64), ("dstate", _I64), ("chunk_size", _I64),
        ("dtype", _I32), ("dt_dtype", _I32), ("flags", _U32),
        ("x", _P), ("dt", _P), ("A", _P), ("B", _P), ("C", _P), ("D", _P), ("z", _P),
        ("dt_bias", _P), ("initial_states", _P),
        ("y", _P), ("final_state", _P),
        ("dy", _P), ("dfinal", _P),
        ("dx", _P), ("ddt", _P), ("dA", _P), ("dB", _P), ("dC", _P), ("dD", _P), ("dz", _P),
        ("ddt_bias", _P), ("dinitial", _P),
        ("saved", _P), ("workspace", _P), ("workspace_bytes", _SZ),
        ("x_token_stride", _I64), ("bc_token_stride", _I64),
        ("status", _P),
    ]


class Ss2dScanParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("channels", _I64), ("height", _I64), ("width", _I64),
        ("groups", _I64), ("dstate", _I64),
        ("act_dtype", _I32), ("bc_dtype", _I32), ("scale", ctypes.c_float),
        ("u", _P), ("dt", _P), ("A", _P), ("B", _P), ("C", _P),
        ("y", _P), ("checkpoints", _P),
        ("dout", _P), ("du", _P), ("ddt", _P), ("dA", _P), ("dB", _P), ("dC", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("status", _P),
    ]


class CausalConv1dParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("channels", _I64), ("length", _I64), ("width", _I64),
        ("dtype", _I32), ("flags", _U32),
        ("x", _P), ("weight", _P), ("bias", _P), ("initial_state", _P),
        ("out", _P), ("final_state", _P),
        ("dout", _P), ("dx", _P), ("dweight", _P), ("dbias", _P), ("dinitial", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("x_row_stride", _I64), ("dout_row_stride", _I64),
        ("status", _P),
    ]


class CausalConv1dUpdateParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("channels", _I64), ("length", _I64), ("width", _I64), ("state_len", _I64),
        ("state_stride_batch", _I64), ("state_stride_channel", _I64),
        ("dtype", _I32), ("flags", _U32),
        ("state", _P), ("x", _P), ("weight", _P), ("bias", _P), ("out", _P),
        ("status", _P),
    ]


class GatedRmsNormParams(ctypes.Structure):
    _fields_ = [
        ("rows", _I64), ("features", _I64), ("group_size", _I64),
        ("dtype", _I32), ("gate", _I32), ("flags", _U32), ("eps", ctypes.c_float),
        ("x", _P), ("z", _P), ("weight", _P), ("bias", _P), ("out", _P), ("rstd", _P),
        ("dy", _P), ("dx", _P), ("dz", _P), ("dweight", _P), ("dbias", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("x_row_stride", _I64), ("z_row_stride", _I64),
        ("status", _P),
    ]


class AddRmsNormParams(ctypes.Structure):
    _fields_ = [
        ("rows", _I64), ("features", _I64),
        ("x_row_stride", _I64), ("residual_row_stride", _I64), ("dy_row_stride", _I64), ("dstream_row_stride", _I64),
        ("dtype", _I32), ("stream_dtype", _I32), ("weight_dtype", _I32), ("eps", ctypes.c_float),
        ("x", _P), ("residual", _P), ("weight", _P), ("stream", _P), ("y", _P), ("q", _P), ("scale", _P),
        ("rstd", _P),
        ("dy", _P), ("dstream", _P), ("dx", _P), ("dresidual", _P), ("dweight", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("status", _P),
    ]


class Int8LinearParams(ctypes.Structure):
    _fields_ = [
        ("tokens", _I64), ("in_features", _I64), ("out_features", _I64),
        ("x_row_stride", _I64), ("w_row_stride", _I64),
        ("out_dtype", _I32), ("flags", _U32),
        ("x", _P), ("x_scale", _P), ("w", _P), ("w_scale", _P), ("bias", _P), ("out", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("status", _P),
    ]


class GatedRecurrenceParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("length", _I64), ("dim", _I64),
        ("x_token_stride", _I64), ("x_batch_stride", _I64),
        ("forget_token_stride", _I64), ("forget_batch_stride", _I64),
        ("z_token_stride", _I64), ("z_batch_stride", _I64),
        ("dy_token_stride", _I64), ("dy_batch_stride", _I64),
        ("dtype", _I32), ("flags", _U32),
        ("x", _P), ("forget", _P), ("z", _P), ("lower", _P), ("initial_state", _P), ("reset", _P),
        ("y", _P), ("final_state", _P), ("states", _P),
        ("dy", _P), ("dfinal", _P), ("dx", _P), ("dforget", _P), ("dz", _P), ("dlower", _P), ("dinitial", _P),
        ("workspace", _P), ("workspace_bytes", _SZ),
        ("status", _P),
    ]


class GatedRecurrenceStepParams(ctypes.Structure):
    _fields_ = [
        ("batch", _I64), ("dim", _I64),
        ("x_batch_stride", _I64), ("forget_batch_stride", _I64), ("z_batch_stride", _I64),
        ("state_batch_stride", _I64),
        ("dtype", _I32), ("flags", _U32),
        ("x", _P), ("forget", _P), ("z", _P), ("lower", _P), ("state", _P), ("y", _P),
        ("status", _P),
    ]


_lib = None
_lock = threading.Lock()


def lib():
    """The loaded library; raises if it was not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise RuntimeError(
                    f"{LIB_PATH.name} is not built; run `python -m metal_kernelops_b200.build` "
                    "(there is no CPU fallback)")
            handle = ctypes.CDLL(str(LIB_PATH))
            handle.ssm_status_string.restype = ctypes.c_char_p
            handle.ssm_status_string.argtypes = [ctypes.c_int]
            handle.ssm_last_error.restype = ctypes.c_char_p
            handle.ssm_last_error.argtypes = []
            for name, struct in (("selective_scan", SelectiveScanParams),
                                 ("state_update", StateUpdateParams),
                                 ("chunk_scan", ChunkScanParams),
                                 ("ss2d_scan", Ss2dScanParams),
                                 ("causal_conv1d", CausalConv1dParams),
                                 ("gated_rmsnorm", GatedRmsNormParams),
                                 ("add_rmsnorm", AddRmsNormParams),
                                 ("gated_recurrence", GatedRecurrenceParams)):
                for suffix in ("fwd", "bwd"):
                    fn = getattr(handle, f"ssm_{name}_{suffix}")
                    fn.restype = ctypes.c_int
                    fn.argtypes = [ctypes.POINTER(struct), ctypes.c_void_p]
            handle.ssm_selective_scan_sizes.argtypes = [
                ctypes.POINTER(SelectiveScanParams), ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)]
            handle.ssm_state_update_sizes.argtypes = [
                ctypes.POINTER(StateUpdateParams), ctypes.POINTER(_SZ)]
            handle.ssm_chunk_scan_sizes.argtypes = [
                ctypes.POINTER(ChunkScanParams), ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)]
            handle.ssm_causal_conv1d_sizes.argtypes = [ctypes.POINTER(CausalConv1dParams), ctypes.POINTER(_SZ)]
            handle.ssm_gated_rmsnorm_sizes.argtypes = [ctypes.POINTER(GatedRmsNormParams), ctypes.POINTER(_SZ)]
            handle.ssm_add_rmsnorm_sizes.argtypes = [ctypes.POINTER(AddRmsNormParams), ctypes.POINTER(_SZ)]
            handle.ssm_gated_recurrence_sizes.argtypes = [
                ctypes.POINTER(GatedRecurrenceParams), ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)]
            handle.ssm_int8_linear_fwd.restype = ctypes.c_int
            handle.ssm_int8_linear_fwd.argtypes = [ctypes.POINTER(Int8LinearParams), ctypes.c_void_p]
            handle.ssm_int8_linear_sizes.argtypes = [ctypes.POINTER(Int8LinearParams), ctypes.POINTER(_SZ)]
            handle.ssm_gated_recurrence_step.restype = ctypes.c_int
            handle.ssm_gated_recurrence_step.argtypes = [ctypes.POINTER(GatedRecurrenceStepParams),
                                                         ctypes.c_void_p]
            handle.ssm_quantize_int8.restype = ctypes.c_int
            handle.ssm_quantize_int8.argtypes = [ctypes.POINTER(AddRmsNormParams), ctypes.c_void_p]
            handle.ssm_causal_conv1d_update.restype = ctypes.c_int
            handle.ssm_causal_conv1d_update.argtypes = [ctypes.POINTER(CausalConv1dUpdateParams), ctypes.c_void_p]
            handle.ssm_selective_scan_fwd_workspace.argtypes = [
                ctypes.POINTER(SelectiveScanParams), ctypes.POINTER(_SZ)]
            handle.ssm_ss2d_scan_sizes.argtypes = [
                ctypes.POINTER(Ss2dScanParams), ctypes.POINTER(_SZ), ctypes.POINTER(_SZ),
                ctypes.POINTER(_SZ)]
            handle.ssm_state_update_bwd_noalloc.restype = ctypes.c_int
            handle.ssm_state_update_bwd_noalloc.argtypes = [ctypes.POINTER(StateUpdateParams),
                                                            ctypes.c_void_p]
            for name in ("ssm_selective_scan_sizes", "ssm_state_update_sizes", "ssm_chunk_scan_sizes",
                         "ssm_ss2d_scan_sizes", "ssm_selective_scan_fwd_workspace",
                         "ssm_causal_conv1d_sizes", "ssm_gated_rmsnorm_sizes", "ssm_add_rmsnorm_sizes",
                         "ssm_gated_recurrence_sizes", "ssm_int8_linear_sizes"):
                getattr(handle, name).restype = ctypes.c_int
            handle.ssm_take_kernel_error.restype = ctypes.c_int
            handle.ssm_take_kernel_error.argtypes = []
            handle.ssm_selftest_bounded_wait.restype = ctypes.c_int
            handle.ssm_selftest_bounded_wait.argtypes = [ctypes.c_void_p, ctypes.c_uint32, ctypes.c_void_p]
            _lib = handle
    return _lib


class NativeError(RuntimeError):
    pass


def check(status: int, what: str) -> None:
    """Map a C-ABI status to the reference's error convention: contract
    violations are ``ValueError``, everything else ``RuntimeError``."""
    if status == SSM_OK:
        return
    L = lib()
    msg = L.ssm_last_error().decode() or L.ssm_status_string(status).decode()
    if status in (SSM_ERR_INVALID, SSM_ERR_UNSUPPORTED):
        raise ValueError(f"{what}: {msg}")
    raise NativeError(f"{what}: {msg} (status {status})")


_DTYPES = {torch.float32: SSM_F32, torch.bfloat16: SSM_BF16, torch.float16: SSM_F16}


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPES[dtype]


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_of(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def like(t: torch.Tensor, shape, dtype) -> torch.Tensor:
    """A dense tensor of ``shape`` (t's, or its rows) and ``dtype`` on t's device:
    ``empty_like`` takes half of ``torch.empty``'s 3 us."""
    if t.shape == shape and t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(shape, dtype=dtype, device=t.device)


def vector(n: int, t: torch.Tensor) -> torch.Tensor:
    """n float32 values on t's device."""
    return torch.empty_strided((n,), (1,), dtype=torch.float32, device=t.device)


def matrix(m: int, n: int, dtype, t: torch.Tensor) -> torch.Tensor:
    """A dense (m, n) tensor on t's device."""
    return torch.empty_strided((m, n), (n, 1), dtype=dtype, device=t.device)


def stream_here(t: torch.Tensor) -> int:
    """The current stream's handle on t's device (as :func:`stream_of`, without
    the 2 us of building a Stream object)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def same_device(name: str, index: int, named) -> None:
    """Raise ``ValueError`` unless every tensor of ``named`` is on CUDA device ``index``
    (negative: the first one is not on a GPU).  Called when a quick look found one that is not."""
    for label, t in named:
        if t is not None and (index < 0 or t.get_device() != index):
            if not t.is_cuda:
                raise ValueError(f"{name} runs CUDA kernels, {label} is on {t.device}")
            raise ValueError(f"{name}: {label} is on {t.device}, {named[0][0]} is on {named[0][1].device}")


def apart(index: int, *tensors) -> bool:
    """Whether one of the tensors is not on CUDA device ``index``."""
    if index < 0:
        return True
    for t in tensors:
        if t is not None and t.get_device() != index:
            return True
    return False


def direct(*tensors) -> bool:
    """Whether a call may go to the library itself (with a gradient: through a
    ``torch.autograd.Function``) instead of the custom op of torch's dispatcher:
    the tensors are plain ones (no fake or other subclass) on the current
    device, and nothing has to see the call as an operator: ``torch.compile``,
    ``torch.jit.trace``, a dispatch mode (``make_fx``, fake tensors, logging and
    counting modes) or a functorch transform (``vmap``).  Their tensors may look plain,
    and a launch beside the dispatcher would leave them with memory that the
    recorded program never writes.  The dispatcher's Python path costs about 15 us
    a call, more than the kernels of a decode step run for."""
    for t in tensors:
        if t is not None and type(t) is not torch.Tensor and type(t) is not torch.nn.Parameter:
            return False
    return not (_is_compiling() or _is_tracing() or _dispatch_modes() or _functorch_level() is not None) \
        and tensors[0].get_device() == torch._C._cuda_getDevice()


_is_compiling = torch.compiler.is_compiling
_is_tracing = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack
_functorch_level = torch._C._functorch.maybe_current_level


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# --------------------------------------------------------------- status words --
# One int32 device word per op family and device, zero-initialised once from
# the caching allocator and handed to every call of that op (params.status).
# A kernel that gives up on a bounded wait writes its code there; nothing is
# cleared until ``check_errors`` reads the words.  Reading is lazy -- one small
# device-to-host copy when the caller asks -- so the ops never synchronise.
STATUS_SLOTS = ("selective_scan", "state_update", "chunk_scan", "ss2d_scan", "causal_conv1d",
                "causal_conv1d_update", "gated_rmsnorm", "selftest", "add_rmsnorm", "int8_linear", "gated_recurrence")
_SLOT_BYTES = {op: 4 * i for i, op in enumerate(STATUS_SLOTS)}
_status = {}


def _status_buffer(device: torch.device) -> torch.Tensor:
    key = device.index if device.index is not None else torch.cuda.current_device()
    buf = _status.get(key)
    if buf is None:
        buf = torch.zeros(len(STATUS_SLOTS), dtype=torch.int32, device=torch.device("cuda", key))
        _status[key] = buf
    return buf


def status_word(device: torch.device, op: str) -> int:
    """Device address of ``op``'s status word on ``device`` (for params.status)."""
    return _status_buffer(device).data_ptr() + _SLOT_BYTES[op]


def check_errors(device=None) -> None:
    """Read the status words of ``device`` (every device used so far when
    None), clear them, and raise ``RuntimeError`` if a kernel gave up on a
    bounded wait since the last check.  Synchronises with those devices."""
    keys = list(_status) if device is None else [torch.device(device).index or 0]
    failed = []
    for key in keys:
        buf = _status.get(key)
        if buf is None:
            continue
        vals = buf.cpu().tolist()
        if any(vals):
            buf.zero_()
            failed += [f"{op} (code {v}) on cuda:{key}" for op, v in zip(STATUS_SLOTS, vals) if v]
    if failed:
        raise NativeError("a kernel gave up on a bounded wait; its outputs are invalid: " + ", ".join(failed))


def selftest_bounded_wait(device=None, polls: int = 16) -> None:
    """Launch the library's failure-path self-test on ``device``: a wait on an
    mbarrier that nothing completes, limited to ``polls`` polls, which gives
    up and writes its code into the self-test status word."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        check(lib().ssm_selftest_bounded_wait(ctypes.c_void_p(status_word(dev, "selftest")),
                                              ctypes.c_uint32(polls), stream), "selftest_bounded_wait")
