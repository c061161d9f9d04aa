"""reef_amd: int8 attention for AMD MI355X behind the reef_hip C ABI.

Host-side mirror of the Reef engine's quantization and attention operators
(inference-engine/reference/cpp/include/inference_engine/quant.hpp and
operator/attention.hpp), running on the HIP kernels of libreef_hip.so through
its C ABI (include/reef_hip/attention.h). Tensors are torch tensors on the GPU;
torch only provides device memory and the current stream. There is no CPU
fallback: without the built library every call raises.

Errors follow the engine: shape and argument errors raise InvalidArgument (a
ValueError, as the engine's std::invalid_argument), non-finite input raises
NonFiniteInput (also a ValueError, quant.hpp:72-74), cache capacity raises
CapacityError (an IndexError, the engine's std::length_error).
"""
from __future__ import annotations

import ctypes as C
import math
import os
import struct

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "libreef_hip.so")

OK, INVALID_ARGUMENT, NON_FINITE_INPUT, CAPACITY, HIP_ERROR, UNSUPPORTED, OVERFLOW = range(7)
PER_TENSOR, PER_HEAD, PER_TOKEN = 0, 1, 2
ATTN_PRECISE_PV = 0x1
# prefill schedules (reef_attention_params.flags bits 4-6)
SCHED_AUTO, SCHED_ONE_ITEM, SCHED_SPLIT, SCHED_BALANCED, SCHED_PACKED = (0x00, 0x10, 0x20,
                                                                         0x30, 0x40)
PAGE = 16
# epilogues of the W8A8 product (reef_activation)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu_tanh": 2, "gelu_erf": 3, "silu": 4}

EXPORTS = [
    "reef_quantize_int8_per_tensor", "reef_quantize_int8_per_head",
    "reef_quantize_int8_per_token", "reef_quantize_int8_per_token_heads",
    "reef_dequantize_int8", "reef_read_status_word",
    "reef_attention_prefill_workspace_bytes", "reef_attention_prefill_int8", "reef_qk_scores_i32",
    "reef_qk_scores_i32_packed_workspace_bytes", "reef_qk_scores_i32_packed",
    "reef_attention_decode_workspace_bytes", "reef_attention_decode_int8",
    "reef_attention_decode_int8_paged", "reef_attention_decode_int8_paged_noalloc",
    "reef_kv_pack_v_pages", "reef_kv_append_int8",
    "reef_kv_append_int8_paged", "reef_attention_int8_integer", "reef_linear_w8a8_workspace_bytes",
    "reef_linear_w8a8", "reef_gemm_w8a8", "reef_linear_w8a8_epilogue", "reef_gemm_w8a8_epilogue",
    "reef_rmsnorm_quantize_int8", "reef_kv_free", "reef_kv_fork",
    "reef_kv_reserve_workspace_bytes", "reef_kv_reserve", "reef_kv_compact_workspace_bytes",
    "reef_attention_decode_tree_workspace_bytes", "reef_attention_decode_tree_int8",
    "reef_attention_decode_tree_int8_paged",
    "reef_kv_compact", "reef_kv_copy_pages", "reef_kv_keep_int8", "reef_kv_keep_int8_paged",
    "reef_attention_prefill_cache_workspace_bytes",
    "reef_attention_prefill_int8_cache",
]


class ReefError(RuntimeError):
    pass


class InvalidArgument(ReefError, ValueError):
    pass


class NonFiniteInput(ReefError, ValueError):
    pass


class CapacityError(ReefError, IndexError):
    pass


class HipError(ReefError):
    pass


class Unsupported(ReefError, NotImplementedError):
    pass


class Overflow(ReefError, OverflowError):
    pass


_ERRORS = {INVALID_ARGUMENT: InvalidArgument, NON_FINITE_INPUT: NonFiniteInput,
           CAPACITY: CapacityError, HIP_ERROR: HipError, UNSUPPORTED: Unsupported,
           OVERFLOW: Overflow}


class Strides(C.Structure):
    _fields_ = [("batch", C.c_int64), ("head", C.c_int64), ("token", C.c_int64)]


class AttentionParams(C.Structure):
    _fields_ = [("batch", C.c_int64), ("q_heads", C.c_int64), ("kv_heads", C.c_int64),
                ("q_len", C.c_int64), ("kv_len", C.c_int64), ("head_dim", C.c_int64),
                ("query_start", C.c_int64), ("window", C.c_int64),
                ("softmax_scale", C.c_float), ("q_granularity", C.c_int32),
                ("kv_granularity", C.c_int32), ("flags", C.c_uint32)]


class DecodeParams(C.Structure):
    _fields_ = [("batch", C.c_int64), ("q_heads", C.c_int64), ("kv_heads", C.c_int64),
                ("head_dim", C.c_int64), ("max_context", C.c_int64), ("window", C.c_int64),
                ("softmax_scale", C.c_float), ("q_granularity", C.c_int32),
                ("num_splits", C.c_int32), ("flags", C.c_uint32)]


class KvAppendParams(C.Structure):
    _fields_ = [("batch", C.c_int64), ("kv_heads", C.c_int64), ("head_dim", C.c_int64),
                ("new_tokens", C.c_int64), ("max_context", C.c_int64)]


class TreeParams(C.Structure):
    _fields_ = [("batch", C.c_int64), ("q_heads", C.c_int64), ("kv_heads", C.c_int64),
                ("head_dim", C.c_int64), ("draft_len", C.c_int64), ("max_context", C.c_int64),
                ("window", C.c_int64), ("softmax_scale", C.c_float), ("q_granularity", C.c_int32),
                ("flags", C.c_uint32), ("reserved", C.c_uint32)]


class Epilogue(C.Structure):
    _fields_ = [("residual", C.c_void_p), ("residual_row_stride", C.c_int64),
                ("activation", C.c_int64)]


_P = C.c_void_p
_I64 = C.c_int64
_ST, _AP = C.POINTER(Strides), C.POINTER(AttentionParams)
_DP, _KP = C.POINTER(DecodeParams), C.POINTER(KvAppendParams)
_EP, _TP = C.POINTER(Epilogue), C.POINTER(TreeParams)
_SIGS = {
    "reef_quantize_int8_per_tensor": [_P, _I64, _P, _P, _P, _P],
    "reef_quantize_int8_per_head": [_P, _I64, _I64, _I64, _I64, _ST, _P, _P, _P, _P],
    "reef_quantize_int8_per_token": [_P, _I64, _I64, _I64, _P, _P, _P, _P],
    "reef_quantize_int8_per_token_heads": [_P, _I64, _I64, _I64, _I64, _ST, _P, _P, _P, _P],
    "reef_dequantize_int8": [_P, _I64, _I64, _P, _P, _P],
    "reef_read_status_word": [_P, C.c_int, _P],
    "reef_attention_prefill_workspace_bytes": [_AP],
    "reef_attention_prefill_int8": [_AP, _P, _ST, _P, _ST, _P, _ST, _P, _P, _P, _P, _ST, _P,
                                    C.c_size_t, _P],
    "reef_qk_scores_i32": [_P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _P, _P],
    "reef_qk_scores_i32_packed_workspace_bytes": [_I64, _I64, _I64, _I64, _I64],
    "reef_qk_scores_i32_packed": [_P, _P, _I64, _I64, _I64, _I64, _I64, _P, _P, C.c_size_t, _P],
    "reef_attention_decode_workspace_bytes": [_DP],
    "reef_attention_decode_int8": [_DP, _P, _P, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, _P,
                                   _P],
    "reef_attention_decode_int8_paged": [_DP, _P, _P, _P, _P, _P, _P, _P,
                                         _I64, _I64, _P, _P, _P, C.c_size_t, _P, _P],
    "reef_attention_decode_int8_paged_noalloc": [_DP, _P, _P, _P, _P, _P, _P,
                                                 _P, _I64, _I64, _P, _P, _P, _P],
    "reef_kv_pack_v_pages": [_P, _I64, _I64, _P, _P],
    "reef_linear_w8a8_workspace_bytes": [_I64, _I64],
    "reef_linear_w8a8": [_P, _I64, _I64, _I64, _P, _P, _P, _I64, _P, _I64, _P, C.c_size_t, _P,
                         _P],
    "reef_gemm_w8a8": [_P, _P, _I64, _I64, _P, _P, _P, _I64, _P, _I64, _P, _P],
    "reef_linear_w8a8_epilogue": [_P, _I64, _I64, _I64, _P, _P, _P, _EP, _I64, _P, _I64, _P,
                                  C.c_size_t, _P, _P],
    "reef_gemm_w8a8_epilogue": [_P, _P, _I64, _I64, _P, _P, _P, _EP, _I64, _P, _I64, _P, _P],
    "reef_rmsnorm_quantize_int8": [_P, _I64, _I64, _I64, _P, _I64, _P, C.c_double, _P, _P, _P,
                                   _I64, _P, _P],
    "reef_attention_int8_integer": [_AP, _P, _ST, _P, _ST, _P, _ST, C.c_uint32, _P, C.c_uint32,
                                    _P, _ST, _P],
    "reef_kv_append_int8": [_KP, _P, _ST, _P, _ST, _P, _P, _P, _P, _P, _P, _P, _P],
    "reef_kv_append_int8_paged": [_KP, _P, _ST, _P, _ST, _P, _P, _I64, _I64, _P, _P, _P, _P, _P,
                                  _P, _P],
    "reef_attention_decode_tree_workspace_bytes": [_TP],
    "reef_attention_decode_tree_int8": [_TP, _P, _ST, _P, _P, _P, _P, _P, _P, _P, _P, _ST, _P,
                                        C.c_size_t, _P, _P],
    "reef_attention_decode_tree_int8_paged": [_TP, _P, _ST, _P, _P, _P, _P, _P, _P, _I64, _I64,
                                              _P, _P, _P, _ST, _P, C.c_size_t, _P, _P],
    "reef_kv_free": [_P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _P],
    "reef_kv_fork": [_P, _P, _I64, _P, _I64, _P, _I64, _P, _I64, _P, _P],
    "reef_kv_reserve_workspace_bytes": [_I64, _I64],
    "reef_kv_reserve": [_P, _I64, _P, _I64, _I64, _P, _I64, _P, _P, _P, C.c_size_t, _P, _P],
    "reef_kv_compact_workspace_bytes": [_I64],
    "reef_kv_compact": [_P, _I64, _I64, _P, _I64, _P, _P, _P, _P, C.c_size_t, _P, _P],
    "reef_kv_copy_pages": [_P, _P, _I64, _I64, _I64, _P, _P, _P, _P, _I64, _P, _P],
    "reef_kv_keep_int8": [_KP, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P],
    "reef_kv_keep_int8_paged": [_KP, _P, _P, _P, _P, _I64, _I64, _P, _P, _P, _P, _P, _P, _P],
    "reef_attention_prefill_cache_workspace_bytes": [_AP],
    "reef_attention_prefill_int8_cache": [_AP, _P, _ST, _P, _P, _P, _P, _P, _I64, _P, _I64, _I64,
                                          _P, _ST, _P, C.c_size_t, _P, _P],
}

_lib_handle = _plain_handle = None


def _load(plain: bool) -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build it with python -m reef_amd._build")
    handle = C.CDLL(LIB_PATH)
    for name, args in _SIGS.items():
        fn = getattr(handle, name)
        fn.argtypes = [_P if plain and issubclass(t, C._Pointer) else t for t in args]
        fn.restype = C.c_size_t if name.endswith("_bytes") else C.c_int
    return handle


def lib() -> C.CDLL:
    """The loaded libreef_hip.so. Raises if it has not been built."""
    global _lib_handle
    if _lib_handle is None:
        _lib_handle = _load(plain=False)
    return _lib_handle


def _lib() -> C.CDLL:
    """The same library with structures as plain addresses, for the wrappers below."""
    global _plain_handle
    if _plain_handle is None:
        _plain_handle = _load(plain=True)
    return _plain_handle


def check(status: int, what: str) -> None:
    if status != OK:
        raise _ERRORS.get(status, ReefError)(f"{what}: reef status {status}")


# --- torch plumbing -------------------------------------------------------------------

# The wrappers below run once per layer and token of a serving loop, so the small calls are
# bound by this file: arguments go to the library as plain addresses and packed bytes
# (a ctypes structure costs four times its bytes), and the stream is read as a handle
# rather than through a torch.cuda.Stream (a 1x1x128x64 prefill: 11.4 us a call against
# 20.5, of which 8 us are the kernel's).

_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def _stream():
    """The current device's current stream, as an address."""
    c = _torch()._C
    try:
        return c._cuda_getCurrentRawStream(c._cuda_getDevice())
    except AttributeError:
        return _torch().cuda.current_stream().cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _packed(layout, structure, *fields):
    """The bytes of `structure` (whose members `layout` gives) for the library to read."""
    try:
        return layout.pack(*fields)
    except (struct.error, OverflowError):  # a value outside its member's range
        return C.byref(structure(*fields))


_STRIDES = struct.Struct("=3q")
_ATTENTION = struct.Struct("=8qf2iI")
_DECODE = struct.Struct("=6qf2iI")
_APPEND = struct.Struct("=5q")
_EPILOGUE = struct.Struct("=3q")
_TREE = struct.Struct("=7qfi2I")


def _require(t, dtype, name):
    torch = _torch()
    if isinstance(t, torch.Tensor) and t.is_cuda:
        if t.dtype == dtype:
            return
        raise InvalidArgument(f"{name} must be {dtype}, got {t.dtype}")
    raise InvalidArgument(f"{name} must be a GPU tensor")


def _expect(what, dtype, *tensors):
    """(tensor, name) pairs: contiguous, of one type, on the current device, whose stream the
    call takes."""
    device = None
    for t, name in tensors:
        try:
            if t.dtype is dtype and t.is_cuda and t.is_contiguous():
                if device is None:
                    device = _torch()._C._cuda_getDevice()
                if t.get_device() == device:
                    continue
        except AttributeError:
            pass
        _require(t, dtype, name)
        raise InvalidArgument(f"{what}: {name} must be contiguous and on the current GPU")


def _on_device(what, *tensors):
    """Every tensor (None: absent) lies on the current device, whose stream the call takes."""
    device = _torch()._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise InvalidArgument(f"{what}: every tensor must be on the current GPU")


def _strides4(t):
    """Strides of a [B, H, S, D] tensor with a contiguous last dimension."""
    st = t.stride()
    if len(st) != 4 or st[3] != 1:
        raise InvalidArgument("expected [batch, heads, tokens, head_dim] with contiguous head_dim")
    return _STRIDES.pack(st[0], st[1], st[2])


class StatusWord:
    """A device status word the kernels flag non-finite input and bad pages in."""

    def __init__(self, device=None):
        torch = _torch()
        self.tensor = torch.zeros(1, dtype=torch.int32, device=device or "cuda")

    @property
    def ptr(self):
        return C.c_void_p(self.tensor.data_ptr())

    def check(self, what: str) -> None:
        check(_lib().reef_read_status_word(self.ptr, 1, _stream()), what)


# --- quantization (quant.hpp) ---------------------------------------------------------

def quantize_per_tensor(x, status: StatusWord | None = None):
    """One scale for the whole tensor (the quant.hpp rule); returns (int8, scale[1])."""
    torch = _torch()
    _require(x, torch.float32, "x")
    x = x.contiguous()
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(1, dtype=torch.float32, device=x.device)
    own = status or StatusWord(x.device)
    check(_lib().reef_quantize_int8_per_tensor(_ptr(x), x.numel(), _ptr(q), _ptr(s), _ptr(own.tensor),
                                              _stream()), "quantize_per_tensor")
    if status is None:
        own.check("quantize_per_tensor requires finite values")
    return q, s


def quantize_per_head(x, status: StatusWord | None = None):
    """x [B, H, S, D] (any strides, contiguous D); one scale per head over batch and
    tokens. Returns packed int8 [B, H, S, D] and scales [H]."""
    torch = _torch()
    _require(x, torch.float32, "x")
    st = _strides4(x)
    B, H, S, D = x.shape
    q = torch.empty((B, H, S, D), dtype=torch.int8, device=x.device)
    s = torch.empty(H, dtype=torch.float32, device=x.device)
    own = status or StatusWord(x.device)
    check(_lib().reef_quantize_int8_per_head(_ptr(x), B, H, S, D, st, _ptr(q), _ptr(s),
                                            _ptr(own.tensor), _stream()), "quantize_per_head")
    if status is None:
        own.check("quantize_per_head requires finite values")
    return q, s


def quantize_rows(x, status: StatusWord | None = None):
    """quantize_rows (quant.hpp:112-133) over the last dimension: one scale per row
    (per token). Returns int8 of x's shape and scales of x.shape[:-1]."""
    torch = _torch()
    _require(x, torch.float32, "x")
    shape = x.shape
    width = shape[-1]
    if len(shape) == 4 and not x.is_contiguous() and x.numel() > 0:
        # heads as a projection lays them out: read in place rather than copied first
        sb, sh, st, sd = x.stride()
        if sd == 1 and (sb | sh | st | width) % 4 == 0 and width <= 1024 and x.data_ptr() % 16 == 0:
            q = torch.empty(shape, dtype=torch.int8, device=x.device)
            s = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
            own = status or StatusWord(x.device)
            ret = _lib().reef_quantize_int8_per_token_heads(
                _ptr(x), *shape, _STRIDES.pack(sb, sh, st), _ptr(q), _ptr(s), _ptr(own.tensor),
                _stream())
            if ret != UNSUPPORTED:  # 2^31 rows or more are copied
                check(ret, "quantize_rows")
                if status is None:
                    own.check("quantize_rows requires finite values")
                return q, s
            del q, s
    x2 = x if len(shape) == 2 else x.reshape(-1, width)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    rows = x2.shape[0]
    q = torch.empty(shape, dtype=torch.int8, device=x.device)
    s = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    own = status or StatusWord(x.device)
    check(_lib().reef_quantize_int8_per_token(_ptr(x2), rows, width, x2.stride(0), _ptr(q),
                                             _ptr(s), _ptr(own.tensor), _stream()), "quantize_rows")
    if status is None:
        own.check("quantize_rows requires finite values")
    return q, s


quantize_per_token = quantize_rows


def dequantize(q, scales, group: int):
    """x[i] = float(q[i]) * scales[i // group]."""
    torch = _torch()
    _require(q, torch.int8, "q")
    _require(scales, torch.float32, "scales")
    q = q.contiguous()
    x = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    scales = scales.contiguous()
    check(_lib().reef_dequantize_int8(_ptr(q), q.numel(), group, _ptr(scales), _ptr(x),
                                     _stream()), "dequantize")
    return x


# --- attention ------------------------------------------------------------------------

_PREFILL_WS = {}


def prefill_workspace(params: AttentionParams, device):
    """The zero-filled workspace of the balanced prefill schedule, one per (device,
    stream): every launch leaves it zero-filled, so the next launch on that stream
    reuses it."""
    n = lib().reef_attention_prefill_workspace_bytes(C.byref(params))
    return _prefill_workspace(n, _torch().device(device), _stream())


def _prefill_workspace(n, device, stream):
    key = (device.index, stream)
    ws = _PREFILL_WS.get(key)
    if ws is None or ws.numel() < n:
        torch = _torch()
        ws = torch.zeros(max(n, 256), dtype=torch.uint8, device=device)
        _PREFILL_WS[key] = ws
    return ws


def attention_prefill(q, k, v, q_scales, k_scales, v_scales, *, query_start=None, window=0,
                      softmax_scale=None, q_granularity=PER_HEAD, kv_granularity=PER_HEAD,
                      precise=False, schedule=SCHED_AUTO, out=None, workspace=None):
    """Attention::context (attention.hpp:374-432) over int8 heads in one launch.

    q [B, Hq, Sq, D], k and v [B, Hkv, Skv, D] int8 (contiguous head_dim, any other
    strides); scales by granularity. softmax_scale defaults to 1/sqrt(D); pass 1.0
    for the engine's unscaled scores. Returns fp32 [B, Hq, Sq, D]. schedule is one
    of the SCHED_* flags (SCHED_AUTO: the library's choice). workspace: None takes
    this stream's cached one (prefill_workspace), False passes none, or a
    zero-filled uint8 tensor of reef_attention_prefill_workspace_bytes bytes.
    """
    torch = _torch()
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _require(t, torch.int8, n)
    for t, n in ((q_scales, "q_scales"), (k_scales, "k_scales"), (v_scales, "v_scales")):
        _require(t, torch.float32, n)
    B, Hq, Sq, D = q.shape
    _, Hkv, Skv, _ = k.shape
    if tuple(v.shape) != tuple(k.shape) or k.shape[0] != B or k.shape[3] != D:
        raise InvalidArgument("attention_prefill shape mismatch")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    start = Skv - Sq if query_start is None else query_start
    p = _packed(_ATTENTION, AttentionParams, B, Hq, Hkv, Sq, Skv, D, start, window, softmax_scale,
                q_granularity, kv_granularity, (ATTN_PRECISE_PV if precise else 0) | schedule)
    device = q.device
    if out is None:
        out = torch.empty((B, Hq, Sq, D), dtype=torch.float32, device=device)
    qs, ks, vs, os_ = _strides4(q), _strides4(k), _strides4(v), _strides4(out)
    stream = _stream()
    if workspace is None:
        n = _lib().reef_attention_prefill_workspace_bytes(p)
        workspace = _prefill_workspace(n, device, stream)
    ws_ptr, ws_n = (None, 0) if workspace is False else (_ptr(workspace), workspace.numel()
                                                          * workspace.element_size())
    # (named, so that a copy that contiguous() makes lives until the launch is queued)
    q_scales, k_scales, v_scales = (q_scales.contiguous(), k_scales.contiguous(),
                                    v_scales.contiguous())
    check(_lib().reef_attention_prefill_int8(
        p, _ptr(q), qs, _ptr(k), ks, _ptr(v), vs, _ptr(q_scales), _ptr(k_scales), _ptr(v_scales),
        _ptr(out), os_, ws_ptr, ws_n, stream), "attention_prefill")
    return out


def attention_prefill_cache(q, q_scales, k_cache, v_cache, k_scales, v_scales, kv_len, *,
                            block_table=None, query_start=None, window=0, softmax_scale=None,
                            q_granularity=PER_HEAD, status: StatusWord | None = None, out=None):
    """A prompt chunk over the int8 cache (Attention::forward with query_len > 1 on a
    non-empty cache, attention.hpp:354-372): the cache already holds the chunk's
    keys (kv_append), kv_len tokens per sequence. Contiguous cache (block_table
    None): k_cache [B, Hkv, L, D], v_cache [B, Hkv, L/16, D, 16] (or the same bytes
    in any shape), scales [B, Hkv, L]. Paged: k_cache [P, Hkv, 16, D], v_cache
    [P, Hkv, D, 16], scales [P, Hkv, 16], block_table [B, max_blocks] int32.
    q [B, Hq, q_len, D] int8; returns fp32 [B, Hq, q_len, D]."""
    torch = _torch()
    _require(q, torch.int8, "q")
    B, Hq, Sq, D = q.shape
    Hkv = k_cache.shape[1]
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    start = kv_len - Sq if query_start is None else query_start
    p = _packed(_ATTENTION, AttentionParams, B, Hq, Hkv, Sq, kv_len, D, start, window,
                softmax_scale, q_granularity, PER_TOKEN, 0)
    if block_table is None:
        max_context, table, max_blocks, pages = k_cache.shape[2], None, 0, 0
    else:
        max_context, table = 0, block_table.contiguous()
        max_blocks, pages = table.shape[1], k_cache.shape[0]
    n = _lib().reef_attention_prefill_cache_workspace_bytes(p)
    device, stream = q.device, _stream()
    key = ("cache", device.index, stream)
    ws = _PREFILL_WS.get(key)
    if ws is None or ws.numel() < n:  # zero-filled once; every call leaves it so
        ws = torch.zeros(max(n, 256), dtype=torch.uint8, device=device)
        _PREFILL_WS[key] = ws
    if out is None:
        out = torch.empty((B, Hq, Sq, D), dtype=torch.float32, device=q.device)
    qs, os_ = _strides4(q), _strides4(out)
    own = status or StatusWord(q.device)
    q_scales, k_cache, v_cache = q_scales.contiguous(), k_cache.contiguous(), v_cache.contiguous()
    k_scales, v_scales = k_scales.contiguous(), v_scales.contiguous()
    check(_lib().reef_attention_prefill_int8_cache(
        p, _ptr(q), qs, _ptr(q_scales), _ptr(k_cache), _ptr(v_cache), _ptr(k_scales),
        _ptr(v_scales), max_context, _ptr(table), max_blocks, pages, _ptr(out), os_, _ptr(ws), n,
        _ptr(own.tensor), stream), "attention_prefill_cache")
    if status is None:
        own.check("attention_prefill_cache")
    return out


def qk_scores_i32(q, k):
    """int32 q . k^T for packed q [B, Hq, Sq, D] and k [B, Hkv, Skv, D]."""
    torch = _torch()
    _require(q, torch.int8, "q")
    _require(k, torch.int8, "k")
    q = q.contiguous()
    k = k.contiguous()
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    acc = torch.empty((B, Hq, Sq, Skv), dtype=torch.int32, device=q.device)
    check(_lib().reef_qk_scores_i32(_ptr(q), _ptr(k), B, Hq, Hkv, Sq, Skv, D, _ptr(acc),
                                   _stream()), "qk_scores_i32")
    return acc


def qk_scores_i32_packed(q, k):
    """int32 q . k^T for packed q [B, Hq, Sq, 128] and k [B, Hkv, Skv, 128], read from
    the packed prefill kernel's own score accumulators."""
    torch = _torch()
    _require(q, torch.int8, "q")
    _require(k, torch.int8, "k")
    q = q.contiguous()
    k = k.contiguous()
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    if D != 128:
        raise ValueError("the packed score hook takes head_dim 128")
    acc = torch.full((B, Hq, Sq, Skv), -1, dtype=torch.int32, device=q.device)
    nbytes = _lib().reef_qk_scores_i32_packed_workspace_bytes(B, Hq, Hkv, Sq, Skv)
    if nbytes == 0:
        raise ValueError("qk_scores_i32_packed: invalid sizes")
    ws = torch.zeros(nbytes, dtype=torch.uint8, device=q.device)
    check(_lib().reef_qk_scores_i32_packed(_ptr(q), _ptr(k), B, Hq, Hkv, Sq, Skv, _ptr(acc),
                                          _ptr(ws), nbytes, _stream()), "qk_scores_i32_packed")
    return acc


def _decode_bytes(q, max_context, kv_heads, window, softmax_scale, q_granularity, num_splits):
    B, Hq, D = q.shape
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    return _packed(_DECODE, DecodeParams, B, Hq, kv_heads, D, max_context, window, softmax_scale,
                   q_granularity, num_splits, 0)


def _decode_params(q, max_context, kv_heads, window, softmax_scale, q_granularity, num_splits):
    B, Hq, D = q.shape
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    return DecodeParams(B, Hq, kv_heads, D, max_context, window, softmax_scale, q_granularity,
                        num_splits, 0)


def decode_workspace(params: DecodeParams, device):
    """A zero-filled decode workspace (its item counters must start at zero; every
    launch leaves them so, so the workspace is reusable without refilling)."""
    return _decode_workspace(lib().reef_attention_decode_workspace_bytes(C.byref(params)), device)


def _decode_workspace(n, device):
    torch = _torch()
    return torch.zeros(max(n, 16) // 4 + 4, dtype=torch.float32, device=device)


def attention_decode(q, q_scales, k_cache, v_pages, k_scales, v_scales, context_lens=None, *,
                     window=0, softmax_scale=None, q_granularity=PER_TOKEN, num_splits=0,
                     workspace=None, status: StatusWord | None = None, out=None):
    """One decode step over a contiguous int8 cache.

    q [B, Hq, D] int8; k_cache [B, Hkv, L, D]; v_pages [B, Hkv, L/16, D, 16] (see
    pack_v_pages); k_scales, v_scales [B, Hkv, L]; context_lens [B] int32 or None.
    """
    torch = _torch()
    _require(q, torch.int8, "q")
    B, Hq, D = q.shape
    Hkv, L = k_cache.shape[1], k_cache.shape[2]
    if tuple(k_cache.shape) != (B, Hkv, L, D) or v_pages.numel() != k_cache.numel():
        raise InvalidArgument("attention_decode cache shape mismatch")
    p = _decode_bytes(q, L, Hkv, window, softmax_scale, q_granularity, num_splits)
    ws = workspace
    if ws is None:
        ws = _decode_workspace(_lib().reef_attention_decode_workspace_bytes(p), q.device)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=q.device)
    own = status or StatusWord(q.device)
    cl = context_lens.contiguous() if context_lens is not None else None
    q, q_scales, k_cache, v_pages = (q.contiguous(), q_scales.contiguous(), k_cache.contiguous(),
                                     v_pages.contiguous())
    k_scales, v_scales = k_scales.contiguous(), v_scales.contiguous()
    check(_lib().reef_attention_decode_int8(
        p, _ptr(q), _ptr(q_scales), _ptr(k_cache), _ptr(v_pages), _ptr(k_scales), _ptr(v_scales),
        _ptr(cl), _ptr(out), _ptr(ws), ws.numel() * 4, _ptr(own.tensor), _stream()), "attention_decode")
    if status is None:
        own.check("attention_decode")
    return out


def attention_decode_paged(q, q_scales, k_pages, v_pages, k_scale_pages, v_scale_pages,
                           block_table, context_lens, *, window=0, softmax_scale=None,
                           q_granularity=PER_TOKEN, num_splits=0, workspace=None,
                           status: StatusWord | None = None, out=None):
    """One decode step over a paged int8 cache: k_pages [P, Hkv, 16, D], v_pages
    [P, Hkv, D, 16], scale pages [P, Hkv, 16], block_table [B, max_blocks] int32,
    context_lens [B] int32."""
    torch = _torch()
    _require(q, torch.int8, "q")
    B, Hq, D = q.shape
    P, Hkv = k_pages.shape[0], k_pages.shape[1]
    max_blocks = block_table.shape[1]
    p = _decode_bytes(q, max_blocks * PAGE, Hkv, window, softmax_scale, q_granularity, num_splits)
    ws = workspace
    if ws is None:
        ws = _decode_workspace(_lib().reef_attention_decode_workspace_bytes(p), q.device)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=q.device)
    own = status or StatusWord(q.device)
    q, q_scales, block_table, context_lens = (q.contiguous(), q_scales.contiguous(),
                                              block_table.contiguous(), context_lens.contiguous())
    check(_lib().reef_attention_decode_int8_paged(
        p, _ptr(q), _ptr(q_scales), _ptr(k_pages), _ptr(v_pages), _ptr(k_scale_pages),
        _ptr(v_scale_pages), _ptr(block_table), max_blocks, P, _ptr(context_lens), _ptr(out),
        _ptr(ws), ws.numel() * 4, _ptr(own.tensor), _stream()), "attention_decode_paged")
    if status is None:
        own.check("attention_decode_paged")
    return out


# --- attention of drafted tokens ------------------------------------------------------------

_TREE_WS = {}


def tree_workspace(params: TreeParams, device):
    """A zero-filled workspace of the tree attention: every launch leaves it ready for the
    next, of any shape it is large enough for."""
    n = lib().reef_attention_decode_tree_workspace_bytes(C.byref(params))
    torch = _torch()
    return torch.zeros(max(n, 256), dtype=torch.uint8, device=device)


def _tree_workspace(n, device, stream):
    """This stream's workspace. A call under graph capture takes one of its own, which lives
    in the graph's memory: graphs that replay at the same time share nothing. Only its
    counters have to be zero, the first 8 KB: not a megabyte of parts at every replay."""
    torch = _torch()
    if torch.cuda.is_current_stream_capturing():
        ws = torch.empty(max(n, 8192), dtype=torch.uint8, device=device)
        ws[:8192].zero_()
        return ws
    key = (device.index, stream)
    ws = _TREE_WS.get(key)
    if ws is None or ws.numel() < n:
        ws = _TREE_WS[key] = torch.zeros(max(n, 256), dtype=torch.uint8, device=device)
    return ws


def _given(workspace):
    _on_device("workspace", workspace)
    if not workspace.is_contiguous():
        raise InvalidArgument("workspace must be contiguous")
    return workspace


def _tree_inputs(what, q, q_scales, tree_mask, window, softmax_scale, q_granularity, kv_heads,
                 max_context, head_dim, context_lens, out):
    torch = _torch()
    _require(q, torch.int8, "q")
    if q.dim() != 4 or q.shape[3] != head_dim:
        raise InvalidArgument(f"{what}: q must be [B, heads, drafts, head_dim of the cache]")
    B, Hq, T, D = shape = q.shape
    if not q_scales.is_contiguous():
        q_scales = q_scales.contiguous()
    _expect(what, torch.float32, (q_scales, "q_scales"))
    scales = B * Hq * T if q_granularity == PER_TOKEN else Hq if q_granularity == PER_HEAD else 1
    if q_scales.numel() != scales:
        raise InvalidArgument(f"{what}: q_scales do not match q_granularity")
    if tree_mask is not None:
        if not tree_mask.is_contiguous():
            tree_mask = tree_mask.contiguous()
        _expect(what, torch.int64, (tree_mask, "tree_mask"))
        if tree_mask.shape != (B, T):
            raise InvalidArgument(f"{what}: tree_mask must be [B, drafts] int64")
    if context_lens is not None:
        _expect(what, torch.int32, (context_lens, "context_lens"))
        if context_lens.shape != (B,):
            raise InvalidArgument(f"{what}: context_lens must be [B]")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
        _on_device(what, q)
    else:
        _require(out, torch.float32, "out")
        if out.shape != shape:
            raise InvalidArgument(f"{what}: out must have q's shape")
        _on_device(what, q, out)
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    p = _packed(_TREE, TreeParams, B, Hq, kv_heads, D, T, max_context, window, softmax_scale,
                q_granularity, 0, 0)
    return p, q_scales, tree_mask, out


def attention_decode_tree(q, q_scales, k_cache, v_pages, k_scales, v_scales, context_lens=None, *,
                          tree_mask=None, window=0, softmax_scale=None, q_granularity=PER_TOKEN,
                          workspace=None, status: StatusWord | None = None, out=None):
    """Attention of T drafted tokens per sequence over a contiguous int8 cache that holds them
    in its last T places (kv_append).

    q [B, Hq, T, D] int8 (any strides with contiguous head_dim), T <= 64; q_scales [B, Hq, T]
    by default; the cache as for attention_decode; context_lens [B] int32 (the drafted
    tokens counted in) or None; tree_mask [B, T] int64, bit j of row i set where token i sees
    drafted token j (itself among them; 0: padding, zeros), None for a chain. Returns fp32
    [B, Hq, T, D].
    """
    H, L, D = _contiguous_cache("attention_decode_tree", q.shape[0], k_cache, v_pages, k_scales,
                                v_scales)
    p, q_scales, tree_mask, out = _tree_inputs(
        "attention_decode_tree", q, q_scales, tree_mask, window, softmax_scale, q_granularity, H, L,
        D, context_lens, out)
    stream = _stream()
    n = _lib().reef_attention_decode_tree_workspace_bytes(p)
    ws = _tree_workspace(n, q.device, stream) if workspace is None else _given(workspace)
    own = status or StatusWord(q.device)
    check(_lib().reef_attention_decode_tree_int8(
        p, _ptr(q), _strides4(q), _ptr(q_scales), _ptr(k_cache), _ptr(v_pages), _ptr(k_scales),
        _ptr(v_scales), _ptr(context_lens), _ptr(tree_mask), _ptr(out), _strides4(out), _ptr(ws),
        ws.numel() * ws.element_size(), _ptr(own.tensor), stream), "attention_decode_tree")
    if status is None:
        own.check("attention_decode_tree")
    return out


def attention_decode_tree_paged(q, q_scales, k_pages, v_pages, k_scale_pages, v_scale_pages,
                                block_table, context_lens, *, tree_mask=None, window=0,
                                softmax_scale=None, q_granularity=PER_TOKEN, workspace=None,
                                status: StatusWord | None = None, out=None):
    """attention_decode_tree over a paged int8 cache: k_pages [P, Hkv, 16, D], v_pages [P,
    Hkv, D, 16], scale pages [P, Hkv, 16], block_table [B, max_blocks] int32, context_lens
    [B] int32."""
    what = "attention_decode_tree_paged"
    P, H, D = _pool_shapes(what, k_pages, v_pages, k_scale_pages, v_scale_pages)
    _expect(what, _torch().int32, (block_table, "block_table"), (context_lens, "context_lens"))
    if block_table.dim() != 2 or block_table.shape[0] != q.shape[0]:
        raise InvalidArgument(f"{what}: block_table must be [B, max_blocks]")
    blocks = block_table.shape[1]
    p, q_scales, tree_mask, out = _tree_inputs(
        what, q, q_scales, tree_mask, window, softmax_scale, q_granularity, H, blocks * PAGE, D,
        context_lens, out)
    stream = _stream()
    n = _lib().reef_attention_decode_tree_workspace_bytes(p)
    ws = _tree_workspace(n, q.device, stream) if workspace is None else _given(workspace)
    own = status or StatusWord(q.device)
    check(_lib().reef_attention_decode_tree_int8_paged(
        p, _ptr(q), _strides4(q), _ptr(q_scales), _ptr(k_pages), _ptr(v_pages),
        _ptr(k_scale_pages), _ptr(v_scale_pages), _ptr(block_table), blocks, P,
        _ptr(context_lens), _ptr(tree_mask), _ptr(out), _strides4(out), _ptr(ws),
        ws.numel() * ws.element_size(), _ptr(own.tensor), stream), what)
    if status is None:
        own.check(what)
    return out


def pack_v_pages(v_tokens):
    """Token-major values [..., pages * 16, D] -> transposed pages [..., pages, D, 16]."""
    torch = _torch()
    _require(v_tokens, torch.int8, "v_tokens")
    *lead, L, D = v_tokens.shape
    if L % PAGE:
        raise InvalidArgument("token count must be a multiple of 16")
    src = v_tokens.contiguous()
    pages = src.numel() // (PAGE * D)
    out = torch.empty((*lead, L // PAGE, D, PAGE), dtype=torch.int8, device=src.device)
    check(_lib().reef_kv_pack_v_pages(_ptr(src), pages, D, _ptr(out), _stream()), "pack_v_pages")
    return out


# --- KV-cache append (attention.hpp:290-352) --------------------------------------------

def _append_inputs(k_new, v_new):
    torch = _torch()
    _require(k_new, torch.float32, "k_new")
    _require(v_new, torch.float32, "v_new")
    if k_new.shape != v_new.shape or k_new.dim() != 4:
        raise InvalidArgument("KV cache append shape mismatch")
    return _strides4(k_new), _strides4(v_new)


def kv_append(k_new, v_new, start_positions, k_cache, v_pages, k_scales, v_scales,
              context_lens=None, status: StatusWord | None = None):
    """Quantize fp32 rows k_new, v_new [B, Hkv, T, D] per token and write them into
    the contiguous cache (k_cache [B, Hkv, L, D], v_pages [B, Hkv, L/16, D, 16],
    scales [B, Hkv, L]) at start_positions[b] + t. context_lens, when given, is set
    to start_positions + T afterwards (it may be start_positions itself)."""
    torch = _torch()
    ks, vs = _append_inputs(k_new, v_new)
    B, H, T, D = k_new.shape
    L = k_cache.shape[2]
    if tuple(k_cache.shape) != (B, H, L, D) or v_pages.numel() != k_cache.numel():
        raise InvalidArgument("KV cache append shape mismatch")
    _require(start_positions, torch.int32, "start_positions")
    p = _packed(_APPEND, KvAppendParams, B, H, D, T, L)
    own = status or StatusWord(k_new.device)
    check(_lib().reef_kv_append_int8(
        p, _ptr(k_new), ks, _ptr(v_new), vs, _ptr(start_positions),
        _ptr(k_cache), _ptr(v_pages), _ptr(k_scales), _ptr(v_scales), _ptr(context_lens),
        _ptr(own.tensor), _stream()), "kv_append")
    if status is None:
        own.check("kv_append")


def kv_append_paged(k_new, v_new, start_positions, block_table, k_pages, v_pages,
                    k_scale_pages, v_scale_pages, context_lens=None,
                    status: StatusWord | None = None, max_context=None):
    """kv_append into the paged cache (k_pages [P, Hkv, 16, D], v_pages [P, Hkv, D, 16],
    scale pages [P, Hkv, 16], block_table [B, max_blocks] int32)."""
    torch = _torch()
    ks, vs = _append_inputs(k_new, v_new)
    B, H, T, D = k_new.shape
    P = k_pages.shape[0]
    max_blocks = block_table.shape[1]
    _require(start_positions, torch.int32, "start_positions")
    _require(block_table, torch.int32, "block_table")
    p = _packed(_APPEND, KvAppendParams, B, H, D, T, max_context or max_blocks * PAGE)
    block_table = block_table.contiguous()
    own = status or StatusWord(k_new.device)
    check(_lib().reef_kv_append_int8_paged(
        p, _ptr(k_new), ks, _ptr(v_new), vs, _ptr(start_positions), _ptr(block_table), max_blocks, P, _ptr(k_pages), _ptr(v_pages),
        _ptr(k_scale_pages), _ptr(v_scale_pages), _ptr(context_lens), _ptr(own.tensor), _stream()),
        "kv_append_paged")
    if status is None:
        own.check("kv_append_paged")


# --- pages of the paged cache ---------------------------------------------------------------
#
# block_table [B, max_blocks], context_lens [B] and page_refs [P] are int32 on the GPU and
# changed in place: a table starts filled with -1, page_refs with 0. See the C header.

def _table(what, block_table, context_lens, page_refs):
    if block_table.dim() != 2 or page_refs.dim() != 1 or (
            context_lens is not None and context_lens.shape != block_table.shape[:1]):
        raise InvalidArgument(f"{what} shapes: block_table [B, max_blocks], context_lens [B], "
                              "page_refs [pages]")
    return block_table.shape


def kv_free(sequences, block_table, context_lens, page_refs, status: StatusWord | None = None):
    """The listed sequences ([n] int32 rows of the table, negative: padding) give their pages
    back; their table rows become -1 and their lengths 0."""
    _expect("kv_free", _torch().int32, (sequences, "sequences"), (block_table, "block_table"),
            (context_lens, "context_lens"), (page_refs, "page_refs"))
    B, blocks = _table("kv_free", block_table, context_lens, page_refs)
    if sequences.numel() == 0:
        return
    own = status or StatusWord(block_table.device)
    check(_lib().reef_kv_free(_ptr(sequences), sequences.numel(), _ptr(block_table), blocks,
                              _ptr(context_lens), B, _ptr(page_refs), page_refs.numel(),
                              _ptr(own.tensor), _stream()), "kv_free")
    if status is None:
        own.check("kv_free")


def kv_fork(parents, children, block_table, context_lens, page_refs,
            status: StatusWord | None = None):
    """Sequence children[i] becomes a copy of parents[i] (both [n] int32, negative: padding)
    that shares its pages. A parent may have many children; a child is listed once and is no
    parent in the same call."""
    _expect("kv_fork", _torch().int32, (parents, "parents"), (children, "children"),
            (block_table, "block_table"), (context_lens, "context_lens"), (page_refs, "page_refs"))
    B, blocks = _table("kv_fork", block_table, context_lens, page_refs)
    if parents.numel() != children.numel():
        raise InvalidArgument("kv_fork: as many parents as children")
    if parents.numel() == 0:
        return
    own = status or StatusWord(block_table.device)
    check(_lib().reef_kv_fork(_ptr(parents), _ptr(children), parents.numel(), _ptr(block_table),
                              blocks, _ptr(context_lens), B, _ptr(page_refs), page_refs.numel(),
                              _ptr(own.tensor), _stream()), "kv_fork")
    if status is None:
        own.check("kv_fork")


def kv_reserve(block_table, context_lens, page_refs, new_tokens: int,
               status: StatusWord | None = None):
    """Pages of its own for every sequence's next new_tokens tokens: absent ones from the free
    pages, and instead of shared ones. Returns (source, destination) pages [B] int32 for
    kv_copy_pages on each layer's pool: a shared page that holds tokens is copied, -1 where
    there is nothing to copy. Lengths are left; kv_append_paged writes the tokens."""
    torch = _torch()
    _expect("kv_reserve", torch.int32, (block_table, "block_table"),
            (context_lens, "context_lens"), (page_refs, "page_refs"))
    B, blocks = _table("kv_reserve", block_table, context_lens, page_refs)
    device = block_table.device
    fits = 0 < new_tokens <= blocks * PAGE  # (refused below otherwise)
    n = _lib().reef_kv_reserve_workspace_bytes(B, new_tokens) if fits else 0
    ints = torch.empty(n // 4 + 2 * B, dtype=torch.int32, device=device)
    source, place = ints[:B], ints[B:2 * B]
    own = status or StatusWord(device)
    check(_lib().reef_kv_reserve(
        _ptr(block_table), blocks, _ptr(context_lens), B, new_tokens, _ptr(page_refs),
        page_refs.numel(), _ptr(source), _ptr(place), ints.data_ptr() + 8 * B, n,
        _ptr(own.tensor), _stream()), "kv_reserve")
    if status is None:
        own.check("kv_reserve")
    return source, place


def kv_compact(block_table, page_refs, status: StatusWord | None = None):
    """The pool's L live pages become its first L: table and counts are rewritten. Returns
    (source, destination) pages [pages // 2] int32 for kv_copy_pages on each layer's pool, -1
    behind the last move, and L as a [1] int32 tensor."""
    torch = _torch()
    _expect("kv_compact", torch.int32, (block_table, "block_table"), (page_refs, "page_refs"))
    B, blocks = _table("kv_compact", block_table, None, page_refs)
    pages, device = page_refs.numel(), block_table.device
    n, half = _lib().reef_kv_compact_workspace_bytes(pages), pages // 2
    ints = torch.empty(n // 4 + 2 * max(half, 1) + 1, dtype=torch.int32, device=device)
    live, source, place = ints[:1], ints[1:1 + half], ints[1 + half:1 + 2 * half]
    own = status or StatusWord(device)
    base = ints.data_ptr()
    check(_lib().reef_kv_compact(
        _ptr(block_table), blocks, B, _ptr(page_refs), pages, base + 4, base + 4 * (1 + half),
        base, base + 4 * (1 + 2 * half), n, _ptr(own.tensor), _stream()), "kv_compact")
    if status is None:
        own.check("kv_compact")
    return source, place, live


def _pool_shapes(what, k_pages, v_pages, k_scale_pages, v_scale_pages):
    """(pages, heads, head_dim) of a paged cache."""
    torch = _torch()
    _expect(what, torch.int8, (k_pages, "k_pages"), (v_pages, "v_pages"))
    _expect(what, torch.float32, (k_scale_pages, "k_scale_pages"),
            (v_scale_pages, "v_scale_pages"))
    if k_pages.dim() != 4 or k_pages.shape[2] != PAGE:
        raise InvalidArgument(f"{what}: k_pages must be [pages, heads, 16, head_dim]")
    P, H, _, D = k_pages.shape
    if (v_pages.numel() != k_pages.numel() or k_scale_pages.numel() != P * H * PAGE
            or v_scale_pages.numel() != P * H * PAGE):
        raise InvalidArgument(f"{what}: pages and scale pages do not match")
    return P, H, D


def kv_copy_pages(source, place, k_pages, v_pages, k_scale_pages, v_scale_pages,
                  status: StatusWord | None = None):
    """Page source[i] of one layer's pool (keys, values, scales) is copied to page place[i]
    (both [n] int32; pairs with a negative page are left out). No page may be a destination
    twice, or a source and a destination."""
    _expect("kv_copy_pages", _torch().int32, (source, "source"), (place, "place"))
    P, H, D = _pool_shapes("kv_copy_pages", k_pages, v_pages, k_scale_pages, v_scale_pages)
    if source.numel() != place.numel():
        raise InvalidArgument("kv_copy_pages: as many sources as destinations")
    if source.numel() == 0:
        return
    own = status or StatusWord(k_pages.device)
    check(_lib().reef_kv_copy_pages(
        _ptr(source), _ptr(place), source.numel(), H, D, _ptr(k_pages), _ptr(v_pages),
        _ptr(k_scale_pages), _ptr(v_scale_pages), P, _ptr(own.tensor), _stream()),
        "kv_copy_pages")
    if status is None:
        own.check("kv_copy_pages")


def _kept(what, kept, kept_lens, context_lens):
    _expect(what, _torch().int32, (kept, "kept"), (kept_lens, "kept_lens"),
            (context_lens, "context_lens"))
    if kept.dim() != 2 or kept_lens.shape != kept.shape[:1] or (
            context_lens.shape != kept_lens.shape):
        raise InvalidArgument(f"{what} shapes: kept [B, drafts], kept_lens [B], context_lens [B]")
    return kept.shape


def kv_keep(kept, kept_lens, context_lens, k_cache, v_pages, k_scales, v_scales,
            status: StatusWord | None = None):
    """Of every sequence's last T tokens (drafted ones, appended before) rows kept[b][:n] with
    n = kept_lens[b] stay and move to the first n of their places (kept [B, T] int32,
    ascending; context_lens [B] counts the drafted tokens in). Contiguous cache as in
    kv_append. Returns the new lengths, context_lens - T + kept_lens."""
    torch = _torch()
    B, T = _kept("kv_keep", kept, kept_lens, context_lens)
    H, L, D = _contiguous_cache("kv_keep", B, k_cache, v_pages, k_scales, v_scales)
    lens = torch.empty_like(context_lens)
    own = status or StatusWord(k_cache.device)
    check(_lib().reef_kv_keep_int8(
        _packed(_APPEND, KvAppendParams, B, H, D, T, L), _ptr(kept), _ptr(kept_lens),
        _ptr(context_lens), _ptr(k_cache), _ptr(v_pages), _ptr(k_scales), _ptr(v_scales),
        _ptr(lens), _ptr(own.tensor), _stream()), "kv_keep")
    if status is None:
        own.check("kv_keep")
    return lens


def _contiguous_cache(what, B, k_cache, v_pages, k_scales, v_scales):
    """(heads, tokens, head_dim) of a contiguous cache of B sequences."""
    torch = _torch()
    _expect(what, torch.int8, (k_cache, "k_cache"), (v_pages, "v_pages"))
    _expect(what, torch.float32, (k_scales, "k_scales"), (v_scales, "v_scales"))
    shape, n = k_cache.shape, k_cache.numel()
    if len(shape) != 4 or shape[0] != B or v_pages.numel() != n or (
            k_scales.numel() * shape[3] != n or v_scales.numel() * shape[3] != n):
        raise InvalidArgument(f"{what}: cache shape mismatch")
    return shape[1:]


def kv_keep_paged(kept, kept_lens, context_lens, block_table, k_pages, v_pages, k_scale_pages,
                  v_scale_pages, status: StatusWord | None = None):
    """kv_keep in the paged cache; the drafted tokens' pages must be the sequence's own."""
    torch = _torch()
    B, T = _kept("kv_keep_paged", kept, kept_lens, context_lens)
    _expect("kv_keep_paged", torch.int32, (block_table, "block_table"))
    P, H, D = _pool_shapes("kv_keep_paged", k_pages, v_pages, k_scale_pages, v_scale_pages)
    if block_table.dim() != 2 or block_table.shape[0] != B:
        raise InvalidArgument("kv_keep_paged: block_table must be [B, max_blocks]")
    blocks = block_table.shape[1]
    lens = torch.empty_like(context_lens)
    own = status or StatusWord(k_pages.device)
    check(_lib().reef_kv_keep_int8_paged(
        _packed(_APPEND, KvAppendParams, B, H, D, T, blocks * PAGE), _ptr(kept), _ptr(kept_lens),
        _ptr(context_lens), _ptr(block_table), blocks, P, _ptr(k_pages), _ptr(v_pages),
        _ptr(k_scale_pages), _ptr(v_scale_pages), _ptr(lens), _ptr(own.tensor), _stream()),
        "kv_keep_paged")
    if status is None:
        own.check("kv_keep_paged")
    return lens


# --- integer-only attention (int8.hpp:156-279) -----------------------------------------

def attention_int8_integer(q, k, v, table, *, score_shift, out_shift=8, query_start=None,
                           window=0):
    """attend_head_int8 for every (batch, head): q [B, Hq, Sq, D], k and v
    [B, Hkv, Skv, D] int8, table [256] uint16 (as int16/uint16 torch tensor) on the
    device; returns int8 [B, Hq, Sq, D], bit-identical to the engine."""
    torch = _torch()
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _require(t, torch.int8, n)
    if table.numel() != 256 or table.element_size() != 2 or not table.is_cuda:
        raise InvalidArgument("table must hold 256 16-bit entries on the GPU")
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    start = Skv - Sq if query_start is None else query_start
    p = _packed(_ATTENTION, AttentionParams, B, Hq, Hkv, Sq, Skv, D, start, window, 1.0, PER_HEAD,
                PER_HEAD, 0)
    out = torch.empty((B, Hq, Sq, D), dtype=torch.int8, device=q.device)
    sq, sk, sv, so = _strides4(q), _strides4(k), _strides4(v), _strides4(out)
    table = table.contiguous()
    check(_lib().reef_attention_int8_integer(
        p, _ptr(q), sq, _ptr(k), sk, _ptr(v), sv, score_shift, _ptr(table), out_shift, _ptr(out),
        so, _stream()), "attention_int8_integer")
    return out


# --- W8A8 projection (operator/linear.hpp:106-132) ---------------------------------------

def _epilogue(activation, residual, rows, fout, what):
    """The packed reef_epilogue of an activation's name and a [rows, fout] residual."""
    if activation not in ACTIVATIONS:
        raise InvalidArgument(f"{what}: activation must be one of {', '.join(ACTIVATIONS)}")
    if residual is None:
        return None if activation == "none" else _EPILOGUE.pack(0, 0, ACTIVATIONS[activation])
    _require(residual, _torch().float32, "residual")
    if tuple(residual.shape) != (rows, fout) or _row_stride(residual) is None:
        raise InvalidArgument(f"{what}: residual must be [rows, out] with contiguous rows")
    _on_device(what, residual)
    return _EPILOGUE.pack(residual.data_ptr(), _row_stride(residual), ACTIVATIONS[activation])


def _row_stride(t):
    """Elements from row to row of a matrix with contiguous rows; None for any other."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        return None
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _product_out(out, rows, fout, device, what):
    torch = _torch()
    if out is None:
        return torch.empty((rows, fout), dtype=torch.float32, device=device), fout
    _require(out, torch.float32, "out")
    _on_device(what, out)
    stride = _row_stride(out)
    if tuple(out.shape) != (rows, fout) or stride is None or stride < fout:
        raise InvalidArgument(f"{what}: out must be [rows, out] with contiguous rows")
    return out, stride


def linear_w8a8(x, weight, w_scales, bias=None, status: StatusWord | None = None, *,
                activation="none", residual=None):
    """y = linear(x, QuantizedWeight{weight, w_scales}, bias): x [rows, in] fp32,
    weight [out, in] int8, w_scales [out] fp32, bias [out] fp32 or None. Rows are
    quantized per row on the device; outputs are bit-identical to the engine's.
    activation (a key of ACTIVATIONS) is applied after the bias, then residual
    [rows, out] fp32 is added."""
    torch = _torch()
    _require(x, torch.float32, "x")
    _require(weight, torch.int8, "weight")
    _require(w_scales, torch.float32, "w_scales")
    if x.dim() != 2 or x.stride(1) != 1 or weight.dim() != 2 or weight.shape[1] != x.shape[1]:
        raise InvalidArgument("linear_w8a8 shapes: x [rows, in], weight [out, in]")
    rows, fin = x.shape
    fout = weight.shape[0]
    epilogue = _epilogue(activation, residual, rows, fout, "linear_w8a8")
    n = _lib().reef_linear_w8a8_workspace_bytes(rows, fin)
    ws = torch.empty(n // 4 + 4, dtype=torch.float32, device=x.device)
    y = torch.empty((rows, fout), dtype=torch.float32, device=x.device)
    own = status or StatusWord(x.device)
    weight, w_scales = weight.contiguous(), w_scales.contiguous()
    bias = bias.contiguous() if bias is not None else None
    check(_lib().reef_linear_w8a8_epilogue(
        _ptr(x), rows, fin, x.stride(0), _ptr(weight), _ptr(w_scales), _ptr(bias), epilogue, fout,
        _ptr(y), fout, _ptr(ws), ws.numel() * 4, _ptr(own.tensor), _stream()), "linear_w8a8")
    if status is None:
        own.check("linear_w8a8")
    return y


def gemm_w8a8(xq, x_scales, weight, w_scales, bias=None, status: StatusWord | None = None, *,
              activation="none", residual=None, out=None):
    """The product of linear_w8a8 on rows that are int8 already: xq [rows, in] int8 with
    x_scales [rows] (quantize_rows, rmsnorm_quantize). y = activation(float(sum) *
    (x_scale * w_scale) + bias) + residual, fp32 [rows, out]; out (contiguous rows) may be
    the residual itself, which then becomes the new residual stream."""
    torch = _torch()
    for t, dtype, name in ((xq, torch.int8, "xq"), (weight, torch.int8, "weight"),
                           (x_scales, torch.float32, "x_scales"),
                           (w_scales, torch.float32, "w_scales")):
        _require(t, dtype, name)
    if xq.dim() != 2 or weight.dim() != 2 or weight.shape[1] != xq.shape[1]:
        raise InvalidArgument("gemm_w8a8 shapes: xq [rows, in], weight [out, in]")
    (rows, fin), fout = xq.shape, weight.shape[0]
    if x_scales.numel() != rows or w_scales.numel() != fout:
        raise InvalidArgument("gemm_w8a8 shapes: x_scales [rows], w_scales [out]")
    if bias is not None:
        _require(bias, torch.float32, "bias")
        if bias.numel() != fout:
            raise InvalidArgument("gemm_w8a8 shapes: bias [out]")
        bias = bias.contiguous()
    _on_device("gemm_w8a8", xq, x_scales, weight, w_scales, bias)
    epilogue = _epilogue(activation, residual, rows, fout, "gemm_w8a8")
    y, y_stride = _product_out(out, rows, fout, xq.device, "gemm_w8a8")
    own = status or StatusWord(xq.device)
    xq, x_scales, weight, w_scales = (xq.contiguous(), x_scales.contiguous(), weight.contiguous(),
                                      w_scales.contiguous())
    check(_lib().reef_gemm_w8a8_epilogue(
        _ptr(xq), _ptr(x_scales), rows, fin, _ptr(weight), _ptr(w_scales), _ptr(bias), epilogue,
        fout, _ptr(y), y_stride, _ptr(own.tensor), _stream()), "gemm_w8a8")
    if status is None:
        own.check("gemm_w8a8")
    return y


# --- norm ---------------------------------------------------------------------------------

def _rows_of(t, width):
    """t's rows as a matrix, and the elements from row to row; copied only where they do not
    lie evenly."""
    if t.is_contiguous():
        return t, width
    m = t if t.dim() == 2 else t.reshape(-1, width)
    stride = _row_stride(m)
    return (m, stride) if stride is not None and stride >= width else (m.contiguous(), width)


def rmsnorm_quantize(x, weight=None, *, residual=None, eps=1e-6, residual_out=None,
                     status: StatusWord | None = None):
    """The root-mean-square norm of x (+ residual) over the last dimension, as int8 rows
    with scales: h = x + residual, y = h * weight / sqrt(mean(h^2) + eps), one scale
    max|y| / 127 per row. x and residual [..., width] fp32, weight [width] fp32 or None.
    Returns (int8 of x's shape, scales of x.shape[:-1]), and h as a third where there is a
    residual: the new residual stream, in residual_out if that is given (contiguous, and x
    or residual itself or apart from both)."""
    torch = _torch()
    _require(x, torch.float32, "x")
    shape = x.shape
    if len(shape) == 0 or x.numel() == 0:
        raise InvalidArgument("rmsnorm_quantize: x must be [..., width] and not empty")
    width = shape[-1]
    if weight is not None:
        _require(weight, torch.float32, "weight")
        if weight.shape != (width,):
            raise InvalidArgument("rmsnorm_quantize: weight must be [width]")
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if residual is not None:
        _require(residual, torch.float32, "residual")
        if residual.shape != shape:
            raise InvalidArgument("rmsnorm_quantize: residual must have x's shape")
    elif residual_out is not None:
        raise InvalidArgument("rmsnorm_quantize: residual_out needs a residual")
    _on_device("rmsnorm_quantize", x, weight, residual)

    x2, x_stride = _rows_of(x, width)
    r2 = h = None
    r_stride = 0
    if residual is not None:
        r2, r_stride = _rows_of(residual, width)
        h = residual_out
        if h is None:
            h = torch.empty(shape, dtype=torch.float32, device=x.device)
        else:
            _expect("rmsnorm_quantize", torch.float32, (h, "residual_out"))
            if h.shape != shape:
                raise InvalidArgument("rmsnorm_quantize: residual_out must have x's shape")
    q = torch.empty(shape, dtype=torch.int8, device=x.device)
    s = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    own = status or StatusWord(x.device)
    check(_lib().reef_rmsnorm_quantize_int8(
        _ptr(x2), s.numel(), width, x_stride, _ptr(r2), r_stride, _ptr(weight), eps, _ptr(q),
        _ptr(s), _ptr(h), width, _ptr(own.tensor), _stream()), "rmsnorm_quantize")
    if status is None:
        own.check("rmsnorm_quantize requires finite values")
    return (q, s) if residual is None else (q, s, h)
