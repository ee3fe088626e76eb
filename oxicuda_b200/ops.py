"""Device-tensor front end of the C ABI: torch tensors supply device memory and the current stream,
every computation happens inside liboxq_b200.so.  Function names follow the C entry points."""
from __future__ import annotations

import ctypes as C
import functools
import threading

import torch

from . import _ffi
from .errors import raise_for_status

F32, BF16, F16 = 0, 1, 2
ROUND_HALF_EVEN, ROUND_HALF_AWAY = 0, 1
FP8_SPEC_RNE, FP8_REFCOMPAT = 0, 1

_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_TORCH_DT = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}


class Handle:
    """One per host thread and device, like BlasHandle (crates/oxicuda-blas/src/handle.rs:41-52)."""

    def __init__(self, device: int | None = None):
        if not torch.cuda.is_available():
            raise RuntimeError("oxicuda_b200 needs a CUDA device (sm_100); there is no CPU fallback")
        self.lib = _ffi.load()
        self.device = torch.cuda.current_device() if device is None else int(device)
        self._h = C.c_void_p()
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream().cuda_stream
            raise_for_status(self.lib.oxq_handle_create(self.device, C.c_void_p(stream), C.byref(self._h)))
        self._stream = stream
        self._lock = threading.Lock()

    def close(self):
        if self._h:
            self.lib.oxq_handle_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync_stream(self):
        """Follow torch's current stream (BlasHandle::set_stream)."""
        s = torch._C._cuda_getCurrentRawStream(self.device)          # current_stream() without building a Stream object
        if s != self._stream:
            raise_for_status(self.lib.oxq_set_stream(self._h, C.c_void_p(s)))
            self._stream = s

    def call(self, name: str, *args):
        with self._lock:                      # the stream is the handle's: threads that share it take turns from setting it to the launch
            self.sync_stream()
            rc = getattr(self.lib, name)(self._h, *args)
            error = self.lib.oxq_last_error_string(self._h).decode() if rc else ""
        if rc:
            raise_for_status(rc, error)

    def device_status(self) -> int:
        v = C.c_int32(0)
        raise_for_status(self.lib.oxq_device_status(self._h, C.byref(v)))
        return v.value


_handles: dict[int, Handle] = {}


def handle(device: int | None = None) -> Handle:
    d = torch.cuda.current_device() if device is None else int(device)
    if d not in _handles:
        _handles[d] = Handle(d)
    return _handles[d]


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _chk(t: torch.Tensor, *dtypes):
    if not t.is_cuda:
        raise TypeError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise TypeError("expected a contiguous tensor")
    if dtypes and t.dtype not in dtypes:
        raise TypeError(f"expected dtype in {dtypes}, got {t.dtype}")


# ------------------------------------------------------------------------------------------- INT8

def int8_quant_rows(x: torch.Tensor, rounding: int = ROUND_HALF_EVEN):
    _chk(x, torch.float32)
    rows, cols = (x.shape[0], x.shape[1]) if x.dim() == 2 else (0, 0)
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    s = torch.empty((rows,), dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_int8_quant_rows", _p(x), rows, cols, _p(q), _p(s), rounding)
    return q, s


def int8_dequant_rows(q: torch.Tensor, scales: torch.Tensor):
    _chk(q, torch.int8)
    _chk(scales, torch.float32)
    rows, cols = q.shape
    y = torch.empty((rows, cols), dtype=torch.float32, device=q.device)
    handle(q.device.index).call("oxq_int8_dequant_rows", _p(q), _p(scales), rows, cols, _p(y))
    return y


# ------------------------------------------------------------------------------------------- FP8

def absmax(x: torch.Tensor, out: torch.Tensor | None = None):
    _chk(x, *_DT)
    out = torch.empty(1, dtype=torch.float32, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_absmax", _p(x), _DT[x.dtype], x.numel(), _p(out))
    return out


def fp8_quant(x: torch.Tensor, scale: torch.Tensor, mode: int = FP8_SPEC_RNE, out: torch.Tensor | None = None):
    _chk(x, *_DT)
    _chk(scale, torch.float32)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_fp8_quant", _p(x), _DT[x.dtype], x.numel(), _p(scale), _p(q), mode)
    return q


def fp8_quant_dynamic(x: torch.Tensor, out: torch.Tensor | None = None, stats: torch.Tensor | None = None):
    """Returns (codes, stats) with stats[0] = absmax and stats[1] = scale = absmax / 448."""
    _chk(x, *_DT)
    q = torch.empty(x.shape, dtype=torch.uint8, device=x.device) if out is None else out
    stats = torch.empty(2, dtype=torch.float32, device=x.device) if stats is None else stats
    handle(x.device.index).call("oxq_fp8_quant_dynamic", _p(x), _DT[x.dtype], x.numel(), _p(q), _p(stats))
    return q, stats


def fp8_dequant(q: torch.Tensor, scale: torch.Tensor, dtype=torch.float32, mode: int = FP8_SPEC_RNE):
    _chk(q, torch.uint8)
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    handle(q.device.index).call("oxq_fp8_dequant", _p(q), q.numel(), _p(scale), _p(y), _DT[dtype], mode)
    return y


# ------------------------------------------------------------------------------------------- INT4

def int4g_quant_pack(x: torch.Tensor, group: int = 128, rounding: int = ROUND_HALF_AWAY):
    _chk(x, *_DT)
    rows, k = (x.shape[0], x.shape[1]) if x.dim() == 2 else (0, 0)
    ng = rows * (k // group) if group > 0 else 0
    # int32 tensors hold the u32 words and uint16 bit patterns are kept in int16 tensors
    codes = torch.empty((rows, max(k // 8, 0)), dtype=torch.int32, device=x.device)
    scales = torch.empty((rows, k // group if group > 0 else 0), dtype=torch.float16, device=x.device)
    zeros = torch.empty(((ng + 7) // 8,), dtype=torch.int32, device=x.device)
    handle(x.device.index).call("oxq_int4g_quant_pack", _p(x), _DT[x.dtype], rows, k, group, _p(codes), _p(scales),
                                _p(zeros), rounding)
    return codes, scales, zeros


def int4g_dequant(codes, scales, zeros, rows: int, k: int, group: int = 128, dtype=torch.float32):
    y = torch.empty((rows, k), dtype=dtype, device=codes.device)
    handle(codes.device.index).call("oxq_int4g_dequant", _p(codes), _p(scales), _p(zeros), rows, k, group, _p(y),
                                    _DT[dtype])
    return y


def int4g_quant_pack_f32(x: torch.Tensor, group: int = 128, rounding: int = ROUND_HALF_AWAY, check_scales: bool = True):
    """MinMaxQuantizer per group, asymmetric, in the reference's own parameter types: (codes u32 words [rows x k/8],
    scales f32 [rows x k/group], zero_points i32 [rows x k/group]).  With check_scales the scales are read back and a
    non-finite or non-positive one raises QuantError InvalidScale, as calibrate does (minmax.rs:234-236)."""
    _chk(x, torch.float32)
    rows, k = (x.shape[0], x.shape[1]) if x.dim() == 2 else (0, 0)
    gpr = k // group if group > 0 else 0
    codes = torch.empty((rows, max(k // 8, 0)), dtype=torch.int32, device=x.device)
    scales = torch.empty((rows, gpr), dtype=torch.float32, device=x.device)
    zps = torch.empty((rows, gpr), dtype=torch.int32, device=x.device)
    handle(x.device.index).call("oxq_int4g_quant_pack_f32", _p(x), rows, k, group, _p(codes), _p(scales), _p(zps), rounding)
    if check_scales and not bool((torch.isfinite(scales) & (scales > 0)).all()):
        from .errors import QuantError
        raise QuantError("InvalidScale", "a group's scale is not finite and positive", 3)
    return codes, scales, zps


def int4g_dequant_f32(codes, scales, zps, rows: int, k: int, group: int = 128):
    y = torch.empty((rows, k), dtype=torch.float32, device=codes.device)
    handle(codes.device.index).call("oxq_int4g_dequant_f32", _p(codes), _p(scales), _p(zps), rows, k, group, _p(y))
    return y


def fp4_microscale_quant(x: torch.Tensor, block: int = 32):
    """MicroScalingQuantizer::quantize_fp4 (crates/oxicuda-blas/src/precision/fp4_fp6_ops.rs:849-876):
    (packed bytes [ceil(n / 2)], f32 scales [ceil(n / block)])."""
    _chk(x, torch.float32)
    n = x.numel()
    packed = torch.empty(max((n + 1) // 2, 1), dtype=torch.uint8, device=x.device)
    scales = torch.empty(max((n + max(block, 1) - 1) // max(block, 1), 1), dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_fp4_microscale_quant", _p(x), n, block, _p(packed), _p(scales))
    return packed[: (n + 1) // 2], scales[: (n + block - 1) // block]


def fp4_microscale_dequant(packed: torch.Tensor, scales: torch.Tensor, n: int, block: int = 32):
    y = torch.empty(max(n, 1), dtype=torch.float32, device=packed.device)
    handle(packed.device.index).call("oxq_fp4_microscale_dequant", _p(packed), _p(scales), n, block, _p(y))
    return y[:n]


class TensorDesc:
    """TensorDesc<T> of the reference's DNN layer (crates/oxicuda-dnn/src/types.rs:108-118) over a torch tensor:
    a borrowed device pointer with dims and strides; numel() and the byte size follow the dims."""

    def __init__(self, tensor: torch.Tensor):
        _chk(tensor, torch.float32, torch.bfloat16, torch.float16)
        self.tensor = tensor
        self.ptr = tensor.data_ptr()
        self.dims = tuple(tensor.shape)
        self.strides = tuple(tensor.stride())

    def numel(self) -> int:
        return self.tensor.numel()

    def nbytes(self) -> int:
        return self.tensor.numel() * self.tensor.element_size()


def _dnn_need(buf: torch.Tensor, elems: int, what: str):
    """DnnError::BufferTooSmall counts bytes (crates/oxicuda-dnn/src/error.rs:33-40)."""
    if buf.numel() < elems:
        from .errors import DnnError
        raise DnnError("BufferTooSmall", what, 11, expected=elems * buf.element_size(), actual=buf.numel() * buf.element_size())


class Int4QuantConfig:
    """Int4QuantConfig of the DNN layer (crates/oxicuda-dnn/src/quantize/int4_quantize.rs:66-104)."""

    def __init__(self, group_size: int, symmetric: bool):
        if group_size == 0:
            from .errors import DnnError
            raise DnnError("InvalidArgument", "INT4 group_size must be non-zero", 15)
        self.group_size, self.symmetric = int(group_size), bool(symmetric)

    def num_groups(self, n: int) -> int:
        return -(-n // self.group_size)

    def packed_bytes(self, n: int) -> int:
        return -(-n // 2)


def quantize_to_int4(x: torch.Tensor, output: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, n: int, config: Int4QuantConfig):
    """quantize_to_int4 (int4_quantize.rs:132-218): fills `output` (ceil(n / 2) bytes), `scales` and, when asymmetric,
    `zeros` (one float per group).  n == 0 does nothing; undersized buffers raise DnnError BufferTooSmall in bytes."""
    if n == 0:
        return
    _chk(x, torch.float32)
    _dnn_need(x, n, "input")
    _dnn_need(output, config.packed_bytes(n), "output")
    _dnn_need(scales, config.num_groups(n), "scales")
    if not config.symmetric:
        if zeros is None:
            from .errors import DnnError
            raise DnnError("BufferTooSmall", "zeros", 11, expected=config.num_groups(n) * 4, actual=0)
        _dnn_need(zeros, config.num_groups(n), "zeros")
    handle(x.device.index).call("oxq_dnn_int4_quant", _p(x), n, config.group_size, 1 if config.symmetric else 0, _p(output), _p(scales),
                                _p(zeros if not config.symmetric else None))


def dequantize_int4(packed: torch.Tensor, scales: torch.Tensor, output: torch.Tensor, n: int, config: Int4QuantConfig):
    """dequantize_int4 (int4_quantize.rs:229-300)."""
    if n == 0:
        return
    _dnn_need(packed, config.packed_bytes(n), "input")
    _dnn_need(scales, config.num_groups(n), "scales")
    _dnn_need(output, n, "output")
    handle(packed.device.index).call("oxq_dnn_int4_dequant", _p(packed), _p(scales), n, config.group_size, 1 if config.symmetric else 0, _p(output))


class Fp4BlockQuantizer:
    """Fp4BlockQuantizer of the DNN layer (crates/oxicuda-dnn/src/quantize/block_scale.rs:346-395): the host-side helper for blocks of
    32 E2M1 codes; compute_scale is max |x| / 6 in f32, or 1 for an all-zero block."""

    MAX_VALUE = 6.0
    REQUIRED_BLOCK_SIZE = 32

    def __init__(self, block_size: int):
        if block_size != self.REQUIRED_BLOCK_SIZE:
            from .errors import DnnError
            raise DnnError("InvalidArgument", f"NVFP4/OCP MXFP4 block size must be {self.REQUIRED_BLOCK_SIZE}, got {block_size}", 15)
        self.block_size = int(block_size)

    def compute_scale(self, block) -> float:
        import numpy as np
        b = np.asarray(block, dtype=np.float32)
        max_abs = np.float32(np.nanmax(np.abs(b))) if b.size and not np.isnan(b).all() else np.float32(0.0)   # f32::max skips NaN
        return 1.0 if max_abs == 0.0 else float(max_abs / np.float32(self.MAX_VALUE))

    def num_scales(self, n: int) -> int:
        return -(-n // self.block_size)


def quantize_block_scaled(desc: TensorDesc, output: torch.Tensor, scales: torch.Tensor, block_size: int):
    """quantize_block_scaled (crates/oxicuda-dnn/src/quantize/block_scale.rs:53-140): one biased byte per element into
    `output`, one f32 scale per block into `scales`."""
    from .errors import DnnError
    n = desc.numel()
    if n == 0:
        return
    if block_size == 0 or (block_size & (block_size - 1)) != 0:
        raise DnnError("InvalidArgument", f"block_size must be a non-zero power of 2, got {block_size}", 15)
    if block_size < 16:
        raise DnnError("InvalidArgument", f"block_size must be >= 16, got {block_size}", 15)
    _dnn_need(output, n, "output")
    _dnn_need(scales, -(-n // block_size), "scales")
    x = desc.tensor
    handle(x.device.index).call("oxq_dnn_block_scaled_quant", _p(x), _DT[x.dtype], n, block_size, _p(output), _p(scales))


def fused_dequant_gemv(packed_w: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, cols: int, group_size: int, bits: int = 4):
    """dnn_fused_dequant_gemv_f32 (crates/oxicuda-dnn/src/quantize/gptq_awq.rs:867-994): y[row] = sum_col (code * scale) * x[col] with
    unsigned codes packed LSB-first in u32 words [rows x cols * bits / 32], f32 scales [rows x cols / group_size], f32 x and y."""
    _chk(x, torch.float32)
    _chk(scales, torch.float32)
    rows = packed_w.shape[0]
    y = torch.empty(rows, dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_dnn_fused_dequant_gemv", _p(packed_w), _p(scales), _p(x), _p(y), rows, cols, group_size, bits)
    return y


# ------------------------------------------------------------------------------------------- block scaled

def sf_mma_bytes(rows: int, sf_cols: int) -> int:
    return int(_ffi.load().oxq_sf_mma_bytes(rows, sf_cols))


def mxfp8_quant(x: torch.Tensor, want_mma_layout: bool = True):
    """Returns (codes [rows x k] u8, sf_rowmajor [rows x k/32] u8, sf_mma bytes or None)."""
    _chk(x, *_DT)
    rows, k = (x.shape[0], x.shape[1]) if x.dim() == 2 else (0, 0)
    codes = torch.empty((rows, k), dtype=torch.uint8, device=x.device)
    sf = torch.empty((rows, k // 32), dtype=torch.uint8, device=x.device)
    sf_mma = torch.empty(sf_mma_bytes(rows, k // 32), dtype=torch.uint8, device=x.device) if want_mma_layout else None
    handle(x.device.index).call("oxq_mxfp8_quant", _p(x), _DT[x.dtype], rows, k, _p(codes), _p(sf), _p(sf_mma))
    return codes, sf, sf_mma


def mxfp8_dequant(codes, sf, dtype=torch.float32):
    rows, k = codes.shape
    y = torch.empty((rows, k), dtype=dtype, device=codes.device)
    handle(codes.device.index).call("oxq_mxfp8_dequant", _p(codes), _p(sf), rows, k, _p(y), _DT[dtype])
    return y


def nvfp4_quant(x: torch.Tensor, want_mma_layout: bool = True, stats: torch.Tensor | None = None):
    """absmax pass + encode pass.  Returns (packed [rows x k/2] u8, sf_rowmajor [rows x k/16] u8, sf_mma, stats)
    with stats[0] = absmax and stats[1] = the f32 tensor scale."""
    _chk(x, *_DT)
    rows, k = (x.shape[0], x.shape[1]) if x.dim() == 2 else (0, 0)
    stats = torch.empty(2, dtype=torch.float32, device=x.device) if stats is None else stats
    packed = torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device)
    sf = torch.empty((rows, k // 16), dtype=torch.uint8, device=x.device)
    sf_mma = torch.empty(sf_mma_bytes(rows, k // 16), dtype=torch.uint8, device=x.device) if want_mma_layout else None
    h = handle(x.device.index)
    if rows > 0 and k > 0:
        h.call("oxq_absmax", _p(x), _DT[x.dtype], x.numel(), _p(stats))
    h.call("oxq_nvfp4_quant", _p(x), _DT[x.dtype], rows, k, _p(stats), _p(packed), _p(sf), _p(sf_mma))
    return packed, sf, sf_mma, stats


def nvfp4_dequant(packed, sf, stats, dtype=torch.float32):
    rows, k = packed.shape[0], packed.shape[1] * 2
    y = torch.empty((rows, k), dtype=dtype, device=packed.device)
    handle(packed.device.index).call("oxq_nvfp4_dequant", _p(packed), _p(sf), _p(stats), rows, k, _p(y), _DT[dtype])
    return y


# ------------------------------------------------------------------------------------------- next to the hot path

def quantize_to_int8(x: torch.Tensor, out: torch.Tensor | None = None, scale: torch.Tensor | None = None):
    """Per-tensor INT8 of oxicuda-dnn (crates/oxicuda-dnn/src/quantize/int8_quantize.rs:33-38): returns (codes, scale[1])."""
    _chk(x, torch.float32, torch.bfloat16, torch.float16)
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device) if out is None else out
    sc = torch.empty(1, dtype=torch.float32, device=x.device) if scale is None else scale
    handle(x.device.index).call("oxq_int8_quant_tensor", _p(x), _DT[x.dtype], x.numel(), _p(q), _p(sc))
    return q, sc


def dequantize_from_int8(q: torch.Tensor, scale: torch.Tensor, dtype=torch.float32):
    """out[i] = (float)q[i] * scale[0] (int8_quantize.rs:101-107)."""
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    handle(q.device.index).call("oxq_int8_dequant_tensor", _p(q), _p(scale), q.numel(), _p(y), _DT[dtype])
    return y


def block_int8_quant(x: torch.Tensor, block: int):
    """BlockQuantizedInt8::quantize on a device tensor (int8_quantize.rs:404-432): (codes, scales[ceil(n / block)])."""
    _chk(x, torch.float32)
    if block <= 0:
        raise ValueError("block_size must be > 0")
    n = x.numel()
    q = torch.empty(n, dtype=torch.int8, device=x.device)
    sc = torch.empty(max((n + block - 1) // block, 1), dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_int8_block_quant", _p(x), n, block, _p(q), _p(sc))
    return q, sc[: (n + block - 1) // block]


def block_int8_dequant(q: torch.Tensor, scales: torch.Tensor, block: int):
    y = torch.empty(q.numel(), dtype=torch.float32, device=q.device)
    handle(q.device.index).call("oxq_int8_block_dequant", _p(q), _p(scales), q.numel(), block, _p(y))
    return y


def nf4_quant(x: torch.Tensor, block: int = 64):
    """Nf4Quantizer::encode (crates/oxicuda-quant/src/scheme/nf4.rs:93-130): (packed bytes [n / 2], absmax [n / block])."""
    _chk(x, torch.float32)
    n = x.numel()
    packed = torch.empty(max(n // 2, 1), dtype=torch.uint8, device=x.device)
    am = torch.empty(max(n // max(block, 1), 1), dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_nf4_quant", _p(x), n, block, _p(packed), _p(am))
    return packed[: n // 2], am[: n // block]


def nf4_dequant(packed: torch.Tensor, absmaxs: torch.Tensor, block: int = 64, dtype=torch.float32):
    """Nf4Quantizer::decode (nf4.rs:137-155)."""
    n = packed.numel() * 2
    if block <= 0 or absmaxs.numel() != n // block:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"expected {n // max(block, 1)} absmax values, got {absmaxs.numel()}", 4)
    y = torch.empty(n, dtype=dtype, device=packed.device)
    handle(packed.device.index).call("oxq_nf4_dequant", _p(packed), _p(absmaxs), n, block, _p(y), _DT[dtype])
    return y


def gemm_nf4(x: torch.Tensor, packed: torch.Tensor, absmaxs: torch.Tensor, n: int, block: int = 64, out: torch.Tensor | None = None):
    """Y = X . dequant(W)^T for up to 8 batch rows; `packed` / `absmaxs` are nf4_quant's tensors of a row-major [n x k] weight."""
    _chk(x, torch.bfloat16)
    _chk(packed, torch.uint8)
    _chk(absmaxs, torch.float32)
    m, k = x.shape
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_gemm_nf4", m, n, k, _p(x), _p(packed), _p(absmaxs), block, _p(y))
    return y


def rmsnorm_int8_quant_rows(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, want_normed: bool = False):
    """RmsNorm::forward (crates/oxicuda-lm/src/layer/norm.rs:73-95) fused with the per-row INT8 quantizer: returns
    (codes int8 [rows x cols], scales f32 [rows]) and, if asked, the normalised activations in x's dtype."""
    _chk(x, torch.float32, torch.bfloat16, torch.float16)
    _chk(weight, torch.float32)
    rows, cols = x.shape
    if weight.numel() != cols:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"expected {cols} weights, got {weight.numel()}", 4)
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    sc = torch.empty(rows, dtype=torch.float32, device=x.device)
    y = torch.empty_like(x) if want_normed else None
    handle(x.device.index).call("oxq_rmsnorm_int8_quant_rows", _p(x), _DT[x.dtype], _p(weight), rows, cols, C.c_float(eps), _p(q), _p(sc), _p(y))
    return (q, sc, y) if want_normed else (q, sc)


def rmsnorm_fp8_quant_rows(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, eps: float = 1e-5):
    """RmsNorm::forward fused with the E4M3 quantizer at a calibrated per-tensor scale: codes uint8 [rows x cols]."""
    _chk(x, torch.float32, torch.bfloat16, torch.float16)
    _chk(weight, torch.float32)
    rows, cols = x.shape
    if weight.numel() != cols:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"expected {cols} weights, got {weight.numel()}", 4)
    q = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    handle(x.device.index).call("oxq_rmsnorm_fp8_quant_rows", _p(x), _DT[x.dtype], _p(weight), rows, cols, C.c_float(eps), _p(scale), _p(q))
    return q


def silu_gate_fp8_quant(gate: torch.Tensor, up: torch.Tensor, scale: torch.Tensor):
    """silu(gate) * up (the reference's silu_gate kernel) fused with the E4M3 quantizer at a calibrated per-tensor scale."""
    _chk(gate, torch.float32, torch.bfloat16, torch.float16)
    _chk(up, gate.dtype)
    if gate.shape != up.shape:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"gate {tuple(gate.shape)} vs up {tuple(up.shape)}", 4)
    q = torch.empty(gate.shape, dtype=torch.uint8, device=gate.device)
    handle(gate.device.index).call("oxq_silu_gate_fp8_quant", _p(gate), _p(up), _DT[gate.dtype], gate.numel(), _p(scale), _p(q))
    return q


def quantize_to_fp8(x: torch.Tensor, out: torch.Tensor | None = None, scale: torch.Tensor | None = None):
    """quantize_to_fp8 of the reference's DNN layer (crates/oxicuda-dnn/src/quantize/fp8_quantize.rs:47-118): per-tensor
    scale = absmax / 448 into a one-element buffer, E4M3 codes.  Returns (codes, scale)."""
    stats = torch.empty(2, dtype=torch.float32, device=x.device)
    q, _ = fp8_quant_dynamic(x, out=out, stats=stats)
    if scale is None:
        scale = stats[1:2]
    else:
        scale[:1].copy_(stats[1:2])
    return q, scale


def dequantize_from_fp8(q: torch.Tensor, scale: torch.Tensor, dtype=torch.float32):
    """dequantize_from_fp8 (fp8_quantize.rs:121-170): out[i] = e4m3(q[i]) * scale[0]."""
    return fp8_dequant(q, scale, dtype=dtype)


class SmoothQuantMigrator:
    """SmoothQuantMigrator of the reference (crates/oxicuda-quant/src/scheme/smooth_quant.rs:54-293) on device tensors."""

    def __init__(self, alpha: float = 0.5):
        self.alpha = float(alpha)

    @staticmethod
    def _col_absmax(x: torch.Tensor) -> torch.Tensor:
        _chk(x, torch.float32)
        if x.dim() != 2:
            from .errors import QuantError
            raise QuantError("DimensionMismatch", f"expected a matrix, got {tuple(x.shape)}", 4)
        st = torch.empty(max(x.shape[1], 1), dtype=torch.float32, device=x.device)
        handle(x.device.index).call("oxq_smooth_col_absmax", _p(x), x.shape[0], x.shape[1], _p(st))
        return st[: x.shape[1]]

    compute_act_stats = _col_absmax
    compute_weight_stats = _col_absmax

    def compute_migration_scales(self, act_max: torch.Tensor, weight_max: torch.Tensor) -> torch.Tensor:
        from .errors import QuantError
        if act_max.numel() == 0:
            raise QuantError("EmptyInput", "SmoothQuantMigrator::compute_migration_scales", 1)
        if act_max.numel() != weight_max.numel():
            raise QuantError("DimensionMismatch", f"expected {act_max.numel()}, got {weight_max.numel()}", 4)
        sc = torch.empty_like(act_max)
        handle(act_max.device.index).call("oxq_smooth_scales", _p(act_max), _p(weight_max), act_max.numel(), C.c_float(self.alpha), _p(sc))
        return sc

    @staticmethod
    def _apply(x: torch.Tensor, scales: torch.Tensor, divide: bool):
        from .errors import QuantError
        _chk(x, torch.float32)
        if x.dim() != 2 or scales.numel() != x.shape[1]:
            raise QuantError("DimensionMismatch", f"expected {x.shape[-1]} scales, got {scales.numel()}", 4)
        handle(x.device.index).call("oxq_smooth_apply", _p(x), x.shape[0], x.shape[1], _p(scales), 1 if divide else 0)
        return x

    @staticmethod
    def smooth_activations(acts: torch.Tensor, scales: torch.Tensor):
        """In place acts[t, j] /= max(scales[j], 1e-12)."""
        return SmoothQuantMigrator._apply(acts, scales, True)

    @staticmethod
    def smooth_weights(weights: torch.Tensor, scales: torch.Tensor):
        """In place weights[r, j] *= scales[j]."""
        return SmoothQuantMigrator._apply(weights, scales, False)

    def smooth_layer(self, acts: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """Smooths both matrices in place and returns the per-channel scales (smooth_quant.rs:274-293)."""
        sc = self.compute_migration_scales(self.compute_act_stats(acts), self.compute_weight_stats(weights))
        self.smooth_activations(acts, sc)
        self.smooth_weights(weights, sc)
        return sc


class GptqConfig:
    """GptqConfig of the reference (crates/oxicuda-quant/src/scheme/gptq.rs:30-54); block_size has no effect there or here."""

    def __init__(self, bits: int = 4, block_size: int = 128, percdamp: float = 0.01, symmetric: bool = True):
        self.bits, self.block_size, self.percdamp, self.symmetric = int(bits), int(block_size), float(percdamp), bool(symmetric)


class GptqOutput:
    """GptqOutput of the reference (gptq.rs:58-96) on device tensors: codes [n_rows, n_cols] i32, per-column scales and zero points."""

    def __init__(self, quantized, scales, zero_points, n_rows, n_cols):
        self.quantized, self.scales, self.zero_points, self.n_rows, self.n_cols = quantized, scales, zero_points, n_rows, n_cols

    def dequantize(self) -> torch.Tensor:
        return (self.quantized.to(torch.float32) - self.zero_points.to(torch.float32)[None, :]) * self.scales[None, :]

    def reconstruction_mse(self, original: torch.Tensor) -> float:
        return float(((self.dequantize() - original.reshape(self.n_rows, self.n_cols)) ** 2).mean())


class GptqQuantizer:
    """GptqQuantizer of the reference (gptq.rs:104-257) on device tensors; the whole layer is quantized on the GPU."""

    def __init__(self, config: GptqConfig | None = None):
        self.config = config or GptqConfig()
        self.workspace: torch.Tensor | None = None      # kept after a call: H^-1 and the factor's inverse, for inspection

    def quantize_layer(self, weights: torch.Tensor, n_rows: int, n_cols: int, hessian: torch.Tensor) -> GptqOutput:
        from .errors import QuantError
        if weights.numel() == 0:
            raise QuantError("EmptyInput", "GptqQuantizer::quantize_layer", 1)
        if weights.numel() != n_rows * n_cols:
            raise QuantError("DimensionMismatch", f"expected {n_rows * n_cols}, got {weights.numel()}", 4)
        if hessian.numel() != n_cols * n_cols:
            raise QuantError("DimensionMismatch", f"expected {n_cols * n_cols}, got {hessian.numel()}", 4)
        _chk(weights, torch.float32)
        _chk(hessian, torch.float32)
        dev = weights.device
        nbytes = C.c_size_t(0)
        raise_for_status(_ffi.load().oxq_gptq_workspace_bytes(n_rows, n_cols, C.byref(nbytes)))
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev)
        q = torch.empty((n_rows, n_cols), dtype=torch.int32, device=dev)
        sc = torch.empty(n_cols, dtype=torch.float32, device=dev)
        zp = torch.empty(n_cols, dtype=torch.int32, device=dev)
        info = torch.zeros(2, dtype=torch.int32, device=dev)
        handle(dev.index).call("oxq_gptq_quantize_layer", _p(weights), n_rows, n_cols, _p(hessian), self.config.bits,
                               1 if self.config.symmetric else 0, C.c_double(self.config.percdamp), _p(q), _p(sc), _p(zp), _p(info),
                               _p(ws), nbytes.value)
        host = info.cpu()                                 # the reference returns the error synchronously: wait for the stream
        if int(host[0]) != 0:
            raise QuantError("SingularHessian", f"min_diag = {float(host[1:2].view(torch.float32)[0]):.3e}", 7)
        self.workspace = ws
        return GptqOutput(q, sc, zp, n_rows, n_cols)


def bias_add_(y: torch.Tensor, bias: torch.Tensor):
    """In place y[m, n] += bias[n] (bf16 matrix, f32 bias)."""
    _chk(bias, torch.float32)
    handle(y.device.index).call("oxq_bias_add_bf16", _p(y), y.stride(0), _p(bias), y.shape[0], y.shape[1])
    return y


# ------------------------------------------------------------------------------------------- between two blocks

def _row_stride(t, shape):
    """Leading dimension of a matrix whose rows are adjacent elements."""
    if t.is_contiguous():
        return shape[1]
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1:
        raise TypeError("expected rows of adjacent elements")
    return stride[0] if shape[0] > 1 else max(stride[0], shape[1])


def _residual_norm_args(y, residual, weight, post_weight, gate, alpha, eps, residual_out):
    from .errors import QuantError
    shape, index = y.shape, y.get_device()
    if len(shape) != 2 or residual.shape != shape:
        raise QuantError("DimensionMismatch", f"y {tuple(shape)} vs residual {tuple(residual.shape)}", 4)
    rows, cols = shape
    dt = y.dtype
    if dt not in _DT or residual.dtype not in (dt, torch.float32):
        raise TypeError(f"y is f32, bf16 or f16 and residual the same or f32, got {dt} and {residual.dtype}")
    if index < 0 or residual.get_device() != index:
        raise TypeError("expected CUDA tensors on one device")
    for w in (weight, post_weight):
        if w is not None:
            if w.dtype is not torch.float32 or not w.is_contiguous() or w.get_device() != index:
                raise TypeError(f"expected contiguous float32 weights on {y.device}")
            if w.numel() != cols:
                raise QuantError("DimensionMismatch", f"expected {cols} weights, got {w.numel()}", 4)
    y_ld = _row_stride(y, shape)
    gate_ptr = gate_ld = 0
    if gate is not None:
        if gate.dtype != dt or tuple(gate.shape) not in ((cols,), (rows, cols)) or gate.get_device() != index:
            raise QuantError("DimensionMismatch", f"gate {tuple(gate.shape)} {gate.dtype} for y {tuple(shape)} {dt} on {y.device}", 4)
        if gate.dim() == 2:
            gate_ld = _row_stride(gate, shape)
        elif not gate.is_contiguous():
            raise TypeError("expected a gate of adjacent elements")
        gate_ptr = gate.data_ptr()
    r_ld = _row_stride(residual, shape)
    if residual_out is None:
        residual_out, ro_ld = torch.empty_like(residual) if r_ld == cols else residual.new_empty(shape), cols
    else:
        if residual_out.shape != shape or residual_out.dtype != residual.dtype or residual_out.get_device() != index:
            raise QuantError("DimensionMismatch", f"residual_out {tuple(residual_out.shape)} {residual_out.dtype} for {tuple(shape)} {residual.dtype} on {y.device}", 4)
        ro_ld = _row_stride(residual_out, shape)
    return residual_out, _ffi.residual_norm(y.data_ptr(), y_ld, _DT[dt], residual.data_ptr(), r_ld, _DT[residual.dtype], gate_ptr, gate_ld,
                                            0 if post_weight is None else post_weight.data_ptr(), weight.data_ptr(), alpha, eps, residual_out.data_ptr(), ro_ld)


def residual_rmsnorm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, post_weight: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, alpha: float = 1.0, residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """The seam between two blocks in one pass: t = y or rms(y; post_weight), t *= gate ([cols] or [rows, cols]), r = residual + alpha * t,
    h = rms(r; weight), RmsNorm::forward (crates/oxicuda-lm/src/layer/norm.rs:73-95) for rms.  Returns (r in residual's dtype, h in y's dtype);
    residual_out may be residual itself.  y, residual, residual_out and gate may be row-strided views."""
    r_out, args = _residual_norm_args(y, residual, weight, post_weight, gate, alpha, eps, residual_out)
    if out is None:
        out = torch.empty_like(y) if y.is_contiguous() else y.new_empty(y.shape)
    else:
        _chk(out, y.dtype)
        if out.shape != y.shape or out.device != y.device:
            raise TypeError(f"out must be {tuple(y.shape)} on {y.device}")
    handle(y.device.index).call("oxq_residual_rmsnorm", args, y.shape[0], y.shape[1], out.data_ptr())
    return r_out, out


def residual_rmsnorm_fp8(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, eps: float = 1e-5,
                         post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, alpha: float = 1.0,
                         residual_out: torch.Tensor | None = None):
    """residual_rmsnorm with h as E4M3 of h / scale[0] (the input of gemm_fp8): returns (r, codes uint8 [rows x cols])."""
    r_out, args = _residual_norm_args(y, residual, weight, post_weight, gate, alpha, eps, residual_out)
    if scale.dtype is not torch.float32 or scale.numel() < 1 or scale.get_device() != y.get_device():
        raise TypeError(f"expected a float32 scale on {y.device}")
    q = y.new_empty(y.shape, dtype=torch.uint8)
    handle(y.get_device()).call("oxq_residual_rmsnorm_fp8", args, y.shape[0], y.shape[1], scale.data_ptr(), q.data_ptr())
    return r_out, q


def residual_rmsnorm_int8_rows(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, post_weight: torch.Tensor | None = None,
                               gate: torch.Tensor | None = None, alpha: float = 1.0, residual_out: torch.Tensor | None = None):
    """residual_rmsnorm with h through the per-row INT8 quantizer (the input of gemm_w8a8): returns (r, codes int8 [rows x cols], scales f32 [rows])."""
    r_out, args = _residual_norm_args(y, residual, weight, post_weight, gate, alpha, eps, residual_out)
    q = y.new_empty(y.shape, dtype=torch.int8)
    sc = y.new_empty(y.shape[0], dtype=torch.float32)
    handle(y.get_device()).call("oxq_residual_rmsnorm_int8_rows", args, y.shape[0], y.shape[1], q.data_ptr(), sc.data_ptr())
    return r_out, q, sc


# ------------------------------------------------------------------------------------------- 4-bit key / value cache

_HALVES = (torch.bfloat16, torch.float16)


class Kv4Cache:
    """A paged pool of 4-bit keys and values: codes uint8 [pages, heads, page_size, dim / 2] and params f16 [pages, heads, page_size, dim / group, 2]
    (step and offset of each group of `group` elements), for keys and for values.  The affine per-group form of MinMaxQuantizer
    (crates/oxicuda-quant/src/scheme/minmax.rs:146-167, :226-232) with a float offset.  dim is 64 or 128, group 64 or 128, page_size a power of two
    from 16 to 4096."""

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "pages", "heads", "page_size", "dim", "group", "device", "_index", "_desc", "_shape")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor):
        cs, ps = k_codes.shape, k_params.shape
        if len(cs) != 4 or len(ps) != 5 or ps[4] != 2 or cs[:3] != ps[:3] or v_codes.shape != cs or v_params.shape != ps:
            from .errors import QuantError
            raise QuantError("DimensionMismatch", f"codes {tuple(cs)}, {tuple(v_codes.shape)} with params {tuple(ps)}, {tuple(v_params.shape)}", 4)
        index = k_codes.get_device()
        if index < 0:
            raise TypeError("expected CUDA tensors")
        if not (k_codes.dtype is v_codes.dtype is torch.uint8 and k_params.dtype is v_params.dtype is torch.float16):
            raise TypeError("expected uint8 codes and float16 params")
        if not (k_codes.is_contiguous() and v_codes.is_contiguous() and k_params.is_contiguous() and v_params.is_contiguous()):
            raise TypeError("expected contiguous tensors")
        if not (k_params.get_device() == v_codes.get_device() == v_params.get_device() == index):
            raise TypeError("expected tensors on one device")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.pages, self.heads, self.page_size, half = cs
        self.dim = 2 * half
        self.group = self.dim // ps[3] if ps[3] and self.dim % ps[3] == 0 else 0
        self.device, self._index = k_codes.device, index
        self._shape = (self.page_size, self.heads, self.dim, self.group)
        self._desc = _ffi.kv4_cache(k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), self.pages, self.page_size, self.heads,
                                    self.dim, self.group)

    @classmethod
    def empty(cls, pages: int, page_size: int, heads: int, dim: int, group: int = 64, device=None):
        """An uninitialised pool; nothing in it is read before it is written."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        codes = [torch.empty((pages, heads, page_size, dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
        params = [torch.empty((pages, heads, page_size, dim // max(group, 1), 2), dtype=torch.float16, device=device) for _ in range(2)]
        return cls(codes[0], params[0], codes[1], params[1])


def _kv4_batch(cache: Kv4Cache, block_table, seq_lens, cu_tokens, tokens: int) -> bytes:
    if not (block_table.dtype is seq_lens.dtype is cu_tokens.dtype is torch.int32):
        raise TypeError("block_table, seq_lens and cu_tokens are int32")
    shape, seqs = block_table.shape, seq_lens.numel()
    if len(shape) != 2 or shape[0] != seqs or cu_tokens.numel() != seqs + 1:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"block_table {tuple(shape)}, seq_lens {tuple(seq_lens.shape)}, cu_tokens {tuple(cu_tokens.shape)}", 4)
    if not (block_table.get_device() == seq_lens.get_device() == cu_tokens.get_device() == cache._index):
        raise TypeError(f"expected block_table, seq_lens and cu_tokens on {cache.device}")
    if not (block_table.is_contiguous() and seq_lens.is_contiguous() and cu_tokens.is_contiguous()):
        raise TypeError("expected contiguous block_table, seq_lens and cu_tokens")
    return _ffi.kv4_batch(block_table.data_ptr(), shape[1], seq_lens.data_ptr(), cu_tokens.data_ptr(), seqs, tokens)


def _kv4_rows(t: torch.Tensor, heads: int, cache: Kv4Cache, what: str, dtypes):
    """The tensor's token and head strides, if it is rows of the cache's kind."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != cache.dim:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"{what} {tuple(shape)}, expected [tokens, {heads}, {cache.dim}]", 4)
    if t.dtype not in dtypes:
        raise TypeError(f"{what}: expected dtype in {tuple(dtypes)}, got {t.dtype}")
    if t.get_device() != cache._index:
        raise TypeError(f"{what}: expected a tensor on {cache.device}")
    stride = t.stride()
    if stride[2] != 1:
        raise TypeError(f"{what}: expected rows of adjacent elements")
    return stride[0], stride[1]


@functools.lru_cache(maxsize=4096)
def _kv4_workspace(device_index: int, cache_shape: tuple, width: int, seqs: int, tokens: int, q_heads: int, max_tokens: int) -> int:
    """A size: it follows from the shapes alone, so it is asked for once."""
    cache = _ffi.kv4_cache(256, 256, 256, 256, 1, *cache_shape)
    batch = _ffi.kv4_batch(256, width, 256, 256, seqs, tokens)
    n = C.c_size_t(0)
    handle(device_index).call("oxq_kv4_attention_workspace_bytes", cache, batch, q_heads, max_tokens, C.byref(n))
    return n.value


def kv4_append(cache: Kv4Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_tokens: torch.Tensor):
    """Quantises keys and values [tokens, heads, dim] (f32, bf16 or f16; any token and head strides) into the pool.  Sequence b owns tokens
    cu_tokens[b]:cu_tokens[b + 1], its last ones of seq_lens[b]; position p lives in page block_table[b, p // page_size].  Rows behind the last
    sequence are not read."""
    kt, kh = _kv4_rows(k, cache.heads, cache, "k", _DT)
    vt, vh = _kv4_rows(v, cache.heads, cache, "v", (k.dtype,))
    if v.shape != k.shape:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"k {tuple(k.shape)} vs v {tuple(v.shape)}", 4)
    batch = _kv4_batch(cache, block_table, seq_lens, cu_tokens, k.shape[0])
    handle(cache._index).call("oxq_kv4_append", cache._desc, batch, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _DT[k.dtype])
    return cache


def kv4_read(cache: Kv4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_tokens: torch.Tensor, tokens: int, dtype=torch.bfloat16,
             k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
    """The last cu_tokens[b + 1] - cu_tokens[b] tokens of every sequence as (k, v) [tokens, heads, dim]; rows behind the last sequence are left as
    they were (uninitialised where the call allocates)."""
    shape = (int(tokens), cache.heads, cache.dim)
    outs = []
    for t, what in ((k_out, "k_out"), (v_out, "v_out")):
        if t is None:
            t = cache.k_codes.new_empty(shape, dtype=dtype)
        else:
            _kv4_rows(t, cache.heads, cache, what, (dtype,))
            if t.shape[0] != shape[0] or not t.is_contiguous():
                raise TypeError(f"{what}: expected a contiguous tensor of {shape}")
        outs.append(t)
    batch = _kv4_batch(cache, block_table, seq_lens, cu_tokens, shape[0])
    handle(cache._index).call("oxq_kv4_read", cache._desc, batch, outs[0].data_ptr(), outs[1].data_ptr(), _DT[dtype])
    return outs[0], outs[1]


def kv4_attention_workspace_bytes(cache: Kv4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_tokens: torch.Tensor, tokens: int, q_heads: int,
                                  max_tokens: int = 0) -> int:
    """Bytes of workspace that kv4_attention needs for `tokens` rows of q_heads heads; depends on the arguments' shapes only, not on their contents."""
    _kv4_batch(cache, block_table, seq_lens, cu_tokens, tokens)
    return _kv4_workspace(cache._index, cache._shape, block_table.shape[1], seq_lens.numel(), tokens, q_heads, max_tokens)


def kv4_attention(q: torch.Tensor, cache: Kv4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_tokens: torch.Tensor, max_tokens: int = 0,
                  scale: float | None = None, causal: bool = True, window: int = 0, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                  want_lse: bool = False, workspace: torch.Tensor | None = None):
    """Attention of queries [tokens, q_heads, dim] (bf16 or f16; any token and head strides) over what the pool holds: softmax(scale * q . k) v, scale
    dim ** -0.5 unless given, over the keys up to each query's own position (causal; the last `window` of them if window > 0) or all of its sequence.
    A query that sees no key gives zeros (and -inf in lse).  max_tokens: the most tokens a sequence has in this call, 0 if it is not known; it
    only chooses kernels.  Returns out, or (out, lse f32 [tokens, q_heads]) if want_lse or lse is given.  Rows behind the last sequence
    are left as they were.  `out` must not lie over the queries.  `workspace` (uint8, kv4_attention_workspace_bytes) may be given to allocate nothing;
    overlapping calls need one each."""
    shape = q.shape
    if len(shape) != 3 or shape[1] == 0 or cache.heads == 0 or shape[1] % cache.heads != 0:
        from .errors import QuantError
        raise QuantError("DimensionMismatch", f"q {tuple(shape)} over {cache.heads} kv heads", 4)
    tokens, heads = shape[0], shape[1]
    qt, qh = _kv4_rows(q, heads, cache, "q", _HALVES)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        ot, oh = heads * cache.dim, cache.dim
    else:
        ot, oh = _kv4_rows(out, heads, cache, "out", (q.dtype,))
        if out.shape[0] != tokens:
            raise TypeError(f"out: expected {tokens} tokens, got {out.shape[0]}")
    if lse is not None:
        _chk(lse, torch.float32)
        if tuple(lse.shape) != (tokens, heads) or lse.get_device() != cache._index:
            raise TypeError(f"lse: expected {(tokens, heads)} on {cache.device}")
    elif want_lse:
        lse = q.new_empty((tokens, heads), dtype=torch.float32)
    batch = _kv4_batch(cache, block_table, seq_lens, cu_tokens, tokens)
    if workspace is None:
        n = _kv4_workspace(cache._index, cache._shape, block_table.shape[1], seq_lens.numel(), tokens, heads, max_tokens)
        workspace = cache.k_codes.new_empty(max(n, 16))
    else:
        _chk(workspace, torch.uint8)
        if workspace.get_device() != cache._index:
            raise TypeError(f"workspace: expected a tensor on {cache.device}")
        n = workspace.numel()
    args = _ffi.kv4_attention_args(q.data_ptr(), qt, qh, out.data_ptr(), ot, oh, 0 if lse is None else lse.data_ptr(), heads, max_tokens, window,
                                   cache.dim ** -0.5 if scale is None else scale, 1 if causal else 0, _DT[q.dtype])
    handle(cache._index).call("oxq_kv4_attention", cache._desc, batch, args, workspace.data_ptr(), n)
    return out if lse is None else (out, lse)


# ------------------------------------------------------------------------------------------- GEMMs

def gemm_fp8(x_q, w_q, sx, sw, out: torch.Tensor | None = None):
    """Y = bf16((X . W^T) * sx * sw); x_q [M x K] u8, w_q [N x K] u8 (E4M3 bytes)."""
    m, k = x_q.shape
    n = w_q.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    handle(x_q.device.index).call("oxq_gemm_fp8", m, n, k, _p(x_q), x_q.stride(0), _p(w_q), w_q.stride(0), _p(sx), _p(sw),
                                  _p(y), y.stride(0))
    return y


def gemm_fp8_ex(alpha: float, x_q, w_q, sx, sw, beta: float, y: torch.Tensor):
    """In place Y = alpha * (X . W^T) * sx * sw + beta * Y (gemm's general form, crates/oxicuda-blas/src/level3/gemm_api.rs:73-82)."""
    m, k = x_q.shape
    n = w_q.shape[0]
    handle(x_q.device.index).call("oxq_gemm_fp8_ex", m, n, k, C.c_float(alpha), _p(x_q), x_q.stride(0), _p(w_q), w_q.stride(0), _p(sx), _p(sw),
                                  C.c_float(beta), _p(y), y.stride(0))
    return y


def gemm_bf16_ex(alpha: float, x, w, beta: float, y: torch.Tensor):
    """In place Y = alpha * (X . W^T) + beta * Y on bf16 matrices."""
    m, k = x.shape
    n = w.shape[0]
    handle(x.device.index).call("oxq_gemm_bf16_ex", m, n, k, C.c_float(alpha), _p(x), x.stride(0), _p(w), w.stride(0), C.c_float(beta), _p(y), y.stride(0))
    return y


OP_K_MAJOR, OP_MN_MAJOR = 0, 1


def gemm_fp8_op(m: int, n: int, k: int, alpha: float, a, a_major: int, b, b_major: int, sa, sb, beta: float, y: torch.Tensor):
    """gemm's operand forms (crates/oxicuda-blas/src/level3/gemm_api.rs:73-82) for E4M3 operands: a is [m x k] (K-major) or
    [k x m] (MN-major) in memory, b is [n x k] (K-major) or [k x n] (MN-major); y [m x n] bf16 is updated in place."""
    handle(a.device.index).call("oxq_gemm_fp8_op", m, n, k, C.c_float(alpha), _p(a), a.stride(0), a_major, _p(b), b.stride(0), b_major,
                                _p(sa), _p(sb), C.c_float(beta), _p(y), y.stride(0))
    return y


def gemm_bf16_op(m: int, n: int, k: int, alpha: float, a, a_major: int, b, b_major: int, beta: float, y: torch.Tensor):
    handle(a.device.index).call("oxq_gemm_bf16_op", m, n, k, C.c_float(alpha), _p(a), a.stride(0), a_major, _p(b), b.stride(0), b_major,
                                C.c_float(beta), _p(y), y.stride(0))
    return y


def gemm_fp8_swiglu(x_q, w_gu_q, sx, sw, out: torch.Tensor | None = None):
    """H = bf16(silu(g) * u); w_gu_q holds gate/up rows interleaved in blocks of 128 (see interleave_gate_up)."""
    m, k = x_q.shape
    n2 = w_gu_q.shape[0]
    y = torch.empty((m, n2 // 2), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    handle(x_q.device.index).call("oxq_gemm_fp8_swiglu", m, n2, k, _p(x_q), x_q.stride(0), _p(w_gu_q), w_gu_q.stride(0),
                                  _p(sx), _p(sw), _p(y), y.stride(0))
    return y


def gemm_bf16(x, w, out: torch.Tensor | None = None):
    m, k = x.shape
    n = w.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_gemm_bf16", m, n, k, _p(x), x.stride(0), _p(w), w.stride(0), _p(y), y.stride(0))
    return y


def gemm_bf16_swiglu(x, w_gu, out: torch.Tensor | None = None):
    m, k = x.shape
    n2 = w_gu.shape[0]
    y = torch.empty((m, n2 // 2), dtype=torch.bfloat16, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_gemm_bf16_swiglu", m, n2, k, _p(x), x.stride(0), _p(w_gu), w_gu.stride(0), _p(y),
                                y.stride(0))
    return y


def swiglu_interleaved(gu: torch.Tensor, out: torch.Tensor | None = None):
    """gu [m x 2n] bf16 in interleaved 128-column blocks -> silu(gate) * up [m x n]."""
    m, n2 = gu.shape
    y = torch.empty((m, n2 // 2), dtype=torch.bfloat16, device=gu.device) if out is None else out
    handle(gu.device.index).call("oxq_swiglu_interleaved", _p(gu), m, n2 // 2, _p(y))
    return y


def interleave_gate_up(w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """[inter x k] gate and up weights -> [2*inter x k] with blocks of 128 gate rows followed by the 128 matching
    up rows (a one-off, load-time layout change; inter must be a multiple of 128)."""
    inter, k = w_gate.shape
    assert inter % 128 == 0 and w_up.shape == w_gate.shape
    g = w_gate.reshape(inter // 128, 128, k)
    u = w_up.reshape(inter // 128, 128, k)
    return torch.stack([g, u], dim=1).reshape(2 * inter, k).contiguous()


def gemm_w8a8(x_q, w_q, sx_rows, sw_rows, out: torch.Tensor | None = None):
    m, k = x_q.shape
    n = w_q.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x_q.device) if out is None else out
    handle(x_q.device.index).call("oxq_gemm_w8a8", m, n, k, _p(x_q), x_q.stride(0), _p(w_q), w_q.stride(0), _p(sx_rows),
                                  _p(sw_rows), _p(y), y.stride(0))
    return y


def gemm_w8a32(x, w_q, sw_rows):
    m, k = x.shape
    n = w_q.shape[0]
    y = torch.empty((m, n), dtype=torch.float32, device=x.device)
    handle(x.device.index).call("oxq_gemm_w8a32", m, n, k, _p(x), _p(w_q), _p(sw_rows), _p(y))
    return y


def gemm_w4a16_workspace(m: int, n: int, k: int, device) -> torch.Tensor:
    """Zero-filled workspace; every call leaves it zero-filled again, so it can be reused."""
    nbytes = int(_ffi.load().oxq_gemm_w4a16_workspace_bytes(m, n, k))
    return torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)


def gemm_w4a16(x, codes, scales, zeros, group: int = 128, workspace: torch.Tensor | None = None,
               out: torch.Tensor | None = None):
    m, k = x.shape
    n = codes.shape[0]
    ws = gemm_w4a16_workspace(m, n, k, x.device) if workspace is None else workspace
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x.device) if out is None else out
    handle(x.device.index).call("oxq_gemm_w4a16", m, n, k, _p(x), _p(codes), _p(scales), _p(zeros), group, _p(y), _p(ws),
                                ws.numel())
    return y


def gemm_mxfp8(x_codes, x_sf_mma, w_codes, w_sf_mma, out: torch.Tensor | None = None):
    m, k = x_codes.shape
    n = w_codes.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x_codes.device) if out is None else out
    handle(x_codes.device.index).call("oxq_gemm_mxfp8", m, n, k, _p(x_codes), _p(x_sf_mma), _p(w_codes), _p(w_sf_mma),
                                      _p(y), y.stride(0))
    return y


def gemm_nvfp4(x_packed, x_sf_mma, x_stats, w_packed, w_sf_mma, w_stats, out: torch.Tensor | None = None):
    """x_stats / w_stats are the 2-float tensors of nvfp4_quant; element 1 is the tensor scale."""
    m, k = x_packed.shape[0], x_packed.shape[1] * 2
    n = w_packed.shape[0]
    y = torch.empty((m, n), dtype=torch.bfloat16, device=x_packed.device) if out is None else out
    handle(x_packed.device.index).call("oxq_gemm_nvfp4", m, n, k, _p(x_packed), _p(x_sf_mma), _p(x_stats[1:]),
                                       _p(w_packed), _p(w_sf_mma), _p(w_stats[1:]), _p(y), y.stride(0))
    return y


# ------------------------------------------------------------------------------------------- collective

def multimem_all_reduce_bf16(multicast_ptr: int, numel: int, rank: int, world: int, device_index: int | None = None):
    """In-place all-reduce over the multicast mapping of a symmetric bf16 buffer; the caller provides the barriers."""
    handle(device_index).call("oxq_multimem_all_reduce_bf16", C.c_void_p(multicast_ptr), numel, rank, world)


def multimem_all_reduce_bf16_2d_sync(multicast_ptr: int, rows: int, cols: int, ld: int, rank: int, world: int, flags_local: torch.Tensor,
                                     flags_multicast_ptr: int, device_index: int | None = None):
    """In-place all-reduce of a column block of a symmetric bf16 matrix with the cross-rank synchronisation inside the kernel."""
    handle(device_index).call("oxq_multimem_all_reduce_bf16_2d_sync", C.c_void_p(multicast_ptr), rows, cols, ld, rank, world, _p(flags_local),
                              C.c_void_p(flags_multicast_ptr))


def gemm_fp8_all_reduce(x_q, w_q, sx, sw, y_local: torch.Tensor, y_multicast_ptr: int, flags_local: torch.Tensor, flags_multicast_ptr: int,
                        rank: int, world: int):
    """FP8 GEMM of this rank's K-shard with the all-reduce over the ranks fused in (RowLinear::forward_partial + all_reduce):
    y_local is this rank's [m x n] view of a symmetric bf16 buffer, flags_local its int32 flag words (zero before the first
    call); the *_multicast_ptr arguments are the multicast addresses of the same two buffers."""
    m, k = x_q.shape
    n = w_q.shape[0]
    handle(x_q.device.index).call("oxq_gemm_fp8_all_reduce", m, n, k, _p(x_q), x_q.stride(0), _p(w_q), w_q.stride(0), _p(sx), _p(sw), _p(y_local),
                                  C.c_void_p(y_multicast_ptr), y_local.stride(0), _p(flags_local), C.c_void_p(flags_multicast_ptr),
                                  flags_local.numel(), rank, world)
    return y_local


def multimem_all_reduce_bf16_2d(multicast_ptr: int, rows: int, cols: int, ld: int, rank: int, world: int, device_index: int | None = None):
    """In-place all-reduce of a [rows x cols] column block (leading dimension ld) of a symmetric bf16 matrix."""
    handle(device_index).call("oxq_multimem_all_reduce_bf16_2d", C.c_void_p(multicast_ptr), rows, cols, ld, rank, world)
