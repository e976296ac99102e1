"""Dense products with 4-bit weights for 1..16 rows over the C ABI (dsgx_linear_decode), torch tensors as device memory.

The engines' products with INT4 matrices outside the experts (altar1 engine/attn/attn.h): projections, dense FFN layers and
heads, next to the experts of moe.py.

    w = linear.LinearW(N, K, torch.from_numpy(weights.pack_linear_int4(codes, scales, zeros)).cuda())
    y = linear.linear_decode(w, x)                        # bf16 [M][N] = x W^T
    y = linear.linear_decode(w, x, res=r)                 # + r, one rounding
    h = linear.linear_decode(linear.LinearW(N, K, gate, up=up), x)   # silu(x Wg^T) * (x Wu^T)
"""
import ctypes as C

import torch

from . import _lib
from ._lib import check, lib
from .moe import raw_stream


class LinearW:
    """An INT4-g32 matrix [N][K], or a gate / up pair, prepared for linear_decode from the experts' blocks of 8 rows x 512 k on
    the device (weights.pack_linear_int4).  The prepared copy is made once, on the current stream; the blocks are not kept.
    status: an int32 word on the device, 0 until a bounded wait of one of its products runs out (DSGX_ERR_DEVICE_WAIT; that product's
    outputs are undefined); it stays until it is cleared."""

    def __init__(self, N, K, blocks, up=None):
        if N < 1 or K < 1:
            raise ValueError(f"LinearW: N = {N}, K = {K}")
        need = -(-N // 8) * -(-K // 512) * 2368
        for b in (blocks,) if up is None else (blocks, up):
            if b.dtype != torch.uint8 or not b.is_contiguous() or b.numel() != need or not b.is_cuda:
                raise ValueError(f"LinearW: {need} contiguous bytes on the device are wanted for [{N}][{K}], got {b.numel()} of {b.dtype} on {b.device}")
        if up is not None and up.device != blocks.device:
            raise ValueError("LinearW: the two matrices are on different devices")
        self.N, self.K, self.glu, self.device = N, K, up is not None, blocks.device
        with torch.cuda.device(self.device):
            self.data = torch.empty(lib().dsgx_linear_bytes(N, K, int(self.glu)), dtype=torch.uint8, device=self.device)
            self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
            check(lib().dsgx_linear_prepare(blocks.data_ptr(), up.data_ptr() if self.glu else None, _lib.FMT_INT4, N, K, self.data.data_ptr(),
                                            torch.cuda.current_stream(self.device).cuda_stream), "dsgx_linear_prepare")
        self.c = _lib.LinearW(self.data.data_ptr(), N, K, _lib.FMT_INT4, int(self.glu))
        self.ref, self.status_ptr = C.byref(self.c), self.status.data_ptr()


def _lead(t, M, width, what, device):
    """The leading dimension of a [M][width] operand, checked."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != M or shape[1] != width or t.device != device:
        raise ValueError(f"linear_decode: {what} {tuple(shape)} on {t.device}; wanted ({M}, {width}) on {device}")
    s0, s1 = t.stride()
    if (s1 != 1 and width > 1) or (s0 < width and M > 1):
        raise ValueError(f"linear_decode: {what} has strides {(s0, s1)}: the last dimension must be contiguous, rows apart")
    return s0 if s0 > width else width


def linear_decode(w, x, res=None, out=None, out_dtype=torch.bfloat16, status=None):
    """x bf16 [M][K], M = 1..16 -> out [M][N] (bf16 or f32): x W^T (+ res bf16 [M][N]), or silu(x W^T) * (x Wup^T) where w has
    an `up` matrix.  x, res and out may be rows of larger tensors (last dimension contiguous); out may be res (bf16, the same rows), and
    shares no memory with x or res otherwise.
    status: an int32 device tensor that gets DSGX_ERR_DEVICE_WAIT where a bounded wait ran out (default: w.status)."""
    dev, bf16 = w.device, torch.bfloat16
    if x.dtype is not bf16 or (res is not None and res.dtype is not bf16):
        raise ValueError(f"linear_decode: x {x.dtype}, res {None if res is None else res.dtype}; wanted bf16")
    if x.dim() != 2 or not 1 <= x.shape[0] <= _lib.MAX_STEP_ROWS:
        raise ValueError(f"linear_decode: x has shape {tuple(x.shape)}; 1..{_lib.MAX_STEP_ROWS} rows of {w.K} are taken")
    M = x.shape[0]
    ldx = _lead(x, M, w.K, "x", dev)
    if out is None:
        out, ldo = (x.new_empty(M, w.N) if out_dtype is bf16 else torch.empty(M, w.N, dtype=out_dtype, device=dev)), w.N
    else:
        ldo = _lead(out, M, w.N, "out", dev)
    if out.dtype is not bf16 and out.dtype is not torch.float32:
        raise ValueError(f"linear_decode: out {out.dtype}; wanted bf16 or f32")
    ldr, resp = (0, None) if res is None else (_lead(res, M, w.N, "res", dev), res.data_ptr())
    if status is not None and (status.dtype != torch.int32 or status.device != dev or status.numel() < 1):
        raise ValueError("linear_decode: status is an int32 tensor on the weights' device")
    args = (w.ref, x.data_ptr(), ldx, M, resp, ldr, out.data_ptr(), ldo, 0 if out.dtype is bf16 else 1,
            w.status_ptr if status is None else status.data_ptr())
    if torch.cuda.current_device() == dev.index:
        rc = _decode()(*args, raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = _decode()(*args, raw_stream(dev.index))
    if rc:
        check(rc, "dsgx_linear_decode")
    return out


_fn = None


def _decode():
    global _fn
    if _fn is None:
        _fn = lib().dsgx_linear_decode
    return _fn
