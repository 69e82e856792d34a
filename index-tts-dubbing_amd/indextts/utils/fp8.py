"""Linear layers in block-scaled 8-bit floating point (csrc/fp8_linear.hip).

Weights and activations are held as e4m3 codes with one power-of-two scale per 128 consecutive values along the
reduction (include/itts_hip.h: "8-bit operators"); products accumulate in f32.  The weights are quantised once
(``Fp8Linear.from_weight``), the activations within the call.  Beside ``HipLinearBank`` (bf16 operands): half the
weight bytes and twice the matrix rate, at e4m3's half step of 2^-4 per value.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _hip

BLOCK = 128
_CODE = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16}


@lru_cache(4096)
def _workspace_bytes(M: int, N: int, K: int) -> int:
    return _hip.load().itts_fp8_linear_workspace_bytes(M, N, K)


def quant_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] f32 or bf16 on the GPU (unit column stride) -> (codes [M, K rounded up to 128] uint8, scale bytes
    [M, K / 128 rounded up to whole dwords] uint8); view the codes as ``torch.float8_e4m3fn`` for their values."""
    if x.dim() != 2 or x.dtype not in _CODE or not x.is_cuda:
        raise ValueError(f"x must be [M, K] f32 or bf16 on the GPU, got {tuple(x.shape)} {x.dtype} on {x.device}")
    M, K = x.shape
    if K < 1:
        raise ValueError("K must be at least 1")
    if x.stride(1) != 1 and K > 1 or x.stride(0) < K and M > 1:
        x = x.contiguous()
    lib = _hip.load()
    kp = -(-K // BLOCK) * BLOCK
    sp = -(-(kp // BLOCK) // 4) * 4
    q = torch.empty(M, kp, dtype=torch.uint8, device=x.device)
    s = torch.empty(M, sp, dtype=torch.uint8, device=x.device)
    _hip.check(lib.itts_fp8_quant_rows(x.data_ptr(), max(x.stride(0), K), _CODE[x.dtype], M, K, q.data_ptr(), kp,
                                       s.data_ptr(), sp, _hip.current_stream_of(x.get_device())), "itts_fp8_quant_rows")
    return q, s


class Fp8Linear:
    """``layer(x)`` = ``F.linear`` of the quantised x and weight (+ bias) for x [..., K] f32 or bf16.

    codes [N, K rounded up to 128] and scales [N, K / 128 rounded up to whole dwords] as ``quant_rows`` gives them (both
    uint8, contiguous); they are held, not copied.  bias [N] f32."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, in_features: int, bias: Optional[torch.Tensor] = None):
        K = int(in_features)
        kp = -(-K // BLOCK) * BLOCK
        sp = -(-(kp // BLOCK) // 4) * 4
        if K < 1 or codes.dim() != 2 or codes.shape[0] < 1 or codes.shape[1] != kp:
            raise ValueError(f"codes must be [N, {kp}] for {K} input features, got {tuple(codes.shape)}")
        N = codes.shape[0]
        if tuple(scales.shape) != (N, sp):
            raise ValueError(f"scales must be [{N}, {sp}], got {tuple(scales.shape)}")
        for t in (codes, scales):
            if t.dtype != torch.uint8 or not t.is_cuda or not t.is_contiguous() or t.device != codes.device:
                raise ValueError("codes and scales must be contiguous uint8 tensors on one GPU")
        if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype != torch.float32 or not bias.is_contiguous()
                                 or bias.device != codes.device):
            raise ValueError(f"bias must be [{N}] f32, contiguous, on {codes.device}")
        self.codes, self.scales, self.bias = codes, scales, bias
        self.in_features, self.out_features, self.dev, self.index = K, N, codes.device, codes.get_device()
        self.lib = _hip.load()
        self._w = (codes.data_ptr(), kp, scales.data_ptr(), sp, _hip.ptr(bias))

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "Fp8Linear":
        """weight [N, K] f32 or bf16 on the GPU, quantised here; bias [N] (any float dtype)."""
        q, s = quant_rows(weight)
        return cls(q, s, weight.shape[1], None if bias is None else bias.detach().float().contiguous().to(q.device))

    def __call__(self, x: torch.Tensor, act: int = 0, residual: Optional[torch.Tensor] = None, bf16_out: bool = False,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """act(x @ W^T + b) (+ residual); act 0 none, 1 gelu_tanh, 2 SiLU; y f32, or bf16 with ``bf16_out``;
        residual f32 [..., N], contiguous, may be ``out`` itself; ``out`` must not overlap x, nor residual otherwise."""
        K, N, dev = self.in_features, self.out_features, self.index
        shape = x.shape
        xd = _CODE.get(x.dtype)
        if xd is None or not shape or shape[-1] != K or x.get_device() != dev:
            raise ValueError(f"x must be [..., {K}] f32 or bf16 on {self.dev}, got {tuple(shape)} {x.dtype} on {x.device}")
        ys = (*shape[:-1], N)
        if len(shape) != 2:
            x = x.reshape(-1, K)
        M = x.shape[0]
        ldx = x.stride(0) if M > 1 else K
        if K > 1 and x.stride(1) != 1 or ldx < K:
            x = x.contiguous()
            ldx = K
        dt, yd = (torch.bfloat16, _hip.BF16) if bf16_out else (torch.float32, _hip.F32)
        if out is None:
            y = x.new_empty(ys, dtype=dt)
        else:
            y = out
            if y.dtype != dt or y.shape != ys or not y.is_contiguous() or y.get_device() != dev:
                raise ValueError(f"out must be a contiguous {dt} tensor of {ys} on {self.dev}")
            if M and x.data_ptr() < y.data_ptr() + M * N * y.element_size() and \
                    y.data_ptr() < x.data_ptr() + ((M - 1) * ldx + K) * x.element_size():
                raise ValueError("out must not overlap x: other columns of a row still read it")
        res = None
        if residual is not None:
            if residual.dtype != torch.float32 or residual.shape != ys or not residual.is_contiguous() or \
                    residual.get_device() != dev:
                raise ValueError(f"residual must be a contiguous f32 tensor of {ys} on {self.dev}")
            res = residual.data_ptr()
            if out is not None and M and (res != y.data_ptr() or bf16_out):  # out itself: each value is read where it is written
                if res < y.data_ptr() + M * N * y.element_size() and y.data_ptr() < res + M * N * 4:
                    raise ValueError("residual must be out itself or not overlap it")
        if M == 0:
            return y
        n = _workspace_bytes(M, N, K)
        ws = x.new_empty(n, dtype=torch.uint8) if n > 0 else None
        wq, ldw, wsc, lds, b = self._w
        rc = self.lib.itts_fp8_linear(x.data_ptr(), ldx, xd, M, K, wq, ldw, wsc, lds, N, b, act, res, N, y.data_ptr(), N, yd,
                                      None if ws is None else ws.data_ptr(), _hip.current_stream_of(dev))
        if rc:
            _hip.check(rc, "itts_fp8_linear")
        return y
