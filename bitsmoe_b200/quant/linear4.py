"""Weight matrices of dense Linear modules in 4 bits: signed codes and one fp16 scale for every ``group_size`` columns of a row, as
``bitsmoe_b200.layer.linear4`` and ``dense_mlp4`` read them.

The reference keeps everything but the routed experts in 16 bits (bitsmoe/models/qwen3next/bitsmoe_block.py:144-147 runs its shared
expert as torch modules); at decode sizes those weights are then most of what a layer reads.

Format: ``payload`` uint32 [N, 4 * ceil(K / 32)], the code of column 8 j + i (-8 .. 7, stored + 8) in bits 4 i .. 4 i + 3 of word j of its
row, rows padded with code 0; ``scale`` fp16 [N, ceil(K / group_size)]; the last group of a row may be short.
"""
from __future__ import annotations

from typing import Tuple

import torch
import torch.nn as nn

GROUP_SIZES = (32, 64, 128)


def _row_words(k: int) -> int:
    return 4 * (-(-k // 32))


def pack_codes4(codes: torch.Tensor) -> torch.Tensor:
    """int8 codes [N, K] in -8 .. 7 -> payload uint32 [N, 4 * ceil(K / 32)]."""
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise ValueError("pack_codes4 expects int8 codes [N, K]")
    n, k = codes.shape
    u = torch.full((n, _row_words(k) * 8), 8, dtype=torch.int32, device=codes.device)
    u[:, :k] = codes.to(torch.int32) + 8
    u = u.reshape(n, -1, 8)
    words = u[..., 0].clone()
    for i in range(1, 8):
        words |= u[..., i] << (4 * i)
    return words.view(torch.uint32)


def unpack_codes4(payload: torch.Tensor, k: int) -> torch.Tensor:
    """payload uint32 [N, words] -> int8 codes [N, k]."""
    words = payload.view(torch.int32)
    codes = torch.stack([((words >> (4 * i)) & 15) - 8 for i in range(8)], dim=-1)
    return codes.reshape(payload.shape[0], -1)[:, :k].to(torch.int8)


def _quantize_groups(x: torch.Tensor, iters: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and fp16 scales of the last axis' vectors.  The scale starts where 7.5 steps reach the largest magnitude and is then fitted
    to the codes by least squares in turn with them, as ``quantize_symmetric`` does from the mean magnitude: a group of 32 to 128
    normal values keeps all 16 codes (relative error 0.08 to 0.11) where that start leaves six or seven of them (0.19)."""
    scale = (x.abs().amax(dim=-1, keepdim=True) / 7.5).half().float()
    codes, best = None, None
    for _ in range(iters + 1):
        # codes for the scale as it is stored; a group of zeros (or of values below fp16's range) has scale 0 and codes 0
        q = torch.clamp(torch.round(x / torch.where(scale > 0, scale, 1.0)), -8, 7)
        q = torch.where(scale > 0, q, torch.zeros_like(q))
        err = (x - q * scale).square().sum(dim=-1, keepdim=True)
        if best is None:
            codes, best, kept = q, err, scale
        else:
            better = err < best
            codes, best, kept = torch.where(better, q, codes), torch.where(better, err, best), torch.where(better, scale, kept)
        qq = q.square().sum(dim=-1, keepdim=True)
        scale = torch.where(qq > 0, (x * q).sum(dim=-1, keepdim=True) / qq.clamp(min=1.0), scale).half().float()
    return codes.to(torch.int8), kept.squeeze(-1).half()


def quantize_linear4(weight: torch.Tensor, group_size: int = 128, iters: int = 10) -> Tuple[torch.Tensor, torch.Tensor]:
    """weight [N, K] -> (payload, scale), every group of ``group_size`` columns of a row on its own."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"quantize_linear4 expects a 2D weight, got shape={tuple(weight.shape)}")
    n, k = weight.shape
    whole = k // group_size * group_size
    payload = torch.empty((n, _row_words(k)), dtype=torch.uint32, device=weight.device)
    scale = torch.empty((n, -(-k // group_size)), dtype=torch.float16, device=weight.device)
    step = max(1, (1 << 24) // k)
    for r in range(0, n, step):
        w = weight.detach()[r:r + step].float()
        codes = torch.empty(w.shape, dtype=torch.int8, device=w.device)
        if whole:
            q, s = _quantize_groups(w[:, :whole].reshape(w.shape[0], -1, group_size), iters)
            codes[:, :whole] = q.reshape(w.shape[0], whole)
            scale[r:r + step, :whole // group_size] = s
        if whole < k:
            codes[:, whole:], scale[r:r + step, -1] = _quantize_groups(w[:, whole:], iters)
        payload[r:r + step].view(torch.int32).copy_(pack_codes4(codes).view(torch.int32))
    return payload, scale


def dequantize_linear4(payload: torch.Tensor, scale: torch.Tensor, k: int, group_size: int = 128) -> torch.Tensor:
    """The matrix that (payload, scale) stands for, fp32 [N, k]."""
    return unpack_codes4(payload, k).float() * scale.float().repeat_interleave(group_size, dim=1)[:, :k]


class Linear4(nn.Module):
    """A bias-free Linear whose weight is held in 4 bits (buffers ``payload`` and ``scale``); inference on the GPU only."""

    def __init__(self, in_features: int, out_features: int, group_size: int = 128, device=None):
        super().__init__()
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
        self.in_features, self.out_features, self.group_size = int(in_features), int(out_features), int(group_size)
        self.register_buffer("payload", torch.empty((out_features, _row_words(in_features)), dtype=torch.uint32, device=device))
        self.register_buffer("scale", torch.empty((out_features, -(-in_features // group_size)), dtype=torch.float16, device=device))

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 128, iters: int = 10) -> "Linear4":
        if not isinstance(linear, nn.Linear) or linear.bias is not None:
            raise ValueError("Linear4.from_linear expects a bias-free nn.Linear")
        m = cls(linear.in_features, linear.out_features, group_size, device=linear.weight.device)
        m.payload, m.scale = quantize_linear4(linear.weight, group_size, iters)
        return m

    def packed(self) -> Tuple[torch.Tensor, torch.Tensor]:
        return self.payload, self.scale

    def _apply(self, fn, recurse=True):
        # .half() / .bfloat16() / .to(dtype) of a surrounding module must not touch the scales: they are fp16 by format
        kept = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float16:
            self.scale = kept.to(device=self.scale.device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from bitsmoe_b200.layer import linear4
        y = linear4(x.reshape(-1, self.in_features), self.payload, self.scale, self.group_size)
        return y.reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group_size={self.group_size}"
