"""Argument checks shared by the operators that branch and trim the INT4 cache."""

from __future__ import annotations

import math

import torch

from kvint4._lib import binding

FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def check_rows(what: str, k_packed, k_scales, v_packed, v_scales) -> None:
    """Four tensors of packed K/V rows: dtypes, ranks, and shapes that agree."""
    ts = (k_packed, k_scales, v_packed, v_scales)
    if any(t.dim() != 4 for t in ts):
        raise ValueError(f"{what} tensors must be 4D: [B, n_kv_heads, tokens, ...]")
    if k_packed.dtype != torch.uint8 or v_packed.dtype != torch.uint8:
        raise ValueError(f"{what}: packed tensors must be uint8")
    if k_scales.dtype not in FLOATS or v_scales.dtype != k_scales.dtype:
        raise ValueError(f"{what}: scales must be bf16/fp16/fp32, K and V alike")
    if k_packed.shape != v_packed.shape or k_scales.shape != v_scales.shape:
        raise ValueError(f"{what}: K and V must have the same shapes")
    if k_packed.shape[:-1] != k_scales.shape[:-1]:
        raise ValueError(f"{what}: packed/scales leading dimensions must match")


def check_query(q, k_packed, k_scales, n_q_heads: int, n_kv_heads: int, group_size: int) -> None:
    if group_size <= 0:
        raise ValueError("group_size must be > 0")
    if n_q_heads <= 0 or n_kv_heads <= 0:
        raise ValueError("n_q_heads and n_kv_heads must be > 0")
    if n_q_heads % n_kv_heads != 0:
        raise ValueError("n_q_heads must be divisible by n_kv_heads")
    if q.dim() != 4:
        raise ValueError("q must be 4D: [B, n_q_heads, n, d_head]")
    if q.dtype not in FLOATS:
        raise ValueError("q must be bf16/fp16/fp32")
    b, hq, _, d = q.shape
    if hq != n_q_heads:
        raise ValueError(f"q head dim {hq} != n_q_heads {n_q_heads}")
    if k_packed.shape[0] != b or k_packed.shape[1] != n_kv_heads:
        raise ValueError("k/v leading dims must be [B, n_kv_heads, ...]")
    groups = math.ceil(d / group_size)
    if k_packed.shape[-1] < groups * ((group_size + 1) // 2):
        raise ValueError("packed last dimension is too small for q d_head")
    if k_scales.shape[-1] < groups:
        raise ValueError("scales last dimension is too small for q d_head/group_size")


def check_out(name: str, t, shape, dtype, like) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != like.device:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on the device of the inputs")


def check_int32(name: str, t, shape, like) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != like.device:
        raise ValueError(f"{name} must be int32 {list(shape)} on the device of the inputs")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def need_cuda(name: str, *ts) -> None:
    if not all(t.is_cuda for t in ts):
        raise ValueError(f"{name} expects CUDA tensors")
    if any(t.device != ts[0].device for t in ts):
        raise ValueError(f"{name} expects all tensors on one device")


def overlap(a, b) -> bool:
    """Whether some element of ``a`` shares a byte with one of ``b`` (views of one
    buffer may interleave without that)."""
    return a.device == b.device and binding().overlap(a, b)


def check_written(name: str, t) -> None:
    if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        raise ValueError(f"{name} must not be an expanded view: it is written")


def check_apart(name: str, t, others: dict) -> None:
    """``t`` is written while ``others`` are read or written."""
    for other, x in others.items():
        if x is not None and overlap(t, x):
            raise ValueError(f"{name} must not overlap {other}")


def same_view(a, b) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()
