"""Linears and routed experts with 4-bit weights in groups, W = scale * q + bias (the format of the reference's q4.zig):
Linear and call beside linear.py's, Experts, Scratch and routed beside moe.py's, over the C ABI."""
from __future__ import annotations

import ctypes as C

import torch

from . import device
from ._lib import Q4Experts as _Experts, Q4Linear as _Linear, Q4Scratch as _Scratch, check, lib
from .linear import _arrays

F16, BF16, F32 = 0, 1, 2
_S_DTYPE = {torch.float16: F16, torch.bfloat16: BF16}


def _source(m, dims: int):
    """A matrix's tensors (words, scales, biases or None) as contiguous ones on the current device, their n, k, group and
    dtype code. words int32 [.., n, k / 8], scales and biases [.., n, k / group]."""
    words, scales, biases = m
    for t in (words, scales) + (() if biases is None else (biases,)):
        if t.dim() != dims or t.shape[:-1] != words.shape[:-1] or t.device != torch.device("cuda", torch.cuda.current_device()):
            raise ValueError("words, scales and biases must be tensors of one leading shape on the current device")
    if words.dtype != torch.int32 or scales.dtype not in _S_DTYPE:
        raise ValueError("words must be int32, scales float16 or bfloat16")
    if biases is not None and (biases.dtype != scales.dtype or biases.shape != scales.shape):
        raise ValueError("biases must have the scales' type and shape")
    n, k = words.shape[-2], 8 * words.shape[-1]
    group = k // scales.shape[-1] if scales.shape[-1] else 0
    if group not in (32, 64, 128) or group * scales.shape[-1] != k:
        raise ValueError(f"groups of {group}: 32, 64 or 128 consecutive values share a scale")
    return words.contiguous(), scales.contiguous(), None if biases is None else biases.contiguous(), n, k, group


def _pack(first, second, n: int, k: int, group: int, s_dtype: int, count: int) -> torch.Tensor:
    size = lib().ea_q4_bytes(n if second is None else 16 * ((n + 7) // 8), k, group)
    out = torch.empty(size * count, dtype=torch.uint8, device="cuda")
    second = (None, None, None) if second is None else second
    check(lib().ea_q4_pack(device.stream(), *(device.addr(t) for t in (*first, *second)),
                           out.data_ptr(), n, k, group, s_dtype, count), "q4.pack")
    return out


class Linear:
    """One matrix W [n, k] in the kernels' layout, from words int32 [n, k / 8] (the first of a word's eight values in its
    lowest bits), scales and biases [n, k / group] in fp16 or bf16 (biases None: -8 * scales). The sources may be freed
    afterwards; the packing is a launch on the current stream."""

    def __init__(self, words: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor | None = None):
        w, s, b, self.n, self.k, self.group = _source((words, scales, biases), 2)
        self.s_dtype = _S_DTYPE[s.dtype]
        self.words = _pack((w, s, b), None, self.n, self.k, self.group, self.s_dtype, 1)
        self.c = _Linear(self.words.data_ptr(), self.k, self.n, self.group, self.s_dtype)


def call(stream: int, ls, x: int, x_dtype: int, x_stride: int, m: int, outs, out_dtypes) -> None:
    """outs[j] [m, n_j] = x [m, k] @ W_j^T for 1..3 linears of one k, group and scale type; x fp16 or bf16, rows x_stride
    apart; outs fp16, bf16 or fp32, contiguous."""
    if len(outs) != len(ls) or len(out_dtypes) != len(ls):
        raise ValueError("an output and a type for each linear")
    arr, o, d = _arrays(ls, outs, out_dtypes)
    check(lib().ea_q4_call(stream, arr, len(ls), x, x_dtype, x_stride, m, o, d), "q4.call")


class Experts:
    """A layer's routed experts in the kernels' layout: gate, up (words int32 [E, width, dims / 8], scales, biases) and down
    ([E, dims, width / 8], ..); all of one group size and scale type."""

    def __init__(self, gate, up, down):
        *g, I, D, group = _source(gate, 3)
        *u, In, Dn, gn = _source(up, 3)
        *d, Dd, Id, gd = _source(down, 3)
        E = g[0].shape[0]
        if (In, Dn, gn) != (I, D, group) or (Dd, Id, gd) != (D, I, group) or u[0].shape[0] != E or d[0].shape[0] != E:
            raise ValueError("gate and up are [E, width, dims], down is [E, dims, width], in groups of one size")
        if len({t[1].dtype for t in (g, u, d)}) != 1 or (g[2] is None) != (u[2] is None):
            raise ValueError("gate, up and down share the scales' type; gate and up both have biases or neither")
        self.count, self.dims, self.width, self.group = E, D, I, group
        self.s_dtype = _S_DTYPE[g[1].dtype]
        self.gu = _pack(g, u, I, D, group, self.s_dtype, E)
        self.down = _pack(d, None, D, I, group, self.s_dtype, E)
        self.c = _Experts(self.gu.data_ptr(), self.down.data_ptr(), E, D, I, group, self.s_dtype, 0)


class Scratch:
    """Device memory for calls of up to `rows` rows with `slots` picks a row; one call at a time."""

    def __init__(self, ex: Experts, rows: int, slots: int):
        n = lib().ea_q4_scratch_bytes(C.byref(ex.c), rows, slots)
        self.buf = torch.empty(n + 256, dtype=torch.uint8, device="cuda")
        base = (self.buf.data_ptr() + 255) & ~255
        self.c = _Scratch()
        check(lib().ea_q4_scratch_init(C.byref(self.c), base, n, C.byref(ex.c), rows, slots), "q4.Scratch")
        self.rows, self.slots = rows, slots


def routed(stream: int, x: int, x_dtype: int, x_stride: int, pick: int, wts: int, ex: Experts, s: Scratch, out: int,
           out_dtype: int, R: int) -> None:
    """out [R, dims] = the picked experts of R rows weighted by wts (moe.routed for 4-bit experts; any number of rows the
    scratch holds). pick int32 / wts fp32 [R, s.slots]; a pick outside the experts is an empty slot."""
    check(lib().ea_q4_routed(stream, x, x_dtype, x_stride, pick, wts, C.byref(ex.c), C.byref(s.c), out, out_dtype, R),
          "q4.routed")
