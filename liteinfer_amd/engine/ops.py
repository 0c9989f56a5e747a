"""The minimal engine's own ops on a ROCm device: fused elementwise work (`li_add_rms_norm`,
`li_silu_mul`), the decode step's projections (`li_skinny_gemm`), projections in 8-bit integers (`li_linear_int8`)
and the step's inputs (`li_rotary_tables`, `li_stage_decode`).

Same results as the model's torch ops (liteinfer/models/llama.py:34-48,
:101-116) up to the order of the fp32 sum of squares and the exponential's
last bit; one launch each instead of a chain of torch kernels. The kernels
read raw pointers, so every operand is checked here first: the projections
leave what they do not serve to `F.linear`, which serves or refuses it, the
others raise ValueError. The model keeps its torch ops for CPU tensors.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch
import torch.nn.functional as F

from liteinfer_amd import _native


def _rows(t: torch.Tensor, name: str) -> tuple[int, int]:
    if t.dim() < 1 or t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last axis")
    flat = t.reshape(-1, t.shape[-1])
    if flat.data_ptr() != t.data_ptr() or (flat.shape[0] > 1 and t.dim() > 2 and not t.is_contiguous()):
        raise ValueError(f"{name} rows must be evenly strided")
    return flat.shape[0], (flat.stride(0) if flat.shape[0] > 1 else t.shape[-1])


def _same_device(what: str, *tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if not t.is_cuda or t.device != device:
            raise ValueError(f"{what} takes tensors on one ROCm device, got {[str(t.device) for t in tensors]}")
    return device


class Partials(NamedTuple):
    """A projection as fp32 sums over runs of its K, ``[splits, rows, n]``: what an op that follows adds and rounds."""

    sums: torch.Tensor
    shape: torch.Size
    """The projection's shape, ``[..., n]``."""


class Int8Weight(NamedTuple):
    """A projection's weight in 8 bits: row j of ``[n, k]`` stands for ``codes[j] * scales[j]``."""

    codes: torch.Tensor
    """int8 ``[n, k]``, rows at multiples of 16 bytes (`quantize_weight` lays them out so)."""
    scales: torch.Tensor
    """float32 ``[n]``."""


# Rows of x up to which the projections may run as this library's kernels
# (LI_SKINNY_MAX_ROWS; li_skinny_gemm_plan says which); torch's GEMMs serve
# the others.
SKINNY_MAX_ROWS = 256


@functools.lru_cache(maxsize=4096)
def _splits(rows: int, n: int, k: int) -> int:
    """Runs of K one projection is cut into (0: torch's GEMM serves it)."""
    if rows > SKINNY_MAX_ROWS or n % 8 or k % 128 or not n or not k:
        return 0
    splits = ctypes.c_int()
    status = _native.load().li_skinny_gemm_plan(rows, n, k, ctypes.byref(splits))
    if status == _native.LI_EUNSUPPORTED:
        return 0
    _native.check(status, "skinny_gemm")
    return splits.value


def _skinny(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x as ``[rows, k]`` and the splits of ``x @ w.T`` (0: not this kernel's, and x as it came)."""
    if (not x.is_cuda or w.device != x.device or x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]
            or (torch.is_grad_enabled() and (x.requires_grad or w.requires_grad))):
        return x, 0
    flat = x.reshape(-1, x.shape[-1])
    if (x.dtype not in (torch.bfloat16, torch.float16) or w.dtype != x.dtype or not w.is_contiguous()
            or flat.stride(-1) != 1 or flat.stride(0) % 8 or flat.data_ptr() % 16 or w.data_ptr() % 16):
        return flat, 0
    return flat, _splits(flat.shape[0], *w.shape)


def _gemm(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None, sums: torch.Tensor | None, splits: int,
          gate_up: bool) -> None:
    status = _native.load().li_skinny_gemm(
        x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), out.data_ptr() if out is not None else None,
        out.stride(0) if out is not None else 0, sums.data_ptr() if sums is not None else None,
        x.shape[0], w.shape[0], w.shape[1], splits, int(gate_up), _native.dtype_code(x.dtype),
        _native.stream_handle(x.device))
    _native.check(status, "skinny_gemm")


def linear_sums(x: torch.Tensor, w: torch.Tensor | Int8Weight) -> torch.Tensor | Partials:
    """``x @ w.T`` for an op that takes `Partials`: those where the kernel cut K, the rounded rows elsewhere."""
    if isinstance(w, Int8Weight):
        return linear_int8(x, *w)
    flat, splits = _skinny(x, w)
    if splits == 0:
        return F.linear(x, w)
    shape = torch.Size((*x.shape[:-1], w.shape[0]))
    if splits > 1:
        sums = torch.empty(splits, flat.shape[0], w.shape[0], dtype=torch.float32, device=x.device)
        _gemm(flat, w, None, sums, splits, False)
        return Partials(sums, shape)
    out = torch.empty(flat.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
    _gemm(flat, w, out, None, 1, False)
    return out.view(shape)


def linear(x: torch.Tensor, w: torch.Tensor | Int8Weight) -> torch.Tensor:
    """``x @ w.T``, the model's projection."""
    got = linear_sums(x, w)
    if not isinstance(got, Partials):
        return got
    splits, rows, n = got.sums.shape
    out = torch.empty(got.shape, dtype=x.dtype, device=x.device)
    status = _native.load().li_skinny_reduce(got.sums.data_ptr(), out.data_ptr(), n, rows, n, splits,
                                             _native.dtype_code(x.dtype), _native.stream_handle(x.device))
    _native.check(status, "skinny_reduce")
    return out


def gate_up_silu(x: torch.Tensor, w: torch.Tensor | Int8Weight) -> torch.Tensor:
    """``silu(gate) * up`` of the fused projection ``x @ w.T = [gate | up]``."""
    if isinstance(w, Int8Weight):
        return silu_mul(linear_int8(x, *w))
    flat, splits = _skinny(x, w)
    if splits == 0 or w.shape[0] % 16:
        return silu_mul(F.linear(x, w))
    rows, ffn = flat.shape[0], w.shape[0] // 2
    out = torch.empty(*x.shape[:-1], ffn, dtype=x.dtype, device=x.device)
    if splits == 1:
        _gemm(flat, w, out.view(rows, ffn), None, 1, True)
        return out
    sums = torch.empty(splits, rows, 2 * ffn, dtype=torch.float32, device=x.device)
    _gemm(flat, w, None, sums, splits, True)
    status = _native.load().li_silu_mul_partials(sums.data_ptr(), splits, out.data_ptr(), rows, ffn, ffn,
                                                 _native.dtype_code(x.dtype), _native.stream_handle(x.device))
    _native.check(status, "silu_mul")
    return out


def _row_scale(largest: torch.Tensor) -> torch.Tensor:
    """A row's scale from its largest magnitude: over 127, 2^-126 at least, NaN for what is not finite."""
    scale = (largest * (1.0 / 127.0)).clamp(min=2.0 ** -126)
    return torch.where(torch.isfinite(largest), scale, float("nan"))


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x ``[..., k]`` as int8 codes with a float32 scale for each row: ``(codes [..., k], scales [...])``.

    ``scale = max(largest magnitude / 127, 2^-126)``, ``code = rint(x / scale)``
    in float32; a row with a value that is not finite gets the scale NaN and
    codes 0. Rows of codes start at multiples of 16 bytes.
    """
    if x.dtype not in _native.DTYPE_CODES or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"quantize_rows takes float32, float16 or bfloat16 rows, got {x.dtype} {list(x.shape)}")
    k = x.shape[-1]
    flat = x.reshape(-1, k)
    if flat.stride(-1) != 1:
        flat = flat.contiguous()
    rows, padded = flat.shape[0], -(-k // 16) * 16
    codes = torch.empty(rows, padded, dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    if x.is_cuda:
        _native.check(_native.on_device(
            x.device, _native.load().li_quantize_rows, flat.data_ptr(), flat.stride(0) if rows > 1 else k,
            codes.data_ptr(), padded, scales.data_ptr(), rows, k, padded, _native.dtype_code(x.dtype),
            _native.stream_handle(x.device)), "quantize_rows")
    else:
        wide = flat.to(torch.float32)
        scales.copy_(_row_scale(wide.abs().amax(dim=-1)))
        lost = torch.isnan(scales)[:, None]
        inv = torch.where(lost, 0.0, 1.0 / scales[:, None])
        codes.zero_()[:, :k] = torch.round(torch.where(lost, 0.0, wide) * inv).clamp(-127, 127).to(torch.int8)
    return codes[:, :k].view(*x.shape[:-1], k), scales.view(x.shape[:-1])


def quantize_weight(w: torch.Tensor) -> Int8Weight:
    """A projection's weight ``[n, k]`` in 8 bits with a scale for each output channel, as `linear_int8` takes it."""
    if w.dim() != 2:
        raise ValueError(f"a weight is [n, k], got {list(w.shape)}")
    return Int8Weight(*quantize_rows(w))


@functools.lru_cache(maxsize=4096)
def _linear_int8_bytes(rows: int, n: int, k: int, device_index: int) -> int:
    need = ctypes.c_size_t()
    _native.check(_native.load().li_linear_int8_plan(rows, n, k, ctypes.byref(need)), "linear_int8")
    return need.value


def linear_int8(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``x @ w.T`` in 8-bit integers: x ``[..., k]`` quantised row by row, w ``codes [n, k]`` times ``scales [n]``.

    x's rows are quantised as `quantize_rows` does; products are summed exactly
    and ``sum * row scale * channel scale`` is rounded once to x's dtype
    (float32, float16 or bfloat16). A row with a value that is not finite gives
    NaN. `codes` rows start at multiples of 16 bytes (`quantize_weight`).
    """
    if x.is_cuda and _native.is_current(x.device):
        # Operands that need no conversion: checked and passed on in C++.
        out = _native.fast_calls().linear_int8(x, codes, scales, _native.stream_handle(x.device))
        if out is not None:
            if isinstance(out, int):
                _native.check(out, "linear_int8")
            return out
    if x.dtype not in _native.DTYPE_CODES or x.dim() < 1:
        raise ValueError(f"linear_int8 takes float32, float16 or bfloat16 rows, got {x.dtype} {list(x.shape)}")
    if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[1] != x.shape[-1] or 0 in codes.shape:
        raise ValueError(f"the weight's codes must be int8 [n, {x.shape[-1]}], got {codes.dtype} {list(codes.shape)}")
    n, k = codes.shape
    if scales.dtype != torch.float32 or scales.shape != (n,) or (n > 1 and scales.stride(0) != 1):
        raise ValueError(f"the weight's scales must be contiguous float32 [{n}], got {scales.dtype} {list(scales.shape)}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("linear_int8 has no gradient: call it under torch.no_grad()")
    if codes.device != x.device or scales.device != x.device:
        raise ValueError(f"linear_int8 takes tensors on one device, got {[str(t.device) for t in (x, codes, scales)]}")
    flat = x.reshape(-1, k)
    if flat.stride(-1) != 1:
        flat = flat.contiguous()
    rows = flat.shape[0]
    if max(rows, n) >= 2 ** 31:
        raise ValueError(f"linear_int8 takes fewer than 2^31 rows and channels, got {rows} and {n}")
    if not x.is_cuda:
        xc, xs = quantize_rows(flat)
        sums = xc.to(torch.float64) @ codes.to(torch.float64).t()  # whole numbers below 2^31: exact
        return (sums.to(torch.float32) * xs[:, None] * scales).to(x.dtype).view(*x.shape[:-1], n)
    stride, padded = codes.stride(0) if n > 1 else -(-k // 16) * 16, -(-k // 16) * 16
    end = codes.storage_offset() + (n - 1) * stride + padded
    if (codes.stride(1) != 1 and k > 1) or stride % 16 or stride < padded or codes.data_ptr() % 16 or end > codes.untyped_storage().nbytes():
        raise ValueError("rows of codes must start at multiples of 16 bytes and be padded to them: quantize_weight lays them out")
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    need = _native.on_device(x.device, _linear_int8_bytes, rows, n, k, x.device.index or 0)
    workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    _native.check(_native.on_device(
        x.device, _native.load().li_linear_int8, flat.data_ptr(), flat.stride(0) if rows > 1 else k, codes.data_ptr(),
        stride, scales.data_ptr(), out.data_ptr(), n, rows, n, k, workspace.data_ptr(), need,
        _native.dtype_code(x.dtype), _native.stream_handle(x.device)), "linear_int8")
    return out


def add_rms_norm(h: torch.Tensor, weight: torch.Tensor, eps: float,
                 delta: torch.Tensor | Partials | None = None) -> torch.Tensor:
    """``h += delta`` in place (when given), then RMSNorm of h times `weight`; returns the normalised rows."""
    if h.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != h.dtype or weight.shape != h.shape[-1:]:
        raise ValueError("add_rms_norm takes bf16 / f16 rows and a weight of their width and dtype")
    if delta is not None and (delta.shape != h.shape or (not isinstance(delta, Partials) and delta.dtype != h.dtype)):
        raise ValueError("delta must match h")
    _same_device("add_rms_norm", h, weight, *(() if delta is None else (delta.sums if isinstance(delta, Partials) else delta,)))
    rows, h_s = _rows(h, "h")
    if isinstance(delta, Partials):
        if (delta.sums.dtype != torch.float32 or delta.sums.dim() != 3 or not delta.sums.is_contiguous()
                or delta.sums.shape[1:] != (rows, h.shape[-1])):
            raise ValueError(f"partial sums must be contiguous float32 [splits, {rows}, {h.shape[-1]}], "
                             f"got {delta.sums.dtype} {list(delta.sums.shape)}")
        out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        status = _native.load().li_add_rms_norm_partials(
            h.data_ptr(), delta.sums.data_ptr(), delta.sums.shape[0], weight.contiguous().data_ptr(), out.data_ptr(),
            rows, h.shape[-1], h_s, h.shape[-1], float(eps), _native.dtype_code(h.dtype),
            _native.stream_handle(h.device))
        _native.check(status, "add_rms_norm")
        return out
    d_s = _rows(delta, "delta")[1] if delta is not None else 0
    out = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    status = _native.load().li_add_rms_norm(
        h.data_ptr(), delta.data_ptr() if delta is not None else None, weight.contiguous().data_ptr(),
        out.data_ptr(), rows, h.shape[-1], h_s, d_s, h.shape[-1], float(eps), _native.dtype_code(h.dtype),
        _native.stream_handle(h.device))
    _native.check(status, "add_rms_norm")
    return out


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` of the fused projection's halves ``gate_up = [gate | up]``."""
    if gate_up.dtype not in (torch.bfloat16, torch.float16) or gate_up.shape[-1] % 2:
        raise ValueError("silu_mul takes bf16 / f16 rows of an even width")
    _same_device("silu_mul", gate_up)
    ffn = gate_up.shape[-1] // 2
    rows, gu_s = _rows(gate_up, "gate_up")
    out = torch.empty(*gate_up.shape[:-1], ffn, dtype=gate_up.dtype, device=gate_up.device)
    status = _native.load().li_silu_mul(gate_up.data_ptr(), out.data_ptr(), rows, ffn, gu_s, ffn,
                                        _native.dtype_code(gate_up.dtype), _native.stream_handle(gate_up.device))
    _native.check(status, "silu_mul")
    return out


def rotary_tables(positions: torch.Tensor, inv_freq: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin ``[..., D]`` of `positions` times `inv_freq` (``[D / 2]`` fp32, each twice), rounded to `dtype`."""
    _same_device("rotary_tables", positions, inv_freq)
    if positions.is_floating_point() or positions.is_complex():
        raise ValueError(f"rotary_tables takes whole positions, got {positions.dtype}")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be contiguous float32 [D / 2], got {inv_freq.dtype} {list(inv_freq.shape)}")
    positions = positions.to(torch.int64).contiguous()
    half = inv_freq.shape[0]
    cos, sin = (torch.empty(*positions.shape, 2 * half, dtype=dtype, device=positions.device) for _ in range(2))
    status = _native.load().li_rotary_tables(
        positions.data_ptr(), inv_freq.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.numel(), half,
        _native.dtype_code(dtype), _native.stream_handle(positions.device))
    _native.check(status, "rotary_tables")
    return cos, sin


def stage_decode(inputs: tuple[torch.Tensor, ...], static: tuple[torch.Tensor, ...], width: int, pad_slot: int) -> None:
    """A decode step's (ids, positions, write slots, slot table, context lengths) into a captured graph's buffers.

    `static` holds the buffers in the same order; rows past the step's, up to
    `width`, become a one-token context in `pad_slot`.
    """
    ids, positions, write_slots, slots, lens = inputs
    n, cols = slots.shape
    device = _same_device("stage_decode", *static)
    ids_out, positions_out, write_out, table_out, lens_out = static
    for t in (ids_out, positions_out, write_out, lens_out):
        if t.numel() < width or not t.is_contiguous() or t.dtype != (torch.int32 if t is lens_out else torch.int64):
            raise ValueError(f"the static columns must be contiguous int64 (lengths int32) of at least {width} rows, "
                             f"got {t.dtype} {list(t.shape)}")
    if (table_out.dtype != torch.int64 or table_out.dim() != 2 or table_out.stride(1) != 1 or n > width
            or width > table_out.shape[0] or max(cols, 1) > table_out.shape[1] or table_out.stride(0) < table_out.shape[1]):
        raise ValueError(f"a step of {n} x {cols} slots, padded to {width} rows, does not fit a "
                         f"{list(table_out.shape)} {table_out.dtype} slot table")

    def column(t: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
        if t.shape == shape and t.dtype == dtype and t.device == device and t.is_contiguous():
            return t  # (as the engine brings it: 0.6 us on the host, the conversions that change nothing 3)
        return torch.broadcast_to(t, shape).to(device=device, dtype=dtype).contiguous()

    ids, positions = column(ids, (n, 1), torch.int64), column(positions, (n, 1), torch.int64)
    write_slots, lens = column(write_slots, (1, n), torch.int64), column(lens, (n,), torch.int32)
    slots = slots.to(device=device, dtype=torch.int64)
    if slots.stride(-1) != 1:
        slots = slots.contiguous()
    status = _native.load().li_stage_decode(
        ids.data_ptr(), positions.data_ptr(), write_slots.data_ptr(), slots.data_ptr(), slots.stride(0), lens.data_ptr(),
        ids_out.data_ptr(), positions_out.data_ptr(), write_out.data_ptr(), table_out.data_ptr(), table_out.stride(0),
        lens_out.data_ptr(), n, cols, width, pad_slot, _native.stream_handle(device))
    _native.check(status, "stage_decode")
