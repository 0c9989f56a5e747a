"""Products in 8-bit integers: the CPU path and what is refused (CPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from liteinfer_amd import _native
from liteinfer_amd.engine import ops
from oracle import int8 as I8


def _operands(m, n, k, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    return x, torch.randn(n, k, generator=g) * 0.02


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 5, 7), (1, 1, 1), (4, 20, 64)])
def test_the_cpu_path_is_the_definition(shape, dtype):
    x, w = _operands(*shape, dtype)
    weight = ops.quantize_weight(w)
    codes, scales = I8.quantize_rows(w.numpy())
    np.testing.assert_array_equal(weight.codes.numpy(), codes)
    np.testing.assert_array_equal(weight.scales.numpy(), scales)
    want = I8.linear(x.float().numpy(), codes, scales)
    assert torch.equal(ops.linear_int8(x, *weight), torch.from_numpy(want).to(dtype))


def test_the_product_is_off_by_half_a_step_of_each_operand():
    """In 64 bits: |x - c s| <= s / 2 on both sides, so a sum is off by at most sum (s_x |w| + s_w |x| + s_x s_w / 2) / 2."""
    x, w = _operands(5, 9, 200)
    out = ops.linear_int8(x, *ops.quantize_weight(w)).double().numpy()
    sx, sw = (np.abs(t.double().numpy()).max(axis=1) / 127 for t in (x, w))
    ax, aw = np.abs(x.double().numpy()).sum(axis=1), np.abs(w.double().numpy()).sum(axis=1)
    bound = (sx[:, None] * aw + ax[:, None] * sw + 200 * sx[:, None] * sw / 2) / 2
    want = x.double().numpy() @ w.double().numpy().T
    assert (np.abs(out - want) <= bound * (1 + 2.0 ** -18)).all()


def test_rows_of_three_dimensions_and_of_none():
    x, w = _operands(12, 6, 10)
    weight = ops.quantize_weight(w)
    flat = ops.linear_int8(x, *weight)
    assert torch.equal(ops.linear_int8(x.view(3, 4, 10), *weight), flat.view(3, 4, 6))
    assert torch.equal(ops.linear_int8(x[0], *weight), flat[0])
    assert ops.linear_int8(x[:0], *weight).shape == (0, 6)
    codes, scales = ops.quantize_rows(x.view(3, 4, 10))
    assert codes.shape == (3, 4, 10) and scales.shape == (3, 4)
    assert codes.stride(-1) == 1 and codes.stride(-2) % 16 == 0


def test_rows_that_are_not_finite_or_zero():
    x, w = _operands(5, 4, 8)
    x[1, 3], x[2, 0], x[3] = float("nan"), float("inf"), 0.0
    out = ops.linear_int8(x, *ops.quantize_weight(w))
    assert torch.isnan(out[1:3]).all() and (out[3] == 0).all() and torch.isfinite(out[[0, 4]]).all()


def test_refusals():
    x, w = _operands(3, 4, 16)
    codes, scales = ops.quantize_weight(w)
    for args, message in (((x.double(), codes, scales), "float32, float16 or bfloat16"), ((x, w, scales), "must be int8"),
                          ((x[:, :8], codes, scales), "must be int8"), ((x, codes, scales.double()), "float32 \\[4\\]"),
                          ((x, codes, scales[:3]), "float32 \\[4\\]"), ((x, codes[:0], scales[:0]), "must be int8"),
                          ((x.to(torch.int8), codes, scales), "float32, float16")):
        with pytest.raises(ValueError, match=message):
            ops.linear_int8(*args)
    with pytest.raises(ValueError, match="no gradient"):
        ops.linear_int8(x.clone().requires_grad_(), codes, scales)
    for bad in (x.to(torch.int32), x[:, :0], torch.tensor(1.0)):
        with pytest.raises(ValueError, match="quantize_rows takes"):
            ops.quantize_rows(bad)
    with pytest.raises(ValueError, match="\\[n, k\\]"):
        ops.quantize_weight(w[0])


def _status(**kw):
    """li_linear_int8 with host pointers: every refusal comes before a launch."""
    a = dict(m=2, n=4, k=16, w_stride=16, out_stride=4, dtype=_native.LI_BF16, null=False, space=1 << 20, shift=0)
    a.update(kw)
    buf = (ctypes.c_char * 256)()
    p = ctypes.addressof(buf)
    p += -p % 16
    w = None if a["null"] else p + a["shift"]
    return _native.load().li_linear_int8(p, 16, w, a["w_stride"], p, p, a["out_stride"], a["m"], a["n"], a["k"],
                                         p if a["space"] else None, a["space"], a["dtype"], None)


@pytest.mark.parametrize(("change", "status"), [
    (dict(m=0), _native.LI_OK), (dict(null=True), _native.LI_EINVAL), (dict(m=-1), _native.LI_EINVAL),
    (dict(n=0), _native.LI_EINVAL), (dict(k=0), _native.LI_EINVAL), (dict(k=131073, w_stride=131088), _native.LI_EUNSUPPORTED),
    (dict(dtype=_native.LI_FP8_E4M3), _native.LI_EINVAL), (dict(dtype=7), _native.LI_EINVAL),
    (dict(w_stride=24), _native.LI_EINVAL), (dict(k=17, w_stride=16), _native.LI_EINVAL), (dict(shift=8), _native.LI_EINVAL),
    (dict(out_stride=3), _native.LI_EINVAL), (dict(space=0), _native.LI_EWORKSPACE), (dict(space=64), _native.LI_EWORKSPACE),
])
def test_the_c_entry_refuses(change, status):
    assert _status(**change) == status


def test_quantize_rows_refuses_in_c():
    lib = _native.load()
    buf = (ctypes.c_char * 256)()
    p = ctypes.addressof(buf)
    p += -p % 16
    good = dict(x=p, codes=p, stride=16, scales=p, rows=1, k=16, padded=16, dtype=_native.LI_F32)
    for change in (dict(x=None), dict(codes=None), dict(scales=None), dict(codes=p + 4), dict(stride=12), dict(padded=8),
                   dict(k=0), dict(rows=-1), dict(dtype=5), dict(padded=20, stride=20)):
        a = good | change
        assert lib.li_quantize_rows(a["x"], 16, a["codes"], a["stride"], a["scales"], a["rows"], a["k"], a["padded"],
                                    a["dtype"], None) == _native.LI_EINVAL, change
    assert lib.li_quantize_rows(p, 16, p, 16, p, 0, 16, 16, _native.LI_F32, None) == _native.LI_OK


def test_the_plan_holds_the_rows_codes_and_scales():
    need = ctypes.c_size_t()
    lib = _native.load()
    for m in (1, 100, 1000, 5000):
        assert lib.li_linear_int8_plan(m, 4096, 4000, ctypes.byref(need)) == _native.LI_OK
        assert need.value >= m * (4096 + 4)
    assert lib.li_linear_int8_plan(0, 4096, 4096, ctypes.byref(need)) == _native.LI_OK and need.value == 0
    assert lib.li_linear_int8_plan(1, 4096, 0, ctypes.byref(need)) == _native.LI_EINVAL
    assert lib.li_linear_int8_plan(1, 4096, 131073, ctypes.byref(need)) == _native.LI_EUNSUPPORTED


def test_more_rows_than_an_int_counts_are_refused():
    rows = torch.zeros(1, 16).expand(2 ** 31 + 5, 16)
    with pytest.raises(ValueError, match="fewer than 2"):
        ops.linear_int8(rows, torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))
