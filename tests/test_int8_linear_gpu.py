"""Products in 8-bit integers on the GPU, bit for bit: whole-number sums, then the definition's float32 products."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from liteinfer_amd.engine import ops
from oracle import int8 as I8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _operands(m, n, k, dtype, seed=0):
    g = np.random.default_rng(seed)
    x = torch.from_numpy((g.normal(size=(m, k)) * np.exp(0.5 * g.normal(size=(m, 1)))).astype(np.float32)).to(dtype)
    codes = g.integers(-127, 128, size=(n, k)).astype(np.int8)
    scales = np.abs(g.normal(size=n)).astype(np.float32) * 1e-4
    return x, codes, scales


def _weight(codes, scales, fill=99):
    """Codes in rows padded to 16 bytes with what must not count."""
    n, k = codes.shape
    held = torch.full((n, -(-k // 16) * 16), fill, dtype=torch.int8, device=DEV)
    held[:, :k] = torch.from_numpy(codes).to(DEV)
    return held[:, :k], torch.from_numpy(scales).to(DEV)


def _check(out, x, codes, scales):
    want = torch.from_numpy(I8.linear(x.float().numpy(), codes, scales)).to(out.dtype)
    got = out.cpu()
    assert got.shape == want.shape and torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num()), (got.float() - want.float()).abs().max()


ROWS = [1, 2, 15, 16, 17, 33, 64, 65, 100, 129, 300]
WEIGHTS = [(1, 1), (3, 5), (16, 64), (65, 255), (130, 256), (257, 257), (777, 1000), (128, 4096), (2048, 512)]


@pytest.mark.parametrize("weight", WEIGHTS, ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("m", ROWS)
def test_every_kind_of_product(m, weight):
    dtype = (BF16, F16, F32)[(m + weight[0]) % 3]
    x, codes, scales = _operands(m, *weight, dtype)
    _check(ops.linear_int8(x.to(DEV), *_weight(codes, scales)), x, codes, scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 6144, 4096), (61, 4096, 14336), (128, 4096, 4096), (1000, 4096, 1024), (2049, 8448, 512)])
def test_sizes_of_the_engine(shape, dtype):
    x, codes, scales = _operands(*shape, dtype)
    _check(ops.linear_int8(x.to(DEV), *_weight(codes, scales)), x, codes, scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(530, 2051, 77), (530, 2051, 2100), (1300, 6147, 131), (1400, 6147, 131), (1283, 6148, 300),
                                   (1290, 6152, 128), (2000, 6147, 131), (2064, 6147, 131), (2051, 6152, 128), (200, 28685, 131),
                                   (68, 40000, 64), (320, 20001, 16)])
def test_large_tiles_at_odd_sizes(shape, dtype):
    """128 x 128 whole and cut along k, 256 x 128 and 256 x 256, with few and with many rows past the last whole tile."""
    x, codes, scales = _operands(*shape, dtype)
    _check(ops.linear_int8(x.to(DEV), *_weight(codes, scales)), x, codes, scales)


def test_rows_of_a_weight_far_apart():
    """A tile of 256 of w's rows spans more than 2^32 bytes."""
    m, n, k = 1400, 6147, 131
    x, codes, scales = _operands(m, n, k, BF16)
    held = torch.empty(n * ((1 << 24) + 16), dtype=torch.int8, device=DEV).view(n, -1)[:, :k]
    held.copy_(torch.from_numpy(codes).to(DEV))
    _check(ops.linear_int8(x.to(DEV), held, torch.from_numpy(scales).to(DEV)), x, codes, scales)
    del held
    torch.cuda.empty_cache()


def test_the_largest_sums():
    """Codes of one sign at the longest k: the sums come near 2^31."""
    k = 131072
    x = torch.ones(3, k, dtype=BF16)
    codes = np.full((20, k), -128, dtype=np.int8)
    codes[3:] = 127
    scales = np.ones(20, dtype=np.float32)
    _check(ops.linear_int8(x.to(DEV), *_weight(codes, scales)), x, codes, scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(5, 1), (3, 7), (300, 4096), (2, 16384), (2, 16390), (2, 40001)])
def test_rows_are_quantised_as_the_definition_says(shape, dtype):
    x, _, _ = _operands(shape[0], 1, shape[1], dtype)
    for t in (x, x[:, 1:]) if shape[1] > 1 else (x,):
        codes, scales = ops.quantize_rows(t.to(DEV) if t is x else x.to(DEV)[:, 1:])
        want = I8.quantize_rows(t.float().numpy())
        np.testing.assert_array_equal(codes.cpu().numpy(), want[0])
        np.testing.assert_array_equal(scales.cpu().numpy(), want[1])
        assert codes.stride(0) % 16 == 0


def test_strided_rows_and_weights_within_wider_ones():
    x, codes, scales = _operands(40, 96, 300, BF16)
    wide = torch.randn(40, 317, device=DEV).to(BF16)
    wide[:, 5:305] = x.to(DEV)
    held = torch.full((96, 640), 77, dtype=torch.int8, device=DEV)
    held[:, 16:316] = torch.from_numpy(codes).to(DEV)
    _check(ops.linear_int8(wide[:, 5:305], held[:, 16:316], torch.from_numpy(scales).to(DEV)), x, codes, scales)
    turned = x.to(DEV).t().contiguous().t()
    _check(ops.linear_int8(turned, held[:, 16:316], torch.from_numpy(scales).to(DEV)), x, codes, scales)
    _check(ops.linear_int8(x.to(DEV).view(4, 10, 300), held[:, 16:316], torch.from_numpy(scales).to(DEV)).flatten(0, 1), x,
           codes, scales)


@pytest.mark.parametrize("m", [3, 40, 100, 600])
def test_rows_that_are_not_finite_zero_large_or_small(m):
    x, codes, scales = _operands(m, 80, 200, BF16)
    x[0, 7], x[1, 199], x[2] = float("nan"), float("-inf"), 0.0
    if m > 3:
        x[3] *= 1e30
        x[4] *= 1e-30
        x[5] = 1e-39
    out = ops.linear_int8(x.to(DEV), *_weight(codes, scales))
    assert torch.isnan(out[:2]).all()
    _check(out, x, codes, scales)


def test_no_rows():
    _, codes, scales = _operands(1, 8, 32, BF16)
    assert ops.linear_int8(torch.zeros(0, 32, dtype=BF16, device=DEV), *_weight(codes, scales)).shape == (0, 8)


def test_the_model_operators_take_an_8_bit_weight():
    x, codes, scales = _operands(9, 64, 128, BF16)
    weight = ops.Int8Weight(*_weight(codes, scales))
    xd = x.to(DEV)
    want = ops.linear_int8(xd, *weight)
    assert torch.equal(ops.linear(xd, weight), want) and torch.equal(ops.linear_sums(xd, weight), want)
    assert torch.equal(ops.gate_up_silu(xd, weight), ops.silu_mul(want))


@pytest.mark.parametrize("m", [1, 50, 200, 3000])
def test_a_captured_product_replays_and_two_graphs_keep_apart(m):
    x, codes, scales = _operands(m, 512, 1024, BF16)
    weight = _weight(codes, scales)
    inputs = [x.to(DEV), (x * 2 - 1).to(DEV)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_int8(inputs[0], *weight)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for t in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.linear_int8(t, *weight))
    for turn in range(3):
        for t in inputs:
            t.mul_(1.25 if turn else 1.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for t, out in zip(inputs, outs):
            assert torch.equal(out, ops.linear_int8(t, *weight))


def test_two_streams():
    streams, got, want = [torch.cuda.Stream() for _ in range(2)], [], []
    cases = [_operands(m, 700, 900, F16, seed=m) for m in (70, 333)]
    placed = [(x.to(DEV), *_weight(c, s)) for x, c, s in cases]
    torch.cuda.synchronize()
    for s, args in zip(streams, placed):
        with torch.cuda.stream(s):
            got.append(ops.linear_int8(*args))
    torch.cuda.synchronize()
    for out, case in zip(got, cases):
        _check(out, *case)


def test_refusals():
    x, codes, scales = _operands(3, 40, 100, BF16)
    w, s = _weight(codes, scales)
    with pytest.raises(ValueError, match="multiples of 16 bytes"):
        ops.linear_int8(x.to(DEV), w.contiguous(), s)
    with pytest.raises(ValueError, match="multiples of 16 bytes"):
        ops.linear_int8(x[:, 1:].to(DEV), w[:, 1:], s)
    cut = torch.zeros(40 * 112 - 12, dtype=torch.int8, device=DEV).as_strided((40, 100), (112, 1))
    with pytest.raises(ValueError, match="padded to them"):  # the last row's padding lies outside the storage
        ops.linear_int8(x.to(DEV), cut, s)
    with pytest.raises(ValueError, match="one device"):
        ops.linear_int8(x.to(DEV), w, s.cpu())
    with pytest.raises(ValueError, match="32 bits"):
        big = torch.zeros(1, 131088, dtype=torch.int8, device=DEV)
        ops.linear_int8(torch.zeros(1, 131088, dtype=BF16, device=DEV), big, torch.ones(1, device=DEV))
