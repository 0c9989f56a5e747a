"""The int8 cache with a scale for every block and head: its format, the CPU path, and what is refused (CPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from liteinfer_amd import _native
from liteinfer_amd.attention import PagedKV, eager_attention, sdpa_attention
from liteinfer_amd.cache.block_pool import BlockPool
from liteinfer_amd.cache.kv_cache import KVCache, append_int8, scatter_into
from liteinfer_amd.paged_kernels import check_block_scales
from oracle import int8 as I8
from oracle.attention import attend

H, D = 3, 16


def _store(blocks=12, block=8, seed=0, heads=H, dim=D):
    g = np.random.default_rng(seed)
    codes = g.integers(-127, 128, size=(blocks * block, heads, dim)).astype(np.int8)
    scales = np.abs(g.normal(size=(blocks, heads))).astype(np.float32) * 0.01
    return codes, scales


def _rows(n, seed, heads=H, dim=D):
    g = np.random.default_rng(seed)
    return (g.normal(size=(n, heads, dim)) * np.exp(g.normal(size=(n, heads, 1)))).astype(np.float32)


# Lists of slots (blocks of 8): one block's stand next to each other.
LISTS = {
    "fresh": list(range(16, 24)),
    "middle": [19, 20, 21],
    "two blocks": [5, 6, 7, 24, 25],
    "one token each": [3, 17, 46, 90],
    "descending": [47, 46, 45, 44],
    "named twice": [41, 42, 41, 60, 60, 60],
    "first slot last": [73, 74, 72],
    "empty": [],
}


@pytest.mark.parametrize("name", LISTS)
def test_append_matches_the_oracle_code_for_code(name):
    codes, scales = _store()
    slots, rows = np.asarray(LISTS[name], dtype=np.int64), _rows(len(LISTS[name]), 1)
    want_codes, want_scales = I8.append(codes, scales, slots, rows)
    got_codes, got_scales = torch.from_numpy(codes.copy()), torch.from_numpy(scales.copy())
    append_int8(got_codes, got_scales, torch.from_numpy(slots), torch.from_numpy(rows))
    np.testing.assert_array_equal(got_scales.numpy(), want_scales)
    np.testing.assert_array_equal(got_codes.numpy(), want_codes)


def test_rows_appended_one_by_one_stay_within_half_a_step_of_each_scale_they_met():
    """The definition in 64 bits: a row is off by half a step of its block's scale when written, and by half a
    step of each larger scale it is re-expressed with."""
    rows = _rows(8, 3) * np.linspace(0.2, 3.0, 8, dtype=np.float32)[:, None, None]
    codes, scales = np.zeros((8, H, D), np.int8), np.zeros((1, H), np.float32)
    bound = np.zeros((8, H))
    for t in range(8):
        before = scales.copy()
        codes, scales = I8.append(codes, scales, np.array([t]), rows[t:t + 1], dtype=np.float32)
        bound[:t] += np.where(scales > before, scales, 0) / 2
        bound[t] = scales[0] / 2
    off = np.abs(I8.dequantize(codes, scales) - rows).max(axis=-1)
    # (fp32 scales and products: a few 2^-24 of the largest code besides.)
    assert (off <= bound + 127 * scales * 8 * 2.0 ** -24).all()


def test_a_blocks_first_slot_starts_it_anew():
    codes, scales = _store()
    scales[2] = 1e6
    got_codes, got_scales = torch.from_numpy(codes), torch.from_numpy(scales)
    append_int8(got_codes, got_scales, torch.tensor([16]), torch.from_numpy(_rows(1, 5)))
    assert (got_scales[2] < 1).all() and (got_codes[17:24] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_value_that_is_not_finite_turns_its_blocks_scale_to_nan_until_it_starts_anew(bad):
    codes, scales = _store()
    want = codes.copy(), scales.copy()
    rows = _rows(2, 6)
    rows[1, 1, 3] = bad
    got_codes, got_scales = torch.from_numpy(codes), torch.from_numpy(scales)
    append_int8(got_codes, got_scales, torch.tensor([17, 18]), torch.from_numpy(rows))
    want = I8.append(*want, np.array([17, 18]), rows)
    np.testing.assert_array_equal(got_scales.numpy(), want[1])
    np.testing.assert_array_equal(got_codes.numpy(), want[0])
    assert torch.isnan(got_scales[2, 1]) and torch.isfinite(got_scales[2, [0, 2]]).all()
    append_int8(got_codes, got_scales, torch.tensor([19]), torch.from_numpy(_rows(1, 7)))
    assert torch.isnan(got_scales[2, 1])
    append_int8(got_codes, got_scales, torch.tensor([16]), torch.from_numpy(_rows(1, 8)))
    assert torch.isfinite(got_scales[2]).all()


def test_zero_rows_keep_a_finite_scale():
    codes, scales = torch.zeros(8, H, D, dtype=torch.int8), torch.zeros(1, H)
    append_int8(codes, scales, torch.tensor([0, 1]), torch.zeros(2, H, D))
    assert (scales == 2.0 ** -126).all() and (codes == 0).all()


def _filled_cache(dtype=torch.float32, block=4, contexts=(9, 1, 14)):
    pool = BlockPool(num_blocks=16, block_size=block, num_layers=2, num_kv_heads=2, head_dim=D, dtype=dtype,
                     device=torch.device("cpu"), cache_quant="int8")
    cache = KVCache(pool)
    ids = [f"s{i}" for i in range(len(contexts))]
    cache.reserve(ids, list(contexts))
    payload = cache.make_packed_payload(ids, [0] * len(ids), list(contexts))
    g = torch.Generator().manual_seed(3)
    total = sum(contexts)
    k, v = (torch.randn(1, 2, total, D, generator=g).to(dtype) for _ in range(2))
    kv = payload.update(k, v, 1)
    return pool, cache, kv, k, v, contexts


def test_the_pool_and_its_payloads_carry_the_scales():
    pool, cache, kv, k, v, contexts = _filled_cache()
    keys, values = pool.slots(1)
    assert keys.dtype == torch.int8 and kv.key_pool is keys
    assert kv.key_scales.shape == (16, 2) and kv.value_scales.shape == (16, 2)
    assert pool.block_scales(0)[0].eq(0).all() and pool.block_scales(1)[0].gt(0).any()
    assert pool.nbytes == 2 * 2 * 16 * (4 * 2 * D + 4 * 2)
    held = I8.dequantize(keys.numpy(), kv.key_scales.numpy())[kv.slot_table[0, :9].numpy()]
    step = kv.key_scales[kv.slot_table[0, :9] // 4].numpy()
    assert (np.abs(held - k[0, :, :9].permute(1, 0, 2).numpy()) <= (step / 2 * (1 + 2.0 ** -20))[..., None]).all()


def test_a_plain_pool_has_no_scales():
    pool = BlockPool(2, 4, 1, 2, D, torch.float32, torch.device("cpu"))
    assert pool.block_scales(0) == (None, None)


@pytest.mark.parametrize("attention", [eager_attention, sdpa_attention])
def test_the_dense_kernels_attend_over_the_values_the_codes_stand_for(attention):
    pool, cache, kv, _, _, contexts = _filled_cache()
    g = torch.Generator().manual_seed(4)
    query = torch.randn(1, 4, sum(contexts), D, generator=g)
    out = attention(query, kv, D ** -0.5, 2)
    want = attend(query[0].transpose(0, 1).numpy(), I8.dequantize(kv.key_pool.numpy(), kv.key_scales.numpy()),
                  I8.dequantize(kv.value_pool.numpy(), kv.value_scales.numpy()), kv.slot_table.numpy(),
                  np.asarray(contexts), D ** -0.5, 2, query_start_loc=kv.query_start_loc.numpy())
    # fp32 dense arithmetic: sums of 16 dims and 14 keys.
    np.testing.assert_allclose(out[0].transpose(0, 1).numpy(), want, atol=64 * 2.0 ** -24 * 8)


def test_a_decode_payload_appends_and_attends():
    pool, cache, _, k, v, contexts = _filled_cache()
    ids = [f"s{i}" for i in range(3)]
    totals = [c + 1 for c in contexts]
    cache.reserve(ids, totals)
    payload = cache.make_decode_payload(cache.newest_slots_for(ids, list(contexts)), cache.slot_table_for(ids, totals),
                                        torch.tensor(totals, dtype=torch.int32))
    before = pool.slots(1)[0].numpy().copy(), pool.block_scales(1)[0].numpy().copy()
    g = torch.Generator().manual_seed(9)
    q, new_k, new_v = (torch.randn(3, n, 1, D, generator=g) for n in (4, 2, 2))
    cos, sin = torch.randn(3, 1, D, generator=g), torch.randn(3, 1, D, generator=g)
    rotated, kv = payload.update_rotated(q, new_k, new_v, cos, sin, 1)
    want_q = I8.rotate(q.transpose(1, 2).numpy(), cos.numpy(), sin.numpy())
    np.testing.assert_allclose(rotated.transpose(1, 2).numpy(), want_q, atol=4 * 8 * 2.0 ** -24)
    want = I8.append(*before, cache.newest_slots_for(ids, list(contexts)).numpy(),
                     I8.rotate(new_k.transpose(1, 2).numpy(), cos.numpy(), sin.numpy())[:, 0])
    np.testing.assert_array_equal(kv.key_pool.numpy(), want[0])
    np.testing.assert_array_equal(kv.key_scales.numpy(), want[1])
    assert torch.isfinite(eager_attention(rotated, kv, D ** -0.5, 2)).all()


def test_a_slot_outside_the_pool_raises_on_the_cpu():
    codes, scales = (torch.from_numpy(t) for t in _store())
    k = torch.zeros(1, H, 1, D)
    for slot in (-1, 96):
        with pytest.raises(IndexError):
            scatter_into(codes, codes.clone(), torch.tensor([[slot]]), k, k, key_scales=scales,
                         value_scales=scales.clone())


def test_scales_are_checked():
    codes, scales = (torch.from_numpy(t) for t in _store())
    assert check_block_scales(codes, scales, scales.clone()) == 8
    assert check_block_scales(codes.float(), None, None) == 0
    for bad, message in (((codes.float(), scales, scales), "int8 pool"), ((codes, None, scales), "needs key_scales"),
                         ((codes, scales.double(), scales), "float32"), ((codes, scales[:, :2], scales), "num_blocks, 3"),
                         ((codes, scales, scales[:6]), "laid out"), ((codes, scales[:7], scales[:7]), "whole number"),
                         ((codes, scales.t().contiguous().t(), scales), "adjacent heads"),
                         ((codes, scales[:0], scales[:0]), "whole number")):
        with pytest.raises(ValueError, match=message):
            check_block_scales(*bad)
    with pytest.raises(ValueError, match="cache_quant"):
        BlockPool(2, 4, 1, 2, D, torch.float32, torch.device("cpu"), cache_quant="int4")


def _append_status(**kw):
    """li_kv_scatter_int8 with host pointers: every refusal comes before a launch."""
    args = dict(batch=1, tokens=4, num_slots=64, block=16, ps_slot=32, ps_head=16, scale_s=2, heads=2, dim=16,
                dtype=_native.LI_BF16, null=False)
    args.update(kw)
    buf = (ctypes.c_int64 * 64)()
    p = None if args["null"] else ctypes.addressof(buf)
    strides = _native.i64_array([128, 64, 16, 1])
    lib = _native.load()
    return lib.li_kv_scatter_int8(p, p, strides, strides, args["batch"], args["tokens"], p, p, p, p, p,
                                  args["num_slots"], args["block"], args["ps_slot"], args["ps_head"], args["scale_s"],
                                  args["heads"], args["dim"], args["dtype"], None, None)


@pytest.mark.parametrize(("change", "status"), [
    (dict(tokens=0), _native.LI_OK), (dict(null=True), _native.LI_EINVAL), (dict(dtype=9), _native.LI_EINVAL),
    (dict(dtype=_native.LI_FP8_E4M3), _native.LI_EINVAL), (dict(batch=-1), _native.LI_EINVAL),
    (dict(block=0), _native.LI_EUNSUPPORTED), (dict(block=2048, num_slots=2048), _native.LI_EUNSUPPORTED),
    (dict(num_slots=60), _native.LI_EINVAL), (dict(num_slots=1 << 31), _native.LI_EUNSUPPORTED),
    (dict(ps_head=8), _native.LI_EINVAL), (dict(scale_s=1), _native.LI_EINVAL), (dict(tokens=1 << 30), _native.LI_EUNSUPPORTED),
])
def test_the_c_entry_refuses(change, status):
    assert _append_status(**change) == status
