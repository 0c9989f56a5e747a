"""The int8 slot-write on the GPU: codes and scales bit for bit as the definition in float32 gives them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from liteinfer_amd.cache.block_pool import BlockPool
from liteinfer_amd.cache.kv_cache import KVCache
from liteinfer_amd.paged_kernels import check_bad_slots, kv_scatter
from liteinfer_amd.rope import rope_kv_write
from oracle import int8 as I8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


class Case:
    """A store in use and a pass's rows: tokens of several sequences, each from a position of its own."""

    def __init__(self, lens, heads, kv_heads, dim, dtype, block=16, seed=0, step=False, spare=3):
        g = np.random.default_rng(seed)
        self.dtype, self.block, self.step = dtype, block, step
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        counts = [(s + c - 1) // block - s // block + 1 for s, c in lens]
        order = g.permutation(sum(counts) + spare)
        slots, at = [], 0
        for (s, c), n in zip(lens, counts):
            table = order[at:at + n]
            at += n
            slots += [int(table[p // block - s // block]) * block + p % block for p in range(s, s + c)]
        self.slots = np.asarray(slots, dtype=np.int64)
        blocks = len(order)
        shape = (blocks * block, kv_heads, dim)
        self.codes = [g.integers(-127, 128, size=shape).astype(np.int8) for _ in range(2)]
        self.scales = [np.abs(g.normal(size=(blocks, kv_heads))).astype(np.float32) * 0.02 for _ in range(2)]
        n = len(slots)
        lead = (n, 1) if step else (1, n)
        qkv = torch.from_numpy(g.normal(size=(*lead, heads + 2 * kv_heads, dim)).astype(np.float32)).to(dtype).to(DEV)
        self.q, self.k, self.v = (t.transpose(1, 2) for t in qkv.split((heads, kv_heads, kv_heads), dim=2))
        angle = torch.from_numpy(g.uniform(0, 6.3, size=(*lead, dim)))
        self.cos, self.sin = angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV)

    def device(self):
        return [torch.from_numpy(t.copy()).to(DEV) for t in (*self.codes, *self.scales)]

    def slots_t(self):
        return torch.from_numpy(self.slots).to(DEV)[None]

    @staticmethod
    def rows(t):  # [B, H, T, D] -> float32 [B * T, H, D]
        return t.float().cpu().transpose(1, 2).flatten(0, 1).numpy()

    def rotated(self, t):
        tables = (x.float().cpu().flatten(0, 1).numpy() for x in (self.cos, self.sin))
        return I8.rotate(self.rows(t), *tables)

    def want(self, rope):
        k = self.rotated(self.k) if rope else self.rows(self.k)
        keys = I8.append(self.codes[0], self.scales[0], self.slots, k)
        values = I8.append(self.codes[1], self.scales[1], self.slots, self.rows(self.v))
        return keys[0], values[0], keys[1], values[1]


def _check(got, want):
    for name, g, w in zip(("keys", "values", "key_scales", "value_scales"), got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)


def _write(case, store, rope=True, **kw):
    keys, values, key_scales, value_scales = store
    kw |= dict(key_scales=key_scales, value_scales=value_scales)
    if rope:
        return rope_kv_write(case.q, case.k, case.v, case.cos, case.sin, case.slots_t(), keys, values, **kw)
    kv_scatter(keys, values, case.slots_t(), case.k, case.v, **kw)
    return None


SHAPES = {
    "decode step": dict(lens=[(p, 1) for p in range(0, 160, 5)], heads=32, kv_heads=8, dim=128, step=True),
    "one token": dict(lens=[(15, 1)], heads=4, kv_heads=2, dim=64, step=True),
    "ragged chunks": dict(lens=[(0, 37), (5, 3), (31, 1), (16, 16), (250, 70)], heads=8, kv_heads=2, dim=128),
    "long pass": dict(lens=[(3, 700), (0, 900), (77, 11)], heads=4, kv_heads=1, dim=64),
    "blocks of 64": dict(lens=[(10, 200), (63, 2)], heads=4, kv_heads=2, dim=128, block=64),
    "blocks of 1": dict(lens=[(3, 9)], heads=4, kv_heads=2, dim=64, block=1),
    "blocks of 100": dict(lens=[(0, 130), (60, 3)], heads=2, kv_heads=1, dim=32, block=100),
    "head_dim 96": dict(lens=[(0, 20), (9, 30)], heads=6, kv_heads=3, dim=96),
    "head_dim 256": dict(lens=[(2, 40)], heads=4, kv_heads=2, dim=256),
    "head_dim 72, element by element": dict(lens=[(2, 40), (0, 1)], heads=4, kv_heads=2, dim=72),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rope", [True, False], ids=["rope", "scatter"])
@pytest.mark.parametrize("name", SHAPES)
def test_codes_and_scales_are_the_definitions(name, rope, dtype):
    case = Case(**SHAPES[name], dtype=dtype)
    store = case.device()
    q = _write(case, store, rope)
    _check(store, case.want(rope))
    if rope:
        want = case.rotated(case.q)
        got = case.rows(q)
        np.testing.assert_array_equal(got, torch.from_numpy(want).to(dtype).float().numpy())


def test_an_odd_head_dim_scatters():
    case = Case(lens=[(2, 20), (40, 3)], heads=2, kv_heads=2, dim=33, dtype=torch.bfloat16)
    store = case.device()
    _write(case, store, rope=False)
    _check(store, case.want(False))


def test_strided_rows_and_pools():
    """Rows that are no 16-byte multiples apart, a pool and scales that are views of wider ones."""
    case = Case(lens=[(3, 30), (0, 5)], heads=4, kv_heads=2, dim=64, dtype=torch.float16)
    case.k = torch.nn.functional.pad(case.k, (0, 3))[..., :64]
    case.q = case.q.transpose(2, 3).contiguous().transpose(2, 3)
    keys, values, ks, vs = case.device()
    wide = [torch.full((t.shape[0], 4, 72), 55, dtype=torch.int8, device=DEV) for t in (keys, values)]
    scales = [torch.full((t.shape[0], 5), 7.0, device=DEV) for t in (ks, vs)]
    for w, t in zip(wide, (keys, values)):
        w[:, 1:3, 8:72] = t
    for w, t in zip(scales, (ks, vs)):
        w[:, :2] = t
    views = [*(w[:, 1:3, 8:72] for w in wide), *(w[:, :2] for w in scales)]
    _write(case, views)
    _check([t.contiguous() for t in views], case.want(True))
    for w in wide:
        assert (w[:, 0] == 55).all() and (w[:, 3] == 55).all() and (w[:, 1:3, :8] == 55).all()
    for w in scales:
        assert (w[:, 2:] == 7.0).all()


def test_slots_outside_the_pool_are_skipped_and_counted_and_do_not_cut_a_run():
    case = Case(lens=[(4, 12), (0, 40)], heads=4, kv_heads=2, dim=128, dtype=torch.bfloat16)
    case.slots[[2, 5, 20]] = [-1, case.codes[0].shape[0], 1 << 40]
    store = case.device()
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    _write(case, store, bad_slots=bad)
    _check(store, case.want(True))
    with pytest.raises(IndexError, match="3 K/V"):
        check_bad_slots(bad)


def test_a_slot_named_many_times_keeps_the_last_token():
    """The padding rows of a captured decode step all name one slot."""
    case = Case(lens=[(0, 1), (7, 2), (0, 300)], heads=4, kv_heads=2, dim=128, dtype=torch.bfloat16)
    case.slots[3:] = case.slots[3] // 16 * 16
    case.slots[1] = case.slots[2]
    store = case.device()
    _write(case, store)
    _check(store, case.want(True))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [128, 72])
def test_values_that_are_not_finite(bad, dim):
    case = Case(lens=[(3, 9), (20, 1), (32, 20)], heads=2, kv_heads=2, dim=dim, dtype=torch.bfloat16)
    case.v[0, 1, 4, 7] = bad
    case.k[0, 0, 9, 70] = bad
    case.scales[0][case.slots[12] // 16, 1] = np.nan  # (started anew by this pass)
    store = case.device()
    _write(case, store)
    want = case.want(True)
    assert np.isnan(want[3]).any() and np.isnan(want[2]).any()
    _check(store, want)


def test_large_and_small_values():
    for scale in (3e38, 1e30, 1e-30, 1e-38, 0.0):
        case = Case(lens=[(3, 9), (20, 1)], heads=2, kv_heads=1, dim=64, dtype=torch.bfloat16)
        case.v[:] = (case.v.float().sign() * scale).to(torch.bfloat16)
        store = case.device()
        _write(case, store, rope=False)
        _check(store, case.want(False))


def test_step_after_step_as_a_sequence_grows():
    case = Case(lens=[(0, 50)], heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16)
    want = [t.copy() for t in (*case.codes, *case.scales)]
    store = case.device()
    k, v = case.rows(case.k), case.rows(case.v)
    at = 0
    for count in (1, 3, 1, 1, 20, 1, 7, 16):
        cut = slice(at, at + count)
        kv_scatter(store[0], store[1], case.slots_t()[:, cut], case.k[:, :, cut], case.v[:, :, cut],
                   key_scales=store[2], value_scales=store[3])
        want[0], want[2] = I8.append(want[0], want[2], case.slots[cut], k[cut])
        want[1], want[3] = I8.append(want[1], want[3], case.slots[cut], v[cut])
        at += count
    _check(store, want)


def test_a_captured_write_replays():
    case = Case(lens=[(p, 1) for p in (3, 16, 40, 7)], heads=8, kv_heads=2, dim=128, dtype=torch.bfloat16, step=True)
    store, fresh, warm, slots = case.device(), case.device(), case.device(), case.slots_t()
    case.slots_t = lambda: slots
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _write(case, warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = _write(case, store)
    want = case.want(True)
    for _ in range(3):
        for s, f in zip(store, fresh):
            s.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        _check(store, want)
        eager = case.device()
        assert torch.equal(q, _write(case, eager))


def test_two_streams_write_their_own_blocks():
    cases = [Case(lens=[(2, 300)], heads=8, kv_heads=2, dim=128, dtype=torch.bfloat16, seed=s) for s in range(2)]
    stores = [c.device() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for c, st, stream in zip(cases, stores, streams):
        with torch.cuda.stream(stream):
            _write(c, st)
    torch.cuda.synchronize()
    for c, st in zip(cases, stores):
        _check(st, c.want(True))


def test_a_cache_writes_through_its_payloads():
    pool = BlockPool(num_blocks=32, block_size=16, num_layers=2, num_kv_heads=2, head_dim=128, dtype=torch.bfloat16,
                     device=DEV, cache_quant="int8")
    cache = KVCache(pool)
    cache.reserve(["a", "b"], [40, 9])
    payload = cache.make_packed_payload(["a", "b"], [0, 0], [40, 9])
    case = Case(lens=[(0, 49)], heads=4, kv_heads=2, dim=128, dtype=torch.bfloat16)
    case.slots = payload.addresses.slots.cpu().numpy().reshape(-1)
    case.codes = [np.zeros((512, 2, 128), np.int8) for _ in range(2)]
    case.scales = [np.zeros((32, 2), np.float32) for _ in range(2)]
    q, kv = payload.update_rotated(case.q, case.k, case.v, case.cos, case.sin, 1)
    _check((kv.key_pool, kv.value_pool, kv.key_scales, kv.value_scales), case.want(True))
    pool.check_slot_writes()


def test_refusals():
    case = Case(lens=[(0, 4)], heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16)
    keys, values, ks, vs = case.device()
    with pytest.raises(ValueError, match="needs key_scales"):
        _write(case, (keys, values, None, None))
    with pytest.raises(ValueError, match="int8 pool"):
        _write(case, (keys.to(torch.bfloat16), values.to(torch.bfloat16), ks, vs))
    with pytest.raises(ValueError, match="whole number"):
        _write(case, (keys[:-1], values[:-1], ks, vs))
    with pytest.raises(ValueError, match="on cuda"):
        _write(case, (keys, values, ks.cpu(), vs.cpu()))
    case.v = case.v.double()
    with pytest.raises(ValueError):
        _write(case, (keys, values, ks, vs))
    with pytest.raises(ValueError, match="int8 pool takes"):
        _write(case, (keys, values, ks, vs), rope=False)
