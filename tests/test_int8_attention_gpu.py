"""Attention over an int8 pool with block scales against the definition in 64 bits.

Bounds, per output element, with A = the same attention over |V| (the sum of
weight times magnitude an element is made of) and h(t) half a step of t
relative to a value (bf16 2^-8, fp16 2^-11, fp32 2^-24):

* decode, MFMA kernels: the weights times their blocks' scales, over the
  largest scale M met, are rounded to fp16, h(fp16) A, and where they are
  below its normal range by at most 2^-25: of n keys, whose codes are at most
  127 and whose weights sum to at least 1, n 2^-25 127 M in all, with M up to
  twice the largest scale n 2^-24 of the largest |V|. The sum of the weights
  is not rounded. Scores: the query in 22 bits of its largest value and fp32
  products and exponentials, under 2^-14 A for the scores here (|score| < 32:
  2^-24 times 32 and log2 e, a few operations over, and D 2^-22 of the largest
  q k, below 2^-15).
* decode and packed passes, general kernel: fp32 throughout, 2^-14 A.
* packed passes, MFMA kernels, with h = h(fp16): K and V are rounded to fp16
  after a division by a power of two that keeps them in its range, weights
  are rounded to it: 2 h A and, as their sum is taken of the rounded weights,
  h |out|; weights below its normal range as in decode. The query, with the
  softmax scale in it, is rounded to fp16 too: with K's rounding this moves a
  score by at most E = scale (2 h times the largest sum of |q k|, and for what
  lies below the normal range 2^-24 times the sums of |q| and of |k|, each in
  its unit), a weight by a factor within e^-E .. e^E, and with its share of the sum the
  output by at most (e^2E - 1) (A + |out|).
* and the output's rounding, h(t) |out|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from liteinfer_amd.attention import PagedKV, eager_attention, paged_attention
from liteinfer_amd.cache.block_pool import BlockPool
from liteinfer_amd.cache.kv_cache import KVCache
from liteinfer_amd.paged_kernels import paged_decode, paged_decode_noalloc, paged_prefill
from oracle import int8 as I8
from oracle.attention import attend

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """A store of random codes and scales, and a table of random slots of it (no block in order)."""

    def __init__(self, contexts, queries=None, dtype=BF16, heads=8, kv_heads=2, dim=128, block=16, blocks=64, seed=0,
                 width=0):
        g = np.random.default_rng(seed)
        self.contexts, self.queries, self.dtype = list(contexts), queries, dtype
        self.heads, self.kv_heads, self.dim, self.block = heads, kv_heads, dim, block
        self.groups, self.scaling = heads // kv_heads, dim ** -0.5
        shape = (blocks * block, kv_heads, dim)
        self.codes = [np.clip(np.rint(g.normal(size=shape) * 40), -127, 127).astype(np.int8) for _ in range(2)]
        self.scales = [(np.exp(0.3 * g.normal(size=(blocks, kv_heads))) / 40).astype(np.float32) for _ in range(2)]
        rows = len(contexts) if queries is None else sum(queries)
        self.query = torch.from_numpy(g.normal(size=(rows, heads, dim)).astype(np.float32)).to(dtype).to(DEV)
        self.table = g.integers(0, blocks * block, size=(len(contexts), max([*contexts, width, 1])))

    def store(self):
        return [torch.from_numpy(t).to(DEV) for t in (*self.codes, *self.scales)]

    @property
    def table_t(self):
        return torch.from_numpy(self.table).to(DEV)

    @property
    def contexts_t(self):
        return torch.tensor(self.contexts, dtype=torch.int32, device=DEV)

    @property
    def starts(self):
        return None if self.queries is None else np.concatenate(([0], np.cumsum(self.queries))).astype(np.int32)

    def decode(self, **kw):
        keys, values, ks, vs = self.store()
        return paged_decode(self.query, keys, values, self.table_t, self.contexts_t, self.scaling, self.groups,
                            key_scales=ks, value_scales=vs, **kw)

    def prefill(self, **kw):
        keys, values, ks, vs = self.store()
        return paged_prefill(self.query, keys, values, self.table_t, self.contexts_t,
                             torch.from_numpy(self.starts).to(DEV), max(self.queries), self.scaling, self.groups,
                             key_scales=ks, value_scales=vs, **kw)

    def want(self):
        """(attention, attention over |V|) in 64 bits."""
        keys, values = (I8.dequantize(c, s) for c, s in zip(self.codes, self.scales))
        q = self.query.double().cpu().numpy()
        return [attend(q, keys, v, self.table, np.asarray(self.contexts), self.scaling, self.groups, self.starts)
                for v in (values, np.abs(values))]

    def moved(self):
        """e^2E - 1 of the packed passes' bound, for each query row and head: [rows, heads, 1]."""
        keys = np.abs(I8.dequantize(self.codes[0], self.scales[0]))
        q = np.abs(self.query.double().cpu().numpy())
        most = np.stack([(q[:, h] @ keys[:, h // self.groups].T).max(axis=1) for h in range(self.heads)], axis=1)
        unit = 2.0 ** (np.floor(np.log2(self.scales[0].max())) + 4)  # K's; of a short context down to 2^-3 of it
        small = 2.0 ** -24 * (q.sum(axis=2) * unit + 8 * keys.sum(axis=2).max() / unit)
        return np.expm1(2 * self.scaling * (2 * half_step(F16) * most + small))[..., None]

    def check(self, out, weight_step, copied=None):
        """`copied`: the rows that read a packed pass's copy of their contexts."""
        want, size = self.want()
        got = out.double().cpu().numpy()
        assert out.dtype == self.dtype and got.shape == want.shape
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        small = max(self.contexts) * 2.0 ** -24 * np.nanmax(np.abs(I8.dequantize(self.codes[1], self.scales[1])))
        step = half_step(self.dtype)
        extra = 0.0
        if copied is not None:
            of = np.asarray(copied).reshape(-1, 1, 1)
            moved = self.moved()
            weight_step = np.where(of, 2 * half_step(F16) + moved, weight_step)
            extra = np.where(of, half_step(F16) + moved, 0.0)
        bound = small + (weight_step + 2.0 ** -14) * size + (step + extra) * np.abs(want) * (1 + 2.0 ** -7)
        bad = np.abs(got - want) > bound + 1e-30
        assert not bad.any(), (np.abs(got - want)[bad].max(), (np.abs(got - want) / bound)[bad].max(), np.argwhere(bad)[:4])


DECODES = {
    "lengths of one to a few tiles": dict(contexts=[1, 2, 31, 32, 33, 64, 100, 500]),
    "one sequence": dict(contexts=[1000], heads=32, kv_heads=8),
    "a wide table": dict(contexts=[37, 500, 1, 4000], width=5000),
    "long contexts": dict(contexts=[9000, 17000, 300], heads=32, kv_heads=8, width=20000),
    "head_dim 64": dict(contexts=[37, 128, 500, 1023], heads=32, kv_heads=8, dim=64),
    "head_dim 64, wide": dict(contexts=[37, 128, 5000, 1023], heads=8, kv_heads=4, dim=64, width=6000),
    "one KV head": dict(contexts=[700, 3, 2500], heads=5, kv_heads=1, width=3000),
    "three KV heads, groups of 16": dict(contexts=[70, 3, 2500], heads=48, kv_heads=3, width=2500),
    "no grouping": dict(contexts=[70, 33], heads=4, kv_heads=4),
    "blocks of 1": dict(contexts=[70, 330], block=1, blocks=500),
    "blocks of 100": dict(contexts=[70, 330, 3000], block=100, blocks=9, width=4000),
    "many sequences": dict(contexts=list(range(1, 260, 2)), heads=8, kv_heads=8),
    "contexts of nothing": dict(contexts=[0, 5, 0, 70]),
    "contexts of nothing, wide": dict(contexts=[0, 5, 0, 7000], width=8000),
}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kernel", ["auto", "equal_splits", "generic"])
@pytest.mark.parametrize("name", DECODES)
def test_decode(name, kernel, dtype):
    batch = Batch(**DECODES[name], dtype=dtype)
    kw = dict(num_splits=3) if kernel == "equal_splits" else {}
    batch.check(batch.decode(kernel=kernel, **kw), 0.0 if kernel == "generic" else half_step(F16))


@pytest.mark.parametrize("shape", [dict(dim=80), dict(dim=256), dict(heads=34, kv_heads=2), dict(dtype=F32), dict(dim=33),
                                   dict(dtype=F32, dim=64, contexts=[3000, 20], width=4000)])
def test_decode_of_other_shapes_runs_the_general_kernel(shape):
    batch = Batch(**(dict(contexts=[1, 70, 700]) | shape))
    batch.check(batch.decode(), 0.0)


PASSES = {
    "whole prompts": dict(contexts=[1, 33, 200, 64], queries=[1, 33, 200, 64]),
    "chunks over a prefix": dict(contexts=[700, 300, 90], queries=[200, 7, 64], heads=32, kv_heads=8),
    "chunks and rows": dict(contexts=[300, 900, 70, 2000, 5], queries=[100, 1, 33, 1, 1], heads=32, kv_heads=8),
    "only rows": dict(contexts=[300, 900, 70], queries=[1, 1, 1]),
    "a sequence without queries": dict(contexts=[300, 90, 70], queries=[100, 0, 33]),
    "small over a long prefix": dict(contexts=[6000], queries=[100], heads=32, kv_heads=8),
    "small over a long prefix, head_dim 64": dict(contexts=[6000], queries=[100], heads=32, kv_heads=8, dim=64),
    "head_dim 64": dict(contexts=[300, 900, 70], queries=[100, 1, 33], heads=8, kv_heads=4, dim=64),
    "many sequences": dict(contexts=[50 + 3 * i for i in range(70)], queries=[1 + (7 * i) % 40 for i in range(70)]),
    "groups of 5": dict(contexts=[400, 90], queries=[300, 90], heads=10, kv_heads=2),
    "blocks of 100": dict(contexts=[400, 90], queries=[300, 1], block=100, blocks=9),
}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens known", "tokens unknown"])
@pytest.mark.parametrize("name", PASSES)
def test_packed_passes(name, tokens, dtype):
    batch = Batch(**PASSES[name], dtype=dtype)
    out = batch.prefill(context_tokens=sum(batch.contexts) if tokens else None)
    _check_packed(batch, out)


def _check_packed(batch, out):
    """Rows of one query are decoded, the others read the copy."""
    batch.check(out, half_step(F16), copied=np.repeat(np.asarray(batch.queries) > 1, batch.queries))
    assert torch.isfinite(out).all()


SPREAD = dict(contexts=[700, 90, 5000, 33], queries=[100, 1, 300, 20], heads=8, kv_heads=2, width=5000)


@pytest.mark.parametrize("power", [-90, -30, 12, 40, 100])
def test_packed_passes_over_values_of_any_size(power):
    """V times a power of two: the output times it, bit for bit (the units are one for each head)."""
    batch = Batch(**SPREAD)
    plain = batch.prefill(one_query_rows=False)
    batch.scales[1][:, 1] *= np.float32(2.0 ** power)
    got = batch.prefill(one_query_rows=False)
    assert torch.equal(got[:, :4], plain[:, :4])
    assert torch.equal(got[:, 4:], plain[:, 4:] * 2.0 ** power)


@pytest.mark.parametrize("power", [-80, -20, 5, 18, 60])
def test_packed_passes_over_keys_of_any_size(power):
    """K times a power of two and the query by its inverse: the same output, bit for bit."""
    batch = Batch(**SPREAD)
    plain = batch.prefill()
    _check_packed(batch, plain)
    batch.scales[0] *= np.float32(2.0 ** power)
    batch.query = batch.query * 2.0 ** -power
    assert torch.equal(batch.prefill(), plain)


@pytest.mark.parametrize("name", PASSES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_passes_of_the_general_kernel(name, dtype):
    batch = Batch(**PASSES[name], dtype=dtype)
    batch.check(batch.prefill(kernel="auto" if dtype == F32 else "generic"), 0.0)


@pytest.mark.parametrize("flag", [True, False, None])
def test_rows_folded_as_queries_of_the_pass(flag):
    batch = Batch(contexts=[300, 900, 70, 2000], queries=[100, 1, 33, 1], heads=32, kv_heads=8)
    out = batch.prefill(one_query_rows=flag)
    if flag is False:  # every sequence reads the copy
        batch.check(out, half_step(F16), copied=np.ones(sum(batch.queries), bool))
    else:
        _check_packed(batch, out)


def test_rows_behind_the_last_sequence_are_left_as_they_were():
    batch = Batch(contexts=[300, 90], queries=[100, 20], heads=8, kv_heads=2)
    wide = torch.full((150, 8, 128), 7.0, dtype=BF16, device=DEV)
    query = torch.cat([batch.query, torch.randn(30, 8, 128, device=DEV).to(BF16)])
    keys, values, ks, vs = batch.store()
    got = paged_prefill(query, keys, values, batch.table_t, batch.contexts_t, torch.from_numpy(batch.starts).to(DEV), 100,
                        batch.scaling, batch.groups, key_scales=ks, value_scales=vs, out=wide)
    assert got is wide and (wide[120:] == 7.0).all()
    _check_packed(batch, wide[:120])


def test_what_lies_past_a_context_does_not_matter():
    """Table columns past a context name blocks whose scale is NaN, and slots that do not exist."""
    for width in (500, 3000):
        batch = Batch(contexts=[70, 33, 1], width=width, blocks=64)
        want = batch.decode()
        batch.scales[0][50:], batch.scales[1][50:] = np.nan, np.inf
        batch.table %= 50 * 16
        want = batch.decode()
        for i, c in enumerate(batch.contexts):
            batch.table[i, c:] = 50 * 16 + i
        assert torch.equal(batch.decode(), want) and torch.isfinite(want).all()


def test_a_block_that_holds_nan_gives_nan_to_its_readers_only():
    for queries in (None, [30, 1, 20]):
        for dim in (128, 80):
            batch = Batch(contexts=[70, 33, 40], queries=queries, dim=dim, blocks=64)
            batch.table %= 32 * 16
            batch.table[1, 3] = 50 * 16 + 2
            batch.scales[1][50, 0] = np.nan
            out = batch.decode() if queries is None else batch.prefill()
            row = slice(1, 2) if queries is None else slice(30, 31)
            nan = torch.isnan(out)
            assert nan[row, :batch.groups].all() and not nan[row, batch.groups:].any()
            nan[row] = False
            assert not nan.any()


@pytest.mark.parametrize("of", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("dim", [128, 64, 80])
@pytest.mark.parametrize("context, queries", [(70, 30), (2100, 300), (900, 900)])
def test_a_token_that_is_not_finite_is_not_seen_before_it(context, queries, dim, of):
    """Causal: a chunk's queries in front of the NaN do not read it, though it lies in their tile."""
    batch = Batch(contexts=[context, 40], queries=[queries, 1], dim=dim, width=3000)
    batch.table %= 32 * 16
    at = context - 10
    batch.table[0, at] = 50 * 16 + 2
    batch.scales[of][50, 0] = np.nan
    nan = torch.isnan(batch.prefill())
    first = queries - 10
    assert nan[first:queries, :batch.groups].all()
    nan[first:queries, :batch.groups] = False
    assert not nan.any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_gives_nan(value):
    for width in (0, 4000):
        batch = Batch(contexts=[70, 33, 40], width=width)
        batch.query[1, 2, 5] = value
        out = batch.decode()
        assert torch.isnan(out[1, 2]).all()
        nan = torch.isnan(out)
        nan[1, 2] = False
        assert not nan.any()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [128, 64])
def test_a_chunks_query_that_is_not_finite_gives_nan(dim, value):
    for context in (70, 2100):
        batch = Batch(contexts=[context, 40], queries=[60, 1], dim=dim, width=3000)
        batch.query[17, 2, 5] = value
        nan = torch.isnan(batch.prefill())
        assert nan[17, 2].all()
        nan[17, 2] = False
        assert not nan.any()


def test_sequences_without_queries_beside_chunks():
    """Nothing is laid out for them, whatever they hold."""
    batch = Batch(contexts=[300, 500, 90, 0, 40], queries=[100, 0, 20, 0, 1], width=1000)
    _check_packed(batch, batch.prefill())
    tokens = batch.prefill(context_tokens=930)
    _check_packed(batch, tokens)


def test_queries_of_very_different_sizes():
    """Outliers in the query and in K, large and small queries: the scores keep the query to 22 bits of its row."""
    for scale in (1e-30, 1e-3, 30.0):
        batch = Batch(contexts=[70, 900, 40], width=4000, dtype=BF16)
        batch.query *= scale
        batch.query[:, :, 7] *= 20
        if scale > 1:
            batch.query *= 0.02
        batch.check(batch.decode(), half_step(F16))
    batch = Batch(contexts=[70, 900, 40], width=4000)
    batch.query.zero_()
    batch.check(batch.decode(), half_step(F16))


def test_scales_of_very_different_sizes():
    for width in (0, 4000):
        batch = Batch(contexts=[70, 900, 40], width=width)
        g = np.random.default_rng(5)
        batch.scales[1] *= np.exp(8 * g.normal(size=batch.scales[1].shape)).astype(np.float32)
        batch.scales[0][::3] = 2.0 ** -126
        batch.check(batch.decode(), half_step(F16))


def test_slots_past_32_bits_of_bytes():
    """A store of over 4 GiB: rows near its end."""
    blocks = 80000
    keys = torch.zeros(blocks * 64, 8, 128, dtype=torch.int8, device=DEV)
    values = torch.zeros_like(keys)
    ks, vs = (torch.ones(blocks, 8, device=DEV) / 40 for _ in range(2))
    batch = Batch(contexts=[300, 70], heads=8, kv_heads=8, block=64, blocks=5)
    far = (blocks - 5) * 64
    keys[far:], values[far:] = (torch.from_numpy(c).to(DEV) for c in batch.codes)
    ks[-5:], vs[-5:] = (torch.from_numpy(s).to(DEV) for s in batch.scales)
    for width in (0, 5000):
        table = torch.nn.functional.pad(batch.table_t + far, (0, max(0, width - batch.table.shape[1])))
        out = paged_decode(batch.query, keys, values, table, batch.contexts_t, batch.scaling, 1, key_scales=ks, value_scales=vs)
        batch.check(out, half_step(F16))
    batch.queries = [1, 1]
    for one_query_rows in (False, True):
        out = paged_prefill(batch.query, keys, values, batch.table_t + far, batch.contexts_t,
                            torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), 1, batch.scaling, 1,
                            one_query_rows=one_query_rows, key_scales=ks, value_scales=vs)
        batch.check(out, half_step(F16))
    batch = Batch(contexts=[300, 70], queries=[30, 2], heads=8, kv_heads=8, block=64, blocks=5)
    keys[far:], values[far:] = (torch.from_numpy(c).to(DEV) for c in batch.codes)
    ks[-5:], vs[-5:] = (torch.from_numpy(s).to(DEV) for s in batch.scales)
    out = paged_prefill(batch.query, keys, values, batch.table_t + far, batch.contexts_t,
                        torch.from_numpy(batch.starts).to(DEV), 30, batch.scaling, 1, key_scales=ks, value_scales=vs)
    batch.check(out, half_step(F16), copied=np.ones(sum(batch.queries), bool))


def test_strided_operands():
    batch = Batch(contexts=[70, 333], width=2000, heads=8, kv_heads=2)
    keys, values, ks, vs = batch.store()
    wide = torch.zeros(2, keys.shape[0], 3, 160, dtype=torch.int8, device=DEV)
    wide[0, :, 1:, 16:144], wide[1, :, 1:, 16:144] = keys, values
    scales = torch.zeros(2, ks.shape[0], 6, device=DEV)
    scales[0, :, 2:4], scales[1, :, 2:4] = ks, vs
    query = torch.zeros(2, 8, 136, dtype=BF16, device=DEV)
    query[..., :128] = batch.query
    out = paged_decode(query[..., :128], wide[0, :, 1:, 16:144], wide[1, :, 1:, 16:144],
                       batch.table_t.to(torch.int32), batch.contexts_t.long(), batch.scaling, 4,
                       key_scales=scales[0, :, 2:4], value_scales=scales[1, :, 2:4])
    batch.check(out, half_step(F16))


def test_a_sequence_of_operators_as_a_layer_runs_them():
    """Prompt, chunk beside a decode row, decode steps: append and attend through a cache's payloads."""
    torch.manual_seed(0)
    pool = BlockPool(num_blocks=64, block_size=16, num_layers=1, num_kv_heads=2, head_dim=128, dtype=BF16, device=DEV,
                     cache_quant="int8")
    plain = BlockPool(num_blocks=64, block_size=16, num_layers=1, num_kv_heads=2, head_dim=128, dtype=BF16, device=DEV)
    caches = [KVCache(pool), KVCache(plain)]
    outs = []
    starts = {"a": 0, "b": 0}
    for step in ([("a", 100)], [("a", 1), ("b", 45)], [("a", 1), ("b", 1)], [("a", 1), ("b", 1)], [("a", 17), ("b", 1)]):
        ids, counts = [i for i, _ in step], [c for _, c in step]
        begin = [starts[i] for i in ids]
        n = sum(counts)
        q, k, v = (torch.randn(1, n, h, 128, device=DEV).to(BF16).transpose(1, 2) for h in (8, 2, 2))
        angle = torch.rand(1, n, 64, device=DEV) * 6
        cos, sin = (torch.cat((t, t), -1).to(BF16) for t in (angle.cos(), angle.sin()))
        got = []
        for cache in caches:
            cache.reserve(ids, [b + c for b, c in zip(begin, counts)])
            payload = cache.make_packed_payload(ids, begin, counts)
            rotated, kv = payload.update_rotated(q, k, v, cos, sin, 0)
            got.append((paged_attention(rotated, kv, 128 ** -0.5, 4), eager_attention(rotated.float(), kv, 128 ** -0.5, 4)
                        if cache is caches[0] else None))
        for i, c in step:
            starts[i] += c
        outs.append(got)
    for (mine, dense), (other, _) in outs:
        # The dense kernel reads the same codes, in fp32: only roundings to bf16 between them (weights, K, V, output).
        assert (mine.float() - dense).abs().max() <= 4 * 2.0 ** -8 * 4.5  # |V| < 4.5
        # And the 16-bit cache: codes are off by up to a few steps of their block's scale.
        assert (mine.float() - other.float()).norm() <= 0.05 * other.float().norm()
    pool.check_slot_writes()


def test_a_captured_step_replays_for_other_contexts():
    for width in (600, 5000):
        batch = Batch(contexts=[500, 300, 17, 64], width=width)
        keys, values, ks, vs = batch.store()
        table, contexts = batch.table_t, batch.contexts_t

        def call():
            return paged_decode(batch.query, keys, values, table, contexts, batch.scaling, batch.groups, key_scales=ks,
                                value_scales=vs)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for lens in ([500, 300, 17, 64], [1, 2, 600, 33], [600, 600, 600, 600]):
            batch.contexts = lens
            contexts.copy_(torch.tensor(lens, dtype=torch.int32))
            batch.table = np.resize(batch.table, (4, max(width, 600)))
            batch.table[:, :table.shape[1]] = table.cpu().numpy()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call())
            batch.check(out, half_step(F16))


def test_a_captured_packed_pass_replays_for_longer_contexts():
    """Through the payload, whose host lengths are those of the capture."""
    batch = Batch(contexts=[300, 90, 40], queries=[100, 20, 1], width=1000)
    keys, values, ks, vs = batch.store()
    contexts, starts = batch.contexts_t, torch.from_numpy(batch.starts).to(DEV)
    query = batch.query.transpose(0, 1).unsqueeze(0)
    kv = PagedKV(keys, values, batch.table_t, contexts, query_start_loc=starts, max_query_len=100,
                 host_context_lens=(300, 90, 40), host_query_lens=(100, 20, 1), key_scales=ks, value_scales=vs)

    def call():
        return paged_attention(query, kv, batch.scaling, batch.groups)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([300, 90, 40], [1000, 700, 999], [100, 20, 1], [640, 1000, 3]):
        batch.contexts = lens
        contexts.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check_packed(batch, out[0].transpose(0, 1))


def test_two_calls_on_two_streams():
    batches = [Batch(contexts=[4000, 300, 77], width=6000, seed=s) for s in range(2)]
    stores = [b.store() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    tables, lens = [b.table_t for b in batches], [b.contexts_t for b in batches]
    torch.cuda.synchronize()
    outs = []
    for b, (k, v, ks, vs), t, c, s in zip(batches, stores, tables, lens, streams):
        with torch.cuda.stream(s):
            outs.append(paged_decode(b.query, k, v, t, c, b.scaling, b.groups, key_scales=ks, value_scales=vs))
    torch.cuda.synchronize()
    for b, out in zip(batches, outs):
        b.check(out, half_step(F16))


def test_refusals():
    batch = Batch(contexts=[70, 33], queries=[20, 1])
    keys, values, ks, vs = batch.store()
    step = Batch(contexts=[70, 33])
    args = (step.query, keys, values, step.table_t, step.contexts_t, step.scaling, step.groups)
    row = torch.zeros(2, 2, 128, dtype=BF16, device=DEV)
    for kw, message in ((dict(), "needs key_scales"), (dict(key_scales=ks, value_scales=vs[:-1]), "laid out"),
                        (dict(key_scales=ks, value_scales=vs.double()), "float32"),
                        (dict(key_scales=ks, value_scales=vs, new_key=row, new_value=row), "kv_scatter"),
                        (dict(key_scales=ks, value_scales=vs, kernel="fast"), "kernel"),
                        (dict(key_scales=ks, value_scales=vs, num_splits=0), "num_splits")):
        with pytest.raises(ValueError, match=message):
            paged_decode(*args, **kw)
    with pytest.raises(ValueError, match="int8 pool"):
        paged_decode(step.query, keys.to(BF16), values.to(BF16), *args[3:], key_scales=ks, value_scales=vs)
    with pytest.raises(ValueError):
        paged_decode(step.query.double(), *args[1:], key_scales=ks, value_scales=vs)
    with pytest.raises(ValueError, match="pool of the query"):
        paged_decode_noalloc(*args, out=torch.empty_like(step.query))
    with pytest.raises(ValueError, match="needs key_scales"):
        paged_attention(step.query.unsqueeze(2), PagedKV(keys, values, step.table_t, step.contexts_t), step.scaling, 4)
    with pytest.raises(ValueError, match="context_tokens"):
        batch.prefill(context_tokens=-1)
