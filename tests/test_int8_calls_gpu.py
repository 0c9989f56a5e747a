"""The int8 calls through their C++ host side and through Python: the same results, the same errors."""

from __future__ import annotations

import pytest
import torch

from liteinfer_amd import _native
from liteinfer_amd.engine.ops import linear_int8
from liteinfer_amd.paged_kernels import paged_decode, paged_prefill
from liteinfer_amd.rope import rope_kv_write

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


class _Counting:
    """The module, counting the int8 calls it served; or one that serves none."""

    def __init__(self, serve):
        self.real, self.serve, self.served = _native.fast_calls(), serve, 0

    def __getattr__(self, name):
        def run(*args):
            out = getattr(self.real, name)(*args) if self.serve else None
            self.served += out is not None
            return out

        return run


def _both(monkeypatch, call):
    got = []
    for serve in (True, False):
        counting = _Counting(serve)
        monkeypatch.setattr(_native, "_fast", counting)
        try:
            got.append(call())
        except Exception as e:  # compared below
            got.append((type(e), str(e)))
        if serve:
            served = counting.served
        monkeypatch.setattr(_native, "_fast", counting.real)
    return got[0], got[1], served


def _same(a, b):
    if isinstance(a, torch.Tensor):
        return a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a.nan_to_num(), b.nan_to_num())
    return a == b


def _store(heads=2, dim=128, blocks=20, block=16):
    g = torch.Generator().manual_seed(0)
    codes = [torch.randint(-127, 128, (blocks * block, heads, dim), generator=g, dtype=torch.int8).to(DEV) for _ in range(2)]
    return codes + [torch.rand(blocks, heads, generator=g).to(DEV) / 50 for _ in range(2)]


def _attend_operands(queries=3):
    g = torch.Generator().manual_seed(1)
    keys, values, ks, vs = _store()
    return dict(query=torch.randn(queries, 8, 128, generator=g).to(BF16).to(DEV), key_pool=keys, value_pool=values,
                slot_table=torch.randint(0, 320, (3, 200), generator=g).to(DEV),
                context_lens=torch.tensor([200, 1, 77], dtype=torch.int32, device=DEV), key_scales=ks, value_scales=vs)


# (changes to the operands, whether C++ serves the call)
DECODES = {
    "plain": (lambda o: {}, True),
    "fp16": (lambda o: {"query": o["query"].to(torch.float16)}, True),
    "fp32": (lambda o: {"query": o["query"].float()}, True),
    "strided query": (lambda o: {"query": o["query"].repeat(1, 1, 2)[..., :128]}, True),
    "int32 table": (lambda o: {"slot_table": o["slot_table"].int()}, False),
    "int64 lengths": (lambda o: {"context_lens": o["context_lens"].long()}, False),
    "scales within wider ones": (lambda o: {k: torch.cat([o[k], o[k]], dim=1)[:, :2] for k in ("key_scales", "value_scales")}, True),
    "no scales": (lambda o: {"key_scales": None, "value_scales": None}, False),
    "scales of one": (lambda o: {"value_scales": None}, False),
    "scales of another shape": (lambda o: {"value_scales": o["value_scales"][:10]}, False),
    "blocks that do not divide": (lambda o: {k: o[k][:19] for k in ("key_scales", "value_scales")}, False),
    "wrong heads": (lambda o: {"query": o["query"][:, :6]}, False),
    "wrong dim": (lambda o: {"query": o["query"][..., :64]}, False),
    "splits": (lambda o: {"num_splits": 4, "kernel": "equal_splits"}, True),
    "bad splits": (lambda o: {"num_splits": 0}, False),
    "bad kernel": (lambda o: {"kernel": "fast"}, False),
    "no sequences": (lambda o: {k: o[k][:0] for k in ("query", "slot_table", "context_lens")}, False),
}


@pytest.mark.parametrize("name", DECODES)
def test_decode(monkeypatch, name):
    change, serves = DECODES[name]
    operands = _attend_operands()
    operands |= change(operands)
    args = [operands.pop(k) for k in ("query", "key_pool", "value_pool", "slot_table", "context_lens")]
    a, b, served = _both(monkeypatch, lambda: paged_decode(*args, 128 ** -0.5, 4, **operands))
    assert _same(a, b), (a, b)
    assert bool(served) == serves


PASSES = {
    "plain": (lambda o: {}, True),
    "tokens known": (lambda o: {"context_tokens": 278}, True),
    "an output": (lambda o: {"out": torch.zeros_like(o["query"])}, True),
    "rows folded": (lambda o: {"one_query_rows": False}, True),
    "general": (lambda o: {"kernel": "generic"}, True),
    "int64 starts": (lambda o: {"starts": o["starts"].long()}, False),
    "negative tokens": (lambda o: {"context_tokens": -3}, False),
    "wrong starts": (lambda o: {"starts": o["starts"][:-1]}, False),
    "an output of another type": (lambda o: {"out": torch.zeros(78, 8, 128, device=DEV)}, False),
}


@pytest.mark.parametrize("name", PASSES)
def test_prefill(monkeypatch, name):
    change, serves = PASSES[name]
    operands = _attend_operands(78) | {"starts": torch.tensor([0, 60, 61, 78], dtype=torch.int32, device=DEV)}
    operands |= change(operands)
    args = [operands.pop(k) for k in ("query", "key_pool", "value_pool", "slot_table", "context_lens", "starts")]
    a, b, served = _both(monkeypatch, lambda: paged_prefill(*args, 60, 128 ** -0.5, 4, **operands))
    assert _same(a, b), (a, b)
    assert bool(served) == serves


ROPES = {
    "plain": (lambda o: {}, True),
    "packed": (lambda o: {k: o[k].permute(2, 1, 0, 3) for k in "qkv"} | {k: o[k].transpose(0, 1) for k in ("cos", "sin")}, True),
    "tables of one row": (lambda o: {k: o[k][:1] for k in ("cos", "sin")}, True),
    "a counter": (lambda o: {"bad_slots": torch.zeros(1, dtype=torch.int32, device=DEV)}, True),
    "int32 slots": (lambda o: {"slots": o["slots"].int()}, False),
    "a wrong counter": (lambda o: {"bad_slots": torch.zeros(1, device=DEV)}, False),
    "types that differ": (lambda o: {"v": o["v"].float()}, False),
    "too many slots": (lambda o: {"slots": o["slots"][:, :2]}, False),
    "no scales": (lambda o: {"key_scales": None, "value_scales": None}, False),
}


@pytest.mark.parametrize("name", ROPES)
def test_rope(monkeypatch, name):
    change, serves = ROPES[name]
    g = torch.Generator().manual_seed(2)
    heads = {"q": 8, "k": 2, "v": 2}
    operands = {k: torch.randn(3, h, 1, 128, generator=g).to(BF16).to(DEV) for k, h in heads.items()}
    operands |= {k: torch.randn(3, 1, 128, generator=g).to(BF16).to(DEV) for k in ("cos", "sin")}
    operands |= {"slots": torch.tensor([[5, 40, 100]], device=DEV)}
    operands |= change(operands | {"key_scales": 0})
    stores = []

    def call():
        keys, values, ks, vs = _store()
        stores.append((keys, values, ks, vs))
        scales = {"key_scales": ks, "value_scales": vs}
        kw = {k: v for k, v in operands.items() if k in ("bad_slots", "key_scales", "value_scales")}
        return rope_kv_write(*(operands[k] for k in ("q", "k", "v", "cos", "sin", "slots")), keys, values, **(scales | kw))

    a, b, served = _both(monkeypatch, call)
    assert _same(a, b), (a, b)
    assert bool(served) == serves
    for s, t in zip(*stores):
        assert torch.equal(s, t)


LINEARS = {
    "plain": (lambda o: {}, True),
    "three axes": (lambda o: {"x": o["x"].view(2, 3, 100)}, True),
    "one row": (lambda o: {"x": o["x"][0]}, True),
    "strided": (lambda o: {"x": o["x"].repeat(1, 2)[:, :100]}, True),
    "turned": (lambda o: {"x": o["x"].t().contiguous().t()}, False),
    "no rows": (lambda o: {"x": o["x"][:0]}, False),
    "another k": (lambda o: {"x": o["x"][:, :50]}, False),
    "unaligned rows": (lambda o: {"codes": o["codes"].contiguous()}, False),
    "padding outside the storage": (lambda o: {"codes": torch.zeros(40 * 112 - 12, dtype=torch.int8, device=DEV).as_strided((40, 100), (112, 1))}, False),
    "scales of another type": (lambda o: {"scales": o["scales"].double()}, False),
    "another type": (lambda o: {"x": o["x"].double()}, False),
    "a gradient": (lambda o: {"x": o["x"].clone().requires_grad_()}, False),
}


@pytest.mark.parametrize("name", LINEARS)
def test_linear(monkeypatch, name):
    change, serves = LINEARS[name]
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(-127, 128, (40, 112), generator=g, dtype=torch.int8).to(DEV)[:, :100]
    operands = {"x": torch.randn(6, 100, generator=g).to(BF16).to(DEV), "codes": codes,
                "scales": torch.rand(40, generator=g).to(DEV)}
    operands |= change(operands)
    a, b, served = _both(monkeypatch, lambda: linear_int8(**operands))
    assert _same(a, b), (a, b)
    assert bool(served) == serves
