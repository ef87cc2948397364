"""An engine takes an adapter bank of its own geometry only (no GPU needed: it is refused before anything is allocated)."""

from __future__ import annotations

import dataclasses
from types import SimpleNamespace

import pytest

from leanstack_b200.config import TINY
from leanstack_b200.engine import DecodeEngine
from leanstack_b200.requests import AdapterBank


def _engine(bank):
    runtime = SimpleNamespace(final_norm_weight=1, lm_head_weight=1, config=TINY, layers=[None] * TINY.num_hidden_layers)
    return DecodeEngine(runtime, 2, 32, adapters=bank)


@pytest.mark.parametrize("change,targets", [
    ({"intermediate_size": 1024}, AdapterBank.TARGETS), ({"intermediate_size": 1024}, ("gate_up",)),
    ({"intermediate_size": 1664}, ("down",)), ({"intermediate_size": 1664}, ("qkv", "gate_up")),
    ({"hidden_size": 1024}, ("qkv",)), ({"hidden_size": 1024}, ("o",)), ({"num_hidden_layers": 3}, ("o",)),
    ({"num_attention_heads": 6, "num_key_value_heads": 1}, ("qkv", "o")),  # q, k and v rows: 8 heads all the same
])
def test_another_geometry_is_refused(change, targets):
    bank = AdapterBank(dataclasses.replace(TINY, **change), 2, 8, "cpu", targets)
    with pytest.raises(ValueError, match="another geometry"):
        _engine(bank)


@pytest.mark.parametrize("change,targets", [({}, AdapterBank.TARGETS), ({"intermediate_size": 1024}, ("qkv", "o"))])
def test_linears_of_the_same_shapes_are_not(change, targets):
    with pytest.raises(Exception) as e:  # (the stand-in runtime has nothing to run)
        _engine(AdapterBank(dataclasses.replace(TINY, **change), 2, 8, "cpu", targets))
    assert "geometry" not in str(e.value)
