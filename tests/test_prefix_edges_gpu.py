"""Edges of the operators for drafted tokens behind a shared prompt: odd numbers of everything, slots that are none, sums of many small weights."""
import ctypes as C

import numpy as np
import pytest
import torch

import ctorch_b200 as B
import prefix_oracle as O
import test_prefix_gpu as T

pytestmark = pytest.mark.gpu

# as in ATTENTIONS: dtype, heads, kv_heads, dim, page, prefixes, group_first, group_prefix, counts, lengths
ODD = {   # rows, heads, splits and head sizes odd: what follows the partial accumulators in the scratch begins off 8-byte boundaries unless it is put there
    "one of everything": ("bf16", 1, 1, 33, 10, [1], [0], [], [1], [20]),
    "f32": ("f32", 1, 1, 5, 7, [1], [0], [], [1], [20]),
    "three heads, three rows": ("bf16", 3, 1, 33, 16, [1], [0], [], [1, 1, 1], [20, 0, 63]),
    "three splits": ("f32", 3, 3, 35, 16, [1], [0], [], [1, 2], [150, 140]),
    "a prefix of one split and own tokens of two": ("f32", 1, 1, 7, 16, [60], [0, 1], [0], [1], [100]),
    "a prefix of two splits": ("bf16", 3, 3, 9, 8, [100], [0, 3], [0], [1, 1, 1], [9, 30, 0]),
    "heads of 255": ("f32", 1, 1, 255, 16, [40], [0, 1], [0], [1], [100]),
}


@pytest.mark.parametrize("name", ODD)
def test_odd_numbers_of_everything(monkeypatch, name):
    monkeypatch.setitem(T.ATTENTIONS, name, ODD[name])
    state, cache, prefix, query, of = T.attention_state(name)
    out = torch.empty((state.rows, of["heads"] * of["dim"]), device="cuda")
    T.Attention(state, cache, prefix, query, of)(out)
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    assert (np.abs(T.host(out).reshape(want.shape) - want) <= T.attention_bound(of, mass, size, keys)).all()
