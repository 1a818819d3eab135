"""Forms of the operators for drafted tokens behind a shared prompt that their rules choose by size: joined and split attention, merges shared by a block,
short rows that share a block, rows of logits in few and in many parts."""
import ctypes as C

import numpy as np
import pytest
import torch

import ctorch_b200 as B
import prefix_oracle as O
import test_prefix_gpu as T

pytestmark = pytest.mark.gpu

SHORT = {  # as in ATTENTIONS: dtype, heads, kv_heads, dim, page, prefixes, group_first, group_prefix, counts, lengths
    "tiles of 16": ("bf16", 8, 2, 64, 16, [64], [0, 3], [0], [1, 3, 1], [0, 63, 64]),
    "tiles of 32": ("bf16", 8, 1, 128, 32, [65, 3], [0, 2, 5], [1, 0], [4, 1, 2, 3, 4], [0, 63, 64, 65, 127]),
    "tiles of 64": ("bf16", 4, 2, 96, 64, [130], [0, 3], [0], [40, 1, 33], [10, 0, 70]),
    "several tiles": ("bf16", 8, 1, 72, 8, [20], [0, 2], [0], [50, 17], [0, 5]),
    "heads of 40": ("bf16", 6, 2, 40, 24, [100], [0, 4], [0], [12, 1, 9, 30], [3, 60, 0, 24]),
    "no prefix": ("bf16", 8, 2, 128, 64, [1], [0], [], [1, 9, 0, 2], [5, 60, 3, 128]),
    "nothing before": ("bf16", 2, 2, 8, 8, [0, 5], [0, 1, 2], [0, 1], [1, 1], [0, 0]),
    "some outside": ("bf16", 8, 2, 64, 16, [80, 60], [1, 3, 4, 4, 5], [1, 9, 0, 0], [1, 2, 1, 3, 1, 2], [20, 3, 40, 0, 7, 100]),
}


def short_state(monkeypatch, name):
    monkeypatch.setitem(T.ATTENTIONS, name, SHORT[name])
    return T.attention_state(name, spare=2)


def near(got, want, bound):
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


@pytest.mark.parametrize("loose", [False, True])
@pytest.mark.parametrize("name", SHORT)
def test_short_prefixes(monkeypatch, name, loose):
    """Joined for bounds as short as the lengths are, split for loose ones; into f32 and both planes, on 16-byte boundaries and off them."""
    state, cache, prefix, query, of = short_state(monkeypatch, name)
    call = T.Attention(state, cache, prefix, query, of, **(dict(max_length=1 << 16, max_prefix=1 << 16) if loose else {}))
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    width = of["heads"] * of["dim"]
    for stride, shift in ((width, 0), (width + 8, 8), (width + 5, 3)):
        out = torch.full((shift + state.rows * stride,), 9.0, device="cuda")
        hi, lo = (torch.full((shift + state.rows * stride,), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        call(out[shift:], hi[shift:], lo[shift:], stride)

        def rows(x):
            x = T.host(x).astype(np.float64)
            x, before = x[shift:].reshape(state.rows, stride), x[:shift]
            assert (before == 9.0).all() and (x[:, width:] == 9.0).all() and (x[state.live:] == 9.0).all()
            return x[:state.live, :width].reshape(want.shape)
        bound = T.attention_bound(of, mass, size, keys)
        got = rows(out)
        near(got, want, bound)
        # two planes of 8 bits each behind the leading one: off by 2^-9 of 2^-8
        near(rows(hi) + rows(lo), got, 2.0 ** -17 * np.abs(got) + 1e-30)
        near(rows(hi), got, 2.0 ** -8 * np.abs(got) + 1e-30)


@pytest.mark.parametrize("name", T.ATTENTIONS)
def test_split_whatever_the_lengths(name):
    """Bounds far above the lengths: every case in the split form."""
    state, cache, prefix, query, of = T.attention_state(name, spare=1)
    out = torch.full((state.rows, of["heads"] * of["dim"]), 9.0, device="cuda")
    T.Attention(state, cache, prefix, query, of, max_length=1 << 16, max_prefix=1 << 16)(out)
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    near(T.host(out)[:state.live].reshape(want.shape), want, T.attention_bound(of, mass, size, keys))
    assert (T.host(out)[state.live:] == 9.0).all()


@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["tiles of 16", "tiles of 32", "tiles of 64", "heads of 40"])
def test_joined_rows_and_what_they_do_not_see(monkeypatch, name, odd):
    """No number in the last position of every sequence: rows that do not see it are as before, the last row is no number."""
    state, cache, prefix, query, of = short_state(monkeypatch, name)
    clean, spoilt = (torch.empty((state.rows, of["heads"] * of["dim"]), device="cuda") for _ in range(2))
    T.Attention(state, cache, prefix, query, of)(clean)
    last = np.zeros(state.live, dtype=bool)
    for s, slot in enumerate(state.slots):
        if state.counts[s] == 0:
            continue
        position = int(state.lengths[slot]) + state.counts[s] - 1
        page_size = cache.key.shape[2]
        cache.value[cache.table[slot, position // page_size], :, position % page_size] = odd
        last[state.first[s] + state.counts[s] - 1] = True
    T.Attention(state, cache, prefix, query, of)(spoilt)
    a, b = T.host(clean)[:state.live], T.host(spoilt)[:state.live]
    assert np.array_equal(a[~last], b[~last]) and not np.isfinite(b[last]).any()


MANY_SPLITS = {
    "f32": ("f32", 4, 2, 80, 64, [5001], [0, 3], [0], [1, 2, 1], [300, 5, 1]),
    "f32 odd heads": ("f32", 2, 1, 33, 7, [3000], [0, 1], [0], [3], [40]),
    "f32 tiles of 32": ("f32", 8, 1, 64, 16, [4000, 2500], [0, 2, 3], [0, 1], [5, 3, 1], [0, 700, 3]),
    "f32 heads of 256": ("f32", 2, 1, 256, 32, [2100], [0, 2], [0], [1, 1], [900, 2]),
    "bf16": ("bf16", 4, 1, 128, 64, [9000], [0, 2], [0], [1, 1], [0, 130]),
}


@pytest.mark.parametrize("name", MANY_SPLITS)
def test_many_splits_of_few_rows(monkeypatch, name):
    monkeypatch.setitem(T.ATTENTIONS, name, MANY_SPLITS[name])
    state, cache, prefix, query, of = T.attention_state(name, spare=2)
    one, two = (torch.full((state.rows, of["heads"] * of["dim"]), 9.0, device="cuda") for _ in range(2))
    call = T.Attention(state, cache, prefix, query, of)
    call(one)
    call(two)
    assert torch.equal(one, two) and (T.host(one)[state.live:] == 9.0).all()
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    near(T.host(one)[:state.live].reshape(want.shape), want, T.attention_bound(of, mass, size, keys))


@pytest.mark.parametrize("dim,rot,pairs,dtype", [(64, 64, 0, "bf16"), (8, 8, 1, "f32"), (6, 4, 0, "bf16"), (128, 64, 1, "bf16")])
def test_append_of_many_short_rows(dim, rot, pairs, dtype):
    """More rows than fill the SMs, several to a block; the last block is not full; one sequence's slot lies outside the cache."""
    rng = np.random.default_rng(dim)
    counts, page, heads, kv_heads = [700, 1, 600], 32, 2, 1
    span = 700 // page + 2
    table = rng.permutation(2 * span).reshape(2, span)
    state = T.Pass(counts, [1, 2, 0], [0, 5, 9], spare=3)   # slot 2 is none of the table's
    cache = T.Paged(dtype, kv_heads, page, dim, 2 * span, table)
    x = rng.standard_normal((state.rows, (heads + 2 * kv_heads) * dim), dtype=np.float32)
    angle = np.arange(800)[:, None] * O.frequencies(0, max(2, rot), 1e4)
    cosine, sine = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    d = [T.dev(x), T.dev(cosine), T.dev(sine), torch.full((state.rows, heads, dim), 9.0, device="cuda")]
    a = B.RotaryAppendArgs(heads=heads, rot_dims=rot, rotate_pairs=pairs, cosine=d[1].data_ptr(), sine=d[2].data_ptr(), positions=800, offset=None, projected=d[0].data_ptr(), stride=0,
                           query_dtype=B.F32, query=d[3].data_ptr(), cache=cache.args())
    B.kcheck(B.lib().b200_rotary_append(C.byref(a), C.byref(state.args), T.stream()))
    query, key, value = T.host(d[3]), T.host(cache.key), T.host(cache.value)
    assert (query[state.live:] == 9.0).all()
    written = np.zeros((2 * span, page), dtype=bool)
    step = T.BF16_STEP if dtype == "bf16" else 0.0
    for s, slot in enumerate([1, 2, 0]):
        for r in range(state.first[s], state.first[s + 1]):
            position = int(state.lengths[slot]) + r - state.first[s] if slot < 2 else 0
            head = x[r].reshape(-1, dim)
            turned = [O.rotate(h, cosine[position], sine[position], rot if slot < 2 else 0, pairs) for h in head]
            bound = 6 * T.F32_STEP * np.abs(head).max()   # |a c| + |b s| with two roundings each
            near(query[r], np.stack(turned[:heads]), bound)
            if slot < 2:
                at = table[slot, position // page], 0, position % page
                written[at[0], at[2]] = True
                near(key[at], turned[heads], bound + step * np.abs(turned[heads]))
                near(value[at], head[heads + kv_heads], step * np.abs(head[heads + kv_heads]))
    assert np.isnan(key[:, 0][~written]).all() and np.isnan(value[:, 0][~written]).all()


@pytest.mark.parametrize("vocab,shift", [(16376, 0), (16377, 1), (20001, 3), (33000, 2)])
def test_verify_of_many_rows(vocab, shift):
    """Rows enough for every SM: one CTA per row, and two, off 16-byte boundaries."""
    counts = [1 + i % 6 for i in range(50)]
    state, logits, draft, ids, accept, draw = T.verify_state(counts, vocab, 0.9, True, vocab)
    want_accepted, want_next, margin = O.verify(logits, draft, ids, [int(f) for f in state.first], 0.9, accept, draw)
    assert margin > 1e-5
    for temperature in (0.9, 0.0):
        accepted, chosen = T.Verify(state, logits, draft, ids, temperature, accept, draw, shift=shift)()
        if temperature == 0.0:
            want_accepted, want_next, _ = O.verify(logits, draft, ids, [int(f) for f in state.first], 0.0, accept, draw)
        assert np.array_equal(accepted, want_accepted) and np.array_equal(chosen, want_next)
