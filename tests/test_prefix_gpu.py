"""Operators for drafted tokens behind a shared prompt on the GPU, against the plain 64-bit forms of prefix_oracle.py.  torch only holds device memory.

Bounds, with n keys, heads of D values, scores s = scale q.k and S = scale sum |q||k| (all of them follow from half a step of rounding, 2^-24 in
f32 and 2^-8 in bf16, relative to the value):
  f32 attention    a score is off by at most (D + 2) 2^-24 S, its exponential by that, by the rounding of s log2(e) (3 S 2^-24) and by 2^-21 of the
                   exponential itself; the two sums add n 2^-24 each, and the splits' merge a few roundings more:
                   |out - exact| <= (2 (D + 8) 2^-24 S + 2^-20 + 2 n 2^-24) sum w|v|
  bf16 attention   the same on the bf16 inputs, and weights rounded to bf16: 2^-8 sum w|v|; a result rounded to bf16: 2^-8 |out|
  rotation         two products and a sum in f32: 3 * 2^-24 (|a c| + |b s|), and 2^-8 of the result where it is stored in bf16
  tables           f64 angles rounded once: 2^-24, and 2^-50 of the angle
Whole numbers (tokens, counts, lengths) are equal: the uniforms are put away from every border by 1e-5, which the f32 weights reach by far.
"""
import ctypes as C

import numpy as np
import pytest

import ctorch_b200 as B
import prefix_oracle as O
from ctorch_b200 import workloads as W

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32_STEP, BF16_STEP = 2.0 ** -24, 2.0 ** -8


def stream():
    return torch.cuda.current_stream().cuda_stream


def dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), device="cuda") if dtype is None else torch.as_tensor(np.ascontiguousarray(a), device="cuda").to(dtype)


def host(t):
    return t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()


TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {"f32": B.F32, "bf16": B.BF16}


class Pass:
    """A packed pass; `spare` rows stand behind the last sequence."""

    def __init__(self, counts, slots, lengths, spare=0):
        self.counts, self.slots, self.first = counts, slots, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.live, self.rows = int(self.first[-1]), int(self.first[-1]) + spare
        self.lengths = np.asarray(lengths, dtype=np.int32)
        sequence = np.repeat(np.arange(len(counts), dtype=np.int32), counts)
        self.d = [dev(np.asarray(slots, dtype=np.int32)), dev(self.first), dev(np.concatenate([sequence, np.full(spare, 1 << 30, dtype=np.int32)])), dev(self.lengths)]
        slot, first, of, length = (t.data_ptr() for t in self.d)
        self.args = B.Rows(rows=self.rows, sequences=len(counts), max_count=max(counts), slot=slot, first=first, sequence=of, lengths=length)


class Paged:
    """Pools with every page filled (NaN where nothing was written) behind a table of page numbers."""

    def __init__(self, dtype, kv_heads, page, dim, pages, table, rng=None):
        self.dtype, self.table = dtype, np.asarray(table, dtype=np.int32)
        shape = (pages, kv_heads, page, dim)
        self.key, self.value = (torch.full(shape, float("nan"), dtype=TORCH[dtype], device="cuda") if rng is None
                                else dev(rng.standard_normal(shape, dtype=np.float32), TORCH[dtype]) for _ in range(2))
        self.d_table = dev(self.table)

    def args(self):
        pages, kv_heads, page, dim = self.key.shape
        return B.KvPages(dtype=CODE[self.dtype], kv_heads=kv_heads, head_dim=dim, page_size=page, sequences=self.table.shape[0], pages_per_sequence=self.table.shape[1],
                         pages=pages, key=self.key.data_ptr(), value=self.value.data_ptr(), table=self.d_table.data_ptr())

    def oracle(self):
        return O.Pages(host(self.key), host(self.value), self.table)

    def spoil(self, lengths):
        """NaN at every position of every slot from its length on."""
        page = self.key.shape[2]
        for slot, n in enumerate(lengths):
            for i in range(int(n), self.table.shape[1] * page):
                number = self.table[slot, i // page]
                if 0 <= number < len(self.key):
                    self.key[number, :, i % page] = float("nan")
                    self.value[number, :, i % page] = float("nan")


# ---- tables ------------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", range(4))
@pytest.mark.parametrize("dims,first,positions", [(2, 0, 1), (64, 0, 300), (50, 131000, 77), (128, 5, 1), (8, 1 << 22, 33), (126, 0, 1031)])
def test_tables(kind, dims, first, positions):
    s = B.RotaryScaling(kind=kind, base=5e5, factor=8.0, original=8192.0, low=1.0, high=4.0, magnitude=1.2 if kind == 3 else 0.0)
    guard = 7   # values behind the tables stay as they are
    cosine, sine = (torch.full((positions * dims // 2 + guard,), 9.0, device="cuda") for _ in range(2))
    B.kcheck(B.lib().b200_rotary_tables(C.byref(s), dims, first, positions, cosine.data_ptr(), sine.data_ptr(), stream()))
    angle = np.arange(first, first + positions)[:, None] * O.frequencies(kind, dims, 5e5, 8.0, 8192.0, 1.0, 4.0)
    for got, want in ((cosine, np.cos(angle)), (sine, np.sin(angle))):
        got = host(got)
        assert (got[-guard:] == 9.0).all()
        # a frequency is off by a few steps of f64 (its exponent is up to 20), the angle by as much of itself
        bound = 1.2 * (F32_STEP + np.abs(angle) * 2.0 ** -46 + 2.0 ** -40)
        assert (np.abs(got[:-guard].reshape(positions, -1) - (1.2 if kind == 3 else 1.0) * want) <= bound).all()


# ---- rotation and append ---------------------------------------------------------------------------------------------------------------------------

APPENDS = [  # dtype, query dtype, heads, kv_heads, dim, rot, pairs, page, counts, spare rows, extra columns, offset
    ("bf16", "bf16", 8, 2, 64, 64, 0, 16, [1, 1, 1], 0, 0, True),
    ("bf16", "f32", 4, 4, 128, 64, 1, 64, [3, 0, 70, 1], 5, 0, True),
    ("f32", "f32", 6, 2, 80, 40, 0, 24, [9, 2], 2, 8, False),
    ("f32", "bf16", 3, 1, 34, 10, 0, 5, [4, 1, 6], 0, 3, True),
    ("bf16", "bf16", 2, 1, 6, 6, 1, 7, [1], 1, 0, False),
    ("bf16", "bf16", 4, 2, 72, 0, 0, 32, [5], 0, 0, False),
    ("f32", "f32", 1, 1, 256, 256, 1, 128, [130], 0, 0, False),
    ("bf16", "bf16", 40, 8, 128, 128, 0, 64, [33, 1, 12], 0, 4, True),
]


@pytest.mark.parametrize("dtype,qtype,heads,kv_heads,dim,rot,pairs,page,counts,spare,extra,offset", APPENDS)
def test_append(dtype, qtype, heads, kv_heads, dim, rot, pairs, page, counts, spare, extra, offset):
    rng = np.random.default_rng(heads * 100 + dim)
    n = len(counts)
    span = 3 + max(counts) // page
    table = rng.permutation(n * span + 2)[:n * span].reshape(n, span)
    table[0, span - 1] = -1        # no page there: nothing is written
    slots = rng.permutation(n)
    lengths = rng.integers(0, 2 * page, n)
    lengths[0] = span * page - 1   # the slot's last position; further rows of it find no room
    state = Pass(counts, slots, lengths, spare)
    cache = Paged(dtype, kv_heads, page, dim, n * span + 2, table)
    width = (heads + 2 * kv_heads) * dim + extra
    x = rng.standard_normal((state.rows, width), dtype=np.float32)
    positions = 40 + int(lengths[1:].max(initial=0)) + max(counts)   # slot 0 lies past the tables where its span is long: it does not turn
    angle = np.arange(positions)[:, None] * O.frequencies(0, max(2, rot), 1e4)
    cosine, sine = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    offsets = rng.integers(0, 30, n).astype(np.int32) if offset else np.zeros(n, dtype=np.int32)
    d = [dev(x), dev(cosine), dev(sine), dev(offsets), torch.full((state.rows, heads, dim), 9.0, dtype=TORCH[qtype], device="cuda")]
    a = B.RotaryAppendArgs(heads=heads, rot_dims=rot, rotate_pairs=pairs, cosine=d[1].data_ptr() if rot else None, sine=d[2].data_ptr() if rot else None,
                           positions=positions if rot else 0, offset=d[3].data_ptr() if offset else None, projected=d[0].data_ptr(), stride=width if extra else 0,
                           query_dtype=CODE[qtype], query=d[4].data_ptr(), cache=cache.args())
    B.kcheck(B.lib().b200_rotary_append(C.byref(a), C.byref(state.args), stream()))
    query, key, value = host(d[4]), host(cache.key), host(cache.value)
    assert (query[state.live:] == 9.0).all()
    written = np.zeros(key.shape[:1] + key.shape[2:3], dtype=bool)

    def near(got, want, size, kind):
        return (np.abs(got - want) <= 3 * F32_STEP * size + (BF16_STEP if kind == "bf16" else 0) * np.abs(want) + 1e-30).all()
    for s in range(n):
        for r in range(state.first[s], state.first[s + 1]):
            position = int(lengths[slots[s]]) + r - state.first[s]
            at = position + int(offsets[s])
            turn = rot if at < positions else 0
            c, sn = (cosine[at], sine[at]) if turn else ([], [])
            head = x[r, :(heads + 2 * kv_heads) * dim].reshape(-1, dim)
            # |a c| + |b s| is at most |a| + |b|
            size = [O.rotate(np.abs(h), np.ones(dim), -np.ones(dim), turn, pairs) for h in head]
            for h in range(heads):
                assert near(query[r, h], O.rotate(head[h], c, sn, turn, pairs), np.abs(size[h]) + np.abs(head[h]).max(), qtype)
            page_number = table[slots[s], position // page] if position < span * page else -1
            if page_number < 0:
                continue
            written[page_number, position % page] = True
            for k in range(kv_heads):
                assert near(key[page_number, k, position % page], O.rotate(head[heads + k], c, sn, turn, pairs), np.abs(size[heads + k]) + np.abs(head[heads + k]).max(), dtype)
                assert near(value[page_number, k, position % page], head[heads + kv_heads + k].astype(np.float64), np.zeros(dim), dtype)
    assert np.isnan(key.transpose(0, 2, 1, 3)[~written]).all() and np.isnan(value.transpose(0, 2, 1, 3)[~written]).all()


# ---- attention --------------------------------------------------------------------------------------------------------------------------------------

ATTENTIONS = {  # dtype, heads, kv_heads, dim, page, prefixes' lengths, first sequence of every group, prefix of every group, counts, earlier lengths
    "one token": ("bf16", 8, 2, 64, 16, [40], [0, 1], [0], [1], [0]),
    "no groups": ("bf16", 8, 2, 64, 64, [1], [0], [], [1, 1, 1], [100, 0, 63]),
    "empty prefix": ("bf16", 4, 4, 128, 64, [0, 70], [0, 2, 4], [0, 1], [1, 2, 1, 1], [5, 64, 63, 200]),
    "one step and a key": ("bf16", 16, 1, 64, 64, [64, 65, 63, 1], [0, 1, 2, 3, 4], [2, 0, 3, 1], [1, 1, 1, 1], [0, 1, 63, 64]),
    "drafts": ("bf16", 32, 8, 64, 32, [301, 150], [0, 3, 6], [0, 1], [5, 1, 3, 4, 2, 5], [70, 0, 130, 31, 32, 33]),
    "wide heads": ("bf16", 8, 2, 128, 64, [700], [0, 9], [0], [1] * 9, list(range(0, 90, 10))),
    "many rows": ("bf16", 8, 2, 128, 64, [390], [0, 3], [0], [50, 1, 70], [20, 500, 3]),
    "many rows of one sequence": ("bf16", 4, 1, 64, 128, [131], [0, 1], [0], [150], [77]),
    "heads of 80": ("bf16", 6, 2, 80, 24, [200], [0, 4], [0], [1, 7, 2, 20], [33, 5, 0, 60]),
    "heads of 96": ("bf16", 4, 4, 96, 16, [100, 90], [0, 1, 3], [1, 0], [3, 3, 30], [15, 16, 17]),
    "heads of 8": ("bf16", 3, 3, 8, 8, [50], [0, 2], [0], [2, 2], [9, 0]),
    "heads of 72 alone": ("bf16", 5, 1, 72, 40, [90], [0, 2], [0], [1, 1], [41, 2]),
    "heads of 256": ("bf16", 4, 2, 256, 16, [60], [0, 2], [0], [1, 3], [20, 5]),
    "odd heads": ("bf16", 4, 2, 33, 10, [47], [0, 2], [0], [1, 30], [12, 3]),
    "17 heads of one": ("bf16", 17, 1, 64, 64, [200], [0, 2], [0], [1, 1], [30, 80]),
    "f32": ("f32", 6, 2, 64, 16, [301], [0, 4], [0], [3, 1, 2, 3], [100, 0, 31, 17]),
    "f32 many rows": ("f32", 4, 1, 128, 64, [100, 40], [0, 1, 3], [0, 1], [40, 1, 5], [3, 64, 0]),
    "f32 odd heads": ("f32", 2, 1, 20, 7, [33], [0, 2], [0], [2, 9], [5, 40]),
    "f32 heads of 256": ("f32", 2, 2, 256, 32, [70], [0, 2], [0], [1, 2], [5, 40]),
    "sequences in no group": ("bf16", 8, 2, 64, 16, [80, 60], [1, 3, 4], [1, 0], [1, 2, 1, 3, 1, 2], [20, 3, 40, 0, 7, 100]),
    "sequences without rows": ("bf16", 8, 2, 64, 16, [80, 60], [0, 2, 5], [0, 1], [0, 2, 0, 0, 3], [20, 3, 40, 0, 7]),
    "a prefix named twice, one that is none": ("bf16", 8, 2, 64, 16, [80, 60], [0, 2, 3, 4], [1, 1, 7], [1, 2, 1, 3], [20, 3, 40, 0]),
    "two tiles and a bit": ("bf16", 16, 2, 128, 32, [1500, 700, 64], [0, 5, 7, 8], [1, 0, 2], [9, 9, 9, 9, 9, 30, 34, 1], [3, 0, 100, 33, 64, 5, 8, 90]),
    "pages of 8": ("bf16", 8, 1, 64, 8, [333, 120], [0, 6, 12], [0, 1], [1 + i % 4 for i in range(12)], [7 * i for i in range(12)]),
    "long prefix": ("bf16", 8, 1, 64, 64, [5000], [0, 20], [0], [2] * 20, [60 + i for i in range(20)]),
    "forty groups": ("bf16", 2, 1, 64, 16, [30 + i for i in range(40)], list(range(41)), list(range(40)), [1 + i % 3 for i in range(40)], [i for i in range(40)]),
}


def attention_state(name, spread=1.0, spare=0):
    dtype, heads, kv_heads, dim, page, prefixes, group_first, group_prefix, counts, lengths = ATTENTIONS[name]
    rng = np.random.default_rng(sum(map(ord, name)))
    n = len(counts)
    slots = rng.permutation(n + 1)[:n]
    of_slot = np.zeros(n + 1, dtype=np.int64)
    of_slot[slots] = lengths
    span = -(-max(c + i for c, i in zip(counts, lengths)) // page) + 1
    prefix_span = max(1, -(-max(prefixes) // page))
    pages = span * (n + 1) + prefix_span * len(prefixes) + 1
    order = rng.permutation(pages)
    table, prefix_table = order[:span * (n + 1)].reshape(n + 1, span), order[span * (n + 1):-1].reshape(len(prefixes), prefix_span)
    state = Pass(counts, slots, of_slot, spare)
    cache = Paged(dtype, kv_heads, page, dim, pages, table, rng)
    totals = of_slot.copy()
    totals[slots] += counts
    cache.spoil(totals)
    prefix = Paged(dtype, kv_heads, page, dim, 1, prefix_table)
    prefix.key, prefix.value = cache.key, cache.value   # tables over the same pools
    prefix.spoil(prefixes)
    query = dev(spread * rng.standard_normal((state.rows, heads, dim), dtype=np.float32), TORCH[dtype])
    return state, cache, prefix, query, dict(heads=heads, dim=dim, prefixes=prefixes, group_first=group_first, group_prefix=group_prefix, dtype=dtype,
                                             max_length=int(totals.max()), max_prefix=max(prefixes))


class Attention:
    def __init__(self, state, cache, prefix, query, of, max_length=None, max_prefix=None, scale=None):
        heads, dim = of["heads"], of["dim"]
        self.keep = [dev(np.asarray(of["group_first"], dtype=np.int32)), dev(np.asarray(of["group_prefix"] or [0], dtype=np.int32)), dev(np.asarray(of["prefixes"], dtype=np.int32)),
                     state, cache, prefix, query]
        self.a = B.PrefixArgs(heads=heads, scale=scale or dim ** -0.5, query=query.data_ptr(), cache=cache.args(), prefix=prefix.args(), groups=len(of["group_prefix"]),
                              group_first=self.keep[0].data_ptr(), group_prefix=self.keep[1].data_ptr(), prefix_length=self.keep[2].data_ptr())
        self.rows, self.max_length, self.max_prefix = state.args, max_length or of["max_length"], of["max_prefix"] if max_prefix is None else max_prefix
        self.need = B.lib().b200_prefix_scratch_bytes(C.byref(self.a), C.byref(self.rows), self.max_length, self.max_prefix)
        self.scratch = torch.full((self.need,), 0xff, dtype=torch.uint8, device="cuda")   # NaN: nothing that the call did not write counts

    def __call__(self, out=None, hi=None, lo=None, stride=0):
        B.kcheck(B.lib().b200_prefix_attention(C.byref(self.a), C.byref(self.rows), self.max_length, self.max_prefix, self.scratch.data_ptr(), self.need,
                                               *(None if t is None else t.data_ptr() for t in (out, hi, lo)), stride, stream()))


def wanted(state, cache, prefix, query, of, scale=None):
    return O.attention(host(query)[:state.live], of["heads"], scale or of["dim"] ** -0.5, cache.oracle(), [int(s) for s in state.slots], [int(f) for f in state.first],
                       [int(n) for n in state.lengths], prefix.oracle(), of["group_first"], of["group_prefix"], of["prefixes"])


def attention_bound(of, mass, size, keys):
    f32 = 2 * (of["dim"] + 8) * F32_STEP * size[..., None] + 2.0 ** -20 + 2 * keys[:, None, None] * F32_STEP
    return (f32 + (BF16_STEP if of["dtype"] == "bf16" else 0)) * mass + 1e-30


@pytest.mark.parametrize("spread", [1.0, 6.0])
@pytest.mark.parametrize("name", ATTENTIONS)
def test_attention(name, spread):
    state, cache, prefix, query, of = attention_state(name, spread, spare=3)
    width = of["heads"] * of["dim"]
    out, hi, lo = (torch.full((state.rows, width + 8), 9.0, dtype=t, device="cuda") for t in (torch.float32, torch.bfloat16, torch.bfloat16))
    Attention(state, cache, prefix, query, of)(out, hi, lo, width + 8)
    want, mass, size, keys = wanted(state, cache, prefix, query, of)
    bound = attention_bound(of, mass, size, keys)
    got = host(out)
    assert (got[state.live:] == 9.0).all() and (got[:, width:] == 9.0).all()
    got = got[:state.live, :width].reshape(want.shape)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
    assert (got[keys == 0] == 0).all()
    planes = host(hi)[:state.live, :width].reshape(want.shape)
    assert (np.abs(planes - got) <= BF16_STEP * np.abs(got) + 1e-38).all()
    # the planes hold 16 bits: what is left of the first one's rounding is rounded once more
    assert (np.abs(planes + host(lo)[:state.live, :width].reshape(want.shape) - got) <= BF16_STEP ** 2 * np.abs(got) + 1e-38).all()


@pytest.mark.parametrize("counts", [[1, 1], [3, 9], [40, 20]])
@pytest.mark.parametrize("own_page,prefix_page", [(16, 64), (128, 24), (7, 32), (32, 9)])
def test_prefix_and_cache_with_pages_of_their_own(own_page, prefix_page, counts):
    rng = np.random.default_rng(own_page)
    lengths, length = [30, 61], 150
    span, prefix_span = -(-110 // own_page), -(-length // prefix_page)
    cache = Paged("bf16", 2, own_page, 64, 2 * span, rng.permutation(2 * span).reshape(2, span), rng)
    prefix = Paged("bf16", 2, prefix_page, 64, prefix_span, rng.permutation(prefix_span).reshape(1, prefix_span), rng)
    state = Pass(counts, [1, 0], lengths)
    cache.spoil([lengths[0] + counts[1], lengths[1] + counts[0]])
    prefix.spoil([length])
    query = dev(rng.standard_normal((state.rows, 8, 64), dtype=np.float32), torch.bfloat16)
    of = dict(heads=8, dim=64, prefixes=[length], group_first=[0, 2], group_prefix=[0], dtype="bf16", max_length=110, max_prefix=length)
    out = torch.empty((state.rows, 512), device="cuda")
    Attention(state, cache, prefix, query, of)(out)
    want, mass, size, keys = wanted(state, cache, prefix, query, of)
    assert (np.abs(host(out).reshape(want.shape) - want) <= attention_bound(of, mass, size, keys)).all()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-6, 0.7])
@pytest.mark.parametrize("name", ["drafts", "many rows", "heads of 80", "f32"])
def test_scales(name, scale):
    state, cache, prefix, query, of = attention_state(name)
    out = torch.empty((state.rows, of["heads"] * of["dim"]), device="cuda")
    call = Attention(state, cache, prefix, query, of)
    call.a.scale = scale
    call(out)
    f, heads = of, of["heads"]
    want, mass, size, keys = O.attention(host(query)[:state.live], heads, float(np.float32(scale)), cache.oracle(), [int(s) for s in state.slots], [int(x) for x in state.first],
                                         [int(n) for n in state.lengths], prefix.oracle(), f["group_first"], f["group_prefix"], f["prefixes"])
    assert (np.abs(host(out).reshape(want.shape) - want) <= attention_bound(of, mass, size, keys)).all()


@pytest.mark.parametrize("name", ["drafts", "many rows", "f32", "long prefix"])
def test_attention_repeats_itself_whatever_the_bounds(name):
    """The same bits each time; looser bounds of the lengths split the work otherwise, which stays within twice the bound."""
    state, cache, prefix, query, of = attention_state(name)
    width = of["heads"] * of["dim"]
    one, two, three = (torch.empty((state.rows, width), device="cuda") for _ in range(3))
    call = Attention(state, cache, prefix, query, of)
    call(one)
    call(two)
    assert torch.equal(one, two)
    Attention(state, cache, prefix, query, of, max_length=1 << 20, max_prefix=1 << 20)(three)
    want, mass, size, keys = wanted(state, cache, prefix, query, of)
    assert (np.abs(host(three).reshape(want.shape) - want) <= attention_bound(of, mass, size, keys)).all()


@pytest.mark.parametrize("name", ["drafts", "many rows", "heads of 80", "f32", "odd heads", "heads of 256"])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_what_a_row_does_not_see_may_be_no_number(name, odd):
    """The last token of one sequence has keys and values that are no numbers: only that token's own row is touched."""
    state, cache, prefix, query, of = attention_state(name)
    s = int(np.argmax(state.counts))
    position = int(state.lengths[state.slots[s]]) + state.counts[s] - 1
    page = cache.key.shape[2]
    number = cache.table[state.slots[s], position // page]
    before = torch.empty((state.rows, of["heads"] * of["dim"]), device="cuda")
    after = torch.empty_like(before)
    call = Attention(state, cache, prefix, query, of)
    call(before)
    cache.key[number, :, position % page] = odd
    cache.value[number, :, position % page] = odd
    call(after)
    last = int(state.first[s + 1]) - 1
    rest = [r for r in range(state.live) if r != last]
    assert torch.equal(before[rest], after[rest])
    assert not torch.isfinite(after[last]).any()


@pytest.mark.parametrize("name", ["drafts", "wide heads", "many rows", "f32", "heads of 80"])
@pytest.mark.parametrize("where", range(0, 24, 3))
def test_one_key_that_is_no_number_spoils_all_that_see_it(name, where):
    """A NaN in a prefix's key, at any place of a step: the rows of that prefix's groups are NaN, the others as before."""
    state, cache, prefix, query, of = attention_state(name)
    before, after = (torch.empty((state.rows, of["heads"], of["dim"]), device="cuda") for _ in range(2))
    call = Attention(state, cache, prefix, query, of)
    call(before)
    page = prefix.key.shape[2]
    shared = of["group_prefix"][0]
    cache.key[prefix.table[shared, where // page], :, where % page, 1] = float("nan")
    call(after)
    spoilt = np.zeros(state.rows, dtype=bool)
    for g, number in enumerate(of["group_prefix"]):
        if number == shared:
            spoilt[state.first[of["group_first"][g]]:state.first[of["group_first"][g + 1]]] = True
    assert torch.isnan(after[spoilt]).all() and torch.equal(after[~spoilt], before[~spoilt])


def test_infinite_values_that_a_row_sees_reach_its_result():
    state, cache, prefix, query, of = attention_state("drafts")
    s, page = 0, cache.key.shape[2]
    position = int(state.lengths[state.slots[s]]) + state.counts[s] - 2   # the last two rows see it
    cache.value[cache.table[state.slots[s], position // page], :, position % page, 3] = float("inf")
    out = torch.empty((state.rows, of["heads"], of["dim"]), device="cuda")
    Attention(state, cache, prefix, query, of)(out)
    sees = np.zeros(state.rows, dtype=bool)
    sees[state.first[s + 1] - 2:state.first[s + 1]] = True
    got = host(out)
    assert (got[sees][:, :, 3] == np.inf).all() and np.isfinite(got[~sees]).all() and np.isfinite(np.delete(got, 3, axis=2)).all()


@pytest.mark.parametrize("name", ["drafts", "f32", "many rows", "long prefix"])
def test_a_page_outside_the_pools_is_zeros(name):
    state, cache, prefix, query, of = attention_state(name)
    for paged in (cache, prefix):
        for bad, slot in ((-1, 0), (1 << 30, len(paged.table) - 1)):
            paged.table[slot, 0] = bad
        paged.d_table = dev(paged.table)
    out = torch.empty((state.rows, of["heads"] * of["dim"]), device="cuda")
    Attention(state, cache, prefix, query, of)(out)
    want, mass, size, keys = wanted(state, cache, prefix, query, of)
    assert (np.abs(host(out).reshape(want.shape) - want) <= attention_bound(of, mass, size, keys)).all()


@pytest.mark.parametrize("value", [-float("inf"), float(np.finfo(np.float32).min)])
def test_scores_at_the_edge_of_the_type(value):
    """Keys whose scores are the lowest there are weigh nothing beside others (-inf) and share the weight evenly where there are no others (f32's lowest)."""
    heads = kv_heads = 1
    state = Pass([1], [0], [7])
    cache = Paged("f32", kv_heads, 8, 4, 2, [[0]], np.random.default_rng(5))
    query = torch.zeros((1, 1, 4), device="cuda")
    query[0, 0, 0] = 1.0
    cache.key[0, 0, :, :] = 0.0
    cache.key[0, 0, :4 if np.isinf(value) else 8, 0] = value
    of = dict(heads=heads, dim=4, prefixes=[0], group_first=[0], group_prefix=[], dtype="f32", max_length=8, max_prefix=0)
    out = torch.empty((1, 4), device="cuda")
    Attention(state, cache, cache, query, of, scale=0.5)(out)
    seen = host(cache.value)[0, 0, 4:] if np.isinf(value) else host(cache.value)[0, 0]
    assert np.abs(host(out)[0] - seen.astype(np.float64).mean(0)).max() <= 2.0 ** -20 * np.abs(seen).max()


def test_pools_of_more_than_2_to_31_values():
    """Pages far into large pools: element offsets pass 32 bits."""
    heads, kv_heads, dim, page = 4, 2, 64, 64
    pages = (1 << 31) // (kv_heads * page * dim) + 64
    rng = np.random.default_rng(3)
    table = np.array([[pages - 1, 5], [pages - 7, pages - 3]], dtype=np.int32)
    prefix_table = np.array([[pages - 20, 0, pages - 2]], dtype=np.int32)
    cache, prefix = (Paged("bf16", kv_heads, page, dim, 1, t) for t in (table, prefix_table))
    cache.key, cache.value = (torch.empty((pages, kv_heads, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    prefix.key, prefix.value = cache.key, cache.value
    used = sorted({int(p) for p in np.concatenate([table.ravel(), prefix_table.ravel()])})
    for pool in (cache.key, cache.value):
        pool[used] = dev(rng.standard_normal((len(used), kv_heads, page, dim), dtype=np.float32), torch.bfloat16)
    lengths, counts = [64, 20], [2, 1]
    state = Pass(counts, [0, 1], lengths)
    x = rng.standard_normal((3, (heads + 2 * kv_heads) * dim), dtype=np.float32)
    d = [dev(x), torch.ones(300, dim // 2, device="cuda"), torch.zeros(300, dim // 2, device="cuda"), torch.empty(3, heads, dim, dtype=torch.bfloat16, device="cuda")]
    a = B.RotaryAppendArgs(heads=heads, rot_dims=dim, rotate_pairs=0, cosine=d[1].data_ptr(), sine=d[2].data_ptr(), positions=300, offset=None, projected=d[0].data_ptr(),
                           stride=0, query_dtype=B.BF16, query=d[3].data_ptr(), cache=cache.args())
    B.kcheck(B.lib().b200_rotary_append(C.byref(a), C.byref(state.args), stream()))
    of = dict(heads=heads, dim=dim, prefixes=[170], group_first=[0, 2], group_prefix=[0], dtype="bf16", max_length=66, max_prefix=170)
    out = torch.empty((3, heads * dim), device="cuda")
    Attention(state, cache, prefix, d[3], of)(out)
    small = {p: i for i, p in enumerate(used)}
    key, value = host(cache.key[used]), host(cache.value[used])
    renumbered = [O.Pages(key, value, np.vectorize(small.get)(t)) for t in (table, prefix_table)]
    for r, (slot, position) in enumerate([(0, 64), (0, 65), (1, 20)]):
        for h in range(kv_heads):
            want = x[r].reshape(-1, dim)
            assert np.array_equal(renumbered[0].row(key, slot, position, h), host(dev(want[heads + h], torch.bfloat16)))
            assert np.array_equal(renumbered[0].row(value, slot, position, h), host(dev(want[heads + kv_heads + h], torch.bfloat16)))
    want, mass, size, keys = O.attention(host(d[3]), heads, dim ** -0.5, renumbered[0], [0, 1], [0, 2, 3], lengths, renumbered[1], [0, 2], [0], [170])
    assert (np.abs(host(out).reshape(want.shape) - want) <= attention_bound(of, mass, size, keys)).all()


# ---- verification --------------------------------------------------------------------------------------------------------------------------------------


class Verify:
    def __init__(self, state, logits, draft, ids, temperature, accept, draw, advance=0, stride=0, shift=0):
        """`shift`: floats before the first row, so that rows begin off 16-byte boundaries."""
        def rows_of(x):
            flat = torch.full((shift + x.size,), float("nan"), device="cuda")
            flat[shift:] = dev(x).reshape(-1)
            return flat
        self.state, n = state, len(state.counts)
        self.keep = [rows_of(logits), None if draft is None else rows_of(draft), dev(ids.astype(np.int64)), dev(np.asarray(accept)), dev(np.asarray(draw))]
        self.accepted, self.next = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7, dtype=torch.int64, device="cuda")
        p = [None if t is None else t.data_ptr() + (4 * shift if i < 2 else 0) for i, t in enumerate(self.keep)]
        self.a = B.VerifyArgs(vocab=logits.shape[1] if not stride else stride[0], stride=stride[1] if stride else 0, logits=p[0], draft_logits=p[1], ids=p[2],
                              temperature=temperature, accept=p[3], draw=p[4], accepted=self.accepted.data_ptr(), next=self.next.data_ptr(), advance=advance)
        self.need = B.lib().b200_verify_scratch_bytes(C.byref(self.a), C.byref(state.args))
        self.scratch = torch.full((self.need,), 0xff, dtype=torch.uint8, device="cuda")

    def __call__(self):
        B.kcheck(B.lib().b200_verify_drafts(C.byref(self.a), C.byref(self.state.args), self.scratch.data_ptr(), self.need, stream()))
        return host(self.accepted), host(self.next)


def verify_state(counts, vocab, temperature, model, seed, spare=0, spread=2.5):
    """Logits, drafts that the draft's distribution has, and uniforms: a draw lies in the middle of the interval of a token that is drawn by share, and
    an accept away from its border."""
    rng = np.random.default_rng(seed)
    state = Pass(counts, list(range(len(counts))), [10 * i for i in range(len(counts))], spare)
    logits = (spread * rng.standard_normal((state.rows, vocab))).astype(np.float32)
    draft = (logits + 0.7 * rng.standard_normal((state.rows, vocab))).astype(np.float32)
    t = temperature or 1.0
    ids = rng.integers(0, vocab, state.rows)
    accept = rng.random(state.rows)
    first = [int(f) for f in state.first]
    for s in range(len(counts)):
        for r in range(first[s], first[s + 1] - 1):
            p, q = O.weights(logits[r], t), O.weights(draft[r], t)
            if temperature == 0:
                ids[r + 1] = np.argmax(logits[r]) if rng.random() < 0.7 else rng.integers(0, vocab)
                continue
            ids[r + 1] = rng.choice(vocab, p=q if model else p)
            border = p[ids[r + 1]] / (q[ids[r + 1]] if model else 1.0)
            while abs(accept[r] - border) < 1e-3 * border:
                accept[r] = rng.random()
    draw = rng.random(len(counts))
    if temperature > 0:
        accepted, _, _ = O.verify(logits, draft if model else None, ids, first, temperature, accept, draw)
        for s in range(len(counts)):
            if counts[s] == 0:
                continue
            row = first[s] + accepted[s]
            left = O.weights(logits[row], t)
            if row < first[s + 1] - 1:
                minus = O.weights(draft[row], t) if model else np.eye(1, vocab, ids[row + 1])[0]
                rest = np.maximum(left - minus, 0)
                left = rest if rest.sum() > 0 else left
            left /= left.sum()
            token = rng.choice(np.flatnonzero(left > 1e-4), p=left[left > 1e-4] / left[left > 1e-4].sum())
            draw[s] = np.cumsum(left)[token] - left[token] / 2
    return state, logits, draft if model else None, ids, accept, draw


COUNTS = {"one row": [1], "no draft": [1, 1, 1], "drafts": [5, 1, 3, 8, 2], "many drafts": [40, 1, 67], "without rows": [0, 3, 0, 2], "batch": [1 + i % 6 for i in range(70)]}


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 1.9])
@pytest.mark.parametrize("vocab", [1, 3, 127, 1000, 4097, 32000, 50257])
@pytest.mark.parametrize("counts", ["drafts", "without rows"])
def test_verify(counts, vocab, temperature, model):
    state, logits, draft, ids, accept, draw = verify_state(COUNTS[counts], vocab, temperature, model, vocab + 7, spare=2)
    want_accepted, want_next, margin = O.verify(logits, draft, ids, [int(f) for f in state.first], temperature, accept, draw)
    assert margin > 1e-5   # the inputs are as they were meant
    accepted, chosen = Verify(state, logits, draft, ids, temperature, accept, draw)()
    assert np.array_equal(accepted, want_accepted) and np.array_equal(chosen, want_next)


@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("vocab,shift", [(2000, 0), (2001, 1), (131075, 3), (262144, 0)])
def test_verify_rows_of_every_kind(counts, vocab, shift):
    if vocab * sum(COUNTS[counts]) > 3e7:
        pytest.skip("more than the oracle does in a few seconds")
    state, logits, draft, ids, accept, draw = verify_state(COUNTS[counts], vocab, 0.9, True, vocab + 11)
    want_accepted, want_next, margin = O.verify(logits, draft, ids, [int(f) for f in state.first], 0.9, accept, draw)
    assert margin > 1e-5
    call = Verify(state, logits, draft, ids, 0.9, accept, draw, advance=1, shift=shift)
    accepted, chosen = call()
    assert np.array_equal(accepted, want_accepted) and np.array_equal(chosen, want_next)
    moved = [n + (a + 1 if c else 0) for n, a, c in zip(state.lengths, accepted, state.counts)]
    assert np.array_equal(host(state.d[3]), moved)
    again = call()
    assert np.array_equal(again[0], accepted) and np.array_equal(again[1], chosen)


def test_verify_rows_with_a_stride():
    state, logits, draft, ids, accept, draw = verify_state([4, 2], 1003, 0.9, True, 5)
    wide = [np.full((state.rows, 1010), np.inf, dtype=np.float32) for _ in range(2)]
    wide[0][:, :1003], wide[1][:, :1003] = logits, draft
    accepted, chosen = Verify(state, wide[0], wide[1], ids, 0.9, accept, draw, stride=(1003, 1010))()
    want = O.verify(logits, draft, ids, [0, 4, 6], 0.9, accept, draw)
    assert np.array_equal(accepted, want[0]) and np.array_equal(chosen, want[1])


@pytest.mark.parametrize("vocab", [5, 700, 40000])
def test_verify_edges(vocab):
    """Rows without finite weights, drafts outside the vocabulary, tokens that are masked off, borders of the uniforms."""
    rng = np.random.default_rng(vocab)
    counts = [2] * 9 + [1] * 4
    state = Pass(counts, list(range(len(counts))), [0] * len(counts))
    first = state.first
    logits, draft = (rng.standard_normal((state.rows, vocab)).astype(np.float32) for _ in range(2))
    ids, accept, draw = np.zeros(state.rows, dtype=np.int64), np.full(state.rows, 0.0), np.full(len(counts), 0.5)
    ids[first[:9] + 1] = 1
    nan, inf = np.float32("nan"), np.float32("inf")
    logits[first[0]] = -inf                                          # nothing allowed
    logits[first[1], vocab - 1] = nan
    logits[first[2], 2] = logits[first[2], 3] = inf
    draft[first[3]] = nan                                            # no draft distribution: refused, the target's own
    ids[first[4] + 1], ids[first[5] + 1] = -1, vocab
    logits[first[6], 1] = -inf                                       # the draft is masked off in the target
    draft[first[7]] = logits[first[7]]                               # the same distributions: always accepted
    accept[first[7]] = 0.999999
    draft[first[8], 1] = -inf                                        # a draft that the draft model cannot have drawn: p > u * 0
    accept[first[8]] = 0.999999
    logits[first[9], :-1] = -inf                                     # one token left
    draw[9] = 0.0
    logits[first[10], 0] = -inf                                      # the first token that has weight
    draw[10] = 0.0
    logits[first[11], -1] = -inf                                     # the last token that has weight
    draw[11] = 1.0 - 2.0 ** -53
    draw[12] = 1.0 - 2.0 ** -53
    accepted, chosen = Verify(state, logits, draft, ids, 1.0, accept, draw)()
    want_accepted, want_next, _ = O.verify(logits, draft, ids, [int(f) for f in first], 1.0, accept, draw)
    assert np.array_equal(accepted, want_accepted), (accepted, want_accepted)
    exact = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10]
    assert np.array_equal(chosen[exact], want_next[exact]), (chosen, want_next)
    assert chosen[0] == 0 and chosen[1] == vocab - 1 and chosen[2] == 2 and accepted[7] == accepted[8] == 1 and chosen[9] == vocab - 1 and chosen[10] == 1
    assert chosen[11] == vocab - 2 and chosen[12] == vocab - 1


def test_greedy_verification_takes_the_first_maximum():
    state = Pass([3, 2, 1], [0, 1, 2], [0, 0, 0])
    logits = np.zeros((6, 9000), dtype=np.float32)
    logits[0, [4500, 8000]] = 2.0
    logits[1, 10] = np.nan
    logits[1, 8999] = np.nan
    logits[2, 77] = 5
    logits[5] = -np.inf
    ids = np.array([3, 4500, 10, 1, 1, 1])
    accepted, chosen = Verify(state, logits, None, ids, 0.0, [0.0] * 6, [0.0] * 3)()
    assert accepted.tolist() == [2, 0, 0] and chosen.tolist() == [77, 0, 0]


# ---- together ------------------------------------------------------------------------------------------------------------------------------------------


class Layer:
    """One attention layer and a head over the framework's entry points: projections, rotation and append, attention, logits."""

    def __init__(self, dtype, width, heads, kv_heads, dim, vocab, rng):
        self.dtype, self.width, self.heads, self.kv_heads, self.dim, self.vocab = dtype, width, heads, kv_heads, dim, vocab
        self.h = {n: (rng.standard_normal(s) * s[-1] ** -0.5).astype(np.float32) for n, s in
                  dict(embed=(vocab, width), qkv=((heads + 2 * kv_heads) * dim, width), out=(width, heads * dim), logits=(vocab, width)).items()}
        if dtype == "bf16":
            self.h = {n: W.bf16_to_f32(W.bf16_bits(w)) for n, w in self.h.items()}
        self.h["logits"] *= 3.0   # exact in bf16 up to its own rounding, which the device's copy shares
        if dtype == "bf16":
            self.h["logits"] = W.bf16_to_f32(W.bf16_bits(self.h["logits"]))
        self.w = {n: dev(w, TORCH[dtype]) for n, w in self.h.items()}

    def linear(self, x, name):
        y = torch.empty((x.shape[0], self.w[name].shape[0]), device="cuda")
        B.kcheck(B.lib().b200_linear(x.data_ptr(), x.shape[0], x.shape[1], self.w[name].data_ptr(), CODE[self.dtype], y.shape[1], None, 0, 0.0, 0, None, None, y.data_ptr(), stream()))
        return y

    def embed(self, ids):
        x = torch.empty((len(ids), self.width), device="cuda")
        B.kcheck(B.lib().b200_embedding(self.w["embed"].data_ptr(), CODE[self.dtype], ids.data_ptr(), len(ids), self.vocab, self.width, x.data_ptr(), stream()))
        return x


def run_pass(layer, ids, state, cache, prefix, of, cosine, sine, offset):
    """Logits of every row of a pass."""
    x = layer.embed(ids)
    query = torch.empty((state.rows, layer.heads, layer.dim), dtype=TORCH[layer.dtype], device="cuda")
    projected = layer.linear(x, "qkv")
    a = B.RotaryAppendArgs(heads=layer.heads, rot_dims=layer.dim, rotate_pairs=0, cosine=cosine.data_ptr(), sine=sine.data_ptr(), positions=len(cosine),
                           offset=None if offset is None else offset.data_ptr(), projected=projected.data_ptr(), stride=0, query_dtype=CODE[layer.dtype], query=query.data_ptr(),
                           cache=cache.args())
    B.kcheck(B.lib().b200_rotary_append(C.byref(a), C.byref(state.args), stream()))
    out = torch.empty((state.rows, layer.heads * layer.dim), device="cuda")
    Attention(state, cache, prefix, query, of)(out)
    return layer.linear(layer.linear(out, "out"), "logits")


def oracle_logits(layer, tokens, cosine, sine):
    """Logits behind every token of one sequence, prefix and all, in 64 bits."""
    x = layer.h["embed"][tokens].astype(np.float64)
    y = (x @ layer.h["qkv"].T.astype(np.float64)).reshape(len(tokens), -1, layer.dim)
    turned = np.stack([[O.rotate(h, cosine[i], sine[i], layer.dim, 0) for h in y[i, :layer.heads + layer.kv_heads]] for i in range(len(tokens))])
    group, out = layer.heads // layer.kv_heads, np.zeros((len(tokens), layer.heads, layer.dim))
    for i in range(len(tokens)):
        for h in range(layer.heads):
            score = turned[:i + 1, layer.heads + h // group] @ turned[i, h] * layer.dim ** -0.5
            w = np.exp(score - score.max())
            out[i, h] = w / w.sum() @ y[:i + 1, layer.heads + layer.kv_heads + h // group]
    return out.reshape(len(tokens), -1) @ layer.h["out"].T.astype(np.float64) @ layer.h["logits"].T.astype(np.float64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_behind_a_shared_prompt(dtype):
    """Two prompts, five answers, drafted tokens: tables, then passes of append, attention and verification.  The accepted tokens of every answer are what
    greedy decoding of its whole text gives, and its logits are those of the whole text."""
    rng = np.random.default_rng(11)
    layer = Layer(dtype, 96, 6, 2, 32, 211, rng)
    cosine, sine = (torch.empty(400, 16, device="cuda") for _ in range(2))
    scaling = B.RotaryScaling(kind=B.ROTARY_PARTS, base=1e4, factor=4.0, original=64.0, low=1.0, high=8.0, magnitude=1.1)
    B.kcheck(B.lib().b200_rotary_tables(C.byref(scaling), 32, 0, 400, cosine.data_ptr(), sine.data_ptr(), stream()))
    prompts = [rng.integers(0, layer.vocab, n) for n in (83, 50)]
    group = [0, 0, 0, 1, 1]
    page, span = 16, 4
    order = rng.permutation(60)
    prefix_table, table = order[:12].reshape(2, 6), order[12:32].reshape(5, span)
    cache = Paged(dtype, 2, page, 32, 60, table)
    prefix = Paged(dtype, 2, page, 32, 1, prefix_table)
    prefix.key, prefix.value = cache.key, cache.value
    # the prompts themselves, through the prefix's table: a pass without groups
    prompt_pass = Pass([len(p) for p in prompts], [0, 1], [0, 0])
    alone = dict(heads=6, dim=32, prefixes=[0, 0], group_first=[0], group_prefix=[], dtype=dtype, max_length=83, max_prefix=0)
    logits = run_pass(layer, dev(np.concatenate(prompts)), prompt_pass, prefix, prefix, alone, cosine, sine, None)
    c, s = host(cosine), host(sine)
    texts = [list(prompts[g]) for g in group]
    tolerance = 1e-4 if dtype == "f32" else 4e-2

    def near(got, want):
        return np.abs(got - want).max() <= tolerance * np.abs(want).max()
    for i, p in enumerate(prompts):
        assert near(host(logits)[prompt_pass.first[i]:prompt_pass.first[i + 1]], oracle_logits(layer, p, c, s))
    for i, g in enumerate(group):   # every answer begins with a token of its own
        texts[i].append(int(rng.integers(0, layer.vocab)))
    lengths = dev(np.zeros(5, dtype=np.int32))
    offset = dev(np.array([len(prompts[g]) for g in group], dtype=np.int32))
    total = 0
    for step in range(4):
        counts = [int(rng.integers(1, 6)) for _ in texts]
        state = Pass(counts, list(range(5)), host(lengths))
        state.args.lengths = lengths.data_ptr()
        ids, drafts = [], []
        for text, n in zip(texts, counts):
            known = list(text)
            for _ in range(n - 1):   # mostly right drafts
                known.append(int(np.argmax(oracle_logits(layer, known, c, s)[-1])) if rng.random() < 0.8 else int(rng.integers(0, layer.vocab)))
            drafts.append(known)
            ids += known[len(text) - 1:]
        of = dict(heads=6, dim=32, prefixes=[83, 50], group_first=[0, 3, 5], group_prefix=[0, 1], dtype=dtype, max_length=page * span, max_prefix=83)
        d_ids = dev(np.array(ids))
        logits = run_pass(layer, d_ids, state, cache, prefix, of, cosine, sine, offset)
        n = len(counts)
        accepted, chosen = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int64, device="cuda")
        a = B.VerifyArgs(vocab=layer.vocab, stride=0, logits=logits.data_ptr(), draft_logits=None, ids=d_ids.data_ptr(), temperature=0.0, accept=None, draw=None,
                         accepted=accepted.data_ptr(), next=chosen.data_ptr(), advance=1)
        need = B.lib().b200_verify_scratch_bytes(C.byref(a), C.byref(state.args))
        scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        B.kcheck(B.lib().b200_verify_drafts(C.byref(a), C.byref(state.args), scratch.data_ptr(), need, stream()))
        got, token = host(accepted), host(chosen)
        for i, known in enumerate(drafts):
            want = oracle_logits(layer, known, c, s)[-counts[i]:]
            have = host(logits)[state.first[i]:state.first[i + 1]]
            assert near(have, want)
            greedy = [int(np.argmax(r)) for r in have]
            taken = 0
            while taken < counts[i] - 1 and known[len(texts[i]) + taken] == greedy[taken]:
                taken += 1
            assert got[i] == taken and token[i] == greedy[taken]
            if dtype == "f32":
                assert greedy == [int(np.argmax(r)) for r in want]
            texts[i] = known[:len(texts[i]) + taken] + [int(token[i])]
            total += taken
        assert host(lengths).tolist() == [len(t) - 1 - len(prompts[g]) for t, g in zip(texts, group)]
    assert total > 5


def test_captured_and_on_another_stream():
    """Append, attention and verification in one graph on a side stream, replayed with other inputs and lengths; a second graph shares the workspaces."""
    layer_heads, kv_heads, dim, vocab, page = 8, 2, 64, 5000, 64
    rng = np.random.default_rng(2)
    counts = [3, 1, 4]
    state = Pass(counts, [2, 0, 1], [70, 10, 30])
    rows = state.rows
    cache = Paged("bf16", kv_heads, page, dim, 20, np.arange(12).reshape(3, 4), rng)
    prefix = Paged("bf16", kv_heads, page, dim, 1, [[12, 13, 14, 15]])
    prefix.key, prefix.value = cache.key, cache.value
    of = dict(heads=layer_heads, dim=dim, prefixes=[200], group_first=[0, 3], group_prefix=[0], dtype="bf16", max_length=256, max_prefix=256)
    projected = dev(rng.standard_normal((rows, (layer_heads + 2 * kv_heads) * dim), dtype=np.float32))
    angle = torch.arange(600, device="cuda")[:, None] * torch.rand(32, device="cuda")
    cosine, sine = angle.cos(), angle.sin()
    query, out = torch.empty((rows, layer_heads, dim), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, layer_heads * dim), device="cuda")
    append = B.RotaryAppendArgs(heads=layer_heads, rot_dims=dim, rotate_pairs=1, cosine=cosine.data_ptr(), sine=sine.data_ptr(), positions=600, offset=None,
                                projected=projected.data_ptr(), stride=0, query_dtype=B.BF16, query=query.data_ptr(), cache=cache.args())
    attend = Attention(state, cache, prefix, query, of)
    _, logits, draft, ids, accept, draw = verify_state(counts, vocab, 1.0, True, 9)
    check = Verify(state, logits, draft, ids, 1.0, accept, draw)

    def work():
        B.kcheck(B.lib().b200_rotary_append(C.byref(append), C.byref(state.args), stream()))
        attend(out)
        B.kcheck(B.lib().b200_verify_drafts(C.byref(check.a), C.byref(state.args), check.scratch.data_ptr(), check.need, stream()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    results = (out, query, cache.key, cache.value, check.accepted, check.next)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            work()
    clean = [cache.key.clone(), cache.value.clone()]
    for number in range(4):
        projected.copy_(torch.randn_like(projected))
        state.d[3].copy_(dev(rng.integers(0, 200, 3).astype(np.int32)))
        check.keep[0].mul_(0.9)
        got = []
        for how in (graphs[number % 2].replay, work):
            cache.key.copy_(clean[0])
            cache.value.copy_(clean[1])
            for t in (out, query, check.accepted, check.next):
                t.zero_()
            check.scratch.fill_(0xff)
            attend.scratch.fill_(0xff)
            how()
            torch.cuda.synchronize()
            got.append([t.clone() for t in results])
        for a, b in zip(*got):
            assert torch.equal(a, b)


def test_pages_of_a_cache():
    """The view of a b200_kv_cache: what its own append wrote is what the attention over the view sees."""
    handle, rng = C.c_void_p(), np.random.default_rng(1)
    l = B.lib()
    B.kcheck(l.b200_kv_cache_create(0, B.BF16, 2, 2, 64, 100, 16, C.byref(handle)))
    try:
        key, value = (rng.standard_normal((2, 2, 40, 64), dtype=np.float32) for _ in range(2))
        d = [dev(key), dev(value)]
        B.kcheck(l.b200_kv_cache_append(handle, d[0].data_ptr(), d[1].data_ptr(), 40, stream()))
        view = B.KvPages()
        B.kcheck(l.b200_kv_cache_pages(handle, C.byref(view)))
        assert (view.dtype, view.kv_heads, view.head_dim, view.page_size, view.sequences, view.pages_per_sequence, view.pages) == (B.BF16, 2, 64, 16, 2, 7, 14)
        state = Pass([1, 1], [0, 1], [39, 39])
        query = dev(rng.standard_normal((2, 4, 64), dtype=np.float32), torch.bfloat16)
        a = B.PrefixArgs(heads=4, scale=0.125, query=query.data_ptr(), cache=view, prefix=view, groups=0, group_first=None, group_prefix=None, prefix_length=None)
        need = l.b200_prefix_scratch_bytes(C.byref(a), C.byref(state.args), 40, 0)
        scratch, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty((2, 256), device="cuda")
        B.kcheck(l.b200_prefix_attention(C.byref(a), C.byref(state.args), 40, 0, scratch.data_ptr(), need, out.data_ptr(), None, None, 0, stream()))
        stored = [host(dev(x, torch.bfloat16)).transpose(0, 2, 1, 3) for x in (key, value)]   # [slot, position, head, dim]: pages of one position
        whole = O.Pages(*(x.reshape(80, 2, 1, 64) for x in stored), np.arange(80).reshape(2, 40))
        want, mass, size, keys = O.attention(host(query), 4, 0.125, whole, [0, 1], [0, 1, 2], [39, 39])
        assert (np.abs(host(out).reshape(want.shape) - want) <= attention_bound(dict(dim=64, dtype="bf16"), mass, size, keys)).all()
    finally:
        torch.cuda.synchronize()
        l.b200_kv_cache_release(handle)
