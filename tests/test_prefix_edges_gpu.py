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


# ---- weights: what they are rounded to, and that it does not hang on the batch -----------------------------------------------------------------------


def weight_bound(of, mass, size, keys):
    """Of f32 and two-plane results: the weights' two bf16 planes hold all but 2^-15 of a weight (the first is cut off, 2^-7, the second rounded, 2^-8 of that) and
    are 2^-23 too large; the rest is what attention_bound says of f32."""
    f32 = T.attention_bound({**of, "dtype": "f32"}, mass, size, keys)
    return f32 + (2.0 ** -15 + 2.0 ** -23) * mass if of["dtype"] == "bf16" else f32


def bf16_bound(of, want, mass, size, keys):
    """Of bf16 results: weights w (1 + e) with |e| <= 2^-8 in the products and in their sum, so that out is off by sum w e v / sum w (1 + e) and by out times
    sum w e / sum w (1 + e); then rounded."""
    weights = 2.0 ** -8 / (1 - 2.0 ** -8) * (mass + np.abs(want)) if of["dtype"] == "bf16" else 0.0
    off = T.attention_bound({**of, "dtype": "f32"}, mass, size, keys) + weights
    return off + 2.0 ** -8 * (np.abs(want) + off)


@pytest.mark.parametrize("loose", [False, True])
@pytest.mark.parametrize("spread", [1.0, 6.0])
@pytest.mark.parametrize("name", T.ATTENTIONS)
def test_results_are_as_good_as_their_form(name, spread, loose):
    """f32 results; two planes alone; one plane alone."""
    state, cache, prefix, query, of = T.attention_state(name, spread, spare=2)
    call = T.Attention(state, cache, prefix, query, of, **(dict(max_length=1 << 16, max_prefix=1 << 16) if loose else {}))
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    width = of["heads"] * of["dim"]
    out, (hi, lo, one) = torch.full((state.rows, width), 9.0, device="cuda"), torch.full((3, state.rows, width), 9.0, dtype=torch.bfloat16, device="cuda")
    call(out)
    call(None, hi, lo)
    call(None, one)
    out, hi, lo, one = (T.host(x).astype(np.float64) for x in (out, hi, lo, one))
    assert (out[state.live:] == 9.0).all() and (one[state.live:] == 9.0).all()
    bound = weight_bound(of, mass, size, keys)
    assert (np.abs(out[:state.live].reshape(want.shape) - want) <= bound).all()
    # the second plane of a result is rounded to 2^-8 of at most 2^-8
    assert (np.abs((hi + lo)[:state.live].reshape(want.shape) - want) <= bound + 2.0 ** -16 * (np.abs(want) + bound)).all()
    assert (np.abs(one[:state.live].reshape(want.shape) - want) <= bf16_bound(of, want, mass, size, keys)).all()


BATCHES = [  # dtype, heads, kv_heads, dim, page, prefix, sequences, rows and earlier tokens of each
    ("bf16", 32, 8, 128, 64, 2000, 40, 1, 512),
    ("bf16", 8, 2, 64, 32, 3001, 30, 5, 700),
    ("bf16", 8, 1, 96, 16, 900, 50, 3, 90),
    ("bf16", 4, 4, 72, 24, 1200, 64, 2, 300),
    ("bf16", 4, 2, 64, 64, 0, 50, 4, 2000),
    ("bf16", 4, 2, 160, 64, 300, 30, 4, 200),
    ("f32", 8, 2, 64, 16, 700, 40, 2, 200),
]


@pytest.mark.parametrize("spread", [1.0, 2.0, 6.0])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,length,sequences,count,earlier", BATCHES)
def test_a_sequence_by_itself_and_among_others(dtype, heads, kv_heads, dim, page, length, sequences, count, earlier, spread):
    """Other splits, tiles and kernels for the same sequence: what f32 results differ by is what f32 allows, and bf16 results are the same but where two such
    f32 values lie on either side of a border.  These differ by some 2^-21 of mass (a few roundings of 2^-24, and of weights near a border 2^-8 once in
    2^12 times) and borders are 2^-8 |out| apart: one result in 2^13 |out| / mass; |out| is a 30th of mass at the least here.  Below 1 % then; it
    was a third with weights rounded relative to the maximum."""
    rng = np.random.default_rng(dim + count)
    prefix_span, span = max(1, -(-length // page)), -(-(earlier + count) // page)
    pages = prefix_span + span * sequences
    order = rng.permutation(pages)
    cache, prefix = T.Paged(dtype, kv_heads, page, dim, 1, order[:span * sequences].reshape(sequences, span)), T.Paged(dtype, kv_heads, page, dim, 1, order[span * sequences:].reshape(1, -1))
    g = torch.Generator(device="cuda").manual_seed(dim)
    cache.key, cache.value = prefix.key, prefix.value = torch.randn((2, pages, kv_heads, page, dim), generator=g, device="cuda").to(T.TORCH[dtype])
    query = (spread * torch.randn((sequences * count, heads, dim), generator=g, device="cuda")).to(T.TORCH[dtype])
    results = []
    for n in (sequences, 1):
        state = T.Pass([count] * n, list(range(n)), [earlier] * sequences)
        of = dict(heads=heads, dim=dim, prefixes=[length], group_first=[0, n], group_prefix=[0], dtype=dtype, max_length=earlier + count, max_prefix=length)
        call = T.Attention(state, cache, prefix, query, of)
        out, one = torch.empty((n * count, heads, dim), device="cuda"), torch.empty((n * count, heads, dim), dtype=torch.bfloat16, device="cuda")
        call(out)
        call(None, one)
        results.append((T.host(out[:count]).astype(np.float64), T.host(one[:count])))
    # mass and size of the sequence's rows
    def keys_of(pool):
        both = [pool[torch.as_tensor(table.astype(np.int64), device="cuda")].double().transpose(0, 1).reshape(kv_heads, -1, dim) for table in (prefix.table[0], cache.table[0])]
        return torch.cat([both[0][:, :length], both[1][:, :earlier + count]], 1)
    key, value = keys_of(cache.key), keys_of(cache.value)
    q = query[:count].double().view(count, kv_heads, heads // kv_heads, dim)
    score = torch.einsum("nkgd,kjd->nkgj", q, key) * dim ** -0.5
    hidden = torch.arange(key.shape[1], device="cuda")[None] > length + earlier + torch.arange(count, device="cuda")[:, None]
    weight = torch.softmax(score.masked_fill(hidden[:, None, None], -float("inf")), -1)
    mass = torch.einsum("nkgj,kjd->nkgd", weight, value.abs()).reshape(count, heads, dim).cpu().numpy()
    size = torch.einsum("nkgd,kjd->nkgj", q.abs(), key.abs()).amax(-1).reshape(count, heads).cpu().numpy() * dim ** -0.5
    bound = weight_bound(dict(dim=dim, dtype=dtype), mass, size, np.full(count, key.shape[1]))
    (many, many_bf16), (alone, alone_bf16) = results
    assert (np.abs(many - alone) <= 2 * bound).all()
    assert np.mean(many_bf16 != alone_bf16) < 0.01


@pytest.mark.parametrize("name", ["drafts", "many rows", "wide heads", "heads of 80", "f32", "heads of 256"])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_infinite_values_of_a_prefix_reach_the_results(name, value):
    """A value that everyone sees and that is infinite: so is its column of the results of the prefix's groups, whatever their form."""
    state, cache, prefix, query, of = T.attention_state(name)
    page, shared, where = prefix.key.shape[2], of["group_prefix"][0], 21
    cache.value[prefix.table[shared, where // page], :, where % page, 3] = value
    sees = np.zeros(state.rows, dtype=bool)
    for g, number in enumerate(of["group_prefix"]):
        if number == shared:
            sees[state.first[of["group_first"][g]]:state.first[of["group_first"][g + 1]]] = True
    call = T.Attention(state, cache, prefix, query, of)
    out, one = torch.empty((state.rows, of["heads"], of["dim"]), device="cuda"), torch.empty((state.rows, of["heads"], of["dim"]), dtype=torch.bfloat16, device="cuda")
    call(out)
    call(None, one)
    for got in (T.host(out), T.host(one)):
        assert (got[sees][:, :, 3] == value).all() and np.isfinite(got[~sees]).all() and np.isfinite(np.delete(got, 3, axis=2)).all()


# ---- verification ------------------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_sequences_without_a_slot_do_not_move_on(temperature):
    """Slot -1 is none, as for append and attention: the values around the lengths stay as they are."""
    counts = [3, 1, 0, 4, 2]
    state, logits, draft, ids, accept, draw = T.verify_state(counts, 600, temperature, True, 17)
    call = T.Verify(state, logits, draft, ids, temperature, accept, draw, advance=1)
    memory = torch.arange(100, 130, dtype=torch.int32, device="cuda")
    slots = T.dev(np.array([-1, 2, -1, 0, -5], dtype=np.int32))
    state.args.slot, state.args.lengths = slots.data_ptr(), memory[12:].data_ptr()
    accepted, chosen = call()
    want = O.verify(logits, draft, ids, [int(f) for f in state.first], temperature, accept, draw)
    assert np.array_equal(accepted, want[0]) and np.array_equal(chosen, want[1])
    moved = np.arange(100, 130)
    moved[12 + 2] += accepted[1] + 1
    moved[12 + 0] += accepted[3] + 1
    assert np.array_equal(T.host(memory), moved)


@pytest.mark.parametrize("tokens", [False, True])
def test_rows_of_no_slot_do_not_move_on(tokens):
    """b200_rows_advance and its form that keeps the last tokens: slot -1 is none, a sequence without rows has no last token."""
    state = T.Pass([0, 3, 1, 0, 4], [0, 1, 2, 3, 4], [0] * 5)
    lengths, last = torch.arange(100, 130, dtype=torch.int32, device="cuda"), torch.arange(200, 230, dtype=torch.int32, device="cuda")
    slots = T.dev(np.array([4, -1, 2, -1, 0], dtype=np.int32))
    state.args.slot, state.args.lengths = slots.data_ptr(), lengths[12:].data_ptr()
    ids = torch.arange(7, 7 + state.rows, device="cuda")
    if tokens:
        B.kcheck(B.lib().b200_rows_advance_tokens(C.byref(state.args), ids.data_ptr(), last[12:].data_ptr(), T.stream()))
    else:
        B.kcheck(B.lib().b200_rows_advance(C.byref(state.args), T.stream()))
    want, want_last = np.arange(100, 130), np.arange(200, 230)
    want[12 + 2] += 1
    want[12 + 0] += 4
    if tokens:
        want_last[12 + 2], want_last[12 + 0] = 7 + 3, 7 + 7
    assert np.array_equal(T.host(lengths), want) and np.array_equal(T.host(last), want_last)


@pytest.mark.parametrize("level", [-12.48, -6.3, -17.9])   # weights of about 2^-18, 2^-9, 2^-26
@pytest.mark.parametrize("vocab", [1001, 5003, 50257, 100001, 300001])
def test_sums_of_many_small_weights(vocab, level):
    """Rows of one token of weight 1 and vocab - 1 of one weight w, at every alignment.  Bisection over `accept` finds the shares 1 / S and w / S that the
    kernel holds to the last bit; their quotient is w, a value of f32, and S = 1 + (vocab - 1) w.  What the sum may be off by: a thread adds at most 64 values in
    three f32 parts, of which two are exact and the third stays below 64 2^-37, so that each addition to it is off by 2^-56 at most; what is added in 64 bits is off
    by 2^-53 of S for each of the less than 64 additions on a value's way."""
    counts = [2, 2, 1, 2, 2]
    state = T.Pass(counts, list(range(5)), [0] * 5)
    logits = np.full((state.rows, vocab), level, dtype=np.float32)
    judged = [int(state.first[s]) for s in range(5) if counts[s] == 2]
    assert {r * vocab % 4 for r in judged} == {0, 1, 2, 3}
    logits[:, 0] = 0.0
    ids = np.zeros(state.rows, dtype=np.int64)

    def shares(token):
        ids[:] = token
        call = T.Verify(state, logits, None, ids, 1.0, np.zeros(state.rows), np.zeros(5))
        low, high = np.zeros(4, dtype=np.int64), np.full(4, np.float64(1.0).view(np.int64))   # bits of uniforms that are accepted, and that are not
        while (high - low > 1).any():
            middle = (low + high) // 2
            u = np.zeros(state.rows)
            u[judged] = middle.view(np.float64)
            call.keep[3].copy_(torch.as_tensor(u))
            accepted = call()[0][[0, 1, 3, 4]] == 1
            low, high = np.where(accepted, middle, low), np.where(accepted, high, middle)
        return high.view(np.float64)   # u < share holds up to the value before
    one, small = shares(0), shares(1)
    weight = (small / one).astype(np.float32)
    assert (np.abs(small / one / weight - 1) < 2.0 ** -50).all() and (weight == weight[0]).all() and abs(np.log(weight[0]) / level - 1) < 1e-6
    exact = 1 + (vocab - 1) * float(weight[0])
    assert (np.abs(one * exact - 1) <= vocab * 2.0 ** -56 / exact + 64 * 2.0 ** -53).all(), np.abs(one * exact - 1).max()


# ---- passes that run part after part -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,counts,lengths,prefixes,group_first,group_prefix", [
    ("bf16", 128, 8, 64, 32, [1500, 1, 900, 3, 0, 2500, 40, 100], [10, 0, 70, 5, 3, 33, 64, 2], [300, 77], [0, 4, 8], [1, 0]),
    ("bf16", 256, 4, 128, 16, [700, 700, 800], [0, 100, 3], [130], [1, 3], [0]),
    ("bf16", 128, 128, 36, 10, [2100, 200], [20, 0], [50], [0, 2], [0]),
    ("f32", 192, 16, 20, 16, [1, 1400, 1, 1700], [20, 0, 50, 31], [90, 10, 33], [0, 1, 2, 4], [2, 0, 1]),
    ("bf16", 256, 2, 64, 64, [1] * 2600, [i % 90 for i in range(2600)], [500], [0, 2600], [0]),
])
def test_passes_of_more_rows_than_partial_results_find_room(dtype, heads, kv_heads, dim, page, counts, lengths, prefixes, group_first, group_prefix):
    """2^18 pairs of a row and a head run at once; these passes have more, with sequences and groups across the borders of the parts."""
    rng = np.random.default_rng(heads + dim)
    n, rows = len(counts), sum(counts)
    assert rows * heads > 1 << 18
    span, prefix_span = -(-max(c + i for c, i in zip(counts, lengths)) // page), -(-max(prefixes) // page)
    pages = n * span + len(prefixes) * prefix_span
    order = rng.permutation(pages)
    slots = rng.permutation(n)
    of_slot = np.empty(n, dtype=np.int64)
    of_slot[slots] = lengths
    cache = T.Paged(dtype, kv_heads, page, dim, 1, order[:n * span].reshape(n, span))
    prefix = T.Paged(dtype, kv_heads, page, dim, 1, order[n * span:].reshape(len(prefixes), prefix_span))
    g = torch.Generator(device="cuda").manual_seed(dim)
    cache.key, cache.value = prefix.key, prefix.value = torch.randn((2, pages, kv_heads, page, dim), generator=g, device="cuda").to(T.TORCH[dtype])
    state = T.Pass(counts, slots, of_slot, spare=5)
    query = torch.randn((state.rows, heads, dim), generator=g, device="cuda").to(T.TORCH[dtype])
    of = dict(heads=heads, dim=dim, prefixes=prefixes, group_first=group_first, group_prefix=group_prefix, dtype=dtype, max_length=1 << 14, max_prefix=1 << 16)
    call = T.Attention(state, cache, prefix, query, of)
    call.scratch = torch.full((call.need + 4096,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full((state.rows, heads, dim), 9.0, device="cuda")
    call(out)
    assert (call.scratch[call.need:] == 0xff).all() and (out[state.live:] == 9.0).all()
    group = heads // kv_heads
    for s in range(n):
        if s >= 60 and s % 97:   # of very many sequences some
            continue
        begin, count = int(state.first[s]), counts[s]
        if not count:
            continue
        owner = [i for i in range(len(group_prefix)) if group_first[i] <= s < group_first[i + 1]]
        shared = prefixes[group_prefix[owner[0]]] if owner else 0

        def keys_of(pool):
            a = pool[torch.as_tensor(prefix.table[group_prefix[owner[0]]] if owner else prefix.table[0], device="cuda").long()].double().transpose(0, 1).reshape(kv_heads, -1, dim)
            b = pool[torch.as_tensor(cache.table[slots[s]], device="cuda").long()].double().transpose(0, 1).reshape(kv_heads, -1, dim)
            return torch.cat([a[:, :shared], b[:, :lengths[s] + count]], 1)
        key, value = keys_of(cache.key), keys_of(cache.value)
        for at in range(0, count, 256):
            part = query[begin + at:begin + min(count, at + 256)].double().view(-1, kv_heads, group, dim)
            m = len(part)
            score = torch.einsum("nkgd,kjd->nkgj", part, key) * dim ** -0.5
            hidden = torch.arange(key.shape[1], device="cuda")[None] > shared + lengths[s] + at + torch.arange(m, device="cuda")[:, None]
            weight = torch.softmax(score.masked_fill(hidden[:, None, None], -float("inf")), -1)
            want, mass = (torch.einsum("nkgj,kjd->nkgd", weight, v).reshape(m, heads, dim).cpu().numpy() for v in (value, value.abs()))
            size = torch.einsum("nkgd,kjd->nkgj", part.abs(), key.abs()).amax(-1).reshape(m, heads).cpu().numpy() * dim ** -0.5
            got = T.host(out[begin + at:begin + at + m])
            assert (np.abs(got - want) <= weight_bound(of, mass, size, np.full(m, key.shape[1]))).all(), (s, at)


# ---- two calls at once -------------------------------------------------------------------------------------------------------------------------------


def at_once(calls, times=400):
    """Every call again and again, each from a thread and on a stream of its own; what they return."""
    import threading
    failed, start = [], threading.Barrier(len(calls))

    def loop(call, stream):
        start.wait()
        for _ in range(times):
            status = call(stream.cuda_stream)
            if status != 0:
                failed.append((status, B.lib().b200_last_error().decode()))
                return
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop, args=a) for a in zip(calls, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_attention_of_different_head_sizes_at_once():
    """The plain kernel's shared memory hangs on the head size: heads of 128 and of 116 share a kernel and need more than the default."""
    calls, checks = [], []
    for dim in (128, 116, 124):
        T.ATTENTIONS["at once"] = ("f32", 16, 1, dim, 16, [40], [0, 3], [0], [2, 1, 2], [10, 0, 31])
        state, cache, prefix, query, of = T.attention_state("at once")
        del T.ATTENTIONS["at once"]
        call, out = T.Attention(state, cache, prefix, query, of), torch.empty((state.rows, 16, dim), device="cuda")
        calls.append(lambda stream, call=call, out=out: B.lib().b200_prefix_attention(C.byref(call.a), C.byref(call.rows), call.max_length, call.max_prefix,
                                                                                        call.scratch.data_ptr(), call.need, out.data_ptr(), None, None, 0, stream))
        checks.append((state, cache, prefix, query, of, out))
    assert at_once(calls) == []
    for state, cache, prefix, query, of, out in checks:
        want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
        assert (np.abs(T.host(out).reshape(want.shape) - want) <= T.attention_bound(of, mass, size, keys)).all()


def test_verification_of_different_vocabularies_at_once():
    """The draw's shared memory hangs on the vocabulary; beyond 6 million values it is more than the default."""
    calls, checks = [], []
    for vocab in (1 << 23, 6_500_000, 7_300_001):
        state = T.Pass([2], [0], [0])
        logits = torch.full((2, vocab), -30.0, device="cuda")
        logits[:, vocab - 5] = 0.0
        check = T.Verify(state, np.zeros((2, 1), dtype=np.float32), None, np.array([3, vocab - 5]), 1.0, [0.5, 0.5], [0.5])
        check.a.vocab, check.a.logits = vocab, logits.data_ptr()
        calls.append(lambda stream, check=check: B.lib().b200_verify_drafts(C.byref(check.a), C.byref(check.state.args), check.scratch.data_ptr(), check.need, stream))
        checks.append((check, logits, vocab))
    assert at_once(calls) == []
    for check, _, vocab in checks:
        assert T.host(check.accepted).tolist() == [1] and T.host(check.next).tolist() == [vocab - 5]


# ---- long contexts, lengths that the pages do not hold -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,length,sequences,count,earlier", [
    ("bf16", 8, 2, 64, 64, 131072, 1, 1, 30),        # few rows: tiles of 16 pairs
    ("bf16", 4, 1, 128, 32, 100003, 40, 3, 100),     # many: the tcgen05 kernel
    ("bf16", 4, 1, 128, 64, 70, 2, 3, 70001),        # own tokens that are long
    ("bf16", 2, 1, 36, 10, 65537, 3, 2, 50),         # plain
    ("f32", 4, 2, 64, 16, 70001, 5, 2, 33000),
])
def test_long_contexts(dtype, heads, kv_heads, dim, page, length, sequences, count, earlier):
    prefix_span, span = -(-length // page), -(-(earlier + count) // page)
    pages = prefix_span + span * sequences
    order = np.random.default_rng(dim).permutation(pages)
    cache, prefix = T.Paged(dtype, kv_heads, page, dim, 1, order[:span * sequences].reshape(sequences, span)), T.Paged(dtype, kv_heads, page, dim, 1, order[span * sequences:].reshape(1, -1))
    g = torch.Generator(device="cuda").manual_seed(dim)
    cache.key, cache.value = prefix.key, prefix.value = torch.randn((2, pages, kv_heads, page, dim), generator=g, device="cuda").to(T.TORCH[dtype])
    query = (2.0 * torch.randn((sequences * count, heads, dim), generator=g, device="cuda")).to(T.TORCH[dtype])
    state = T.Pass([count] * sequences, list(range(sequences)), [earlier] * sequences)
    of = dict(heads=heads, dim=dim, prefixes=[length], group_first=[0, sequences], group_prefix=[0], dtype=dtype, max_length=earlier + count, max_prefix=length)
    out = torch.empty((sequences * count, heads, dim), device="cuda")
    T.Attention(state, cache, prefix, query, of)(out)
    for s in range(0, sequences, 7):
        def keys_of(pool):
            both = [pool[torch.as_tensor(t.astype(np.int64), device="cuda")].double().transpose(0, 1).reshape(kv_heads, -1, dim) for t in (prefix.table[0], cache.table[s])]
            return torch.cat([both[0][:, :length], both[1][:, :earlier + count]], 1)
        key, value = keys_of(cache.key), keys_of(cache.value)
        q = query[s * count:(s + 1) * count].double().view(count, kv_heads, heads // kv_heads, dim)
        hidden = torch.arange(key.shape[1], device="cuda")[None] > length + earlier + torch.arange(count, device="cuda")[:, None]
        weight = torch.softmax((torch.einsum("nkgd,kjd->nkgj", q, key) * dim ** -0.5).masked_fill(hidden[:, None, None], -float("inf")), -1)
        want, mass = (torch.einsum("nkgj,kjd->nkgd", weight, v).reshape(count, heads, dim).cpu().numpy() for v in (value, value.abs()))
        size = torch.einsum("nkgd,kjd->nkgj", q.abs(), key.abs()).amax(-1).reshape(count, heads).cpu().numpy() * dim ** -0.5
        got = T.host(out[s * count:(s + 1) * count])
        assert (np.abs(got - want) <= weight_bound(of, mass, size, np.full(count, key.shape[1]))).all(), s


@pytest.mark.parametrize("loose", [False, True])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,counts", [
    ("bf16", 8, 2, 64, 16, [1, 2, 1, 3]), ("bf16", 16, 1, 128, 64, [9, 7, 20, 11]), ("bf16", 4, 2, 33, 10, [1, 9, 2, 2]), ("f32", 4, 2, 64, 16, [3, 1, 2, 2]),
])
def test_lengths_that_the_pages_do_not_hold(dtype, heads, kv_heads, dim, page, counts, loose):
    """Prefix lengths below 0 and past the table, lengths past the slot's pages: what the pages hold is what there is."""
    rng = np.random.default_rng(page)
    cache, prefix = (T.Paged(dtype, kv_heads, page, dim, 24, t, rng) for t in (rng.permutation(24)[:12].reshape(4, 3), rng.permutation(24)[:12].reshape(4, 3)))
    prefix.key, prefix.value = cache.key, cache.value
    state = T.Pass(counts, [2, 0, 3, 1], [3 * page - 1, 5 * page, 0, 3 * page])
    query = T.dev(rng.standard_normal((state.rows, heads, dim), dtype=np.float32), T.TORCH[dtype])
    of = dict(heads=heads, dim=dim, prefixes=[-5, 10 * page, 3 * page, 1], group_first=[0, 1, 2, 3, 4], group_prefix=[1, 0, 2, 3], dtype=dtype,
              max_length=1 << 16 if loose else 6 * page, max_prefix=1 << 16 if loose else 10 * page)
    out = torch.empty((state.rows, heads, dim), device="cuda")
    T.Attention(state, cache, prefix, query, of)(out)
    want, mass, size, keys = T.wanted(state, cache, prefix, query, of)
    assert (np.abs(T.host(out) - want) <= weight_bound(of, mass, size, keys)).all()


@pytest.mark.parametrize("vocab", [300, 40000])
def test_temperatures_at_their_ends(vocab):
    """Towards 0 sampling becomes the argmax; towards infinity all tokens have the same share."""
    counts = [4, 1, 3]
    state, logits, draft, ids, accept, draw = T.verify_state(counts, vocab, 0.0, True, vocab)
    want = O.verify(logits, None, ids, [int(f) for f in state.first], 0.0, accept, draw)
    for temperature in (1e-6, 1e-36):
        accepted, chosen = T.Verify(state, logits, None, ids, temperature, np.full(state.rows, 0.5), [0.5] * 3)()
        assert np.array_equal(accepted, want[0]) and np.array_equal(chosen, want[1])
    # no draft is taken by uniforms above 1 / vocab; the residual leaves the refused token out, so vocab - 1 tokens share the draw (and vocab of them behind no draft)
    accepted, chosen = T.Verify(state, logits, None, ids, 1e36, np.full(state.rows, 0.5), [0.25 + 0.5 / vocab] * 3)()
    assert accepted.tolist() == [0, 0, 0]
    for s in range(3):
        left = [x for x in range(vocab) if counts[s] == 1 or x != ids[state.first[s] + 1]]
        at = (0.25 + 0.5 / vocab) * len(left)
        assert abs(at - round(at)) > 1e-3 and chosen[s] == left[int(at)]


def test_a_pass_in_parts_is_captured_and_replayed():
    """Three launches for every part in one graph: the same bits as by the call itself, with other queries and lengths."""
    rng = np.random.default_rng(1)
    heads, kv_heads, dim, page, counts = 256, 4, 64, 64, [500, 1, 700, 30]
    table, prefix_table = np.arange(60).reshape(4, 15), np.arange(60, 64).reshape(1, 4)
    cache, prefix = T.Paged("bf16", kv_heads, page, dim, 64, table, rng), T.Paged("bf16", kv_heads, page, dim, 1, prefix_table)
    prefix.key, prefix.value = cache.key, cache.value
    state = T.Pass(counts, [2, 0, 3, 1], [0, 7, 64, 100])
    assert state.rows * heads > 1 << 18
    query = T.dev(rng.standard_normal((state.rows, heads, dim), dtype=np.float32), torch.bfloat16)
    of = dict(heads=heads, dim=dim, prefixes=[250], group_first=[0, 3], group_prefix=[0], dtype="bf16", max_length=1 << 14, max_prefix=1 << 16)
    call = T.Attention(state, cache, prefix, query, of)
    out, one = torch.empty((state.rows, heads, dim), device="cuda"), torch.empty((state.rows, heads, dim), dtype=torch.bfloat16, device="cuda")

    def both():
        call(out)
        call(None, one)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(3):
        query.copy_(torch.randn_like(query, dtype=torch.float32))
        state.d[3].copy_(T.dev(rng.integers(0, 200, 4).astype(np.int32)))
        got = []
        for how in (graph.replay, both):
            call.scratch.fill_(0xff)
            out.zero_()
            one.zero_()
            how()
            torch.cuda.synchronize()
            got.append((out.clone(), one.clone()))
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*got))
