"""What the operators of speculative serving behind a shared prompt are measured on.

A program that answers many requests over one long prompt (a system prompt, a document, several samples of one question) runs, in every layer of a
pass, `b200_rotary_append` on the projected rows and `b200_prefix_attention` on the caches, and at the end of the pass `b200_verify_drafts` on the
logits; `b200_rotary_tables` makes the angles once per model or context length.  A case names its `path`:

  tables     cosines and sines of rotary positions, with the usual ways to stretch them for long contexts.
  append     rotation of queries and keys of a packed pass, keys and values into the paged cache.
  attention  grouped-query attention of a packed pass over a prefix that a group of sequences shares and over every sequence's own tokens.
  verify     drafted tokens against the target's probabilities, from given random numbers.

Lengths of a case come from its own `shape` number, so that every input of the case has the same work; values come from the seed."""
from __future__ import annotations

import ctypes as C
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a small model's tables at its start: the smallest call
        {"name": "tables_2k", "path": "tables", "kind": 0, "dims": 64, "positions": 2048, "base": 10000.0, "factor": 1.0},
        # a context stretched by parts to 128k positions
        {"name": "tables_128k_parts", "path": "tables", "kind": 3, "dims": 128, "positions": 131072, "base": 500000.0, "factor": 8.0},
        # one user's next token
        {"name": "append_step_1", "path": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 64, "rot": 64, "pairs": True, "page": 64,
         "sequences": 1, "count": 1, "length": 300, "ragged": False, "shape": 1},
        # a full decode batch, projections in f32 as the linear kernels leave them, part of the head turning
        {"name": "append_step_256", "path": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "pairs": False, "page": 64,
         "sequences": 256, "count": 1, "length": 1024, "ragged": False, "shape": 2},
        # prompts of unequal length in one pass
        {"name": "append_prompts", "path": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "pairs": False, "page": 64,
         "sequences": 24, "count": 1024, "length": 500, "ragged": True, "shape": 3},
        # a few answers to one short prompt: latency
        {"name": "attention_step_4", "path": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 64, "page": 64, "groups": 1,
         "sequences": 4, "count": 1, "prefix": 700, "length": 90, "shape": 4},
        # a decode batch behind one system prompt
        {"name": "attention_step_64", "path": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "groups": 1,
         "sequences": 64, "count": 1, "prefix": 8192, "length": 512, "shape": 5},
        # several samples of each of a few questions, with drafted tokens
        {"name": "attention_drafts_8x12", "path": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "groups": 8,
         "sequences": 96, "count": 5, "prefix": 3001, "length": 700, "shape": 6},
        # the f32 configuration
        {"name": "attention_f32", "path": "attention", "dtype": "f32", "heads": 12, "kv_heads": 4, "dim": 64, "page": 16, "groups": 1,
         "sequences": 9, "count": 3, "prefix": 1201, "length": 200, "shape": 7},
        # questions about one long document, read in one pass: the largest
        {"name": "attention_prompts", "path": "attention", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "groups": 1,
         "sequences": 16, "count": 200, "prefix": 8000, "length": 64, "shape": 8},
        # four drafted tokens of one sequence
        {"name": "verify_1", "path": "verify", "vocab": 32000, "sequences": 1, "drafts": 4, "model": True, "temperature": 0.8, "shape": 9},
        # a batch with a large vocabulary and up to seven drafts each
        {"name": "verify_64", "path": "verify", "vocab": 128256, "sequences": 64, "drafts": 7, "model": True, "temperature": 1.0, "shape": 10},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    path = rng.choice(["tables", "append", "append", "attention", "attention", "attention", "verify", "verify"])
    shape = rng.randrange(1 << 30)
    if path == "tables":
        dims = 2 * _log(rng, 8, 64)
        return {"path": path, "kind": rng.randrange(4), "dims": dims, "positions": _log(rng, 100, 131072), "base": rng.choice([10000.0, 500000.0, 1e6]),
                "factor": rng.choice([2.0, 4.0, 8.0, 32.0])}
    group = rng.choice([1, 2, 3, 4, 4, 8])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 80, 96])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    page = rng.choice([16, 32, 64, 64, 128, 24])
    if path == "append":
        ragged = rng.random() < 0.5
        sequences = _log(rng, 1, 24 if ragged else 256)
        return {"path": path, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "dim": dim, "rot": rng.choice([dim, dim // 2]), "pairs": rng.random() < 0.5,
                "page": page, "sequences": sequences, "count": _log(rng, 2, 1024) if ragged else 1, "length": _log(rng, 1, 2048), "ragged": ragged, "shape": shape}
    if path == "attention":
        sequences = _log(rng, 1, 64)
        count = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 8, 100)])
        case = {"path": path, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page, "groups": rng.choice([1, 1, min(sequences, rng.randint(2, 8))]),
                "sequences": sequences, "count": count, "prefix": _log(rng, 16, 8192), "length": _log(rng, 1, 1024), "shape": shape}
        while work(case)["flops"] > 1.5e10 * (10 if dtype == "bf16" else 1) and case["count"] > 1:
            case["count"] = max(1, case["count"] // 2)
        return case
    return {"path": path, "vocab": rng.choice([1000, 32000, 50257, 128256, _log(rng, 500, 128256)]), "sequences": _log(rng, 1, 64), "drafts": rng.randint(1, 7),
            "model": rng.random() < 0.7, "temperature": rng.choice([0.0, 0.6, 1.0, 1.3]), "shape": shape}


# ---- sizes of a case -----------------------------------------------------------------------------------------------------------------------------


def _counts(case):
    """Rows, earlier tokens and group sizes of the sequences of a packed pass."""
    r = random.Random(case["shape"])
    n = case["sequences"]
    ragged = case.get("ragged", case["path"] == "attention")
    counts = [r.randint(max(1, case["count"] // 3), case["count"]) if ragged else case["count"] for _ in range(n)]
    lengths = [r.randint(case["length"] // 2, case["length"]) for _ in range(n)]
    groups = case.get("groups", 1)
    cuts = sorted(r.sample(range(1, n), groups - 1))
    prefixes = [case.get("prefix", 0) - r.randint(0, case.get("prefix", 0) // 4) if g else case.get("prefix", 0) for g in range(groups)]
    return counts, lengths, [0, *cuts, n], prefixes


def _drafts(case):
    r = random.Random(case["shape"])
    return [case["drafts"] if case["sequences"] < 4 else r.randint(case["drafts"] // 2, case["drafts"]) for _ in range(case["sequences"])]


def work(case):
    if case["path"] == "tables":
        return {"bytes": 4.0 * case["positions"] * case["dims"], "flops": 20.0 * case["positions"] * case["dims"]}
    if case["path"] == "verify":
        rows = [d + 1 for d in _drafts(case)]
        read = sum(rows) + (sum(rows) - len(rows) if case["model"] and case["temperature"] > 0 else 0)   # a sequence's last row has no draft
        return {"bytes": 4.0 * read * case["vocab"], "flops": 4.0 * read * case["vocab"]}
    counts, lengths, first_of_group, prefixes = _counts(case)
    size = 4 if case["dtype"] == "f32" else 2
    h, k, d = case["heads"], case["kv_heads"], case["dim"]
    rows = sum(counts)
    if case["path"] == "append":
        # projected rows in f32, queries and cached keys and values out, the angles of the rows' positions
        return {"bytes": float(rows * (4 * (h + 2 * k) * d + size * (h + 2 * k) * d + 4 * case["rot"])), "flops": 3.0 * rows * (h + k) * case["rot"]}
    keys = sum(prefixes) + sum(c + n for c, n in zip(counts, lengths))
    pairs = sum(c * n + c * (c + 1) // 2 for c, n in zip(counts, lengths))
    for g, p in enumerate(prefixes):
        pairs += p * sum(counts[first_of_group[g]:first_of_group[g + 1]])
    return {"bytes": float(size * (2 * keys * k * d + 2 * rows * h * d)), "flops": 4.0 * pairs * h * d}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------------


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _packed(counts, lengths, g):
    """A packed pass: slots in a shuffled order, the first row of every sequence, every row's sequence."""
    n = len(counts)
    slots = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    first = [0]
    for c in counts:
        first.append(first[-1] + c)
    of_slot = torch.empty(n, dtype=torch.int32, device="cuda")
    of_slot[slots.long()] = _ints(lengths)
    return {"rows": first[-1], "sequences": n, "max_count": max(counts), "slot": slots, "first": _ints(first),
            "sequence": torch.repeat_interleave(torch.arange(n, device="cuda", dtype=torch.int32), _ints(counts).long()), "lengths": of_slot}


def _scaling(case):
    return {"kind": case["kind"], "base": case["base"], "factor": case["factor"], "original": 8192.0, "low": 1.0, "high": 4.0,
            "magnitude": 0.1 * math.log(case["factor"]) + 1.0 if case["kind"] == 3 else 1.0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    path = case["path"]
    state = {"case": case}

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    def uniform(n):
        return torch.rand(n, generator=g, device="cuda", dtype=torch.float64)

    if path == "tables":
        # tables of another range of positions each time: a window that a long context moves through
        state["start"] = seed % 1000
        state["cosine"], state["sine"] = (torch.empty(case["positions"], case["dims"] // 2, device="cuda") for _ in range(2))
        return state
    if path == "verify":
        counts = [d + 1 for d in _drafts(case)]
        p = _packed(counts, [100 + 3 * i for i in range(len(counts))], g)
        v = case["vocab"]
        logits = normal(p["rows"], v, scale=2.5)
        draft = logits + normal(p["rows"], v, scale=0.6)
        # every row's token is drawn from the draft's distribution of the row before it
        t = max(case["temperature"], 1e-3)
        drawn = (draft / t - torch.empty_like(draft).exponential_(generator=g).log_()).argmax(1)
        ids = torch.randint(0, v, (p["rows"],), generator=g, device="cuda")
        ids[1:] = torch.where(p["sequence"][1:] == p["sequence"][:-1], drawn[:-1], ids[1:])
        state |= {"pass": p, "logits": logits, "draft": draft if case["model"] else None, "ids": ids, "accept": uniform(p["rows"]), "draw": uniform(p["sequences"]),
                  "accepted": torch.empty(p["sequences"], dtype=torch.int32, device="cuda"), "next": torch.empty(p["sequences"], dtype=torch.int64, device="cuda")}
        return state
    counts, lengths, first_of_group, prefixes = _counts(case)
    p = _packed(counts, lengths, g)
    h, k, d, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], TYPES[case["dtype"]]
    span = -(-max(c + n for c, n in zip(counts, lengths)) // page)                       # pages of a slot, and of a prefix
    prefix_span = max(1, -(-max(prefixes) // page)) if path == "attention" else 0
    pages = span * p["sequences"] + prefix_span * len(prefixes)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    state |= {"pass": p, "table": order[:span * p["sequences"]].view(p["sequences"], span).contiguous(), "pages": pages, "max_length": max(c + n for c, n in zip(counts, lengths))}
    if path == "append":
        state["key"], state["value"] = (torch.zeros(pages, k, page, d, dtype=dtype, device="cuda") for _ in range(2))
        state["projected"] = normal(p["rows"], (h + 2 * k) * d)
        reach = case["length"] + case["count"] + 4096
        angle = torch.arange(reach, device="cuda", dtype=torch.float64)[:, None] * (10000.0 ** (-2.0 * torch.arange(case["rot"] // 2, device="cuda") / case["rot"]).double())
        state["cosine"], state["sine"], state["positions"] = angle.cos().float(), angle.sin().float(), reach
        state["offset"] = torch.randint(0, 4096, (p["sequences"],), generator=g, device="cuda", dtype=torch.int32)   # lengths of the prefixes before the slots
        state["query"] = torch.empty(p["rows"], h, d, dtype=dtype, device="cuda")
        return state
    # values with a mean per channel, as they have in trained models; scores with a spread of about two
    state["key"] = normal(pages, k, page, d, dtype=dtype)
    state["value"] = (normal(pages, k, page, d) + 0.5 * normal(1, k, 1, d)).to(dtype)
    state["query"] = normal(p["rows"], h, d, scale=2.0, dtype=dtype)
    state["prefix_table"] = order[span * p["sequences"]:].view(len(prefixes), prefix_span).contiguous()
    state["group_prefix"] = torch.randperm(len(prefixes), generator=g, device="cuda").to(torch.int32)
    state["prefix_length"] = torch.empty(len(prefixes), dtype=torch.int32, device="cuda")
    state["prefix_length"][state["group_prefix"].long()] = _ints(prefixes)
    state["group_first"], state["groups"], state["max_prefix"] = _ints(first_of_group), len(prefixes), max(prefixes)
    state["most_rows"] = max(sum(counts[first_of_group[i]:first_of_group[i + 1]]) for i in range(len(prefixes)))   # of one group
    state["out"] = torch.empty(p["rows"], h * d, dtype=dtype, device="cuda")
    return state


# ---- the framework's calls -----------------------------------------------------------------------------------------------------------------------


def _pointer(t):
    return None if t is None else t.data_ptr()


def _call(state):
    """The argument structs of a state, as a program that runs the operator again and again keeps them, and the call."""
    import ctorch_b200 as B
    l, case, path = B.lib(), state["case"], state["case"]["path"]
    if path == "tables":
        s = B.RotaryScaling(**_scaling(case))
        held = (s, state)
        args = (C.byref(s), case["dims"], state["start"], case["positions"], state["cosine"].data_ptr(), state["sine"].data_ptr())
        return l.b200_rotary_tables, args, B.kcheck, held
    p = state["pass"]
    rows = B.Rows(rows=p["rows"], sequences=p["sequences"], max_count=p["max_count"], slot=p["slot"].data_ptr(), first=p["first"].data_ptr(),
                  sequence=p["sequence"].data_ptr(), lengths=p["lengths"].data_ptr())
    if path == "verify":
        a = B.VerifyArgs(vocab=case["vocab"], stride=0, logits=state["logits"].data_ptr(), draft_logits=_pointer(state["draft"]), ids=state["ids"].data_ptr(),
                         temperature=case["temperature"], accept=state["accept"].data_ptr(), draw=state["draw"].data_ptr(), accepted=state["accepted"].data_ptr(),
                         next=state["next"].data_ptr(), advance=0)
        need = l.b200_verify_scratch_bytes(C.byref(a), C.byref(rows))
        scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        return l.b200_verify_drafts, (C.byref(a), C.byref(rows), scratch.data_ptr(), need), B.kcheck, (a, rows, scratch)
    code = B.F32 if case["dtype"] == "f32" else B.BF16

    def pages(table):
        return B.KvPages(dtype=code, kv_heads=case["kv_heads"], head_dim=case["dim"], page_size=case["page"], sequences=table.shape[0],
                         pages_per_sequence=table.shape[1], pages=state["pages"], key=state["key"].data_ptr(), value=state["value"].data_ptr(), table=table.data_ptr())

    cache = pages(state["table"])
    if path == "append":
        a = B.RotaryAppendArgs(heads=case["heads"], rot_dims=case["rot"], rotate_pairs=int(case["pairs"]), cosine=state["cosine"].data_ptr(), sine=state["sine"].data_ptr(),
                               positions=state["positions"], offset=state["offset"].data_ptr(), projected=state["projected"].data_ptr(), stride=0,
                               query_dtype=code, query=state["query"].data_ptr(), cache=cache)
        return l.b200_rotary_append, (C.byref(a), C.byref(rows)), B.kcheck, (a, rows)
    a = B.PrefixArgs(heads=case["heads"], scale=case["dim"] ** -0.5, query=state["query"].data_ptr(), cache=cache, prefix=pages(state["prefix_table"]),
                     groups=state["groups"], group_first=state["group_first"].data_ptr(), group_prefix=state["group_prefix"].data_ptr(),
                     prefix_length=state["prefix_length"].data_ptr())
    need = l.b200_prefix_scratch_bytes(C.byref(a), C.byref(rows), state["max_length"], state["max_prefix"])
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = state["out"].data_ptr()
    return l.b200_prefix_attention, (C.byref(a), C.byref(rows), state["max_length"], state["max_prefix"], scratch.data_ptr(), need,
                                     out if code == B.F32 else None, out if code == B.BF16 else None, None, 0), B.kcheck, (a, rows, scratch)


def run(state):
    path = state["case"]["path"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        call, args, check, _ = state["call"]
        check(call(*args, torch.cuda.current_stream().cuda_stream))
    else:
        {"tables": _tables, "append": _append, "attention": _attention, "verify": _verify}[path](state)
    if path == "tables":
        return state["cosine"], state["sine"]
    if path == "append":
        return state["query"], state["key"], state["value"]
    if path == "attention":
        return state["out"]
    return state["accepted"], state["next"]


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------------


def _tables(state):
    case = state["case"]
    s, dims = _scaling(case), case["dims"]
    i = torch.arange(dims // 2, device="cuda", dtype=torch.float64)
    base = s["base"] * s["factor"] ** (dims / (dims - 2)) if s["kind"] == 2 else s["base"]
    frequency = torch.exp(-2.0 * i / dims * math.log(base))
    if s["kind"] == 1:
        frequency = frequency / s["factor"]
    if s["kind"] == 3:
        kept = ((s["original"] * frequency / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        frequency = frequency * (kept + (1 - kept) / s["factor"])
    angle = torch.arange(state["start"], state["start"] + case["positions"], device="cuda", dtype=torch.float64)[:, None] * frequency
    state["cosine"].copy_(s["magnitude"] * angle.cos())
    state["sine"].copy_(s["magnitude"] * angle.sin())


def _places(state):
    """Sequence, slot and position in the slot of every row."""
    p = state["pass"]
    sequence = p["sequence"].long()
    slot = p["slot"].long()[sequence]
    return sequence, slot, p["lengths"].long()[slot] + torch.arange(p["rows"], device="cuda") - p["first"].long()[sequence]


def _append(state):
    case = state["case"]
    h, k, d, rot, page = case["heads"], case["kv_heads"], case["dim"], case["rot"], case["page"]
    sequence, slot, position = _places(state)
    at = position + state["offset"].long()[sequence]
    cosine, sine = state["cosine"][at][:, None], state["sine"][at][:, None]
    heads = state["projected"].view(-1, h + 2 * k, d)
    turned = heads[:, :h + k]
    if case["pairs"]:
        a, b = turned[..., 0:rot:2], turned[..., 1:rot:2]
        head = torch.stack([a * cosine - b * sine, b * cosine + a * sine], -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:rot]
        head = torch.cat([a * cosine - b * sine, b * cosine + a * sine], -1)
    turned = torch.cat([head, turned[..., rot:]], -1)
    state["query"].copy_(turned[:, :h])
    where = state["table"].long()[slot, position // page]
    state["key"][where, :, position % page] = turned[:, h:].to(state["key"].dtype)
    state["value"][where, :, position % page] = heads[:, h + k:].to(state["value"].dtype)


def _keys(state, pool, table):
    """The pages of a table as [sequences, kv_heads, keys, dim] in f32."""
    return pool[table.long()].transpose(1, 2).flatten(2, 3).float()


def _attention(state):
    case, p = state["case"], state["pass"]
    h, k, d = case["heads"], case["kv_heads"], case["dim"]
    sequence, slot, position = _places(state)
    group = torch.searchsorted(state["group_first"].long(), sequence, right=True) - 1
    in_group = torch.arange(p["rows"], device="cuda") - p["first"].long()[state["group_first"].long()[group]]
    in_sequence = torch.arange(p["rows"], device="cuda") - p["first"].long()[sequence]
    query = state["query"].float().view(-1, k, h // k, d)

    def scores(index, place, sets, most, table):
        """Products with the keys of a table, the rows gathered by set: [rows, kv_heads, heads per kv head, keys]."""
        rows = query.new_zeros(sets, most, k, h // k, d)
        rows[index, place] = query
        keys = _keys(state, state["key"], table)
        s = torch.matmul(rows.permute(0, 2, 1, 3, 4).flatten(2, 3), keys.transpose(-1, -2))
        return s.view(sets, k, most, h // k, -1).transpose(1, 2)[index, place] * d ** -0.5

    def sums(weights, index, place, sets, most, table):
        rows = weights.new_zeros(sets, most, k, h // k, weights.shape[-1])
        rows[index, place] = weights
        values = _keys(state, state["value"], table)
        s = torch.matmul(rows.permute(0, 2, 1, 3, 4).flatten(2, 3), values)
        return s.view(sets, k, most, h // k, d).transpose(1, 2)[index, place]

    prefix_table = state["prefix_table"][state["group_prefix"].long()]
    table = state["table"][p["slot"].long()]
    first = (group, in_group, state["groups"], state["most_rows"], prefix_table)
    second = (sequence, in_sequence, p["sequences"], p["max_count"], table)
    shared = scores(*first)
    seen = torch.arange(shared.shape[-1], device="cuda") < state["prefix_length"].long()[state["group_prefix"].long()][group][:, None]
    shared = shared.masked_fill(~seen[:, None, None], -math.inf)
    mine = scores(*second)
    mine = mine.masked_fill((torch.arange(mine.shape[-1], device="cuda") > position[:, None])[:, None, None], -math.inf)
    top = torch.maximum(shared.amax(-1, keepdim=True), mine.amax(-1, keepdim=True))
    shared, mine = (shared - top).exp_(), (mine - top).exp_()
    total = shared.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)
    state["out"].copy_(((sums(shared, *first) + sums(mine, *second)) / total).flatten(1))


def _verify(state):
    case, p = state["case"], state["pass"]
    logits, ids, first = state["logits"], state["ids"], p["first"].long()
    sequence = p["sequence"].long()
    row = torch.arange(p["rows"], device="cuda")
    last = row == first[sequence + 1] - 1
    token = torch.where(last, 0, ids.roll(-1))
    if case["temperature"] == 0:
        best = logits.argmax(1)
        rejects = last | (token != best)
        stop = torch.full((p["sequences"],), p["rows"], device="cuda").scatter_reduce(0, sequence, torch.where(rejects, row, p["rows"]), "amin")
        state["accepted"].copy_(stop - first[:-1])
        state["next"].copy_(best[stop])
        return
    inverse = torch.tensor(1.0 / case["temperature"], dtype=torch.float32)

    def weights(x):
        """exp((x - max) / T) in f32, as b200_sample has its weights, and their sums, which are border values' scale, in f64."""
        e = ((x - x.amax(1, keepdim=True)) * inverse).exp()
        return e, e.sum(1, dtype=torch.float64)

    e, total = weights(logits)
    p_token = e.gather(1, token[:, None])[:, 0].double() / total
    if state["draft"] is not None:
        f, draft_total = weights(state["draft"])
        q_token = f.gather(1, token[:, None])[:, 0].double() / draft_total
    else:
        q_token = torch.ones_like(p_token)
    rejects = last | ~(state["accept"] * q_token < p_token)
    stop = torch.full((p["sequences"],), p["rows"], device="cuda").scatter_reduce(0, sequence, torch.where(rejects, row, p["rows"]), "amin")
    # what is left of the target's distribution where the draft was refused; all of it behind the last draft
    target = e[stop].double() / total[stop][:, None]
    if state["draft"] is not None:
        minus = f[stop].double() / draft_total[stop][:, None]
    else:
        minus = torch.zeros_like(target).scatter_(1, token[stop][:, None], 1.0)
    left = torch.where(last[stop][:, None], target, (target - minus).clamp(min=0))
    left = torch.where(left.sum(1, keepdim=True) > 0, left, target)
    running = left.cumsum(1)
    state["accepted"].copy_(stop - first[:-1])
    state["next"].copy_((running <= state["draw"][:, None] * running[:, -1:]).sum(1).clamp(max=case["vocab"] - 1))


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    path = case["path"]
    if path == "verify":
        return None   # whole numbers
    state = prepare(case, seed)
    if path == "tables":
        s, half = _scaling(case), case["dims"] // 2
        frequencies = []
        for i in range(half):
            if s["kind"] == 2:
                f = (s["base"] * s["factor"] ** (case["dims"] / (case["dims"] - 2))) ** (-i / half)
            else:
                f = s["base"] ** (-i / half)
            if s["kind"] == 1:
                f /= s["factor"]
            if s["kind"] == 3:
                turns = s["original"] * f / math.tau
                share = 1.0 if turns >= s["high"] else 0.0 if turns <= s["low"] else (turns - s["low"]) / (s["high"] - s["low"])
                f = share * f + (1 - share) * f / s["factor"]
            frequencies.append(f)
        turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"),
                           torch.outer(torch.arange(case["positions"], dtype=torch.float64, device="cuda") + state["start"], torch.tensor(frequencies, dtype=torch.float64, device="cuda")))
        return turn.real.contiguous(), turn.imag.contiguous()
    p, h, k, d, page = state["pass"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    slots, first, lengths = p["slot"].tolist(), p["first"].tolist(), p["lengths"].tolist()
    if path == "append":
        key, value = state["key"].double(), state["value"].double()
        query = torch.empty(p["rows"], h, d, dtype=torch.float64, device="cuda")
        rot, offsets = case["rot"], state["offset"].tolist()
        low = torch.arange(0, rot, 2, device="cuda") if case["pairs"] else torch.arange(rot // 2, device="cuda")
        high = low + 1 if case["pairs"] else low + rot // 2
        for s, slot in enumerate(slots):
            x = state["projected"][first[s]:first[s + 1]].double().view(-1, h + 2 * k, d)
            at = lengths[slot] + torch.arange(len(x), device="cuda")
            turn = torch.complex(state["cosine"][at + offsets[s]].double(), state["sine"][at + offsets[s]].double())[:, None]
            z = torch.complex(x[:, :h + k, low], x[:, :h + k, high]) * turn
            y = x[:, :h + k].clone()
            y[..., low], y[..., high] = z.real, z.imag
            query[first[s]:first[s + 1]] = y[:, :h]
            where = state["table"][slot].long()[at // page]
            key[where, :, at % page], value[where, :, at % page] = y[:, h:], x[:, h + k:]
        return query, key, value
    out = torch.empty(p["rows"], h, d, dtype=torch.float64, device="cuda")
    group_first, group_prefix, prefix_length = (state[n].tolist() for n in ("group_first", "group_prefix", "prefix_length"))
    for g, prefix in enumerate(group_prefix):
        for s in range(group_first[g], group_first[g + 1]):
            n = first[s + 1] - first[s]
            mine = lengths[slots[s]] + n

            def keys(pool):
                a, b = (pool[table.long()].double().transpose(0, 1).reshape(k, -1, d) for table in (state["prefix_table"][prefix], state["table"][slots[s]]))
                return torch.cat([a[:, :prefix_length[prefix]], b[:, :mine]], 1)

            q = state["query"][first[s]:first[s + 1]].double().view(n, k, h // k, d).permute(1, 2, 0, 3)
            score = torch.einsum("kgnd,kjd->kgnj", q, keys(state["key"])) / math.sqrt(d)
            hidden = torch.ones(n, mine, device="cuda", dtype=torch.bool).triu(mine - n + 1)
            score[..., prefix_length[prefix]:].masked_fill_(hidden, -math.inf)
            out[first[s]:first[s + 1]] = torch.einsum("kgnj,kjd->nkgd", torch.softmax(score, -1), keys(state["value"])).reshape(n, h, d)
    return out.flatten(1)
