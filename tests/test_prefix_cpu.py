"""Operators for drafted tokens behind a shared prompt, without a GPU: what they refuse, what their workspaces need, and the oracle's own sense."""
import ctypes as C

import numpy as np
import pytest

import ctorch_b200 as B
import prefix_oracle as O

HERE = 0x1000   # an address that is never followed: every call here ends before its launch


def pages(**changes):
    fields = dict(dtype=B.BF16, kv_heads=2, head_dim=64, page_size=16, sequences=4, pages_per_sequence=8, pages=32, key=HERE, value=HERE, table=HERE)
    return B.KvPages(**{**fields, **changes})


def rows(**changes):
    fields = dict(rows=6, sequences=4, max_count=3, slot=HERE, first=HERE, sequence=HERE, lengths=HERE)
    return B.Rows(**{**fields, **changes})


def error():
    return B.lib().b200_last_error().decode()


BAD_PAGES = [dict(dtype=4), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0), dict(sequences=0), dict(pages_per_sequence=0), dict(pages=0), dict(pages=1 << 31),
             dict(key=None), dict(value=None), dict(table=None), dict(pages_per_sequence=1 << 24, page_size=1 << 10)]
BAD_ROWS = [dict(rows=0), dict(sequences=0), dict(sequences=7), dict(max_count=0), dict(max_count=7), dict(slot=None), dict(first=None), dict(sequence=None), dict(lengths=None)]


def test_tables_refuse():
    l = B.lib()
    good = dict(kind=B.ROTARY_PARTS, base=1e4, factor=8.0, original=8192.0, low=1.0, high=4.0, magnitude=1.0)

    def call(dims=64, first=0, positions=8, cosine=HERE, sine=HERE, **changes):
        return l.b200_rotary_tables(C.byref(B.RotaryScaling(**{**good, **changes})), dims, first, positions, cosine, sine, None)
    for bad in (dict(dims=0), dict(dims=7), dict(dims=-2), dict(first=-1), dict(positions=-1), dict(cosine=None), dict(sine=None), dict(kind=4), dict(kind=-1), dict(base=0.0),
                dict(base=-1.0), dict(base=float("nan")), dict(base=float("inf")), dict(factor=0.0), dict(factor=-2.0), dict(factor=float("nan")), dict(original=0.0),
                dict(low=4.0), dict(low=float("nan")), dict(high=float("inf")), dict(magnitude=float("nan")), dict(first=1 << 60)):
        assert call(**bad) == -1 and "b200_rotary_tables" in error(), bad
    assert l.b200_rotary_tables(None, 64, 0, 8, HERE, HERE, None) == -1
    assert call(positions=0) == 0


def test_append_refuses():
    l = B.lib()
    good = dict(heads=4, rot_dims=64, rotate_pairs=0, cosine=HERE, sine=HERE, positions=100, offset=None, projected=HERE, stride=0, query_dtype=B.BF16, query=HERE)

    def call(cache=None, of=None, **changes):
        return l.b200_rotary_append(C.byref(B.RotaryAppendArgs(**{**good, **changes}, cache=cache or pages())), C.byref(of or rows()), None)
    for bad in (dict(heads=0), dict(rot_dims=66), dict(rot_dims=63), dict(rot_dims=-2), dict(cosine=None), dict(sine=None), dict(positions=0), dict(projected=None),
                dict(stride=511), dict(stride=-512), dict(query_dtype=4), dict(query=None), dict(cache=pages(head_dim=63), rot_dims=0), dict(heads=1 << 26)):
        assert call(**bad) == -1 and "b200_rotary_append" in error(), bad
    for bad in BAD_PAGES:
        assert call(cache=pages(**bad)) == -1 and "b200_rotary_append" in error(), bad
    for bad in BAD_ROWS:
        assert call(of=rows(**bad)) == -1 and "b200_rows" in error(), bad
    assert l.b200_rotary_append(None, C.byref(rows()), None) == -1 and l.b200_rotary_append(C.byref(B.RotaryAppendArgs()), None, None) == -1


def test_attention_refuses():
    l = B.lib()
    good = dict(heads=4, scale=0.125, query=HERE, groups=1, group_first=HERE, group_prefix=HERE, prefix_length=HERE)

    def call(cache=None, prefix=None, of=None, max_length=100, max_prefix=100, scratch=HERE, size=1 << 40, out=None, hi=HERE, lo=None, stride=0, **changes):
        a = B.PrefixArgs(**{**good, **changes}, cache=cache or pages(), prefix=prefix or pages())
        return l.b200_prefix_attention(C.byref(a), C.byref(of or rows()), max_length, max_prefix, scratch, size, out, hi, lo, stride, None)
    for bad in (dict(heads=0), dict(heads=3), dict(query=None), dict(scale=float("nan")), dict(scale=float("inf")), dict(groups=-1), dict(group_first=None),
                dict(group_prefix=None), dict(prefix_length=None), dict(max_length=0), dict(max_prefix=-1), dict(scratch=None), dict(scratch=HERE + 8), dict(size=16),
                dict(hi=None), dict(hi=None, out=HERE, lo=HERE), dict(stride=255), dict(prefix=pages(head_dim=128)), dict(prefix=pages(kv_heads=4)),
                dict(prefix=pages(dtype=B.F32))):
        assert call(**bad) == -1 and "b200_prefix_attention" in error(), bad
    for bad in BAD_PAGES:
        assert call(cache=pages(**bad)) == -1 and call(prefix=pages(**bad)) == -1 and "b200_prefix_attention" in error(), bad
    for bad in BAD_ROWS:
        assert call(of=rows(**bad)) == -1 and "b200_rows" in error(), bad
    assert call(cache=pages(head_dim=264), prefix=pages(head_dim=264)) == -2 and "head_dim" in error()
    a = B.PrefixArgs(**good, cache=pages(), prefix=pages())
    need = l.b200_prefix_scratch_bytes(C.byref(a), C.byref(rows()), 100, 100)
    assert need >= 6 * 4 * 66 * 4 and call(size=need - 1) == -1 and str(need) in error()
    assert l.b200_prefix_scratch_bytes(C.byref(a), C.byref(rows()), 0, 100) == 0 and l.b200_prefix_scratch_bytes(None, C.byref(rows()), 1, 1) == 0


def test_verify_refuses():
    l = B.lib()
    good = dict(vocab=100, stride=0, logits=HERE, draft_logits=HERE, ids=HERE, temperature=1.0, accept=HERE, draw=HERE, accepted=HERE, next=HERE, advance=0)

    def call(of=None, scratch=HERE, size=1 << 40, **changes):
        return l.b200_verify_drafts(C.byref(B.VerifyArgs(**{**good, **changes})), C.byref(of or rows()), scratch, size, None)
    for bad in (dict(vocab=0), dict(vocab=-5), dict(stride=99), dict(logits=None), dict(ids=None), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(temperature=1e-300), dict(temperature=1e300), dict(accept=None), dict(draw=None), dict(accepted=None), dict(next=None),
                dict(scratch=None), dict(scratch=HERE + 4), dict(size=16)):
        assert call(**bad) == -1 and "b200_verify_drafts" in error(), bad
    for bad in BAD_ROWS:
        assert call(of=rows(**bad)) == -1 and "b200_rows" in error(), bad
    assert call(vocab=(1 << 23) + 1) == -2 and "2^23" in error()
    assert l.b200_verify_drafts(None, C.byref(rows()), HERE, 1 << 30, None) == -1


def test_cache_pages_refuses():
    l = B.lib()
    assert l.b200_kv_cache_pages(None, C.byref(B.KvPages())) == -1 and "b200_kv_cache_pages" in error()


@pytest.mark.parametrize("seed", range(3))
def test_verified_tokens_follow_the_target(seed):
    """The rule that the oracle states draws from p: over all values of the two uniforms, in steps, the first token has p's shares."""
    r = np.random.default_rng(seed)
    logits, draft = r.normal(size=(2, 5)) * 1.5, r.normal(size=(2, 5)) * 1.5
    p, q = O.weights(logits[0], 0.8), O.weights(draft[0], 0.8)
    steps, share = 40, np.zeros(5)
    for x in range(5):
        for i in range(steps):
            for j in range(steps):
                accepted, chosen, _ = O.verify(logits, draft, [0, x], [0, 2], 0.8, [(i + 0.5) / steps] * 2, [(j + 0.5) / steps])
                share[x if accepted[0] else chosen[0]] += q[x] / steps ** 2
    assert np.abs(share - p).max() < 5 * 2 / steps   # a step's width per border, five borders, two uniforms


def test_parts_scaling_of_the_oracle():
    """Entries that turn often in the training's positions stay, those that hardly turn are stretched by the factor."""
    plain, parts = O.frequencies(0, 64, 1e4), O.frequencies(3, 64, 1e4, 8.0, 8192.0, 1.0, 32.0)
    assert parts[0] == plain[0] and np.isclose(parts[-1], plain[-1] / 8) and ((parts <= plain) & (parts >= plain / 8)).all()
    base = O.frequencies(2, 64, 1e4, 8.0)
    assert base[0] == 1 and np.isclose(base[-1], plain[-1] / 8)
