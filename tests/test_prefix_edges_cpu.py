"""Workspaces of the attention over a shared prefix, without a GPU: what is enough for the largest pass is enough for all."""
import ctypes as C
import math
import random

import pytest

import ctorch_b200 as B

HERE = 0x1000   # an address that is never followed


def need(rows, sequences, max_count, groups, max_length, max_prefix, heads, kv_heads, dim, dtype=B.BF16, page=64, at=HERE):
    def pages():
        return B.KvPages(dtype=dtype, kv_heads=kv_heads, head_dim=dim, page_size=page, sequences=4, pages_per_sequence=8, pages=32, key=at, value=at, table=HERE)
    a = B.PrefixArgs(heads=heads, scale=0.1, query=at, cache=pages(), prefix=pages(), groups=groups, group_first=HERE, group_prefix=HERE, prefix_length=HERE)
    of = B.Rows(rows=rows, sequences=sequences, max_count=max_count, slot=HERE, first=HERE, sequence=HERE, lengths=HERE)
    return B.lib().b200_prefix_scratch_bytes(C.byref(a), C.byref(of), max_length, max_prefix)


def test_fewer_rows_need_no_more():
    sizes = [need(n, n, 1, 1, 512, 8192, 32, 8, 128) for n in range(1, 300)]
    assert sizes[0] > 0 and sizes == sorted(sizes)


@pytest.mark.parametrize("seed", range(4))
def test_the_largest_pass_and_bounds_are_enough(seed):
    """A pass of fewer rows, however they are shared out, behind shorter bounds, with or without groups and at other addresses, needs no more."""
    r = random.Random(seed)

    def log(low, high):
        return int(round(math.exp(r.uniform(math.log(low), math.log(high)))))
    for _ in range(400):
        kv_heads, group, dim = r.choice([1, 2, 8]), r.choice([1, 4, 5, 16]), r.choice([33, 64, 80, 128, 256])
        dtype = r.choice([B.BF16, B.F32])
        rows, length, prefix = log(1, 40000), log(1, 131072), log(1, 131072)

        def of(rows, length, prefix, groups, at):
            sequences = log(1, rows)
            return need(rows, sequences, r.randint(-(-rows // sequences), rows - sequences + 1), groups, length, prefix, kv_heads * group, kv_heads, dim, dtype, r.choice([7, 16, 64]), at)
        largest = of(rows, length, prefix, r.randint(1, 4), HERE)
        for _ in range(5):
            assert 0 < of(log(1, rows), log(1, length), r.choice([0, log(1, prefix)]), r.randint(0, 4), HERE + r.choice([0, 4])) <= largest


def test_the_workspace_is_bounded():
    """2^19 partial results of head_dim + 2 values, however many rows a pass has."""
    for rows in (1000, 16384, 1 << 20):
        assert need(rows, 16, rows - 15, 1, 1 << 17, 1 << 17, 32, 8, 128) <= 4 * (1 << 19) * 130 + 1024
