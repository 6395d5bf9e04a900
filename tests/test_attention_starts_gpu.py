"""attention_packed where the starts of its sequences fall, and with very many
empty sequences."""
import pytest
import torch

import mlk2_b200 as mb
from attention_util import check, packed, starts
from mlk2_b200 import api

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("again,heads", [(1, 1), (1, 4), (9, 1), (40, 2)])
def test_starts_that_fall_over_long_sequences(cuda, again, heads, causal):
    """The first 2000 rows claimed many times over, more work than the rows could hold:
    the sequences behind them are computed all the same."""
    g = gen(1)
    n, last = 2000, [5, 1, 40]
    rows = n + sum(last)
    q, k, v = normal(g, rows, heads, 64), normal(g, rows, 1, 64), normal(g, rows, 1, 64)
    s = [0, n] * (again + 1)
    for m in last:
        s.append(s[-1] + m)
    y = torch.full_like(q, 5)
    assert api.take_device_error() == 0
    api.attention_packed(q, k, v, y, ints(s), ints(s), 0.125, causal=causal)
    assert api.take_device_error() == mb.ERR_INVALID
    want, bound = packed(q, k, v, [n, *last], [n, *last], 0.125, causal)
    # every claim of the first rows is the same sequence
    check(y, want, bound)


@pytest.mark.parametrize("again", [3, 30])
def test_starts_that_fall_over_cut_keys(cuda, again):
    """The same with few queries over many keys, which are cut and joined."""
    g = gen(2)
    nq, nk, last = 300, 4000, [2, 1]
    q, k, v = normal(g, nq + 3, 1, 64), normal(g, nk + 300, 1, 64), normal(g, nk + 300, 1, 64)
    qs, ks = [0, nq] * (again + 1) + [nq + 2, nq + 3], [0, nk] * (again + 1) + [nk + 250, nk + 300]
    assert api.attention_packed_workspace(q, k, ints(qs)) > 0
    need = api.attention_packed_workspace(q, k, ints(qs))
    y = torch.full_like(q, 5)
    api.attention_packed(q, k, v, y, ints(qs), ints(ks), 0.125,
                         workspace=torch.full((need // 4,), torch.nan, device="cuda"))
    assert api.take_device_error() == mb.ERR_INVALID
    check(y, *packed(q, k, v, [nq, *last], [nk, 250, 50], 0.125))


@pytest.mark.parametrize("rows,heads,kv,seqs", [(1, 8, 1, 3000), (7, 3, 3, 700), (5, 8, 8, 40), (4, 1, 1, 1500),
                                                (3, 8, 2, 50000)])
def test_few_rows_among_empty_sequences(cuda, rows, heads, kv, seqs):
    """Single tokens over many keys (cut where the sequences are not too many), each a
    sequence among empty ones; rows of none are left."""
    g = gen(3)
    keys, pad = 4000, 9
    q = normal(g, rows + pad, heads, 64, dtype=F16)
    k, v = normal(g, keys, kv, 64, dtype=F16), normal(g, keys, kv, 64, dtype=F16)
    nq, nk = torch.zeros(seqs, dtype=torch.int64), torch.zeros(seqs, dtype=torch.int64)
    at = [1 + i * (seqs - 2) // rows for i in range(rows)]
    lengths = [1 + (keys - rows) * (i + 1) // (rows * (rows + 1) // 2) for i in range(rows)]
    for i, n in zip(at, lengths):
        nq[i], nk[i] = 1, n
    qs, ks = starts(nq.tolist(), "cuda"), starts(nk.tolist(), "cuda")
    y = torch.full_like(q, 5)
    api.attention_packed(q, k, v, y, qs, ks, 0.125)
    check(y[:rows], *packed(q[:rows], k, v, [1] * rows, lengths, 0.125))
    assert (y[rows:] == 5).all() and api.take_device_error() == 0


@pytest.mark.parametrize("rows,heads,extra", [(2000, 2, 0), (300, 1, 4000)])  # whole; cut and joined
@pytest.mark.parametrize("again", [1, 20, 500])
def test_rows_belong_to_the_first_sequence_that_claims_them(cuda, again, rows, heads, extra):
    """Sequences that begin below an earlier start are refused, in the same 32 and far behind."""
    g = gen(4)
    keys = rows + extra
    q = normal(g, rows + 20, heads, 64)
    k, v = normal(g, 2 * keys + 20, 1, 64), normal(g, 2 * keys + 20, 1, 64)
    qs, ks = [0, rows], [0, keys]
    for i in range(again):  # the same rows, all or a part, with other keys
        qs += [i % 7 * 10, rows - i % 3]
        ks += [keys, 2 * keys]
    qs += [rows + 3, rows + 10, rows + 10, rows + 13]
    ks += [2 * keys, 2 * keys + 7, 2 * keys + 7, 2 * keys + 10]
    y = torch.full_like(q, 5)
    assert api.take_device_error() == 0
    api.attention_packed(q, k, v, y, ints(qs), ints(ks), 0.125)
    assert api.take_device_error() == mb.ERR_INVALID
    check(y[:rows], *packed(q[:rows], k, v, [rows], [keys], 0.125))
    # once, the sequence behind it begins on the highest start (and has no keys), else one below
    assert (y[rows:rows + 3] == (0 if again == 1 else 5)).all()
    check(y[rows + 3:rows + 10], *packed(q[rows + 3:rows + 10], k[2 * keys:], v[2 * keys:], [7], [7], 0.125))
    check(y[rows + 10:rows + 13], *packed(q[rows + 10:rows + 13], k[2 * keys + 7:], v[2 * keys + 7:], [3], [3], 0.125))
    assert (y[rows + 13:] == 5).all()


def test_captured_call_with_cut_keys_follows_the_starts(cuda):
    """One graph, replayed with other sequences, with none, and with refused ones."""
    g = gen(5)
    q, k, v = normal(g, 6, 8, 64), normal(g, 6000, 2, 64), normal(g, 6000, 2, 64)
    qs, ks = ints([0, 1, 2, 6]), ints([0, 2000, 2500, 6000])
    assert api.attention_packed_workspace(q, k, qs) > 0
    y = torch.zeros_like(q)
    api.attention_packed(q, k, v, y, qs, ks, 0.125)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        api.attention_packed(q, k, v, y, qs, ks, 0.125)
    for nq, nk in (([1, 1, 4], [2000, 500, 3500]), ([0, 0, 1], [0, 0, 6000]), ([6, 0, 0], [1, 0, 5]),
                   ([0, 0, 0], [0, 0, 0]), ([2, 2, 2], [6000, 0, 0])):
        qs.copy_(starts(nq, "cuda"))
        ks.copy_(starts(nk, "cuda"))
        y.fill_(5)
        graph.replay()
        n = sum(nq)
        check(y[:n], *packed(q[:n], k, v, nq, nk, 0.125))
        assert (y[n:] == 5).all() and api.take_device_error() == 0
    qs.copy_(ints([0, 4, 2, 6]))
    ks.copy_(ints([0, 3000, 3000, 6000]))
    y.fill_(5)
    graph.replay()
    check(y[:4], *packed(q[:4], k, v, [4], [3000], 0.125))
    assert (y[4:] == 5).all() and api.take_device_error() == mb.ERR_INVALID
