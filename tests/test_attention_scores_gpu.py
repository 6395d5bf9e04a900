"""Scores at the ends of their range in attention_packed and attention_prefix:
NaN and infinities in visible keys."""
import pytest
import torch

from attention_util import check, packed, prefix, starts
from mlk2_b200 import api

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- NaN and infinities in keys that are seen -------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", [NAN, INF, -INF])
def test_packed_key_of_a_full_tile(cuda, what, dtype):
    """One element of one key, at each place of 16 in a tile that every row sees whole; V stays finite."""
    g = gen(1)
    nq, nk, d = 300, 384, 64
    q, k, v = normal(g, nq, 2, d, dtype=dtype), normal(g, nk, 1, d, dtype=dtype), normal(g, nk, 1, d, dtype=dtype)
    q[:, :, 3] = q[:, :, 3].abs() + 0.5
    qs, ks = starts([nq], "cuda"), starts([nk], "cuda")
    for tile in (0, 128):
        for at in range(tile + 32, tile + 48):
            bad = k.clone()
            bad[at, 0, 3] = what
            y = torch.full_like(q, 5)
            api.attention_packed(q, bad, v, y, qs, ks, 0.125, causal=False)
            if what == -INF:  # its score is -inf: the key is not there
                keep = torch.arange(nk, device="cuda") != at
                check(y, *packed(q, k[keep], v[keep], [nq], [nk - 1], 0.125, False))
            else:
                assert y.isnan().all(), (at, int((~y.isnan()).sum()))
    assert api.take_device_error() == 0


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("nq", [1, 40, 200])
def test_packed_key_of_a_causal_prompt(cuda, what, nq):
    """Only the queries from the key on are NaN, in whole tiles and in the one that the mask cuts."""
    g = gen(2)
    nk, d = 1500, 128
    q, k, v = normal(g, nq, 2, d), normal(g, nk, 1, d), normal(g, nk, 1, d)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    for workspace in (None, torch.empty(0, device="cuda")):
        for at in (1, 5, 130, 771, 1026, 1310, 1440, 1499):
            bad = k.clone()
            bad[at, 0, 0] = what
            y = torch.empty_like(q)
            api.attention_packed(q, bad, v, y, starts([nq], "cuda"), starts([nk], "cuda"), 0.1,
                                 workspace=workspace)
            first = max(0, at - (nk - nq))
            clean = k.clone()
            clean[at] = 0
            want, bound = packed(q, clean, v, [nq], [nk], 0.1)
            check(y[:first], want[:first], bound[:first])
            assert y[first:].isnan().all()


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("batch,steps", [(3, 1), (40, 1), (3, 9)])
def test_prefix_key(cuda, what, batch, steps):
    """In the prefix and among a request's own keys, in few (spread) rows and in many."""
    g = gen(3)
    heads, kv, d, size, length = 8, 2, 64, 64, 300
    q = normal(g, batch, steps, heads, d)
    q[..., 0] = q[..., 0].abs() + 0.5
    pk, pv = normal(g, length, kv, d), normal(g, length, kv, d)
    kp, vp = normal(g, batch * 5, size, kv, d), normal(g, batch * 5, size, kv, d)
    pages = torch.randperm(batch * 5, generator=g, device="cuda").view(batch, 5).int()
    lens = [320] + [20 + b for b in range(batch - 1)]
    want, bound = prefix(q, pk, pv, kp, vp, lens, 0.125, pages)
    for at in range(16):
        y = torch.empty_like(q)
        bad = pk.clone()
        bad[128 + at, 1, 0] = what  # of the second kv head
        api.attention_prefix(q, bad, pv, kp, vp, y, ints(lens), 0.125, pages=pages)
        assert y[:, :, 4:].isnan().all()
        check(y[:, :, :4], want[:, :, :4], bound[:, :, :4])
        own = kp.clone()
        own[pages[0, 2], at, 0, 0] = what
        api.attention_prefix(q, pk, pv, own, vp, y, ints(lens), 0.125, pages=pages)
        assert y[0, :, :4].isnan().all()
        check(y[1:], want[1:], bound[1:])
        check(y[:, :, 4:], want[:, :, 4:], bound[:, :, 4:])
    assert api.take_device_error() == 0
