"""Scores at the ends of their range in attention_packed and attention_prefix:
NaN and infinities in visible keys, scores whose rounded products with
scale log2 e are far from 0, and small probabilities of long flat tails."""
import pytest
import torch

from attention_util import check, half_step, packed, prefix, starts
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


def mean_bound(y, size, n, dtype):
    """Error of a mean over n values of which `size` is the largest magnitude,
    from probabilities that differ by exactly known factors: each is rounded to
    the element type (u), taken by an exponential of at most 2.7e-6, summed in
    f32 (n 2^-24, twice), and the result is rounded (u |y|)."""
    u = half_step(dtype)
    return (u + 2 * 2.7e-6 + 2 * (n + 16) * 2.0 ** -24) * size + u * (1 + u) * y.abs() + u * u * size


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


# ---- large scores ------------------------------------------------------------------

SIZES = [(F16, 64), (F16, 300), (F16, 725), (F16, 1100), (F16, 5736), (F16, 12128), (F16, 60000),
         (BF16, 2.0 ** 11), (BF16, 2.0 ** 30), (BF16, 1.5 * 2.0 ** 58)]


def large_inputs(g, nq, nk, kv, d, dtype, size):
    """Queries and keys of one value each in all elements: every third key points the other way."""
    q = torch.full((nq, 2 * kv, d), size, device="cuda", dtype=dtype)
    k = torch.full((nk, kv, d), size, device="cuda", dtype=dtype)
    away = torch.arange(nk, device="cuda") % 3 == 1
    k[away] *= -1
    return q, k, normal(g, nk, kv, d, dtype=dtype), away


def means(q, v, away, nq, nk, causal):
    """The mean of the values seen that have the largest score, for each query."""
    seen = torch.arange(nk, device="cuda")[None] <= torch.arange(nq, device="cuda")[:, None] + nk - nq if causal \
        else torch.ones(nq, nk, dtype=torch.bool, device="cuda")
    near = seen & ~away
    near = torch.where(near.any(-1, keepdim=True), near, seen)
    w = near.double() / near.sum(-1, keepdim=True)
    y = torch.einsum("qk,kcd->qcd", w, v.double())
    return y.repeat_interleave(q.shape[1] // v.shape[1], 1)


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("nq,nk,causal", [(300, 300, True), (90, 300, False), (300, 700, False), (1, 5000, True)])
def test_packed_large_scores(cuda, nq, nk, causal, dtype, size):
    q, k, v, away = large_inputs(gen(4), nq, nk, 1, 128, dtype, size)
    want = means(q, v, away, nq, nk, causal)
    bound = mean_bound(want, v.abs().max().double(), nk, dtype)
    for workspace in (None, torch.empty(0, device="cuda")):
        y = torch.empty_like(q)
        api.attention_packed(q, k, v, y, starts([nq], "cuda"), starts([nk], "cuda"), 128 ** -0.5, causal=causal,
                             workspace=workspace)
        check(y, want, bound)


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("batch", [2, 40])
def test_prefix_large_scores(cuda, batch, dtype, size):
    g = gen(5)
    length, own, kv, d = 500, 300, 1, 128
    q, k, v, away = large_inputs(g, batch, length + own, kv, d, dtype, size)
    kp = k[length:, None].transpose(0, 1).repeat(batch, 1, 1, 1)
    vp = v[length:, None].transpose(0, 1).repeat(batch, 1, 1, 1)
    y = torch.empty_like(q[:, None])
    api.attention_prefix(q[:, None], k[:length], v[:length], kp, vp, y, ints([own] * batch), 128 ** -0.5)
    want = means(q, v, away, 1, length + own, True)[:1].expand(batch, -1, -1)
    check(y[:, 0], want, mean_bound(want, v.abs().max().double(), length + own, dtype))


@pytest.mark.parametrize("dtype,base", [(F16, 0), (F16, 256), (F16, 1024), (F16, 1700), (F16, 1920), (BF16, 1024),
                                        (BF16, 1920)])
@pytest.mark.parametrize("nq,nk", [(300, 700), (90, 400), (1, 5000)])
def test_packed_small_differences_of_large_scores(cuda, nq, nk, dtype, base):
    """Scores base^2 + t, exact in f32: the weights are e^t whatever the base, across tiles,
    streams and joined chunks."""
    g = gen(6)
    d = 64
    q = torch.zeros(nq, 2, d, device="cuda", dtype=dtype)
    k = torch.zeros(nk, 1, d, device="cuda", dtype=dtype)
    q[:, :, 0], k[:, :, 0] = base, base
    q[:, :, 1] = 1
    t = torch.randint(-8, 4, (nk,), generator=g, device="cuda").double() / 2 + torch.arange(nk, device="cuda") // 100 % 3
    k[:, 0, 1] = t.to(dtype)
    v = normal(g, nk, 1, d, dtype=dtype)
    p = torch.softmax(t, 0)
    want = torch.einsum("k,kcd->cd", p, v.double()).expand(nq, 2, d)
    weight = torch.einsum("k,kcd->cd", p, v.double().abs()).expand(nq, 2, d)
    # u for each probability; the exponent's product is rounded once, |t - max| 2^-23 at most
    # beside the exponential's 2.7e-6; the f32 sums; log-sums of chunks of up to 2^14 keys,
    # 15 2^-23 in the exponent; the result's rounding
    u = half_step(dtype)
    e = 2 * (2.7e-6 + 16 * 2.0 ** -23 + 15 * 2.0 ** -23) + 4 * (nk + 16) * 2.0 ** -24
    bound = (u + e) * (1 + u) * weight + u * want.abs() + e * weight
    for workspace in (None, torch.empty(0, device="cuda")):
        y = torch.empty_like(q)
        api.attention_packed(q, k, v, y, starts([nq], "cuda"), starts([nk], "cuda"), 1.0, causal=False,
                             workspace=workspace)
        check(y, want, bound)


# ---- small probabilities ---------------------------------------------------------------

@pytest.mark.parametrize("gap", [14.0, 17.5, 19.0])
@pytest.mark.parametrize("nq", [1, 300])
def test_packed_flat_tail(cuda, nq, gap):
    """One key far above 2^18 equal others: each of those has a probability at the
    lower end of f16 (e^-17.5 = 2^-25.2), all together a visible share."""
    n, d = 2 ** 18, 16
    q = torch.zeros(nq, 1, d, device="cuda", dtype=F16)
    k = torch.zeros(n, 1, d, device="cuda", dtype=F16)
    v = torch.ones(n, 1, d, device="cuda", dtype=F16)
    q[:, :, 0] = 1
    k[77, 0, 0] = gap
    v[77] = 0
    y = torch.empty_like(q)
    api.attention_packed(q, k, v, y, starts([nq], "cuda"), starts([n], "cuda"), 1.0, causal=False,
                         workspace=torch.empty(0, device="cuda"))
    tail = (n - 1) * torch.exp(torch.tensor(-gap, dtype=torch.float64, device="cuda"))
    want = (tail / (1 + tail)).expand(y.shape)
    # Probabilities are held 2^7 above their value against the largest: a step of 2^-24
    # there is 2^-31, half of it an error; u where they are normal. The f32 sums: the
    # tile's sum joins a running one each 128 keys, 2^-24 a join and 128 2^-24 within;
    # the product with V adds 16 keys at a time, at most 2^-23 an addition if truncated.
    u = half_step(F16)
    sums = (n / 128 + 128) * 2.0 ** -24 + n / 16 * 2.0 ** -23
    check(y, want, n * 2.0 ** -32 + (2 * u + 2.7e-6 + sums) * want)


# ---- large values -------------------------------------------------------------------------

@pytest.mark.parametrize("size", [2.0 ** 118, 3.3895313892515355e38])
@pytest.mark.parametrize("nq,nk,causal", [(300, 300, True), (90, 300, False), (1, 5000, True)])
def test_packed_values_near_the_largest(cuda, nq, nk, causal, size):
    """Sums of such values leave the f32 range; their weighted mean does not."""
    g = gen(7)
    q, k = normal(g, nq, 2, 64), normal(g, nk, 1, 64)
    v = torch.full((nk, 1, 64), size, device="cuda", dtype=BF16)
    v[:, :, 1] = -size
    v[:, 0, 2] *= torch.where(torch.arange(nk, device="cuda") % 3 == 1, -1, 1)
    want, bound = packed(q, k, v, [nq], [nk], 0.125, causal)
    for workspace in (None, torch.empty(0, device="cuda")):
        y = torch.empty_like(q)
        api.attention_packed(q, k, v, y, starts([nq], "cuda"), starts([nk], "cuda"), 0.125, causal=causal,
                             workspace=workspace)
        check(y, want, bound)


@pytest.mark.parametrize("batch,steps", [(2, 1), (40, 1), (3, 9)])
def test_prefix_values_near_the_largest(cuda, batch, steps):
    g = gen(8)
    q, pk, kp = normal(g, batch, steps, 4, 64), normal(g, 600, 2, 64), normal(g, batch, 300, 2, 64)
    top = torch.finfo(BF16).max
    pv, vp = torch.full_like(pk, top), torch.full_like(kp, top)
    vp[1::2] = -top
    lens = [300 - 7 * b for b in range(batch)]
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, ints(lens), 0.125)
    check(y, *prefix(q, pk, pv, kp, vp, lens, 0.125))
