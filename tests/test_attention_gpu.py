"""norm_rope, attention_packed and attention_prefix against plain 64-bit
implementations, at the sizes and masks where they can go wrong."""
import random

import pytest
import torch

import mlk2_b200 as mb
from attention_util import check, norm_rope, packed, prefix, starts, table
from mlk2_b200 import api

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- norm_rope -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,heads,kv,d,rot,norm,interleaved", [
    (1, 1, 1, 16, 16, True, False), (3, 5, 1, 64, 64, True, False), (17, 8, 2, 128, 128, True, True),
    (129, 3, 3, 80, 80, True, False), (130, 7, 1, 96, 48, False, True), (5, 4, 2, 256, 64, True, False),
    (2, 3, 2, 512, 256, True, True), (700, 32, 8, 128, 128, True, False), (33, 2, 0, 32, 16, True, False),
    (1000, 16, 4, 48, 32, False, False)])
def test_norm_rope(cuda, dtype, tokens, heads, kv, d, rot, norm, interleaved):
    g = gen(tokens + d)
    q, k = normal(g, tokens, heads, d, dtype=dtype), normal(g, tokens, max(kv, 1), d, dtype=dtype)
    wq, wk = normal(g, d, dtype=dtype), normal(g, d, dtype=dtype)
    t = table(400, rot, "cuda")
    pos = torch.randint(0, 400, (tokens,), generator=g, device="cuda").int()
    qo, ko = torch.full_like(q, 9), torch.full_like(k, 9)
    api.norm_rope(q, k if kv else None, qo, ko if kv else None, t, pos, q_weight=wq if norm else None,
                  k_weight=wk if norm else None, eps=1e-5, interleaved=interleaved)
    check(qo, *norm_rope(q, wq if norm else None, 1e-5, t, pos, None, interleaved))
    if kv:
        check(ko, *norm_rope(k, wk if norm else None, 1e-5, t, pos, None, interleaved))
    assert api.take_device_error() == 0


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [[16, 24, 24], [1, 0, 63], [5, 59], [7, 9, 11, 37]])
def test_norm_rope_axes(cuda, sections, interleaved):
    g = gen(len(sections))
    q, k = normal(g, 77, 6, 128), normal(g, 77, 2, 128)
    w = normal(g, 128)
    t = table(50, 128, "cuda")
    pos = torch.randint(0, 50, (len(sections), 77), generator=g, device="cuda").int()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    api.norm_rope(q, k, qo, ko, t, pos, sections=sections, q_weight=w, k_weight=w,
                  interleaved=interleaved)
    for x, y in ((q, qo), (k, ko)):
        check(y, *norm_rope(x, w, 1e-6, t, pos, sections, interleaved))


def test_norm_rope_in_place_on_a_projection(cuda):
    """q and k as slices of one [tokens, (q + k + v) heads, d] buffer, turned where they lie; v stays."""
    g = gen(4)
    qkv = normal(g, 219, 14, 96)
    before = qkv.clone()
    w, t = normal(g, 96), table(300, 96, "cuda")
    pos = torch.arange(219, device="cuda", dtype=torch.int32)
    q, k = qkv[:, :8], qkv[:, 8:11]
    api.norm_rope(q, k, q, k, t, pos, q_weight=w, k_weight=w)
    check(q, *norm_rope(before[:, :8], w, 1e-6, t, pos, None, False))
    check(k, *norm_rope(before[:, 8:11], w, 1e-6, t, pos, None, False))
    assert torch.equal(qkv[:, 11:], before[:, 11:])


def test_norm_rope_head_major(cuda):
    g = gen(5)
    q, k = normal(g, 8, 45, 64).transpose(0, 1), normal(g, 2, 45, 64).transpose(0, 1)
    w, t = normal(g, 64), table(64, 64, "cuda")
    pos = torch.arange(45, device="cuda", dtype=torch.int32)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    api.norm_rope(q, k, qo, ko, t, pos, q_weight=w, k_weight=w)
    check(qo, *norm_rope(q, w, 1e-6, t, pos, None, False))
    check(ko, *norm_rope(k, w, 1e-6, t, pos, None, False))


def test_norm_rope_extremes(cuda):
    """Rows of the largest and smallest values, of zeros, and with an infinity or a NaN."""
    big = torch.finfo(BF16).max
    q = torch.ones(6, 1, 64, device="cuda", dtype=BF16)
    q[0] *= big
    q[1] *= 1e-30
    q[2] = 0
    q[3, 0, 5] = torch.inf
    q[4, 0, 7] = torch.nan
    q[5] *= 3e19                      # squares past the f32 range
    q[5, 0, 0] = -1e20
    w, t = torch.ones(64, device="cuda", dtype=BF16), table(8, 64, "cuda")
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    y = torch.empty_like(q)
    api.norm_rope(q, None, y, None, t, pos, q_weight=w)
    want, bound = norm_rope(q, w, 1e-6, t, pos, None, False)
    for r in (0, 1, 2, 5):
        check(y[r], want[r], bound[r])
    assert y[4].isnan().all()
    assert torch.equal(y[3].isnan(), want[3].isnan())


def test_norm_rope_positions_outside_the_table(cuda):
    g = gen(6)
    q, t = normal(g, 5, 2, 64), table(10, 64, "cuda")
    y = torch.full_like(q, 7)
    pos = ints([0, -1, 9, 10, 3])
    assert api.take_device_error() == 0
    api.norm_rope(q, None, y, None, t, pos)
    assert api.take_device_error() == mb.ERR_INVALID
    want, bound = norm_rope(q[[0, 2, 4]], None, 0, t, pos[[0, 2, 4]], None, False)
    check(y[[0, 2, 4]], want, bound)
    assert (y[[1, 3]] == 7).all()
    y.fill_(7)
    api.norm_rope(q, None, y, None, t, torch.stack([pos, pos * 0]), sections=[32, 0])
    assert api.take_device_error() == mb.ERR_INVALID
    assert (y[[1, 3]] == 7).all() and (y[0] != 7).any()


# ---- attention_packed --------------------------------------------------------------

def run_packed(nq, nk, heads, kv, d, dtype=BF16, causal=True, seed=0, pad=3):
    g = gen(seed)
    q = normal(g, sum(nq) + pad, heads, d, dtype=dtype)
    k, v = normal(g, sum(nk), kv, d, dtype=dtype), normal(g, sum(nk), kv, d, dtype=dtype)
    y = torch.full_like(q, 5)
    api.attention_packed(q, k, v, y, starts(nq, "cuda"), starts(nk, "cuda"), d ** -0.5, causal=causal)
    n = sum(nq)
    want, bound = packed(q[:n], k, v, nq, nk, d ** -0.5, causal)
    check(y[:n], want, bound)
    assert (y[n:] == 5).all()
    assert api.take_device_error() == 0


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400, 1023])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_lengths(cuda, n, causal):
    run_packed([n], [n], 4, 2, 128, causal=causal, seed=n)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,d", [
    (1, 1, 8), (2, 1, 64), (3, 1, 72), (5, 1, 80), (6, 2, 96), (7, 1, 128), (8, 8, 120), (24, 3, 64),
    (16, 2, 56), (128, 1, 128), (70, 1, 64), (40, 2, 40)])
def test_packed_heads(cuda, heads, kv, d, dtype):
    run_packed([150, 9], [150, 9], heads, kv, d, dtype=dtype, seed=d)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [
    ([0, 5, 0], [0, 5, 3]), ([7, 1, 200], [0, 300, 200]), ([1], [1000]), ([1, 1, 1], [129, 1, 640]),
    ([200], [30]), ([300], [1]), ([130, 60], [900, 61]), ([0], [4]), ([33, 400, 2], [513, 400, 2])])
def test_packed_uneven(cuda, nq, nk, causal):
    """Pieces of prompts, single tokens, queries that see nothing, empty sequences."""
    run_packed(nq, nk, 8, 2, 64, causal=causal, seed=len(nq))
    run_packed(nq, nk, 3, 3, 128, dtype=F16, causal=causal, seed=len(nq))


def test_packed_many_sequences(cuda):
    r = random.Random(3)
    nq = [r.choice([0, 1, 2, 5, 17, 40, 130]) for _ in range(150)]
    nk = [n + r.choice([0, 0, 3, 200]) for n in nq]
    run_packed(nq, nk, 4, 2, 64, seed=9)
    run_packed(nq, nk, 4, 2, 64, seed=9, causal=False)


def test_packed_long(cuda):
    run_packed([2500, 1], [2500, 4100], 4, 2, 128, seed=11)


@pytest.mark.parametrize("nq,nk,heads,kv,d,causal", [
    ([1], [5000], 8, 1, 128, True), ([1, 1, 0, 3], [2000, 130, 700, 3], 4, 4, 64, True),
    ([40, 7], [1500, 2200], 16, 2, 80, True), ([40, 7], [1500, 2200], 16, 2, 80, False),
    ([100, 2], [60, 1700], 2, 1, 128, True), ([300], [1400], 4, 1, 96, True),
    ([2, 2], [9000, 3], 3, 1, 72, True), ([1], [33000], 4, 1, 64, True)])
def test_packed_few_queries_over_many_keys(cuda, nq, nk, heads, kv, d, causal):
    """Cut along the keys and joined; without a workspace the same values uncut."""
    g = gen(18)
    q = normal(g, sum(nq) + 5, heads, d)
    k, v = normal(g, sum(nk), kv, d), normal(g, sum(nk), kv, d)
    qs, ks = starts(nq, "cuda"), starts(nk, "cuda")
    assert api.attention_packed_workspace(q, k, qs) > 0
    n = sum(nq)
    want, bound = packed(q[:n], k, v, nq, nk, d ** -0.5, causal)
    for workspace in (None, torch.empty(0, device="cuda")):
        y = torch.full_like(q, 5)
        api.attention_packed(q, k, v, y, qs, ks, d ** -0.5, causal=causal, workspace=workspace)
        check(y[:n], want, bound)
        assert (y[n:] == 5).all()
    need = api.attention_packed_workspace(q, k, qs)
    y = torch.full_like(q, 5)
    api.attention_packed(q, k, v, y, qs, ks, d ** -0.5, causal=causal,
                         workspace=torch.full((need // 4,), torch.nan, device="cuda"))
    check(y[:n], want, bound)
    assert (y[n:] == 5).all()


def test_packed_cut_keys_with_nan(cuda):
    """A NaN value among cut keys reaches the queries that see it, and a bad sequence stays out."""
    g = gen(19)
    q, k, v = normal(g, 8, 4, 64), normal(g, 3000, 2, 64), normal(g, 3000, 2, 64)
    v[2997] = torch.nan  # seen by the last three queries of sequence 1
    y = torch.full_like(q, 5)
    qs, ks = ints([0, 3, 7, 20]), ints([0, 1400, 3000, 3000])
    api.attention_packed(q, k, v, y, qs, ks, 0.125)
    assert api.take_device_error() == mb.ERR_INVALID
    clean = v.clone()
    clean[2997] = 0
    want, bound = packed(q[:7], k, clean, [3, 4], [1400, 1600], 0.125)
    check(y[:4], want[:4], bound[:4])
    assert y[4:7].isnan().all() and (y[7] == 5).all()


def test_packed_growing_scores(cuda):
    """Row maxima that rise by far more than 2^8 from tile to tile, and fall again."""
    g = gen(12)
    q, k, v = normal(g, 700, 2, 64), normal(g, 700, 1, 64), normal(g, 700, 1, 64)
    q = q.abs()
    ramp = torch.cat([torch.linspace(-3, 3, 400), torch.linspace(2, -3, 300)]).cuda()
    k = (k.float() * 0.1 + ramp[:, None, None]).to(BF16)
    y = torch.empty_like(q)
    s = starts([700], "cuda")
    for causal in (True, False):
        api.attention_packed(q, k, v, y, s, s, 0.5, causal=causal)
        check(y, *packed(q, k, v, [700], [700], 0.5, causal))


def test_packed_strided(cuda):
    """q, k and v in one projection's output; q, y stored head by head."""
    g = gen(13)
    qkv = normal(g, 333, 12, 80)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    y = torch.empty(8, 333, 80, device="cuda", dtype=BF16).transpose(0, 1)
    s = starts([300, 33], "cuda")
    want, bound = packed(q, k, v, [300, 33], [300, 33], 0.2)
    api.attention_packed(q, k, v, y, s, s, 0.2)
    check(y, want, bound)
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
    k2 = k.transpose(0, 1).contiguous().transpose(0, 1)
    y2 = torch.empty_like(q)
    api.attention_packed(q2, k2, v, y2, s, s, 0.2)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_packed_masked_values_have_no_effect(cuda, what):
    """Keys and values that a query may not see hold a NaN, an infinity or the lowest number."""
    g = gen(14)
    nq = [100, 230]
    q, k, v = normal(g, 330, 4, 128), normal(g, 345, 2, 128), normal(g, 345, 2, 128)
    what = torch.finfo(BF16).min if what == "lowest" else what
    k[330:] = what  # behind the last sequence
    v[330:] = what
    k[320:330], v[320:330] = what, what  # the last ten of sequence 1: seen by its last ten only
    k[95:100], v[95:100] = what, what    # and the last five of sequence 0
    y = torch.empty_like(q)
    api.attention_packed(q, k, v, y, starts(nq, "cuda"), starts(nq, "cuda"), 0.1)
    clean_k, clean_v = k.clone(), v.clone()
    for c in (clean_k, clean_v):
        c[320:], c[95:100] = 0, 0
    want, bound = packed(q, clean_k, clean_v, nq, nq, 0.1)
    for a, b in ((0, 95), (100, 320)):
        check(y[a:b], want[a:b], bound[a:b])
    if what != what:
        assert y[95:100].isnan().all() and y[320:330].isnan().all()


def test_packed_nan_query_stays_in_its_row(cuda):
    g = gen(15)
    q, k, v = normal(g, 140, 4, 64), normal(g, 140, 2, 64), normal(g, 140, 2, 64)
    q[17, 1] = torch.nan
    y = torch.empty_like(q)
    s = starts([140], "cuda")
    api.attention_packed(q, k, v, y, s, s, 0.125)
    assert y[17, 1].isnan().all()
    q[17, 1] = 0
    y[17, 1] = 0
    want, bound = packed(q, k, v, [140], [140], 0.125)
    want[17, 1] = 0
    check(y, want, bound)


def test_packed_scores_of_minus_infinity(cuda):
    """Visible keys whose score is -inf add nothing; a row with no others is zeros."""
    q = torch.ones(4, 1, 64, device="cuda", dtype=BF16)
    k = torch.ones(4, 1, 64, device="cuda", dtype=BF16)
    v = torch.arange(1, 5, device="cuda", dtype=BF16)[:, None, None].expand(4, 1, 64).contiguous()
    k[:2] = -torch.inf
    y = torch.empty_like(q)
    s = starts([4], "cuda")
    api.attention_packed(q, k, v, y, s, s, 0.1)
    assert (y[:2] == 0).all() and (y[2] == 3).all() and (y[3] == 3.5).all()


def test_packed_bad_starts(cuda):
    """A sequence whose starts fall or leave the operands is skipped; the others are computed."""
    g = gen(16)
    q, k, v = normal(g, 50, 2, 64), normal(g, 50, 2, 64), normal(g, 50, 2, 64)
    want, bound = packed(q[:40], k[:40], v[:40], [20, 20], [20, 20], 0.125)
    for qs, ks, good in (([0, 20, -1, 20, 40, 51], [0, 20, 20, 20, 40, 50], ((0, 20), (20, 40))),
                         ([0, 20, 20, 40, 50], [0, 20, 20, 51, 50], ((0, 20),)),
                         ([2 ** 31 - 1, 20, 20, 40], [-2 ** 31, 2 ** 31 - 1, 20, 40], ((20, 40),))):
        y = torch.full_like(q, 5)
        assert api.take_device_error() == 0
        api.attention_packed(q, k, v, y, ints(qs), ints(ks), 0.125)
        assert api.take_device_error() == mb.ERR_INVALID
        left = torch.ones(50, dtype=torch.bool)
        for m, n in good:
            check(y[m:n], want[m:n], bound[m:n])
            left[m:n] = False
        assert (y[left.cuda()] == 5).all()


def test_packed_largest_rows_address(cuda):
    """Keys more than 2^31 elements into their buffer."""
    rows, d = 2 ** 21 + 500, 128
    g = gen(17)
    k = torch.zeros(rows, 8, d, device="cuda", dtype=F16)
    v = torch.zeros(rows, 8, d, device="cuda", dtype=F16)
    at = rows - 300
    k[at:], v[at:] = normal(g, 300, 8, d, dtype=F16), normal(g, 300, 8, d, dtype=F16)
    q = normal(g, 30, 16, d, dtype=F16)
    y = torch.empty_like(q)
    api.attention_packed(q, k, v, y, ints([0, 30]), ints([at, rows]), 0.1)
    check(y, *packed(q, k[at:], v[at:], [30], [300], 0.1))


# ---- attention_prefix ----------------------------------------------------------------

def make_prefix(batch, steps, length, lens, heads, kv, d, page, dtype=BF16, seed=0, spare=2):
    g = gen(seed)
    cap = max(max(lens), 1)
    size = page or cap
    wide = -(-cap // size)
    n = batch * wide + (spare if page else 0)
    q = normal(g, batch, steps, heads, d, dtype=dtype)
    pk, pv = normal(g, length, kv, d, dtype=dtype), normal(g, length, kv, d, dtype=dtype)
    kp, vp = normal(g, n, size, kv, d, dtype=dtype), normal(g, n, size, kv, d, dtype=dtype)
    pages = torch.randperm(n, generator=g, device="cuda")[:batch * wide].view(batch, wide).int() \
        if page else None
    return q, pk, pv, kp, vp, ints(lens), pages


def run_prefix(*args, **kw):
    q, pk, pv, kp, vp, lens, pages = make_prefix(*args, **kw)
    y = torch.full_like(q, 5)
    scale = q.shape[-1] ** -0.5
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, scale, pages=pages)
    check(y, *prefix(q, pk, pv, kp, vp, lens.tolist(), scale, pages))
    assert api.take_device_error() == 0


@pytest.mark.parametrize("page", [0, 16, 64, 128, 256])
@pytest.mark.parametrize("length", [0, 1, 127, 128, 129, 700])
def test_prefix_lengths(cuda, length, page):
    run_prefix(5, 1, length, [1, 300, 17, 128, 129], 8, 2, 128, page, seed=length)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,d,batch,steps", [
    (1, 1, 8, 1, 1), (3, 1, 72, 2, 1), (8, 1, 64, 40, 1), (5, 5, 80, 3, 4), (16, 2, 96, 9, 5),
    (64, 1, 128, 3, 3), (128, 1, 64, 2, 2), (4, 4, 128, 150, 1), (6, 2, 120, 70, 2)])
def test_prefix_heads(cuda, heads, kv, d, batch, steps, dtype):
    r = random.Random(heads + batch)
    run_prefix(batch, steps, 333, [r.randint(0, 180) for _ in range(batch)], heads, kv, d, 32,
               dtype=dtype, seed=batch)


def test_prefix_empty_requests(cuda):
    """Requests with no keys of their own see the prefix alone; without one they get zeros."""
    run_prefix(4, 2, 50, [0, 1, 2, 9], 4, 2, 64, 16)
    run_prefix(4, 2, 0, [0, 1, 2, 9], 4, 2, 64, 16)
    run_prefix(2, 1, 40, [0, 0], 4, 2, 64, 0)


def test_prefix_long(cuda):
    run_prefix(3, 1, 9000, [4000, 5, 2300], 8, 2, 128, 64, seed=1)
    run_prefix(2, 1, 100, [9001, 130], 8, 1, 64, 0, seed=2)


def test_prefix_unused_pages_are_not_read(cuda):
    """Table entries behind the last key hold anything, and so do the pages' rows there."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(3, 1, 200, [70, 200, 1], 8, 2, 128, 64, seed=3)
    want, bound = prefix(q, pk, pv, kp, vp, lens.tolist(), 0.1, pages)
    for b, n in enumerate(lens.tolist()):
        last = n // 64
        kp[pages[b, last], n % 64:] = torch.nan
        vp[pages[b, last], n % 64:] = torch.inf
        pages[b, last + 1:] = 2 ** 31 - 1
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.1, pages=pages)
    check(y, want, bound)
    assert api.take_device_error() == 0


def test_prefix_nan_of_a_later_draft(cuda):
    """A drafted token's NaN value is seen by the drafts after it only."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(2, 4, 100, [60, 10], 4, 2, 64, 16, seed=4)
    want, bound = prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125, pages)
    vp[pages[0, 58 // 16], 58 % 16] = torch.nan
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=pages)
    check(y[0, :2], want[0, :2], bound[0, :2])
    assert y[0, 2:].isnan().all()
    check(y[1], want[1], bound[1])


def test_prefix_bad_pages_and_lengths(cuda):
    """A page index outside the pages reads as zeros, a length outside the table as its end."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(3, 1, 64, [40, 20, 48], 4, 2, 64, 16, seed=5)
    y = torch.empty_like(q)
    assert api.take_device_error() == 0
    zero_k, zero_v = (torch.cat([x, torch.zeros_like(x[:1])]) for x in (kp, vp))
    for bad in (-1, kp.shape[0], 2 ** 31 - 1, -2 ** 31):
        p = pages.clone()
        p[1, 0] = bad
        api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=p)
        assert api.take_device_error() == mb.ERR_INVALID
        p[1, 0] = kp.shape[0]
        check(y, *prefix(q, pk, pv, zero_k, zero_v, lens.tolist(), 0.125, p))
    api.attention_prefix(q, pk, pv, kp, vp, y, ints([-3, 10 ** 9, 48]), 0.125, pages=pages)
    assert api.take_device_error() == mb.ERR_INVALID
    check(y, *prefix(q, pk, pv, kp, vp, [0, 48, 48], 0.125, pages))


def test_prefix_given_workspace_and_strides(cuda):
    """A caller's workspace full of NaN; caches that hold k and v side by side."""
    g = gen(6)
    q, pk, pv, kp, vp, lens, pages = make_prefix(6, 2, 300, [30, 2, 100, 64, 65, 7], 8, 2, 64, 32, seed=6)
    want, bound = prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125, pages)
    cache = normal(g, *kp.shape[:2], 4, 64)
    cache[:, :, :2], cache[:, :, 2:] = kp, vp
    need = api.attention_prefix_workspace(q, pk, cache[:, :, :2], pages)
    ws = torch.full((need // 4 + 4,), torch.nan, device="cuda")
    y = torch.full_like(q, 5)
    api.attention_prefix(q, pk, pv, cache[:, :, :2], cache[:, :, 2:], y, lens, 0.125, pages=pages,
                         workspace=ws)
    check(y, want, bound)
    with pytest.raises(mb.MLKBError):
        api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=pages, workspace=ws[:need // 8])


# ---- streams, graphs and a run of them together --------------------------------------------

def test_same_bits_again_and_on_another_stream(cuda):
    q, pk, pv, kp, vp, lens, pages = make_prefix(30, 1, 900, list(range(1, 301, 10)), 8, 2, 128, 16)
    s = starts([400, 30], "cuda")
    x = normal(gen(1), 430, 8, 128)
    outs = []
    for stream in (None, torch.cuda.Stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        y, z = torch.empty_like(q), torch.empty_like(x)
        torch.cuda.synchronize()
        handle = stream.cuda_stream if stream else None
        api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.1, pages=pages, stream=handle)
        api.attention_packed(x, x[:, :2], x[:, 2:4], z, s, s, 0.1, stream=handle)
        torch.cuda.synchronize()
        outs.append((y, z))
    for y, z in outs[1:]:
        assert torch.equal(y, outs[0][0]) and torch.equal(z, outs[0][1])


def test_two_calls_at_once(cuda):
    """Two streams, each with a workspace of its own."""
    ins = [make_prefix(20, 1, 2000, [100] * 20, 8, 2, 64, 0, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [torch.empty_like(i[0]) for i in ins]
    torch.cuda.synchronize()
    for _ in range(5):
        for (q, pk, pv, kp, vp, lens, _), st, y in zip(ins, streams, outs):
            with torch.cuda.stream(st):
                api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125)
    torch.cuda.synchronize()
    for (q, pk, pv, kp, vp, lens, _), y in zip(ins, outs):
        check(y, *prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125))


class Layer:
    """One attention layer of a server: projections given, norms, rotation,
    a paged cache behind a shared prefix."""

    def __init__(self, heads=8, kv=2, d=64, batch=3, page=16, wide=8, dtype=BF16):
        g = gen(20)
        self.h, self.kv, self.d, self.page, self.batch = heads, kv, d, page, batch
        self.w = [normal(g, d, dtype=dtype), normal(g, d, dtype=dtype)]
        self.table = table(1024, d, "cuda")
        self.k = torch.full((batch * wide, page, kv, d), torch.nan, device="cuda", dtype=dtype)
        self.v = torch.full_like(self.k, torch.nan)
        self.pages = torch.randperm(batch * wide, generator=g, device="cuda").view(batch, wide).int()

    def split(self, qkv):
        return qkv[:, :self.h], qkv[:, self.h:self.h + self.kv], qkv[:, self.h + self.kv:]

    def turn(self, qkv, pos):
        q, k, v = self.split(qkv)
        api.norm_rope(q, k, q, k, self.table, pos, q_weight=self.w[0], k_weight=self.w[1])
        return q, k, v

    def store(self, b, at, k, v):
        page, row = self.pages[b, at // self.page].long(), at % self.page
        self.k[page, row], self.v[page, row] = k, v


def test_prompt_then_decoding_steps(cuda):
    """A shared instruction and three prompts in one packed call, then three
    decoding steps over the shared prefix and the pages: the steps give what
    one packed call over the whole sequences gives."""
    L = Layer()
    g = gen(21)
    shared, prompts, steps = 70, [5, 40, 17], 3
    total = [n + steps for n in prompts]
    raw = [normal(g, shared, 12, 64)] + [normal(g, n, 12, 64) for n in total]
    scale = 64 ** -0.5
    # the whole of it: every request as instruction + its own tokens
    whole = torch.cat([torch.cat([raw[0], r]) for r in raw[1:]])
    pos = torch.cat([torch.arange(shared + n) for n in total]).int().cuda()
    q, k, v = L.turn(whole.clone(), pos)
    n = [shared + t for t in total]
    full = torch.empty(q.shape, device="cuda", dtype=BF16)
    api.attention_packed(q, k, v, full, starts(n, "cuda"), starts(n, "cuda"), scale)
    check(full, *packed(q, k, v, n, n, scale))
    # the instruction once
    pq, pk, pv = L.turn(raw[0].clone(), torch.arange(shared).int().cuda())
    # then step by step, from the prompts' ends
    for b, m in enumerate(prompts):
        _, kb, vb = L.turn(raw[1 + b][:m].clone(), torch.arange(shared, shared + m).int().cuda())
        L.store(b, torch.arange(m, device="cuda"), kb, vb)
    for step in range(steps):
        at = torch.tensor([m + step for m in prompts], device="cuda")
        qkv = torch.stack([raw[1 + b][m + step] for b, m in enumerate(prompts)])
        q1, k1, v1 = L.turn(qkv.clone(), (at + shared).int())
        L.store(torch.arange(3, device="cuda"), at, k1, v1)
        y = torch.empty(3, 1, 8, 64, device="cuda", dtype=BF16)
        lens = (at + 1).int()
        api.attention_prefix(q1[:, None], pk, pv, L.k, L.v, y, lens, scale, pages=L.pages)
        check(y, *prefix(q1[:, None], pk, pv, L.k, L.v, lens.tolist(), scale, L.pages))
        ends = [sum(n[:b]) + shared + m + step for b, m in enumerate(prompts)]
        # both round their probabilities and results: within two bounds of one another
        want, bound = packed(q, k, v, n, n, scale)
        check(y[:, 0], full[ends].double(), 2 * bound[ends])
    assert api.take_device_error() == 0


def test_captured_decoding_step(cuda):
    """norm_rope and attention_prefix in one graph, replayed as the lengths and inputs change."""
    L = Layer(batch=4)
    g = gen(22)
    L.k.copy_(normal(g, *L.k.shape))
    L.v.copy_(normal(g, *L.v.shape))
    pk, pv = normal(g, 150, 2, 64), normal(g, 150, 2, 64)
    raw, qkv = normal(g, 4, 12, 64), torch.empty(4, 12, 64, device="cuda", dtype=BF16)
    pos, lens = ints([5, 6, 7, 8]), ints([1, 2, 3, 4])
    y = torch.empty(4, 1, 8, 64, device="cuda", dtype=BF16)

    def step():
        qkv.copy_(raw)
        q, _, _ = L.turn(qkv, pos)
        api.attention_prefix(q[:, None], pk, pv, L.k, L.v, y, lens, 0.125, pages=L.pages)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        raw.copy_(normal(g, *raw.shape))
        lens.copy_(ints([1 + 30 * i, 128, 100 - i, 16 * (i + 1)]))
        pos.copy_(lens)
        graph.replay()
        torch.cuda.synchronize()
        q = qkv[:, :8]
        want, _ = norm_rope(raw[:, :8], L.w[0], 1e-6, L.table, pos, None, False)
        assert (q.double() - want).abs().max() < 0.05
        check(y, *prefix(q[:, None], pk, pv, L.k, L.v, lens.tolist(), 0.125, L.pages))


def test_captured_prompt(cuda):
    """A captured packed call follows the starts on the device."""
    g = gen(23)
    q, k, v = normal(g, 400, 4, 128), normal(g, 400, 2, 128), normal(g, 400, 2, 128)
    y = torch.zeros_like(q)
    s = starts([400, 0, 0], "cuda")
    api.attention_packed(q, k, v, y, s, s, 0.1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        api.attention_packed(q, k, v, y, s, s, 0.1)
    for n in ([400, 0, 0], [1, 398, 1], [0, 100, 200]):
        s.copy_(starts(n, "cuda"))
        y.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        t = sum(n)
        check(y[:t], *packed(q[:t], k[:t], v[:t], n, n, 0.1))
        assert (y[t:] == 5).all()


FIRST_CALLS = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
from attention_util import check, norm_rope, packed, prefix, starts, table
from mlk2_b200 import api
g = torch.Generator(device="cuda").manual_seed(1)
q, k, v = (torch.randn(40, h, 64, generator=g, device="cuda").half() for h in (4, 2, 2))
t, pos = table(64, 64, "cuda"), torch.arange(40, device="cuda", dtype=torch.int32)
s, lens = starts([30, 10], "cuda"), torch.full((5,), 8, device="cuda", dtype=torch.int32)
qo, ko, y, z = (torch.zeros_like(x) for x in (q, k, q, q))
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    api.norm_rope(q, k, qo, ko, t, pos)
    api.attention_packed(qo, ko, v, y, s, s, 0.125)
    api.attention_prefix(qo.view(5, 8, 4, 64), ko, v, ko.view(5, 8, 2, 64), v.view(5, 8, 2, 64),
                         z.view(5, 8, 4, 64), lens, 0.125)
graph.replay()
torch.cuda.synchronize()
check(qo, *norm_rope(q, None, 0, t, pos, None, False))
check(y, *packed(qo, ko, v, [30, 10], [30, 10], 0.125))
want, bound = prefix(qo.view(5, 8, 4, 64), ko, v, ko.view(5, 8, 2, 64), v.view(5, 8, 2, 64), [8] * 5, 0.125)
check(z.view(5, 8, 4, 64), want, bound)
assert api.take_device_error() == 0
print("captured first calls ok")
"""


def test_first_calls_of_a_process_captured(cuda):
    """Nothing that a first call sets up gets in the way of a capture."""
    import os
    import subprocess
    import sys

    tests = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=os.path.dirname(tests), tests=tests)],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "captured first calls ok" in r.stdout, r.stdout + r.stderr


def test_empty_operands(cuda):
    q, k = torch.empty(0, 4, 64, device="cuda", dtype=F16), torch.empty(0, 2, 64, device="cuda", dtype=F16)
    api.norm_rope(q, k, q, k, table(4, 64, "cuda"), torch.empty(0, device="cuda", dtype=torch.int32))
    api.attention_packed(q, k, k, q, ints([0]), ints([0]), 0.1)
    api.attention_packed(q, k, k, q, ints([0, 0]), ints([0, 0]), 0.1)
    api.attention_prefix(q[:, None], k, k, k[:, None], k[:, None], q[:, None], ints([]), 0.1)
    x = torch.full((3, 4, 64), 7, device="cuda", dtype=F16)
    y = torch.full_like(x, 5)
    api.attention_packed(x, k, k, y, ints([0, 2]), ints([0, 0]), 0.1)  # no keys at all
    assert (y[:2] == 0).all() and (y[2] == 5).all()
    api.attention_prefix(x[:, None], k, k, k[:, None], k[:, None], y[:, None], ints([0, 0, 0]), 0.1)
    assert (y == 0).all() and api.take_device_error() == 0


def test_prefix_pages_shared_between_requests(cuda):
    """Requests may name the same page, and one request a page twice."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(3, 1, 40, [60, 64, 33], 4, 2, 64, 16, seed=7)
    pages[1] = pages[0]
    pages[2, 1] = pages[2, 0]
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=pages)
    check(y, *prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125, pages))


def test_prefix_batch_stride(cuda):
    """q, y and the caches as views with a common stride over their first two dimensions."""
    q, pk, pv, kp, vp, lens, _ = make_prefix(4, 3, 100, [50, 3, 200, 70], 8, 2, 64, 0, seed=8)
    wide = normal(gen(9), 4, 3, 16, 64)
    wide[:, :, 4:12] = q
    out = torch.full((4, 3, 8, 128), 5, device="cuda", dtype=BF16)
    y = out[..., :64]
    api.attention_prefix(wide[:, :, 4:12], pk, pv, kp, vp, y, lens, 0.125)
    check(y, *prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125))
    assert (out[..., 64:] == 5).all()
    with pytest.raises(ValueError, match="common stride"):
        api.attention_prefix(normal(gen(9), 4, 4, 8, 64)[:, :3], pk, pv, kp, vp, q, lens, 0.125)


def test_wrappers_refuse(cuda):
    q, k = torch.zeros(4, 8, 64, device="cuda", dtype=F16), torch.zeros(4, 2, 64, device="cuda", dtype=F16)
    pos, t, s = ints([0, 1, 2, 3]), table(9, 64, "cuda"), ints([0, 4])
    for call in (lambda: api.norm_rope(q, k, q[:3], k, t, pos), lambda: api.norm_rope(q, k, q, None, t, pos),
                 lambda: api.norm_rope(q, k[:3], q, k[:3], t, pos), lambda: api.norm_rope(q, k, q, k, t, pos[:3]),
                 lambda: api.norm_rope(q, k, q, k, t, pos.long()), lambda: api.norm_rope(q, k, q, k, t.half(), pos),
                 lambda: api.norm_rope(q, k.bfloat16(), q, k, t, pos),
                 lambda: api.norm_rope(q, k, q, k, t, pos, sections=[16, 16]),
                 lambda: api.norm_rope(q, k, q, k, t, pos, q_weight=t[0], k_weight=t[0]),
                 lambda: api.attention_packed(q, k, k[:3], q.clone(), s, s, 0.1),
                 lambda: api.attention_packed(q, k, k, q[:, :4], s, s, 0.1),
                 lambda: api.attention_packed(q, k, k, q.clone(), s, ints([0, 4, 4]), 0.1),
                 lambda: api.attention_packed(q, k, k, q.clone(), ints([]), ints([]), 0.1),
                 lambda: api.attention_packed(q.transpose(1, 2), k, k, q, s, s, 0.1),
                 lambda: api.attention_prefix(q[:, None], k, k, k[:2, None], k[:2, None], q[:, None].clone(), pos, 0.1),
                 lambda: api.attention_prefix(q[:, None], k, k, k[:, None], k[:, None], q[:, None].clone(), pos[:2], 0.1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(mb.MLKBError):
        api.attention_packed(q, k, k, q.clone(), s, s, -0.1)
    with pytest.raises(mb.MLKBError):
        api.norm_rope(q, k, q, k, t, pos, q_weight=t[0].half(), k_weight=None)
    with pytest.raises(mb.MLKBError, match="overlap"):
        api.attention_packed(q, k, k, q, s, s, 0.1)
    with pytest.raises(mb.MLKBError, match="overlap"):
        api.attention_prefix(q[:, None], k, k, k[:, None], k[:, None], q[:, None], pos, 0.1)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_without_eps(cuda, interleaved):
    """eps 0: rows whose squares leave the f32 range downwards, to the smallest bf16 values."""
    g = gen(21)
    q = normal(g, 6, 3, 96)
    for r, size in enumerate((1.0, 1e-18, 1e-25, 1e-37, 3e-39, 1e19)):
        q[r] = (q[r].double() * size).to(BF16)
    w, t = normal(g, 96), table(8, 64, "cuda")
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    y = torch.empty_like(q)
    api.norm_rope(q, None, y, None, t, pos, q_weight=w, eps=0.0, interleaved=interleaved)
    check(y, *norm_rope(q, w, 0.0, t, pos, None, interleaved))


@pytest.mark.parametrize("d,dtype", [(64, BF16), (40, F16), (128, F16)])
def test_packed_every_value_infinite_or_nan(cuda, d, dtype):
    """Every row is computed again, and the columns stay apart."""
    g = gen(22)
    n = [300, 77]
    q, k, v = normal(g, 377, 6, d, dtype=dtype), normal(g, 377, 2, d, dtype=dtype), normal(g, 377, 2, d, dtype=dtype)
    v[:, 0, 3] = torch.inf
    v[:, 1, d - 1] = torch.nan
    y = torch.empty_like(q)
    s = starts(n, "cuda")
    api.attention_packed(q, k, v, y, s, s, 0.1)
    assert y[:, :3, 3].isinf().all() and (y[:, :3, 3] > 0).all() and y[:, 3:, d - 1].isnan().all()
    clean = v.clone()
    clean[:, 0, 3] = clean[:, 1, d - 1] = 0
    want, bound = packed(q, k, clean, n, n, 0.1)
    y[:, :3, 3] = y[:, 3:, d - 1] = 0
    check(y, want, bound)


@pytest.mark.parametrize("heads,steps", [(4, 1), (16, 5)])
def test_prefix_infinite_value(cuda, heads, steps):
    """An infinity in the prefix and one of a request's own, in few (spread) rows and in many."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(5, steps, 500, [40, 300, 9, 170, 33], heads, 2, 64, 32, seed=9)
    want, bound = prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125, pages)
    pv[77, 0, 9] = torch.inf
    vp[pages[1, 2], 5, 1, 11] = -torch.inf
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=pages)
    group = heads // 2
    assert (y[:, :, :group, 9] == torch.inf).all() and (y[1, :, group:, 11] == -torch.inf).all()
    for z in (y, want):
        z[:, :, :group, 9] = 0
        z[1, :, group:, 11] = 0
    check(y, want, bound)


def test_prefix_table_without_pages(cuda):
    """Page indices into an empty cache read as zeros."""
    q, pk, pv, _, _, lens, pages = make_prefix(3, 1, 64, [40, 20, 48], 4, 2, 64, 16, seed=10)
    none = torch.empty(0, 16, 2, 64, device="cuda", dtype=BF16)
    zeros = torch.zeros(1, 16, 2, 64, device="cuda", dtype=BF16)
    y = torch.empty_like(q)
    for index in (0, 1, -1, 2 ** 31 - 1):
        api.attention_prefix(q, pk, pv, none, none, y, lens, 0.125, pages=torch.full_like(pages, index))
        assert api.take_device_error() == mb.ERR_INVALID
        check(y, *prefix(q, pk, pv, zeros, zeros, lens.tolist(), 0.125, torch.zeros_like(pages)))


def test_calls_at_once_given_streams(cuda):
    """Streams by handle, the workspaces allocated by the calls."""
    ins = [make_prefix(20, 1, 2000, [100] * 20, 8, 2, 64, 0, seed=s) for s in (1, 2, 3)]
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [[torch.empty_like(i[0]) for _ in range(6)] for i in ins]
    torch.cuda.synchronize()
    for r in range(6):
        for (q, pk, pv, kp, vp, lens, _), st, y in zip(ins, streams, outs):
            api.attention_prefix(q, pk, pv, kp, vp, y[r], lens, 0.125,
                                 stream=st.cuda_stream if r % 3 else torch.cuda.default_stream().cuda_stream)
    torch.cuda.synchronize()
    for (q, pk, pv, kp, vp, lens, _), y in zip(ins, outs):
        want, bound = prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125)
        for z in y:
            check(z, want, bound)


def test_wrappers_refuse_other_ranks(cuda):
    q, s = torch.zeros(8, 64, device="cuda", dtype=F16), ints([0, 8])
    for x in (q, q[0], q[None, None, None]):
        with pytest.raises(ValueError):
            api.attention_packed(x, x, x, x.clone(), s, s, 0.1)
        with pytest.raises(ValueError):
            api.norm_rope(x, None, x, None, table(9, 64, "cuda"), s)
    with pytest.raises(ValueError):
        api.attention_packed(q[None, None], q[None, None], q[None, None], q[None, None].clone(), s, s, 0.1)


@pytest.mark.parametrize("offset", [16, 32])
def test_prefix_workspace_alignment(cuda, offset):
    """A workspace that is a multiple of 16 bytes only."""
    q, pk, pv, kp, vp, lens, pages = make_prefix(6, 2, 300, [30, 2, 100, 64, 65, 7], 8, 2, 72, 32, seed=11)
    need = api.attention_prefix_workspace(q, pk, kp, pages)
    ws = torch.full((need + 64,), 255, device="cuda", dtype=torch.uint8)
    y = torch.empty_like(q)
    api.attention_prefix(q, pk, pv, kp, vp, y, lens, 0.125, pages=pages, workspace=ws[offset:offset + need])
    check(y, *prefix(q, pk, pv, kp, vp, lens.tolist(), 0.125, pages))
    assert (ws[:offset] == 255).all() and (ws[offset + need:] == 255).all()


@pytest.mark.parametrize("causal", [True, False])
def test_packed_very_many_sequences(cuda, causal):
    """Enough sequences that costs are compared in units of several key tiles."""
    r = random.Random(5)
    nq = [r.choice([0, 1, 1, 1, 2, 140]) for _ in range(1500)]
    nk = [n + r.choice([0, 0, 1, 40, 300, 700]) for n in nq]
    nk[700] += 6000
    run_packed(nq, nk, 2, 1, 64, seed=12, causal=causal)
