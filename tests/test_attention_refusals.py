"""Calls of norm_rope and the attention entries that are refused before any
device work, through the C ABI; no GPU needed."""
import pytest

import mlk2_b200 as mb
from test_attention_abi import P, Y, accepted, heads, no_device, norm_rope, packed, prefix, refused

K = P + (1 << 22)


# ---- rows of one request ----------------------------------------------------------

def many(steps, heads_, batch=1):
    q = heads(steps * batch, row=8 * heads_, head=8)
    y = heads(steps * batch, row=8 * heads_, head=8, data=Y)
    return {"batch": batch, "steps": steps, "heads_": heads_, "kv": heads_ // 2, "d": 8, "q": q, "y": y,
            "pk": heads(30, row=4 * heads_, head=8), "pv": heads(30, row=4 * heads_, head=8),
            "kp": heads(320, row=4 * heads_, head=8), "vp": heads(320, row=4 * heads_, head=8),
            "size": 2 ** 62}


@pytest.mark.parametrize("steps,heads_", [(2 ** 29, 4), (2 ** 30, 4), (2 ** 27, 64), (2 ** 22, 2 ** 10)])
def test_prefix_rows_of_a_request_fit_32_bits(steps, heads_):
    refused(prefix(**many(steps, heads_)), "too much work")


@no_device
def test_prefix_most_rows_of_a_request():
    accepted(prefix(**many(2 ** 29 - 1, 4)))


def test_workspace_of_refused_shapes_is_negative():
    packed_size, prefix_size = mb.lib().mlkb_attention_packed_workspace, mb.lib().mlkb_attention_prefix_workspace
    for bad in ((1, 16384, 1, 8, 2, 12), (1, 16384, 1, 2 ** 18, 2 ** 17, 64)):
        assert packed_size(*bad) < 0
    for bad in ((1, 2 ** 29, 4, 2, 8, 30, 16, 3), (4, 1, 8, 2, 12, 5, 16, 1), (4, 1, 2 ** 18, 2 ** 17, 64, 5, 16, 1),
                (4, 1, 8, 2, 64, 5, 2 ** 20, 2 ** 20)):
        assert prefix_size(*bad) < 0
    assert prefix_size(1, 2 ** 29 - 1, 4, 2, 8, 30, 16, 3) > 0


# ---- outputs that are inputs --------------------------------------------------------

@pytest.mark.parametrize("operand,rows", [("pk", 30), ("pv", 30), ("kp", 320), ("vp", 320)])
def test_prefix_y_may_not_be_a_cache(operand, rows):
    refused(prefix(**{operand: heads(rows, data=Y)}), "overlap")


@no_device
def test_prefix_empty_caches_have_no_address():
    none = heads(0, data=Y)
    accepted(prefix(pk=none, pv=none))
    accepted(prefix(kp=none, vp=none, page=0, wide=0, pages=None, lens=None))


@pytest.mark.parametrize("kw", [
    {"qo": heads(row=2048)},                    # q's address, other strides
    {"qo": heads(row=1024, head=256)},
    {"ko": heads(row=512, data=K)},             # k's
    {"qo": heads(data=K)}, {"ko": heads(data=P)},  # the other operand's
    {"qo": heads(data=Y), "ko": heads(data=Y)}])
def test_norm_rope_outputs_over_other_operands(kw):
    refused(norm_rope(**{"k": heads(data=K), "ko": heads(data=K), "heads_": 2, **kw}), "overlap")


@no_device
def test_norm_rope_outputs_in_place_or_apart():
    apart = {"k": heads(data=K), "ko": heads(data=K)}
    accepted(norm_rope(**apart))
    accepted(norm_rope(**{**apart, "qo": heads(data=Y, row=2048)}))
    # strides of dimensions with one entry do not count
    accepted(norm_rope(**{**apart, "heads_": 1, "qo": heads(head=4096)}))
    one = {"k": heads(rows=1, data=K), "ko": heads(rows=1, data=K, row=8)}
    accepted(norm_rope(**one, q=heads(rows=1), qo=heads(rows=1, row=4096)))


@pytest.mark.parametrize("eps", [3.1e38, 1e300, float("inf"), -1e-300])
def test_norm_rope_eps(eps):
    refused(norm_rope(eps=eps), "eps")


# ---- when keys are cut -----------------------------------------------------------------

def test_packed_keys_are_not_cut_among_very_many_sequences():
    """Every block looks through the sequences for each key count there may be."""
    size = mb.lib().mlkb_attention_packed_workspace
    assert size(1, 16384, 8192, 8, 1, 128) == size(1, 16384, 1, 8, 1, 128) > 0
    assert size(1, 16384, 8193, 8, 1, 128) == 0
    assert size(40, 16384, 40, 8, 1, 128) > 0
    assert size(8, 16384, 2000, 8, 2, 128) == 0
