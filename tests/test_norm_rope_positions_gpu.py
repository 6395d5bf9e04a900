"""norm_rope with many tokens whose positions lie outside the table."""
import pytest
import torch

import mlk2_b200 as mb
from attention_util import check, norm_rope, table
from mlk2_b200 import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("every", [2, 5])
def test_tokens_without_a_position_among_others(cuda, every, axes):
    """They are left as they are, their copies landed before the block ends; the others are turned."""
    g = torch.Generator(device="cuda").manual_seed(every)
    n, heads, d = 30011, 6, 128
    q = torch.randn(n, heads, d, generator=g, device="cuda").bfloat16()
    w = torch.ones(d, device="cuda", dtype=torch.bfloat16)
    t = table(64, d, "cuda")
    pos = torch.randint(0, 64, (axes, n), generator=g, device="cuda").int()
    bad = torch.arange(n, device="cuda") % every == 1
    pos[-1, bad] = 64
    sections = [32, 16, 16] if axes == 3 else None
    y = torch.full_like(q, 7)
    assert api.take_device_error() == 0
    api.norm_rope(q, None, y, None, t, pos if axes > 1 else pos[0], sections=sections, q_weight=w)
    assert api.take_device_error() == mb.ERR_INVALID
    assert (y[bad] == 7).all()
    check(y[~bad], *norm_rope(q[~bad], w, 1e-6, t, pos[:, ~bad], sections, False))
