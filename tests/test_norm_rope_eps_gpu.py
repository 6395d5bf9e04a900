"""norm_rope at the ends of eps: values that f32 holds as 0, and values that
matter beside rows whose squares leave the f32 range."""
import pytest
import torch

from attention_util import check, norm_rope, table
from mlk2_b200 import api

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def rows(sizes, d, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(len(sizes), 2, d, generator=g, device="cuda", dtype=torch.float64)
    return (x * torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None, None]).to(BF16)


@pytest.mark.parametrize("eps", [1e-30, 1e-37, 1e-46, 1e-50, 1e-60, 1e-80, 1e-300])
@pytest.mark.parametrize("d", [64, 96])
def test_eps_below_the_f32_range(cuda, d, eps):
    """Zeros stay zeros, and rows of about sqrt(eps) see its share."""
    q = rows([0, 1, 1e-15, 1e-23, 1e-25, 1e-30, 1e-37], d)
    t, pos = table(8, 64, "cuda"), torch.arange(7, device="cuda", dtype=torch.int32)
    w = torch.ones(d, device="cuda", dtype=BF16)
    y = torch.full_like(q, 5)
    api.norm_rope(q, None, y, None, t, pos, q_weight=w, eps=eps)
    check(y, *norm_rope(q, w, eps, t, pos, None, False))


@pytest.mark.parametrize("eps", [1e36, 1e34, 1e20])
@pytest.mark.parametrize("d", [16, 512])
def test_large_eps(cuda, d, eps):
    """Beside rows whose squares are, or sum, past the f32 range."""
    q = rows([1, 1e10, 3e17, 1e18, 5e18, 2e19, 1e25, 1e37], d)
    t, pos = table(8, 16, "cuda"), torch.arange(8, device="cuda", dtype=torch.int32)
    w = torch.ones(d, device="cuda", dtype=BF16)
    y = torch.full_like(q, 5)
    api.norm_rope(q, None, y, None, t, pos, q_weight=w, eps=eps)
    check(y, *norm_rope(q, w, eps, t, pos, None, False))
