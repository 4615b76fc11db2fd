"""Edges of serving sequences of different lengths: calls that the documentation allows and a formula decides, at the borders of
types, sizes, masks and states.  Sampling has no tolerance: the token is the one of the 64-bit definition."""
import math

import pytest
import torch

import ragged_check as R
from smlm_hip import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
bf16, f32 = torch.bfloat16, torch.float32
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=bf16):
    return torch.randn(*shape, generator=g).to(dtype)


# ------------------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("V", [1 << 18, 261_500])
def test_the_last_tokens_of_very_large_flat_rows_are_drawn(V, dtype):
    """Equal logits, masks alone and a temperature that leaves no difference: token n holds the share [n, n + 1) / V of u.  (u has
    24 bits, so u V is exact in 64.)"""
    u = torch.tensor([0.5, 0.998, 0.999, 1 - 2.0 ** -24])
    want = [int(float(a) * V) for a in u]
    for x, T in ((torch.full((4, V), -1.5), 1.0), (torch.full((4, V), -math.inf), 1.0), (torch.randn(4, V, generator=gen(V)), 1e30)):
        assert K.sample_tokens(x.to(DEV, dtype), u.to(DEV), T).tolist() == want
    for outside in (1.0, 7.0, math.inf):              # the last token all the same
        assert K.sample_tokens(x.to(DEV, dtype), torch.full((4,), outside, device=DEV), T).tolist() == [V - 1] * 4
