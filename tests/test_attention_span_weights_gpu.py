"""What the 16-bit weights of the span attentions keep of a softmax.

Tolerance, as in the other span tests: u the unit roundoff of the type (2^-9
BF16, 2^-12 F16), |error| <= (2u + 2^-12) max|v| + u |e|, unless a test says
less."""

import math

import pytest
import torch

from forma_b200 import api
from forma_b200.api import AttentionOptions

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}


def rnd(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,lq", [(150, 20), (300, 1)])
@pytest.mark.parametrize("place", [0, 70000])
def test_many_keys_far_below_one(cuda, dtype, b, lq, place):
    """131072 keys 18 nats below one key: 0.2% of the row, in the sum and in the output alike."""
    keys, d, below = 131072, 64, 18.0
    q = torch.zeros((b, 1, lq, d), dtype=dtype, device=cuda)
    k = torch.zeros((1, 1, keys, d), dtype=dtype, device=cuda)
    q[..., 0], k[:, :, place, 0] = 1.0, below
    k, options = k.expand(b, -1, -1, -1), AttentionOptions(scale=1.0, causal=keys)
    u = UNIT[dtype]
    rest = (keys - 1) * math.exp(-below)
    for v0 in (1.0, -1.0):
        v = torch.ones((1, 1, keys, d), dtype=dtype, device=cuda)
        v[:, :, place] = v0
        got = api.attention_window(q, k, v.expand(b, -1, -1, -1), 1 << 31, 0, options=options).double()
        exp = (v0 + rest) / (1 + rest)
        assert (got - exp).abs().max() <= 2 * u + 2.0**-12 + u * abs(exp)
    assert api.device_status() == 0
