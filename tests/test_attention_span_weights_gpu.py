"""What the 16-bit weights of the span attentions keep of a softmax.

Tolerance, as in the other span tests: |error| <= (2u + 2^-12) max|v| + u |e|
with u = 2^-9 (BF16) and 2^-12 (F16), half the type's unit roundoff, unless a
test says less."""

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


def ones_case(dtype, b, h, hk, d, lq, keys, window, sinks, pre, spread):
    """Values of one: whatever the weights, P V and their sum are the same sum.
    f32 output; both are f32 sums of at most `keys` terms: 2^-24 of the whole each."""
    q, k = rnd((b, h, lq, d), dtype, 1), rnd((b, hk, keys, d), dtype, 2) * spread
    v = torch.ones((b, hk, keys, d), dtype=dtype, device="cuda")
    out = torch.empty((b, h, lq, d), device="cuda")
    if pre:
        pk = rnd((hk, pre, d), dtype, 3) * spread
        api.attention_prefix(q, pk, torch.ones_like(pk), k, v, out=out)
    else:
        api.attention_window(q, k, v, window, sinks, out=out)
    assert (out.double() - 1).abs().max() <= (keys + pre) * 2.0**-24
    assert api.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq", [1, 60])
@pytest.mark.parametrize("spread", [0.1, 1.0, 3.0])
def test_sums_are_of_the_weights_that_multiply(cuda, dtype, d, lq, spread):
    for keys, window, sinks in ((90, 1000, 0), (700, 300, 4), (1500, 5000, 0)):
        ones_case(dtype, 2, 4, 2, d, lq, keys, window, sinks, 0, spread)
    ones_case(dtype, 3, 4, 2, d, lq, 80, 0, 0, 900, spread)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("logit", [1.3, 3.7, 5.0, 5.45, 11.0])
def test_dominant_key_in_a_late_tile(cuda, dtype, lq, logit):
    """A key that outweighs the rest, with and without passing the 2^8 below
    which the running maximum stays: its weight's rounding cancels.  The other
    key's share s of the row is off by its own and the dominant one's rounding,
    2u s; f32 output."""
    keys, d = 300, 64
    q, k, v = (torch.zeros((1, 2, n, d), dtype=dtype, device=cuda) for n in (lq, keys, keys))
    q[..., 0], k[..., 0] = 1.0, -200.0
    k[:, :, 0, 0], k[:, :, 200, 0] = 0.0, logit
    v[:, :, 0], v[:, :, 200] = -1.0, 1.0
    out = torch.empty((1, 2, lq, d), device=cuda)
    api.attention_window(q, k, v, 1000, 0, options=AttentionOptions(scale=1.0, causal=keys), out=out)
    share = 1.0 / (1.0 + math.exp(float(k[0, 0, 200, 0])))
    exp = 1.0 - 2.0 * share
    # exponentials: 7.5e-5 of a weight where the polynomial takes it, 2^-22 otherwise
    assert (out.double() - exp).abs().max() <= 2 * share * (2 * UNIT[dtype] + 1e-4) + 2.0**-22


def definition(q, k, v, seen, scale):
    g = q.shape[1] // k.shape[1]
    s = q.double() @ k.double().repeat_interleave(g, 1).transpose(-1, -2) * scale
    return torch.softmax(s.masked_fill(~seen, -torch.inf), -1) @ v.double().repeat_interleave(g, 1)


def window_seen(lq, keys, window, sinks):
    p = torch.arange(keys - lq, keys, device="cuda")[:, None]
    j = torch.arange(keys, device="cuda")[None]
    return (j <= p) & ((j > p - window) | (j < sinks))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_large_scores_move_by_their_own_error_only(cuda, dtype, lq, d):
    """Scores in the hundreds.  Each is off by at most e = D 2^-24 sum |q k|
    scale (f32 sums of D products), which moves the weights of a row by at most
    exp(2e) - 1 in all; the rest as for small scores."""
    keys, scale = 300, d**-0.5
    q, k, v = rnd((1, 4, lq, d), dtype, 1) * 20, rnd((1, 2, keys, d), dtype, 2) * 20, rnd((1, 2, keys, d), dtype, 3)
    got = api.attention_window(q, k, v, 150, 2).double()
    exp = definition(q, k, v, window_seen(lq, keys, 150, 2), scale)
    e = d * 2.0**-24 * scale * (q.double().abs() @ k.double().abs().repeat_interleave(2, 1).transpose(-1, -2)).amax(-1, keepdim=True)
    u, top = UNIT[dtype], float(v.double().abs().max())
    bound = (torch.expm1(2 * e) + 2 * u + 2.0**-12) * top + u * exp.abs()
    assert bound.max() < 0.1 * top
    assert ((got - exp).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("step", [0.125, 0.03125, 0.0078125, -0.125, -0.03125])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_maximum_rises_from_tile_to_tile(cuda, dtype, lq, d, step, scale):
    """Logits that rise (or fall) along the keys, by more and by less than 2^8
    a tile, so that the running maximum and O are rescaled often or seldom."""
    keys, pre = 600, 400
    q, k, v = rnd((1, 4, lq, d), dtype, 1) * 0.05, rnd((1, 2, keys, d), dtype, 2), rnd((1, 2, keys, d), dtype, 3)
    q[..., 0] = 1.0
    k[..., 0] = (torch.arange(keys, device=cuda) * (step * scale)).to(dtype)
    options = AttentionOptions(scale=scale)
    u, top = UNIT[dtype], float(v.double().abs().max())
    for window, sinks in ((1000, 0), (300, 4)):
        got = api.attention_window(q, k, v, window, sinks, options=options).double()
        exp = definition(q, k, v, window_seen(lq, keys, window, sinks), scale)
        assert ((got - exp).abs() <= (2 * u + 2.0**-12) * top + u * exp.abs()).all()
    got = api.attention_prefix(q, k[0, :, :pre], v[0, :, :pre], k[:, :, pre:], v[:, :, pre:], options=options).double()
    exp = definition(q, k, v, window_seen(lq, keys, 1000, 0), scale)
    assert ((got - exp).abs() <= (2 * u + 2.0**-12) * top + u * exp.abs()).all()
    assert api.device_status() == 0
