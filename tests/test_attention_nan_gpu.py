"""A NaN or an infinity that a query row sees reaches that row, and no other.

Rows whose visible scores hold a NaN are NaN in every column, as an elementwise
max / exp / sum over the row gives it; rows that see none keep their bits.
Exact comparisons: no tolerance."""

import pytest
import torch

from forma_b200 import api
from forma_b200.api import AttentionOptions, Mask

pytestmark = pytest.mark.gpu


def rnd(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def rows_are(got, want, poisoned):
    """NaN in every column of the poisoned rows [B, H, L]; the others as without the poison."""
    nan = torch.isnan(got)
    assert nan[poisoned].all()
    assert not nan[~poisoned].any()
    assert torch.equal(got[~poisoned], want[~poisoned])
    assert api.device_status() == 0


GENERIC = [(torch.float32, 64), (torch.float32, 20), (torch.bfloat16, 40)]  # types and depths the tensor cores leave alone


@pytest.mark.parametrize("dtype,d", GENERIC)
@pytest.mark.parametrize("keys", [1, 31, 33, 65, 300])
def test_window_generic_query_nan(cuda, dtype, d, keys):
    """A NaN query row over key counts that end inside a 32-key tile."""
    for lq, window, sinks in ((1, 400, 0), (3, 17, 2), (40, 33, 1)):
        q, k, v = rnd((2, 4, lq, d), dtype, 1), rnd((2, 2, keys, d), dtype, 2), rnd((2, 2, keys, d), dtype, 3)
        want = api.attention_window(q, k, v, window, sinks)
        assert api.last_route() == ["span_simt_kernel"]
        poisoned = torch.zeros((2, 4, lq), dtype=torch.bool, device=cuda)
        poisoned[1, 2, lq - 1] = poisoned[0, 0, lq - 1] = True  # the last query sees every key of its window
        q[..., d // 2] = torch.where(poisoned, torch.nan, q[..., d // 2])
        rows_are(api.attention_window(q, k, v, window, sinks), want, poisoned)


@pytest.mark.parametrize("dtype,d", GENERIC)
@pytest.mark.parametrize("keys", [1, 31, 33, 65, 300])
def test_window_generic_key_nan(cuda, dtype, d, keys):
    """A NaN key, first or last of its tile, alone in the tile or not: the rows that see it."""
    lq = min(keys, 50)
    q, k, v = rnd((2, 4, lq, d), dtype, 4), rnd((2, 2, keys, d), dtype, 5), rnd((2, 2, keys, d), dtype, 6)
    window, sinks = 20, 2
    want = api.attention_window(q, k, v, window, sinks)
    p = torch.arange(keys - lq, keys, device=cuda)
    for j in sorted({0, keys // 2, keys - 1, min(keys - 1, 31), min(keys - 1, 32)}):
        bad = k.clone()
        bad[1, 0, j, 0] = torch.nan
        sees = (j <= p) & ((j > p - window) | (j < sinks))
        poisoned = torch.zeros((2, 4, lq), dtype=torch.bool, device=cuda)
        poisoned[1, :2] = sees
        rows_are(api.attention_window(q, bad, v, window, sinks), want, poisoned)


@pytest.mark.parametrize("dtype,d", GENERIC)
def test_window_generic_infinite_scores(cuda, dtype, d):
    """+inf scores give NaN; a key at -inf has no weight; a row with nothing else is zeros."""
    keys = 45
    q, k, v = rnd((1, 2, 1, d), dtype, 7).abs() + 0.1, rnd((1, 1, keys, d), dtype, 8), rnd((1, 1, keys, d), dtype, 9)
    up, down, all_down = k.clone(), k.clone(), k.clone()
    up[0, 0, 33, 1], down[0, 0, 33, 1], all_down[..., 1] = torch.inf, -torch.inf, -torch.inf
    assert torch.isnan(api.attention_window(q, up, v, 100)).all()
    without = [torch.cat([t[:, :, :33], t[:, :, 34:]], 2) for t in (k, v)]
    want = api.attention_window(q, *without, 100).double()
    err = (api.attention_window(q, down, v, 100).double() - want).abs().max()
    # f64 states; the order of the keys over the warps differs: one rounding of the output's type each
    assert err <= 2 * torch.finfo(dtype).eps * float(want.abs().max())
    assert (api.attention_window(q, all_down, v, 100) == 0).all()
    assert api.device_status() == 0


@pytest.mark.parametrize("dtype,d", GENERIC)
@pytest.mark.parametrize("pre,keys", [(1, 0), (31, 5), (33, 1), (100, 70)])
def test_prefix_generic_nan(cuda, dtype, d, pre, keys):
    """A NaN query, a NaN prefix key (every sequence's rows of its head), a NaN own key."""
    b, lq = 3, 2
    q, pk, pv = rnd((b, 4, lq, d), dtype, 10), rnd((2, pre, d), dtype, 11), rnd((2, pre, d), dtype, 12)
    k, v = rnd((b, 2, keys, d), dtype, 13), rnd((b, 2, keys, d), dtype, 14)
    want = api.attention_prefix(q, pk, pv, k, v)
    assert api.last_route() == ["span_simt_kernel"]
    none = torch.zeros((b, 4, lq), dtype=torch.bool, device=cuda)
    poisoned, bad = none.clone(), q.clone()
    poisoned[1, 3, 0], bad[1, 3, 0, 5] = True, torch.nan
    rows_are(api.attention_prefix(bad, pk, pv, k, v), want, poisoned)
    poisoned, bad = none.clone(), pk.clone()
    poisoned[:, 2:], bad[1, pre - 1, 0] = True, torch.nan
    rows_are(api.attention_prefix(q, bad, pv, k, v), want, poisoned)
    if keys:
        poisoned, bad = none.clone(), k.clone()
        poisoned[2, :2, lq - 1], bad[2, 0, keys - 1, 0] = True, torch.nan  # the newest key: the last query alone
        rows_are(api.attention_prefix(q, pk, pv, bad, v), want, poisoned)


@pytest.mark.parametrize("dtype,d", GENERIC)
@pytest.mark.parametrize("keys", [1, 31, 33, 65, 700])
@pytest.mark.parametrize("kind", ["plain", "causal", "keep", "additive"])
def test_dense_generic_nan(cuda, dtype, d, keys, kind):
    """The same for the general dense kernel and its split over long key ranges."""
    lq = 5
    q, k, v = rnd((2, 4, lq, d), dtype, 15), rnd((2, 2, keys, d), dtype, 16), rnd((2, 2, keys, d), dtype, 17)
    sees = torch.ones((lq, keys), dtype=torch.bool, device=cuda)
    mask, options = None, AttentionOptions()
    if kind == "causal":
        options = AttentionOptions(causal=keys - 3)
        sees = torch.arange(keys, device=cuda)[None] <= torch.arange(lq, device=cuda)[:, None] + keys - 3
    elif kind != "plain":
        sees[1, keys // 2:] = False
        sees[3] = False
        mask = Mask("keep", sees.int()) if kind == "keep" else Mask("additive", torch.where(sees, 0.25, -torch.inf))
    run = (lambda q, k: api.attention(q, k, v, mask, options)) if dtype == torch.float32 else \
          (lambda q, k: api.attention_low_f32(q, k, v, mask, options))
    want = run(q, k)
    assert all("simt" in r or "attention_part" in r or "attention_merge" in r for r in api.last_route()), api.last_route()
    poisoned, bad = torch.zeros((2, 4, lq), dtype=torch.bool, device=cuda), q.clone()
    poisoned[1, 3] = sees.any(1)
    bad[1, 3, :, 2] = torch.nan
    rows_are(run(bad, k), want, poisoned)
    for j in sorted({0, keys // 2, keys - 1}):
        poisoned, bad = torch.zeros((2, 4, lq), dtype=torch.bool, device=cuda), k.clone()
        poisoned[0, 2:], bad[0, 1, j, 0] = sees[:, j], torch.nan
        rows_are(run(q, bad), want, poisoned)


# Tensor-core kernels: part of the exponentials are polynomials, chosen by the
# key's place in its tile, so every place is tried.

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,kernel", [(40, "span_tile_kernel"), (2, "span_decode_kernel")])
def test_window_tensor_core_nan_and_infinity(cuda, dtype, d, lq, kernel):
    keys, window, sinks = 200, 90, 3
    q, k, v = rnd((1, 4, lq, d), dtype, 20), rnd((1, 2, keys, d), dtype, 21), rnd((1, 2, keys, d), dtype, 22)
    want = api.attention_window(q, k, v, window, sinks)
    assert all(r.startswith(kernel) for r in api.last_route()), api.last_route()
    p = torch.arange(keys - lq, keys, device=cuda)
    for j in [0, 1, 2, keys - 1] + list(range(130, 162)):
        sees = (j <= p) & ((j > p - window) | (j < sinks))
        poisoned, bad = torch.zeros((1, 4, lq), dtype=torch.bool, device=cuda), k.clone()
        poisoned[0, 2:], bad[0, 1, j, 3] = sees, torch.nan
        rows_are(api.attention_window(q, bad, v, window, sinks), want, poisoned)
        # an infinite score: NaN where it is +inf, no weight where it is -inf
        bad = k.clone()
        bad[0, 1, j, 3] = torch.inf
        got = api.attention_window(q, bad, v, window, sinks)
        up = torch.zeros((1, 4, lq), dtype=torch.bool, device=cuda)
        up[0, 2:] = sees & (q[0, 2:, :, 3] > 0)
        assert torch.equal(torch.isnan(got).any(-1), up) and torch.equal(torch.isnan(got).all(-1), up)


@pytest.mark.parametrize("lq,d", [(1, 128), (30, 64)])
def test_prefix_tensor_core_nan(cuda, lq, d):
    """A NaN in the shared prefix passes the records and their join."""
    dt, b, pre, keys = torch.bfloat16, 3, 300, 40
    q, pk, pv = rnd((b, 8, lq, d), dt, 23), rnd((2, pre, d), dt, 24), rnd((2, pre, d), dt, 25)
    k, v = rnd((b, 2, keys, d), dt, 26), rnd((b, 2, keys, d), dt, 27)
    want = api.attention_prefix(q, pk, pv, k, v)
    assert api.last_route()[0].startswith("span_tile_kernel"), api.last_route()
    for j in list(range(16)) + [142, 143, 298, 299]:
        poisoned, bad = torch.zeros((b, 8, lq), dtype=torch.bool, device=cuda), pk.clone()
        poisoned[:, :4], bad[0, j, 0] = True, torch.nan
        rows_are(api.attention_prefix(q, bad, pv, k, v), want, poisoned)


@pytest.mark.parametrize("lq,keys,d,kernel", [(300, 300, 128, "attn_fwd_kernel"), (190, 190, 64, "attn_short_kernel"),
                                              (120, 120, 64, "attn_short_kernel")])
def test_dense_tensor_core_nan(cuda, lq, keys, d, kernel):
    dt = torch.bfloat16
    q, k, v = rnd((1, 2, lq, d), dt, 28), rnd((1, 2, keys, d), dt, 29), rnd((1, 2, keys, d), dt, 30)
    want = api.attention_low_f32(q, k, v)
    assert any(r.startswith(kernel) for r in api.last_route()), api.last_route()
    for j in list(range(32)) + [keys - 1]:
        poisoned, bad = torch.zeros((1, 2, lq), dtype=torch.bool, device=cuda), k.clone()
        poisoned[0, 1], bad[0, 1, j, 0] = True, torch.nan
        rows_are(api.attention_low_f32(q, bad, v), want, poisoned)
