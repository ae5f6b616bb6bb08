"""Windowed attention and attention over a shared prefix against a plain
64-bit implementation with dense masks.

Tolerance.  f32 operands: 1e-5 of max(|e|, 1), the package's f32 bound.
16-bit operands, u the unit roundoff of the type (2^-9 BF16, 2^-12 F16, both
as half an ulp relative to the leading digit's binade): the weights are
rounded to the operands' type before they multiply V, and the row sum adds
them before or after that, so numerator and denominator are each off by at most u
relative to sum p |v| <= max|v|; exponentials and f32 scores add less than
2^-12 of the same; a 16-bit result is rounded once more:
|error| <= (2u + 2^-12) max|v| + u |e|."""

import itertools

import pytest
import torch

from forma_b200 import api
from forma_b200.api import AttentionOptions, TensorError

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}


def rnd(shape, dtype, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, device=device, generator=g, dtype=torch.float32).to(dtype)


def attend64(q, parts, scale):
    """softmax over the joined parts [(k, v, seen or None)]: q [B, H, L, D], k [B, Hkv, K, D], seen [B, L, K]."""
    b, h, lq, d = q.shape
    logits, values = [], []
    for k, v, seen in parts:
        g = h // k.shape[1]
        kk, vv = k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
        s = torch.einsum("bhqd,bhkd->bhqk", q.double(), kk) * scale
        if seen is not None:
            s = s.masked_fill(~seen[:, None], -torch.inf)
            vv = torch.where(seen.any(1)[:, None, :, None], vv, torch.zeros_like(vv))
        logits.append(s)
        values.append(vv)
    p = torch.nan_to_num(torch.softmax(torch.cat(logits, -1), -1), nan=0.0)
    return p @ torch.cat(values, 2)


def seen_mask(b, lq, keys, window, sinks, lengths, offset, device="cuda"):
    n = lengths.long().clamp(max=keys) if lengths is not None else torch.full((b,), keys, device=device)
    base = n - lq if lengths is not None else torch.full((b,), keys - lq if offset is None else offset, device=device)
    p = (base[:, None] + torch.arange(lq, device=device))[:, :, None]
    j = torch.arange(keys, device=device)[None, None]
    return (j < n[:, None, None]) & (j <= p) & ((j > p - window) | (j < sinks))


def check(got, exp, dtype, v_max):
    assert got.shape == exp.shape
    err = (got.double() - exp).abs()
    if dtype == torch.float32:
        bound = 1e-5 * exp.abs().clamp(min=1.0)
    else:
        u = UNIT[dtype]
        bound = (2 * u + 2.0**-12) * v_max + (u * exp.abs() if got.dtype == dtype else 0.0)
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (err / bound).max()


def window_case(b, h, hk, d, lq, keys, window, sinks, dtype, lengths=None, offset=None, seed=0, out=None):
    q, k, v = rnd((b, h, lq, d), dtype, seed), rnd((b, hk, keys, d), dtype, seed + 1), rnd((b, hk, keys, d), dtype, seed + 2)
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths is not None else None
    got = api.attention_window(q, k, v, window, sinks, ln, AttentionOptions(causal=offset), out)
    exp = attend64(q, [(k, v, seen_mask(b, lq, keys, window, sinks, ln, offset))], d**-0.5)
    check(got, exp, dtype, float(v.double().abs().max()) if keys else 1.0)
    assert api.device_status() == 0
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("lq,keys", [(1, 1), (1, 129), (3, 300), (17, 17), (130, 257), (257, 700)])
def test_window_sizes(cuda, dtype, d, lq, keys):
    for window, sinks in ((1, 0), (1, 1), (33, 4), (128, 130), (1000, 0)):
        window_case(2, 4, 2, d, lq, keys, window, sinks, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (8, 1), (32, 8), (48, 2)])
@pytest.mark.parametrize("lq", [1, 2, 40])
def test_window_heads(cuda, dtype, heads, lq):
    window_case(2, *heads, 128, lq, 523, 200, 5, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 4, 70, 300])
def test_window_lengths(cuda, dtype, lq):
    """Empty caches, shorter than the queries (leading rows empty: zeros), full, and beyond the allocation (clamped)."""
    got = window_case(6, 8, 2, 64, lq, 640, 100, 3, dtype, lengths=[0, 1, 2, 333, 640, 700])
    assert got[0].abs().max() == 0
    if lq > 1:
        assert got[1, :, : lq - 1].abs().max() == 0


@pytest.mark.parametrize("offset", [-5, -400, 0, 77, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_offsets(cuda, offset, dtype):
    """Positions before the first key (empty rows), inside, and far past the last key (only the sinks stay)."""
    for lq in (6, 300):
        window_case(1, 4, 4, 128, lq, 400, 64, 2, dtype, offset=offset)
    got = window_case(1, 4, 4, 128, 6, 400, 64, 0, dtype, offset=5000)
    assert got.abs().max() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_unfilled_cache_is_not_read(cuda, dtype):
    """NaN and infinities past the filled keys do not reach the result."""
    for lq in (1, 5, 150):
        q, k, v = rnd((3, 8, lq, 64), dtype, 1), rnd((3, 2, 600, 64), dtype, 2), rnd((3, 2, 600, 64), dtype, 3)
        ln = torch.tensor([160, 401, 599], dtype=torch.int32, device=cuda)
        want = api.attention_window(q, k, v, 200, 4, ln)
        for i, n in enumerate(ln.tolist()):
            k[i, :, n:] = float("nan")
            v[i, :, n:] = float("inf")
            v[i, :, n + 1 :: 2] = float("nan")
        got = api.attention_window(q, k, v, 200, 4, ln)
        assert torch.equal(got, want)


@pytest.mark.parametrize("lq", [1, 3])
def test_window_single_token_reads_only_its_window(cuda, lq):
    """Keys that no query of the call sees may hold anything."""
    q, k, v = rnd((2, 8, lq, 128), torch.bfloat16, 1), rnd((2, 2, 900, 128), torch.bfloat16, 2), rnd((2, 2, 900, 128), torch.bfloat16, 3)
    want = api.attention_window(q, k, v, 100, 4)
    v[:, :, 4 : 900 - lq - 99] = float("nan")
    k[:, :, 4 : 900 - lq - 99] = float("inf")
    assert torch.equal(api.attention_window(q, k, v, 100, 4), want)


@pytest.mark.parametrize("lq", [1, 2, 33, 200])
def test_window_strides(cuda, lq):
    """[B, L, H, D] storage, keys and values inside one wider buffer, a broadcast key batch, strided output and lengths."""
    dt = torch.bfloat16
    q = rnd((2, lq, 8, 64), dt, 1).transpose(1, 2)
    kv = rnd((2, 500, 2, 2, 64), dt, 2)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    ln = torch.tensor([450, 7, 500, 7], dtype=torch.int32, device=cuda)[::2]
    out = torch.empty((2, lq, 8, 64), dtype=dt, device=cuda).transpose(1, 2)
    got = api.attention_window(q, k, v, 90, 2, ln, out=out)
    exp = attend64(q, [(k, v, seen_mask(2, lq, 500, 90, 2, ln, None))], 64**-0.5)
    check(got, exp, dt, float(v.double().abs().max()))
    kb, vb = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    got = api.attention_window(q, kb, vb, 90, 2, ln)
    check(got, attend64(q, [(kb, vb, seen_mask(2, lq, 500, 90, 2, ln, None))], 64**-0.5), dt, float(v.double().abs().max()))
    # a layout the tensor cores refuse: depth strided by two
    q2, k2, v2 = (rnd((2, h, n, 128), dt, s)[..., ::2] for h, n, s in ((8, lq, 4), (2, 500, 5), (2, 500, 6)))
    got = api.attention_window(q2, k2, v2, 90, 2, ln)
    check(got, attend64(q2, [(k2, v2, seen_mask(2, lq, 500, 90, 2, ln, None))], 64**-0.5), dt, float(v2.double().abs().max()))


def test_window_f32_output_rank_two_and_scale(cuda):
    q, k, v = rnd((40, 64), torch.float16, 1), rnd((90, 64), torch.float16, 2), rnd((90, 64), torch.float16, 3)
    out = torch.empty((40, 64), dtype=torch.float32, device=cuda)
    for scale in (0.3, -0.2, 0.0):
        got = api.attention_window(q, k, v, 20, 1, options=AttentionOptions(scale=scale), out=out)
        seen = seen_mask(1, 40, 90, 20, 1, None, None)
        check(got, attend64(q[None, None], [(k[None, None], v[None, None], seen)], scale)[0, 0], torch.float16,
              float(v.double().abs().max()))
    five = [rnd(s, torch.float32, i) for i, s in enumerate(((2, 3, 4, 5, 16), (3, 2, 9, 16), (2, 1, 2, 9, 16)))]
    got = api.attention_window(*five, 4)
    q5, k5, v5 = five[0].reshape(6, 4, 5, 16), five[1].expand(2, 3, 2, 9, 16).reshape(6, 2, 9, 16), five[2].expand(2, 3, 2, 9, 16).reshape(6, 2, 9, 16)
    check(got.reshape(6, 4, 5, 16), attend64(q5, [(k5, v5, seen_mask(6, 5, 9, 4, 0, None, None))], 0.25), torch.float32, 1.0)


def test_window_equals_causal_attention_when_it_covers_everything(cuda):
    q, k, v = (rnd((1, 4, 300, 64), torch.bfloat16, s) for s in (1, 2, 3))
    got = api.attention_window(q, k, v, 300)
    want = api.attention_low(q, k, v, None, AttentionOptions(causal=0))
    assert (got.float() - want.float()).abs().max() <= 2.0**-7 * float(v.abs().max())


def test_window_large_scores_and_values(cuda):
    """Scores of +-1e4 (one key takes all the weight) and values near the type's maximum stay finite."""
    for dt in (torch.bfloat16, torch.float16):
        q, k, v = rnd((1, 4, 200, 64), dt, 1) * 20, rnd((1, 2, 300, 64), dt, 2) * 20, rnd((1, 2, 300, 64), dt, 3)
        big = 3e38 if dt == torch.bfloat16 else 6e4
        v = (v.sign() * big).to(dt)
        for lq in (1, 200):
            got = api.attention_window(q[:, :, :lq], k, v, 150, 2)
            exp = attend64(q[:, :, :lq], [(k, v, seen_mask(1, lq, 300, 150, 2, None, None))], 0.125)
            err = (got.double() - exp).abs()
            assert torch.isfinite(got).all()
            # scores near 1e4 carry an f32 accumulation error of 64 * 2^-24 * 1e4 * 2 < 0.1 in the exponent
            assert (err <= 0.25 * big).all()


def prefix_case(b, h, hk, d, lq, pre, keys, dtype, lengths=None, offset=None, seed=0):
    q, pk, pv = rnd((b, h, lq, d), dtype, seed), rnd((hk, pre, d), dtype, seed + 1), rnd((hk, pre, d), dtype, seed + 2)
    k, v = rnd((b, hk, keys, d), dtype, seed + 3), rnd((b, hk, keys, d), dtype, seed + 4)
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda") if lengths is not None else None
    got = api.attention_prefix(q, pk, pv, k, v, ln, AttentionOptions(causal=offset))
    parts = [(pk.expand(b, hk, pre, d), pv.expand(b, hk, pre, d), None),
             (k, v, seen_mask(b, lq, keys, 1 << 40, 0, ln, offset))]
    vm = max([float(t.double().abs().max()) for t in (pv, v) if t.numel()] + [1.0])
    check(got, attend64(q, parts, d**-0.5), dtype, vm)
    assert api.device_status() == 0
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("b,lq,pre,keys", [(1, 1, 1, 1), (3, 1, 130, 7), (5, 2, 1000, 65), (2, 33, 257, 33), (40, 1, 513, 200),
                                           (3, 140, 300, 150), (2, 4, 64, 0), (2, 4, 0, 9)])
def test_prefix_sizes(cuda, dtype, d, b, lq, pre, keys):
    prefix_case(b, 8, 2, d, lq, pre, keys, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (12, 1), (32, 8), (40, 2), (144, 1)])
@pytest.mark.parametrize("lq", [1, 3])
def test_prefix_heads(cuda, dtype, heads, lq):
    prefix_case(9, *heads, 64, lq, 300, 40, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq", [1, 2, 30])
def test_prefix_lengths(cuda, dtype, lq):
    """Nothing sampled yet, fewer keys than queries, full, and beyond the allocation (clamped)."""
    prefix_case(5, 8, 2, 128, lq, 400, 96, dtype, lengths=[0, 1, 95, 96, 200])
    prefix_case(5, 8, 2, 128, lq, 0, 96, dtype, lengths=[0, 1, 95, 96, 200])
    prefix_case(2, 8, 2, 128, lq, 200, 96, dtype, offset=3)


def test_prefix_unfilled_cache_is_not_read(cuda):
    for dtype, lq in itertools.product((torch.float32, torch.bfloat16), (1, 20)):
        q, pk, pv = rnd((3, 8, lq, 64), dtype, 1), rnd((2, 333, 64), dtype, 2), rnd((2, 333, 64), dtype, 3)
        k, v = rnd((3, 2, 150, 64), dtype, 4), rnd((3, 2, 150, 64), dtype, 5)
        ln = torch.tensor([20, 77, 130], dtype=torch.int32, device=cuda)
        want = api.attention_prefix(q, pk, pv, k, v, ln)
        for i, n in enumerate(ln.tolist()):
            k[i, :, n:] = float("nan")
            v[i, :, n:] = float("nan")
        assert torch.equal(api.attention_prefix(q, pk, pv, k, v, ln), want)


@pytest.mark.parametrize("lq", [1, 3, 50])
def test_prefix_strides(cuda, lq):
    """[tokens, heads, depth] storage of the prefix, [B, tokens, heads, depth] of the sequences, strided f32 output."""
    dt = torch.float16
    q = rnd((3, lq, 8, 128), dt, 1).transpose(1, 2)
    pkv = rnd((700, 2, 2, 128), dt, 2)
    pk, pv = pkv[:, 0].transpose(0, 1), pkv[:, 1].transpose(0, 1)
    k, v = rnd((3, 60, 2, 128), dt, 3).transpose(1, 2), rnd((3, 60, 2, 128), dt, 4).transpose(1, 2)
    out = torch.empty((3, lq, 8, 128), dtype=torch.float32, device=cuda).transpose(1, 2)
    got = api.attention_prefix(q, pk, pv, k, v, out=out)
    parts = [(pk.expand(3, -1, -1, -1), pv.expand(3, -1, -1, -1), None), (k, v, seen_mask(3, lq, 60, 1 << 40, 0, None, None))]
    check(got, attend64(q, parts, 128**-0.5), dt, 6.0)


def test_prefix_matches_the_joined_cache(cuda):
    """The same call as attention over one cache that repeats the prefix per sequence."""
    q, pk, pv = rnd((4, 8, 1, 64), torch.bfloat16, 1), rnd((2, 900, 64), torch.bfloat16, 2), rnd((2, 900, 64), torch.bfloat16, 3)
    k, v = rnd((4, 2, 100, 64), torch.bfloat16, 4), rnd((4, 2, 100, 64), torch.bfloat16, 5)
    whole = [torch.cat([p.expand(4, -1, -1, -1), t], 2) for p, t in ((pk, k), (pv, v))]
    want = api.attention_low_f32(q, *whole)
    got = api.attention_prefix(q, pk, pv, k, v, out=torch.empty(want.shape, device=cuda))
    assert (got - want).abs().max() <= 2.0**-7 * float(pv.abs().max())


def test_repeated_calls_streams_and_programs(cuda):
    """The same bits call after call, on another stream, and replayed as a recorded program."""
    from forma_b200.program import Program

    q, pk, pv = rnd((6, 8, 1, 128), torch.bfloat16, 1), rnd((2, 3000, 128), torch.bfloat16, 2), rnd((2, 3000, 128), torch.bfloat16, 3)
    k, v = rnd((6, 2, 1500, 128), torch.bfloat16, 4), rnd((6, 2, 1500, 128), torch.bfloat16, 5)
    ln = torch.tensor([1500, 3, 700, 64, 65, 1111], dtype=torch.int32, device=cuda)
    a, b = torch.empty_like(q), torch.empty_like(q)

    def step():
        api.attention_prefix(q, pk, pv, k, v, ln, out=a)
        api.attention_window(q, k, v, 900, 4, ln, out=b)

    step()
    want = a.clone(), b.clone()
    for _ in range(20):
        step()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        step()
        step()
    s.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    p = Program(step)
    a.zero_(), b.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        p.run()
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert api.device_status() == 0


def test_refusals(cuda):
    q, k = rnd((2, 4, 3, 64), torch.bfloat16, 1), rnd((2, 2, 9, 64), torch.bfloat16, 2)
    pk = rnd((2, 5, 64), torch.bfloat16, 3)
    ln = torch.tensor([9, 9], dtype=torch.int32, device=cuda)

    def refused(kind, fn, *args, **kw):
        with pytest.raises(TensorError) as e:
            fn(*args, **kw)
        assert e.value.kind == kind, e.value

    w, p = api.attention_window, api.attention_prefix
    refused("InvalidAttention", w, q, k, k, 0)
    refused("InvalidAttention", w, q, k, k, -1)
    refused("InvalidAttention", w, q, k, k, 4, -1)
    refused("InvalidAttention", w, q, k, k, 4, 0, ln, AttentionOptions(causal=0))
    refused("InvalidAttentionScale", w, q, k, k, 4, options=AttentionOptions(scale=float("nan")))
    refused("LowDtypeMismatch", w, q, k.half(), k, 4)
    refused("Dtype", w, q.float(), k, k, 4)
    refused("Dtype", w, q, k, k, 4, 0, ln.float())
    refused("InvalidInput", w, q, k, k, 4, 0, ln[:1])
    refused("InvalidInput", w, q, k, k, 4, 0, ln.cpu())
    refused("Dtype", w, q, k, k, 4, out=torch.empty_like(q, dtype=torch.float16))
    refused("InvalidInput", w, q, k, k, 4, out=torch.empty((2, 4, 3, 63), dtype=q.dtype, device=cuda))
    refused("InvalidAttention", w, q, k[..., :32], k, 4)
    refused("InvalidAttention", p, q, pk[:1], pk, k, k)
    refused("InvalidAttention", p, q, pk, pk[:, :4], k, k)
    refused("InvalidAttention", p, q, pk[..., :32], pk, k, k)
    refused("InvalidAttention", p, q, pk, pk, k[:1], k[:1])
    refused("InvalidAttention", p, q[0], pk, pk, k[0], k[0])
    refused("LowDtypeMismatch", p, q, pk.half(), pk, k, k)
    refused("InvalidAttention", p, q, pk, pk, k, k, ln, AttentionOptions(causal=1))
    # empty outputs return before any launch
    assert w(q[:, :, :0], k, k, 4).shape == (2, 4, 0, 64)
    assert p(q[:0], pk, pk, k[:0], k[:0]).shape == (0, 4, 3, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,sinks,window,offset", [(40, 5, 30, 100), (200, 5, 30, 60), (40, 0, 30, 100), (70, 17, 9, 200),
                                                    (33, 130, 20, 135), (40, 3, 500, 20), (50, 7, 4, 5000), (1, 5, 30, 100)])
def test_window_keys_hidden_from_every_query_may_hold_anything(cuda, dtype, d, lq, sinks, window, offset):
    """NaN and infinities between the first keys and the windows and past the
    last position (a cache whose middle was given away) do not reach the result."""
    keys = 400
    q, k, v = rnd((2, 4, lq, d), dtype, 40), rnd((2, 2, keys, d), dtype, 41), rnd((2, 2, keys, d), dtype, 42)
    seen = seen_mask(2, lq, keys, window, sinks, None, offset)
    exp = attend64(q, [(k, v, seen)], d**-0.5)
    top = float(v.double().abs().max())
    hidden = ~seen.any(1)[0]
    assert hidden.any()
    k[:, :, hidden], v[:, :, hidden] = torch.nan, torch.inf
    v[:, 0, hidden] = torch.nan
    check(api.attention_window(q, k, v, window, sinks, None, AttentionOptions(causal=offset)), exp, dtype, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq", [20, 90])
def test_window_lengths_and_hidden_middle(cuda, dtype, lq):
    """The same for filled lengths, a sequence each."""
    keys, sinks, window = 600, 9, 50
    ln = torch.tensor([600, 333, 150, lq], dtype=torch.int32, device="cuda")
    q, k, v = rnd((4, 2, lq, 128), dtype, 43), rnd((4, 1, keys, 128), dtype, 44), rnd((4, 1, keys, 128), dtype, 45)
    seen = seen_mask(4, lq, keys, window, sinks, ln, None)
    exp = attend64(q, [(k, v, seen)], 128**-0.5)
    top = float(v.double().abs().max())
    for b in range(4):
        hidden = ~seen[b].any(0)
        k[b, :, hidden], v[b, :, hidden] = torch.inf, torch.nan
    check(api.attention_window(q, k, v, window, sinks, ln), exp, dtype, top)


@pytest.mark.parametrize("lq", [2, 40])
def test_prefix_keys_past_the_last_query_may_hold_anything(cuda, lq):
    q, pk, pv = rnd((2, 4, lq, 64), torch.bfloat16, 46), rnd((2, 70, 64), torch.bfloat16, 47), rnd((2, 70, 64), torch.bfloat16, 48)
    k, v = rnd((2, 2, 100, 64), torch.bfloat16, 49), rnd((2, 2, 100, 64), torch.bfloat16, 50)
    seen = seen_mask(2, lq, 100, 1 << 30, 0, None, 3)
    exp = attend64(q, [(pk[None].expand(2, -1, -1, -1), pv[None].expand(2, -1, -1, -1), None), (k, v, seen)], 64**-0.5)
    top = max(float(v.double().abs().max()), float(pv.double().abs().max()))
    k[:, :, 3 + lq:], v[:, :, 3 + lq:] = torch.nan, torch.nan
    check(api.attention_prefix(q, pk, pv, k, v, None, AttentionOptions(causal=3)), exp, torch.bfloat16, top)


def routes(fn):
    fn()
    return api.last_route()


def test_routes(cuda):
    """Which kernels serve which shapes: tiles from 17 rows per key/value head
    on, the streaming kernel below, the generic one for other geometries."""
    def window(lq, d, dtype, keys=300, b=2):
        q, k = rnd((b, 4, lq, d), dtype, 1), rnd((b, 2, keys, d), dtype, 2)
        return routes(lambda: api.attention_window(q, k, k, 100, 4))

    def prefix(lq, d, dtype):
        q, k, pk = rnd((2, 4, lq, d), dtype, 1), rnd((2, 2, 30, d), dtype, 2), rnd((2, 500, d), dtype, 3)
        return routes(lambda: api.attention_prefix(q, pk, pk, k, k))

    assert window(9, 128, torch.bfloat16) == ["span_tile_kernel<128,0>"]
    assert window(9, 64, torch.float16) == ["span_tile_kernel<64,0>"]
    assert window(8, 128, torch.bfloat16) == ["span_decode_kernel<128,1,4>"]
    assert window(1, 64, torch.float16) == ["span_decode_kernel<64,0,4>"]
    assert window(1, 64, torch.float16, b=400) == ["span_decode_kernel<64,0,2>"]
    assert window(9, 40, torch.bfloat16) == ["span_simt_kernel"]
    assert window(1, 128, torch.float32) == ["span_simt_kernel"]
    got = prefix(1, 128, torch.bfloat16)
    assert got[0] == "span_tile_kernel<128,1>" and got[1].startswith("span_decode_kernel<128,1,"), got
    got = prefix(40, 64, torch.float16)
    assert got == ["span_tile_kernel<64,1>", "span_tile_kernel<64,0>", "span_merge_kernel<64>"], got
    assert prefix(3, 24, torch.bfloat16) == ["span_simt_kernel"]


@pytest.mark.parametrize("lq,d", [(1, 128), (40, 128), (2, 40)])
def test_caches_past_32_bit_offsets(cuda, lq, d):
    """Windows behind 2^32 elements of one head's cache; what lies between the
    first keys and the windows is whatever the memory held."""
    keys, window, sinks = (1 << 32) // d + 5000, 300, 4
    q = rnd((1, 2, lq, d), torch.bfloat16, 60)
    k, v = (torch.empty((1, 1, keys, d), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    first, tail = sinks, window + lq - 1
    for t, s in ((k, 61), (v, 62)):
        t[:, :, :first], t[:, :, keys - tail:] = rnd((1, 1, first, d), torch.bfloat16, s), rnd((1, 1, tail, d), torch.bfloat16, s + 5)
    got = api.attention_window(q, k, v, window, sinks, torch.tensor([keys], dtype=torch.int32, device=cuda))
    kk, vv = (torch.cat([t[:, :, :first], t[:, :, keys - tail:]], 2) for t in (k, v))
    exp = attend64(q, [(kk, vv, seen_mask(1, lq, first + tail, window, sinks, None, None))], d**-0.5)
    check(got, exp, torch.bfloat16, float(vv.double().abs().max()))
    assert api.device_status() == 0
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("b,lq", [(300, 1), (700, 1), (150, 6), (37, 20)])
def test_window_many_ragged_sequences(cuda, b, lq):
    """More sequences than a block scans at once, lengths from 0 to all keys."""
    keys = 900
    g = torch.Generator().manual_seed(b)
    ln = torch.randint(0, keys + 1, (b,), generator=g).tolist()
    ln[0], ln[-1] = 0, keys
    for dtype in (torch.bfloat16, torch.float16):
        window_case(b, 4, 2, 64, lq, keys, 200, 3, dtype, ln)


@pytest.mark.parametrize("b", [3, 130])
@pytest.mark.parametrize("lq", [1, 17])
def test_prefix_ragged_sequences(cuda, b, lq):
    keys = 600
    g = torch.Generator().manual_seed(b)
    ln = torch.randint(0, keys + 1, (b,), generator=g, dtype=torch.int32)
    ln[0] = 0
    q, pk, pv = rnd((b, 8, lq, 128), torch.bfloat16, 70), rnd((2, 777, 128), torch.bfloat16, 71), rnd((2, 777, 128), torch.bfloat16, 72)
    k, v = rnd((b, 2, keys, 128), torch.bfloat16, 73), rnd((b, 2, keys, 128), torch.bfloat16, 74)
    got = api.attention_prefix(q, pk, pv, k, v, ln.cuda())
    seen = seen_mask(b, lq, keys, 1 << 30, 0, ln.cuda(), None)
    exp = attend64(q, [(pk[None].expand(b, -1, -1, -1), pv[None].expand(b, -1, -1, -1), None), (k, v, seen)], 128**-0.5)
    check(got, exp, torch.bfloat16, max(float(v.double().abs().max()), float(pv.double().abs().max())))
    assert api.device_status() == 0


@pytest.mark.parametrize("lq,b,low", [(300, 900, True), (120, 1300, False)])
def test_prefix_more_records_than_are_kept_at_once(cuda, lq, b, low):
    """A batch whose intermediate results exceed the scratch bound runs in
    parts: sequences of every part against the same sequences alone."""
    keys = lq + 10
    g = torch.Generator().manual_seed(9)
    ln = torch.randint(lq // 2, keys + 1, (b,), generator=g, dtype=torch.int32).cuda()
    q = rnd((b, 8, lq, 64 if low else 128), torch.bfloat16, 90)
    d = q.shape[-1]
    pk, pv = rnd((2, 200, d), torch.bfloat16, 91), rnd((2, 200, d), torch.bfloat16, 92)
    k, v = rnd((b, 2, keys, d), torch.bfloat16, 93), rnd((b, 2, keys, d), torch.bfloat16, 94)
    out = torch.full(q.shape, torch.nan, dtype=torch.bfloat16 if low else torch.float32, device=cuda)
    api.attention_prefix(q, pk, pv, k, v, ln, out=out)
    assert len(api.last_route()) > 3
    assert torch.isfinite(out).all()
    some = [0, 1, b // 3, b // 2, (2 * b) // 3, b - 2, b - 1]
    exp = attend64(q[some], [(pk[None].expand(len(some), -1, -1, -1), pv[None].expand(len(some), -1, -1, -1), None),
                             (k[some], v[some], seen_mask(len(some), lq, keys, 1 << 30, 0, ln[some], None))], d**-0.5)
    top = max(float(v.double().abs().max()), float(pv.double().abs().max()))
    got = out[some]
    check(got, exp, torch.bfloat16, top)
    assert api.device_status() == 0


@pytest.mark.parametrize("lengths,causal", [([39990], None), (None, None), (None, 100)])
def test_prefix_one_sequence_past_the_record_bound(cuda, lengths, causal):
    """One sequence whose intermediate results exceed the scratch bound runs in
    parts of its queries: rows around the parts' borders against the plain
    form, and no more scratch than the bound on a stream of its own."""
    h, hk, d, lq, pre, keys = 32, 4, 128, 40000, 300, 40000
    q, pk, pv = rnd((1, h, lq, d), torch.bfloat16, 100), rnd((hk, pre, d), torch.bfloat16, 101), rnd((hk, pre, d), torch.bfloat16, 102)
    k, v = rnd((1, hk, keys, d), torch.bfloat16, 103), rnd((1, hk, keys, d), torch.bfloat16, 104)
    ln = torch.tensor(lengths, dtype=torch.int32, device=cuda) if lengths else None
    got = torch.full_like(q, torch.nan)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    free = torch.cuda.mem_get_info()[0]
    with torch.cuda.stream(s):
        api.attention_prefix(q, pk, pv, k, v, ln, AttentionOptions(causal=causal), out=got)
    s.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= (1 << 30) + (64 << 20)
    assert len(api.last_route()) > 3
    assert torch.isfinite(got).all()
    rows = [0, 1, 9, 10, 11, 127, 128, 20000, 32127, 32128, 32255, 32256, 32257, 39871, 39999]
    n = (lengths or [keys])[0]
    p = torch.tensor(rows, device=cuda) + (n - lq if causal is None else causal)
    j = torch.arange(keys, device=cuda)
    seen = ((j[None] <= p[:, None]) & (j[None] < n))[None]
    exp = attend64(q[:, :, rows], [(pk[None], pv[None], None), (k, v, seen)], d**-0.5)
    check(got[:, :, rows], exp, torch.bfloat16, max(float(v.double().abs().max()), float(pv.double().abs().max())))
    assert api.device_status() == 0
