"""Token log probabilities, entropy, alternatives and the gradient against the
definitions in 64 bits.

Tolerance.  With n classes and |x - lse| <= R over the classes that carry
weight: each exponential is off by at most 2^-21 relative (2 ulp of the
hardware exponential, the rounding of x - m and of its scaling), sums add
2^-24 per level of their trees, so S0 is off by less than 2^-20 relative, lse
by 2^-20 + 2^-24 |lse|, the entropy (a weighted mean of |z| <= R plus lse's
error) by 2^-20 (1 + 2 R).  The gradient adds exp's error at z: p is off by
2^-20 (1 + |z| 2^-3) relative, and is rounded once to a 16-bit type."""

import math

import numpy as np
import pytest
import torch

from forma_b200 import api
from forma_b200.api import NO_TOKEN, TensorError

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rnd(shape, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def targets_for(x, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda", generator=g, dtype=torch.int32)
    return t


def order(x, k):
    """Top k by (IEEE total order, lowest index)."""
    bits = x.float().cpu().numpy().view(np.uint32).reshape(-1, x.shape[-1])
    keys = np.where(bits & 0x80000000, ~bits, bits | 0x80000000).astype(np.int64)
    idx = np.argsort(-keys, axis=1, kind="stable")[:, :k]
    return idx.reshape(*x.shape[:-1], k)


def check_forward(x, t, k, r=None):
    r = r or api.token_logprobs(x, t, k)
    y = x.double()
    lse = torch.logsumexp(y, -1)
    logp = y - lse[..., None]
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    span = float(ent.max()) + 2 * math.log(x.shape[-1]) + 1
    e0 = 2.0**-20
    assert ((r.logsumexp.double() - lse).abs() <= e0 + 2.0**-23 * lse.abs()).all()
    assert ((r.entropy.double() - ent).abs() <= e0 * (1 + 2 * span)).all(), ((r.entropy.double() - ent).abs().max(), span)
    if t is not None:
        want = logp.gather(-1, t.long().clamp(min=0)[..., None])[..., 0] * (t >= 0)
        assert ((r.logprob.double() - want).abs() <= e0 + 2.0**-23 * (lse.abs() + want.abs())).all()
        assert (r.logprob[t < 0] == 0).all()
    if k:
        idx = order(x, k)
        assert (r.top_index.cpu().numpy() == idx).all()
        want = logp.gather(-1, torch.from_numpy(idx.astype(np.int64)).cuda())
        got = r.top_logprob.double()
        fine = torch.isfinite(want)
        assert (got[~fine] == want[~fine]).all()
        assert ((got - want)[fine].abs() <= (e0 + 2.0**-23 * (lse.abs()[..., None] + want.abs()))[fine]).all()
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (5, 64, 64), (2, 1000, 20), (300, 1024, 3), (7, 4099, 33),
                                           (1, 50021, 20), (40, 32000, 8), (3, 131072, 32), (2, 300001, 64), (200, 9000, 1)])
def test_forward_sizes(cuda, dtype, rows, cols, top):
    x = rnd((rows, cols), dtype, rows + cols)
    t = targets_for(x, 1)
    t[-1] = NO_TOKEN
    check_forward(x, t, top)
    check_forward(x, t, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_masked_classes(cuda, dtype):
    """-inf and the type's lowest value in most places, weight on one class, a shift far from zero."""
    x = rnd((6, 20000), dtype, 3)
    x[0, 100:] = -torch.inf
    x[1, :19999] = -torch.inf
    x[2, ::2] = torch.finfo(dtype).min
    x[3, 1:] = torch.finfo(dtype).min
    x[4] -= 3000.0
    x[5, 777] = 60.0
    t = torch.tensor([5, 19999, 1, 0, 17, 777], dtype=torch.int32, device=cuda)
    r = check_forward(x, t, 12)
    assert float(r.entropy[1]) == 0.0 and float(r.logprob[1]) == 0.0
    r = api.token_logprobs(x, torch.tensor([200, 5, 0, 9, 17, 777], dtype=torch.int32, device=cuda))
    assert float(r.logprob[0]) == -math.inf  # a masked class has no probability


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_extreme_rows(cuda, dtype):
    """NaN, +inf and all -inf rows give NaN; their neighbours are untouched."""
    x = rnd((5, 5000), dtype, 4)
    x[1, 4321] = torch.nan
    x[2, 17] = torch.inf
    x[3] = -torch.inf
    t = targets_for(x, 2)
    r = api.token_logprobs(x, t, 4)
    for i in (1, 2, 3):
        assert torch.isnan(r.entropy[i]) and torch.isnan(r.logprob[i])
    check_forward(x[[0, 4]], t[[0, 4]], 4)
    assert (r.top_index.cpu().numpy() == order(x, 4)).all()
    assert torch.equal(r.logsumexp[[0, 4]], api.token_logprobs(x[[0, 4]], t[[0, 4]], 4).logsumexp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [70, 5000, 131072])
def test_forward_ties(cuda, dtype, cols):
    """Equal logits: the lowest indices, in order; both zeros (-0 < +0); few distinct values; ascending and descending rows."""
    x = torch.zeros((6, cols), dtype=dtype, device=cuda)
    x[1, cols // 2 :] = 1.0
    x[2] = -0.0
    x[2, cols - 3] = 0.0
    x[3] = (torch.arange(cols, device=cuda) % 7).to(dtype)
    x[4] = torch.linspace(-8, 8, cols, device=cuda).to(dtype)
    x[5] = torch.linspace(8, -8, cols, device=cuda).to(dtype)
    check_forward(x, targets_for(x, 3), 64)
    check_forward(x, targets_for(x, 3), 5)


def test_forward_out_of_range_targets(cuda):
    x = rnd((3, 100), torch.bfloat16, 5)
    r = api.token_logprobs(x, torch.tensor([100, -2, NO_TOKEN], dtype=torch.int32, device=cuda))
    assert torch.isnan(r.logprob[:2]).all() and float(r.logprob[2]) == 0.0
    assert torch.isfinite(r.entropy).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_forward_layouts(cuda, dtype):
    """Leading dims, row strides that break alignment, an offset, a class stride, transposed targets."""
    base = rnd((4, 3, 5003), dtype, 6)
    check_forward(base, targets_for(base, 1), 6)
    check_forward(base[:, :, 1:], targets_for(base, 2), 6)
    check_forward(base[..., ::3], targets_for(base[..., ::3], 3), 6)
    wide = rnd((4, 8192), dtype, 7)
    check_forward(wide[:, :5000], targets_for(wide[:, :5000], 4), 6)
    check_forward(wide[:, 8:4104], targets_for(wide[:, 8:4104], 5), 6)
    check_forward(base.transpose(0, 1), targets_for(base, 6).t(), 6)
    check_forward(wide[:, :1].expand(4, 4096), targets_for(wide[:, :4096], 8), 6)
    vec = rnd((5003,), dtype, 8)
    check_forward(vec, torch.tensor(9, dtype=torch.int32, device=cuda), 6)
    assert api.token_logprobs(base[:0], targets_for(base, 1)[:0], 2).top_index.shape == (0, 3, 2)


def test_forward_equals_the_package_s_row_operators(cuda):
    x = rnd((64, 4096), torch.float32, 9)
    r = api.token_logprobs(x, None, 1)
    assert r.logprob is None
    assert (r.logsumexp - api.logsumexp(x, [1])).abs().max() <= 2e-6
    assert torch.equal(r.top_index[:, 0], api.argmax(x, 1))


def grad64(x, t, gl, gh):
    y = x.double()
    logp = y - torch.logsumexp(y, -1, keepdim=True)
    p = logp.exp()
    g = torch.where(t >= 0, gl.double(), torch.zeros_like(gl, dtype=torch.float64))
    d = -p * g[..., None]
    d.scatter_add_(-1, t.long().clamp(min=0)[..., None], g[..., None])
    if gh is not None:
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        d -= gh.double()[..., None] * (plogp - p * plogp.sum(-1, keepdim=True))
    return d, p, logp


def check_grad(x, t, gl, gh, out=None):
    st = api.token_logprobs(x, t)
    want, p, logp = grad64(x, t, gl, gh)
    got = api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy if gh is not None else None, gh, out)
    z = torch.where(p > 0, logp.abs(), torch.zeros_like(p))
    lse = torch.logsumexp(x.double(), -1, keepdim=True).abs()
    rel = 2.0**-20 * (1 + z / 8) + 2.0**-23 * (lse + z)  # of p: the exponential's error and z's rounding
    bound = rel * p * gl.double().abs()[..., None] + 2.0**-22 * want.abs()
    if gh is not None:
        h = -(torch.where(p > 0, p * logp, torch.zeros_like(p))).sum(-1, keepdim=True)
        bound = bound + gh.double().abs()[..., None] * p * ((z + h) * rel * 2 + 2.0**-20 * (2 + z + 4 * h))
    if got.dtype != torch.float32:
        u, tiny = (2.0**-8, 1e-38) if got.dtype == torch.bfloat16 else (2.0**-11, 2.0**-25)
        bound = bound * 2 + u * want.abs() + tiny
    else:
        bound = bound + 1e-38
    err = (got.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 1000), (300, 1024), (7, 4099), (1, 50021), (40, 32000), (3, 131072)])
@pytest.mark.parametrize("entropy", [False, True])
def test_grad_sizes(cuda, dtype, rows, cols, entropy):
    x = rnd((rows, cols), dtype, rows + cols)
    t = targets_for(x, 1)
    gl, gh = rnd((rows,), torch.float32, 2), rnd((rows,), torch.float32, 3) if entropy else None
    if rows > 1:
        t[1] = NO_TOKEN
    got = check_grad(x, t, gl, gh)
    if rows > 1 and not entropy:
        assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_masked_rows_and_layouts(cuda, dtype):
    x = rnd((4, 9000), dtype, 4)
    x[0, 10:] = -torch.inf
    x[1, ::2] = torch.finfo(dtype).min
    t = torch.tensor([3, 1, 8999, NO_TOKEN], dtype=torch.int32, device=cuda)
    gl, gh = rnd((4,), torch.float32, 5), rnd((4,), torch.float32, 6)
    check_grad(x, t, gl, gh)
    check_grad(x, t, gl, gh, torch.empty(x.shape, device=cuda))  # f32 gradient
    check_grad(x[:, 1:], t.clamp(max=8998), gl, gh)
    check_grad(x[:, ::2], t.clamp(max=4499), gl, gh)
    wide = rnd((4, 9008), dtype, 7)
    check_grad(wide[:, :9000], t, gl, gh)
    check_grad(wide[:, 8:], t, gl, gh, torch.empty((9000, 4), dtype=dtype, device=cuda).t())
    check_grad(x, t, gl[:1].expand(4), gh)
    # a row without a probability: zeros where its gradients are zero
    x[2] = -torch.inf
    gl[2] = gh[2] = 0.0
    st = api.token_logprobs(x, t)
    assert (api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy, gh)[2] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_in_place(cuda, dtype):
    x = rnd((50, 5000), dtype, 8)
    t, gl, gh = targets_for(x, 1), rnd((50,), torch.float32, 2), rnd((50,), torch.float32, 3)
    st = api.token_logprobs(x, t)
    want = api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy, gh)
    got = api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy, gh, out=x)
    assert got is x and torch.equal(got, want)


def test_grad_against_differences(cuda):
    """Central differences of the forward operator in f32: the step's rounding
    error 2^-20 (|lse| + 1) / h and its curvature h^2 bound the difference."""
    x = rnd((2, 40), torch.float32, 9, 1.0)
    t = torch.tensor([3, 39], dtype=torch.int32, device=cuda)
    gl, gh = torch.tensor([1.0, -0.5], device=cuda), torch.tensor([0.7, 2.0], device=cuda)
    st = api.token_logprobs(x, t)
    g = api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy, gh)
    h = 2.0**-6
    steps = torch.eye(40, device=cuda)[:, None] * h
    def f(y):
        r = api.token_logprobs(y, t.expand(40, 2).contiguous())
        return r.logprob.double() * gl + r.entropy.double() * gh
    num = ((f(x + steps) - f(x - steps)) / (2 * h)).t()
    assert (num - g.double()).abs().max() <= 2.0**-20 * 12 * 3 / h + 3 * h * h


def test_same_bits_every_call_and_on_other_streams(cuda):
    for rows, cols in ((1, 131072), (3, 50021), (70, 32000), (600, 2000)):
        x = rnd((rows, cols), torch.bfloat16, 10)
        t = targets_for(x, 1)
        a = api.token_logprobs(x, t, 20)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs = [api.token_logprobs(x, t, 20) for _ in range(5)]
        s.synchronize()
        for b in outs:
            assert all(torch.equal(getattr(a, n), getattr(b, n)) for n in ("logprob", "entropy", "logsumexp", "top_logprob", "top_index"))
    assert api.device_status() == 0


def test_refusals(cuda):
    x = rnd((4, 100), torch.bfloat16, 1)
    t = targets_for(x, 1)

    def refused(kind, fn, *args, **kw):
        with pytest.raises(TensorError) as e:
            fn(*args, **kw)
        assert e.value.kind == kind, e.value

    f, g = api.token_logprobs, api.token_logprobs_grad
    st = f(x, t)
    refused("InvalidInput", f, x, t[:3])
    refused("Dtype", f, x, t.float())
    refused("Dtype", f, x.int(), t)
    refused("InvalidInput", f, x, t, 65)
    refused("InvalidInput", f, x[:, :10], t, 11)
    refused("EmptyReduction", f, x[:, :0], t)
    refused("InvalidInput", f, x, t.cpu())
    gl = torch.ones(4, device=cuda)
    refused("InvalidInput", g, x, t, st.logsumexp[:2], gl)
    refused("Dtype", g, x, t, st.logsumexp, gl.double())
    refused("Dtype", g, x, t, st.logsumexp, gl.half())
    refused("InvalidInput", g, x, t, st.logsumexp, gl, None, gl)  # an entropy gradient needs the entropy
    refused("Dtype", g, x, t, st.logsumexp, gl, out=torch.empty_like(x, dtype=torch.float16))
    refused("InvalidInput", g, x, t, st.logsumexp, gl, out=torch.empty((4, 99), dtype=x.dtype, device=cuda))
    both = torch.empty((5, 100), dtype=x.dtype, device=cuda)
    refused("InvalidInput", g, both[:4], t, st.logsumexp, gl, out=both[1:])


@pytest.mark.parametrize("dtype,cols", [(torch.float32, 1_100_003), (torch.bfloat16, 2_200_001), (torch.float16, 2_200_000)])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_forward_many_classes(cuda, dtype, cols, top):
    """Rows longer than a maximum per segment is kept for."""
    x = rnd((2, cols), dtype, 80)
    check_forward(x, targets_for(x, 81), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(700, 900), (700, 9001), (1300, 20000)])
@pytest.mark.parametrize("top", [0, 5, 33])
def test_forward_rows_that_fill_the_gpu(cuda, dtype, rows, cols, top):
    """More rows than eight-warp blocks are resident: odd columns break the
    rows' alignment; a NaN, a -inf and a constant row among them."""
    x = rnd((rows, cols), dtype, 82)
    t = targets_for(x, 83)
    t[3] = NO_TOKEN
    check_forward(x, t, top)
    x[5, cols // 2], x[6], x[7] = torch.nan, -torch.inf, 1.5
    r = api.token_logprobs(x, t, top)
    assert r.logsumexp[5:7].isnan().all() and r.entropy[5:7].isnan().all()
    keep = [i for i in range(rows) if i not in (5, 6)]
    check_forward(x[keep], t[keep], top, api.TokenLogprobs(*(None if f is None else f[keep] for f in vars(r).values())))


def test_logits_past_32_bit_offsets(cuda):
    """More than 2^32 logits: the last rows' results are those of the rows alone."""
    rows, cols = 33000, 131072
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=cuda)
    for i in range(0, rows, 3000):
        x[i:i + 3000] = rnd((min(3000, rows - i), cols), torch.bfloat16, 84 + i)
    t = torch.arange(rows, device=cuda, dtype=torch.int32) % cols
    r = api.token_logprobs(x, t, 5)
    for part in (slice(0, 3), slice(rows - 3, rows)):
        check_forward(x[part], t[part], 5, api.TokenLogprobs(*(f[part] for f in vars(r).values())))
    gl = torch.ones(rows, device=cuda)
    ends = x[-3:].clone()
    exp = api.token_logprobs_grad(ends, t[-3:], r.logsumexp[-3:], gl[-3:], r.entropy[-3:], gl[-3:])
    api.token_logprobs_grad(x, t, r.logsumexp, gl, r.entropy, gl, out=x)
    assert torch.equal(x[-3:], exp)
    assert api.device_status() == 0
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(3, 7), (5, 4099), (60, 9001), (2, 32000)])
def test_grad_in_f32(cuda, dtype, rows, cols):
    """f32 gradients of 16-bit logits: odd columns move the rows' alignment, an
    offset that keeps it and one that does not."""
    x = rnd((rows, cols), dtype, 85)
    t = targets_for(x, 86)
    gl, gh = rnd((rows,), torch.float32, 87), rnd((rows,), torch.float32, 88)
    check_grad(x, t, gl, gh, torch.empty((rows, cols), device=cuda))
    assert api.last_route() == ["token_grad_stream_kernel"]
    n = rows * cols
    check_grad(x, t, gl, None, torch.empty(n + 4, device=cuda)[4:].view(rows, cols))
    assert api.last_route() == ["token_grad_stream_kernel"]
    got = torch.full((n + 3,), 7.0, device=cuda)
    check_grad(x, t, gl, None, got[1:1 + n].view(rows, cols))
    assert api.last_route() == ["token_grad_rows_kernel"]
    assert got[0] == 7 and (got[1 + n:] == 7).all()


@pytest.mark.parametrize("dtype,cols", [(torch.bfloat16, 16500), (torch.float16, 25000), (torch.float32, 8300), (torch.float32, 16700)])
@pytest.mark.parametrize("top", [17, 20, 21, 50, 64])
def test_forward_parts_with_few_values(cuda, dtype, cols, top):
    """Rows cut into parts whose last one is short: fewer groups of lanes with
    values than alternatives."""
    x = rnd((9, cols), dtype, 89)
    x[2, 40:] = -torch.inf
    t = targets_for(x, 90)
    t[2] = 7
    check_forward(x, t, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,view", [((50, 5000), lambda w: w[:, :4990]), ((50, 5000), lambda w: w[:, 3:4001]),
                                        ((20, 7, 1000), lambda w: w[:, -1]), ((9, 6, 515), lambda w: w[:, ::2, 1:514]),
                                        ((30, 2000), lambda w: w[:, ::2]), ((1, 70000), lambda w: w[:, 8:69999])])
def test_grad_into_rows_of_something_wider(cuda, dtype, shape, view):
    """In place on a part of a padded buffer, and into a part of another: what
    lies between the rows keeps its bits."""
    wide = rnd(shape, dtype, 11)
    x = view(wide)
    t = targets_for(x, 1)
    gl, gh = rnd(t.shape, torch.float32, 2), rnd(t.shape, torch.float32, 3)
    st = api.token_logprobs(x, t)
    untouched = torch.ones(shape, dtype=torch.bool, device=cuda)
    view(untouched).fill_(False)
    for out_dtype in (torch.float32, dtype):
        other = torch.full(shape, 7.0, dtype=out_dtype, device=cuda)
        got = check_grad(x, t, gl, gh, view(other))
        assert (other[untouched] == 7.0).all()
    before = wide.clone()
    again = api.token_logprobs_grad(x, t, st.logsumexp, gl, st.entropy, gh, out=x)
    assert again is x and torch.equal(x, got) and torch.equal(wide[untouched], before[untouched])
    assert api.device_status() == 0
