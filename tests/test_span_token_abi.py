"""Checks of the span attentions and the token log probabilities that need no
GPU: argument errors come before any device work.  The descriptors point at
no real memory, so a launch would fail differently (FB_ERR_DRIVER)."""

import ctypes as C

import pytest

from forma_b200 import _lib, api
from forma_b200.api import AttentionOptions



def desc(dims, dtype=_lib.BF16, strides=None, storage=None, ptr=0x10000):
    d = _lib.FbTensor()
    d.data, d.dtype, d.rank = ptr, dtype, len(dims)
    st = strides
    if st is None:
        st, s = [0] * len(dims), 1
        for i in range(len(dims) - 1, -1, -1):
            st[i] = s
            s *= dims[i]
    n = 1
    for x in dims:
        n *= x
    for i, (x, s) in enumerate(zip(dims, st)):
        d.dims[i], d.strides[i] = x, s
    d.storage_len = storage if storage is not None else n
    return d


def ref(d):
    return None if d is None else C.byref(d)



def window(q, k, v, o, lengths=None, window=4, sinks=0, **opts):
    return api.lib().fb_attention_window(ref(q), ref(k), ref(v), ref(lengths), window, sinks,
                                         api._attn_options(AttentionOptions(**opts)), ref(o), None)


def prefix(q, pk, pv, k, v, o, lengths=None, **opts):
    return api.lib().fb_attention_prefix(ref(q), ref(pk), ref(pv), ref(k), ref(v), ref(lengths),
                                         api._attn_options(AttentionOptions(**opts)), ref(o), None)


def raises(code, kind):
    with pytest.raises(api.TensorError) as e:
        api._check(code)
    assert e.value.kind == kind, e.value


def test_window_arguments():
    q, k, o = desc([2, 4, 3, 64]), desc([2, 2, 9, 64]), desc([2, 4, 3, 64])
    raises(window(None, k, k, o), "InvalidInput")
    raises(window(q, k, k, None), "InvalidInput")
    raises(window(q, k, k, o, window=0), "InvalidAttention")
    raises(window(q, desc([2, 3, 9, 64]), desc([2, 3, 9, 64]), o), "InvalidAttention")        # 4 heads over 3
    raises(window(q, k, desc([2, 2, 8, 64]), o), "InvalidAttention")                          # key and value lengths
    raises(window(q, desc([2, 2, 9, 32]), k, o), "InvalidAttention")                          # depths
    raises(window(q, desc([2, 2, 9, 64], _lib.F16), k, o), "LowDtypeMismatch")
    raises(window(desc([2, 4, 3, 64], _lib.F32), k, k, o), "Dtype")
    raises(window(q, k, k, desc([2, 4, 3, 64], _lib.F16)), "Dtype")
    raises(window(q, k, k, desc([2, 4, 2, 64])), "InvalidInput")
    raises(window(q, k, k, desc([2, 4, 3, 64], strides=[768, 0, 64, 1])), "InvalidInput")     # rows on one another
    raises(window(q, k, k, o, scale=float("inf")), "InvalidAttentionScale")
    ln = desc([2], _lib.U32)
    raises(window(q, k, k, o, ln, causal=1), "InvalidAttention")
    raises(window(q, k, k, o, desc([2], _lib.F32)), "Dtype")
    raises(window(q, k, k, o, desc([3], _lib.U32)), "InvalidInput")
    raises(window(q, k, k, o, desc([2, 1], _lib.U32)), "InvalidInput")
    assert window(desc([2, 4, 3, 64], storage=100), k, k, o) == 7                             # storage bounds
    # empty results return before any device work, whatever the window and the lengths
    assert window(desc([2, 4, 0, 64]), k, k, desc([2, 4, 0, 64]), ln, 1 << 63, 1 << 63) == 0
    assert window(desc([0, 4, 3, 64]), desc([0, 2, 9, 64]), desc([0, 2, 9, 64]), desc([0, 4, 3, 64])) == 0


def test_prefix_arguments():
    q, k, o = desc([2, 4, 3, 64]), desc([2, 2, 9, 64]), desc([2, 4, 3, 64])
    p = desc([2, 70, 64])
    raises(prefix(q, None, p, k, k, o), "InvalidInput")
    raises(prefix(q, p, desc([2, 69, 64]), k, k, o), "InvalidAttention")
    raises(prefix(q, desc([1, 70, 64]), desc([1, 70, 64]), k, k, o), "InvalidAttention")      # heads
    raises(prefix(q, desc([2, 70, 32]), p, k, k, o), "InvalidAttention")
    raises(prefix(q, desc([1, 2, 70, 64]), p, k, k, o), "InvalidAttention")                   # rank
    raises(prefix(q, desc([2, 70, 64], _lib.F16), p, k, k, o), "LowDtypeMismatch")
    raises(prefix(q, p, p, desc([1, 2, 9, 64]), k, o), "InvalidAttention")                    # one batch
    raises(prefix(desc([4, 3, 64]), p, p, desc([2, 9, 64]), desc([2, 9, 64]), desc([4, 3, 64])), "InvalidAttention")
    raises(prefix(q, p, p, k, k, o, desc([2], _lib.U32), causal=0), "InvalidAttention")
    assert prefix(desc([0, 4, 3, 64]), p, p, desc([0, 2, 9, 64]), desc([0, 2, 9, 64]), desc([0, 4, 3, 64])) == 0


def test_token_logprob_arguments():
    lib = api.lib()
    x, t, f = desc([5, 100]), desc([5], _lib.U32), desc([5], _lib.F32)
    tl, ti = desc([5, 7], _lib.F32), desc([5, 7], _lib.U32)

    def fwd(x=x, t=t, lp=f, h=f, lse=f, tl=None, ti=None):
        return lib.fb_token_logprobs(ref(x), ref(t), ref(lp), ref(h), ref(lse), ref(tl), ref(ti), None)

    raises(fwd(x=None), "InvalidInput")
    raises(fwd(t=None), "InvalidInput")                        # a log probability needs targets
    raises(fwd(x=desc([5, 100], _lib.U32)), "Dtype")
    raises(fwd(x=desc([], _lib.F32), t=desc([], _lib.U32)), "InvalidInput")
    raises(fwd(t=desc([4], _lib.U32)), "InvalidInput")
    raises(fwd(t=desc([5], _lib.F32)), "Dtype")
    raises(fwd(h=desc([5], _lib.BF16)), "Dtype")
    raises(fwd(lse=desc([6], _lib.F32)), "InvalidInput")
    raises(fwd(tl=tl), "InvalidInput")                         # the two go together
    raises(fwd(tl=desc([5, 65], _lib.F32), ti=desc([5, 65], _lib.U32)), "InvalidInput")
    raises(fwd(x=desc([5, 6]), tl=tl, ti=ti), "InvalidInput")  # more alternatives than classes
    raises(fwd(tl=tl, ti=desc([5, 6], _lib.U32)), "InvalidInput")
    raises(fwd(tl=desc([5, 7], _lib.F32, strides=[8, 1], storage=40), ti=ti), "InvalidInput")
    raises(fwd(tl=tl, ti=desc([5, 7], _lib.F32)), "Dtype")
    raises(fwd(x=desc([5, 0])), "EmptyReduction")
    e = desc([0], _lib.F32)
    assert fwd(x=desc([0, 100]), t=desc([0], _lib.U32), lp=e, h=e, lse=e) == 0
    assert fwd(lp=None, h=None, lse=None) == 0                 # nothing asked for


def test_token_gradient_arguments():
    lib = api.lib()
    x, t, f, g = desc([5, 100]), desc([5], _lib.U32), desc([5], _lib.F32), desc([5, 100], ptr=0x900000)

    def bwd(x=x, t=t, lse=f, gl=f, h=None, gh=None, g=g):
        return lib.fb_token_logprobs_grad(ref(x), ref(t), ref(lse), ref(gl), ref(h), ref(gh), ref(g), None)

    raises(bwd(t=None), "InvalidInput")
    raises(bwd(lse=None), "InvalidInput")
    raises(bwd(gl=None), "InvalidInput")
    raises(bwd(g=None), "InvalidInput")
    raises(bwd(gh=f), "InvalidInput")                          # an entropy gradient needs the entropy
    raises(bwd(gl=desc([5], _lib.F16)), "Dtype")
    raises(bwd(g=desc([5, 100], _lib.F16)), "Dtype")
    raises(bwd(g=desc([5, 99], ptr=0x900000)), "InvalidInput")
    raises(bwd(x=desc([5, 0]), g=desc([5, 0])), "EmptyReduction")
    raises(bwd(g=desc([5, 100], ptr=0x10000 + 64)), "InvalidInput")                  # overlaps the logits
    raises(bwd(g=desc([5, 100], strides=[1, 5], ptr=0x10000)), "InvalidInput")       # the same memory, another view
    raises(bwd(g=desc([5, 100], _lib.F32, ptr=0x10000)), "InvalidInput")             # in place needs the logits' type
    e = desc([0], _lib.F32)
    assert bwd(x=desc([0, 9]), t=desc([0], _lib.U32), lse=e, gl=e, g=desc([0, 9])) == 0


def test_token_gradient_layouts():
    """Rows with gaps are an output (the launch then needs a GPU); rows on one another are not."""
    lib = api.lib()
    x, t, f = desc([5, 100]), desc([5], _lib.U32), desc([5], _lib.F32)

    def bwd(g):
        return lib.fb_token_logprobs_grad(ref(x), ref(t), ref(f), ref(f), None, None, ref(g), None)

    raises(bwd(desc([5, 100], strides=[99, 1], storage=600, ptr=0x900000)), "InvalidInput")
    raises(bwd(desc([5, 100], strides=[0, 1], ptr=0x900000)), "InvalidInput")
    raises(bwd(desc([5, 100], strides=[1, 4], storage=600, ptr=0x900000)), "InvalidInput")
