"""The encoder operators without a GPU: exports, and refusals before any device call."""
import ctypes as C

import pytest

from beam_search_collab_amd import _lib
from test_abi import declared

PTR = 1 << 20  # never dereferenced: every call here is refused before it launches


def refused(rc, text):
    assert rc == -1
    assert text in _lib.hip().bs_last_error().decode()


def test_exports():
    names = declared("bs_embed.h")
    assert set(names) == set(_lib.EMBED_API)
    for n in names:
        assert hasattr(_lib.hip(), n)


@pytest.mark.parametrize("change,text", [
    (dict(type=3), "type must be"),
    (dict(type=1, wtype=2), "wtype must be"),
    (dict(cols=0), "cols must be"),
    (dict(cols=16385, x_stride=20000, y_stride=20000), "cols must be"),
    (dict(rows=1 << 31), "rows must be"),
    (dict(eps=-1.0), "eps must be"),
    (dict(eps=float("nan")), "eps must be"),
    (dict(x=None), "x and y must be given"),
    (dict(y=None), "x and y must be given"),
    (dict(x_stride=63), "rows overlap"),
    (dict(y_stride=0), "rows overlap"),
])
def test_layer_norm_refuses(change, text):
    a = dict(x=PTR, x_stride=64, w=None, b=None, wtype=0, eps=1e-5, y=PTR, y_stride=64, mean=None, rstd=None, rows=4, cols=64,
             type=0, stream=None) | change
    refused(_lib.hip().bs_layer_norm(*a.values()), text)


@pytest.mark.parametrize("change,text", [
    (dict(dw=None), "given together"),
    (dict(db=None), "given together"),
    (dict(mean=None), "must be given"),
    (dict(dy=None), "must be given"),
    (dict(dx_stride=5), "rows overlap"),
    (dict(ws=None), "the workspace must hold"),
    (dict(size=16), "the workspace must hold"),
    (dict(ws=PTR + 4), "16-byte aligned"),
    (dict(wtype=1), "wtype must be"),
])
def test_layer_norm_backward_refuses(change, text):
    a = dict(dy=PTR, dys=64, x=PTR, xs=64, mean=PTR, rstd=PTR, w=None, wtype=0, dx=PTR, dx_stride=64, dw=PTR, db=PTR, rows=4,
             cols=64, type=0, ws=PTR, size=1 << 20, stream=None) | change
    refused(_lib.hip().bs_layer_norm_backward(*a.values()), text)


@pytest.mark.parametrize("change,text", [
    (dict(type=0, out_type=0), "type must be"),
    (dict(out_type=1), "out_type must be"),
    (dict(act=5), "unknown activation"),
    (dict(act=-1), "unknown activation"),
    (dict(inner=0), "inner and cols"),
    (dict(cols=(1 << 24) + 1), "inner and cols"),
    (dict(rows=1 << 31), "rows must be"),
    (dict(w=None), "must be given"),
    (dict(xs=31), "rows overlap"),
    (dict(os=47), "rows overlap"),
    (dict(r=PTR, rs=47), "rows overlap"),
    (dict(ws_=1 << 24), "strides must be"),
])
def test_linear_refuses(change, text):
    a = dict(x=PTR, xs=32, w=PTR, ws_=32, b=None, r=None, rs=0, out=PTR, os=48, rows=4, inner=32, cols=48, type=2, out_type=2,
             act=0, ws=None, size=0, stream=None) | change
    refused(_lib.hip().bs_linear(*a.values()), text)


def attention_args(**change):
    a = _lib.AttentionArgs()
    d = dict(q=PTR, k=PTR, v=PTR, out=PTR, q_stride=64, q_head_stride=32, k_stride=32, k_head_stride=32, v_stride=32,
             v_head_stride=32, out_stride=64, out_head_stride=32, q_tokens=3, k_tokens=5, sequences=1, heads=2, kv_heads=1,
             head_dim=32, type=2, causal=1, scale=1.0) | change
    for n, x in d.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(type=0), "type must be"),
    (dict(head_dim=20), "head_dim must be"),
    (dict(head_dim=136), "head_dim must be"),
    (dict(head_dim=0), "head_dim must be"),
    (dict(heads=3, kv_heads=2), "multiple of kv_heads"),
    (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(heads=1025), "heads must be"),
    (dict(q_tokens=1 << 31), "must be < 2^31"),
    (dict(sequences=0), "sequences must be"),
    (dict(sequences=2), "need q_offsets"),
    (dict(sequences=1 << 24), "too many tiles"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(k=None), "must be given"),
    (dict(out=None), "must be given"),
    (dict(q=PTR + 8), "multiples of 16 bytes"),
    (dict(q_stride=36), "multiples of 8"),
    (dict(v_stride=24), "multiples of 8"),
])
def test_attention_refuses(change, text):
    refused(_lib.hip().bs_attention(C.byref(attention_args(**change)), None, 0, None), text)


def test_attention_asks_for_its_workspace():
    a = attention_args(k_tokens=100000, q_tokens=1)
    n = C.c_uint64(0)
    assert _lib.hip().bs_attention_workspace(C.byref(a), C.byref(n)) == 0 and n.value > 0
    refused(_lib.hip().bs_attention(C.byref(a), None, 0, None), "the workspace must hold")
    refused(_lib.hip().bs_attention(C.byref(a), PTR, n.value - 1, None), "the workspace must hold")
    refused(_lib.hip().bs_attention(C.byref(a), PTR + 4, n.value, None), "16-byte aligned")
    refused(_lib.hip().bs_attention_workspace(None, C.byref(n)), "args is null")
    refused(_lib.hip().bs_attention_workspace(C.byref(a), None), "bytes is null")
    refused(_lib.hip().bs_linear_workspace(4, 4, 4, None), "bytes is null")
    refused(_lib.hip().bs_layer_norm_backward_workspace(4, 4, 0, None), "bytes is null")


def test_calls_without_rows_do_nothing():
    assert _lib.hip().bs_layer_norm(None, 0, None, None, 0, 1e-5, None, 0, None, None, 0, 64, 0, None) == 0
    assert _lib.hip().bs_linear(None, 0, None, 0, None, None, 0, None, 0, 0, 32, 32, 2, 2, 0, None, 0, None) == 0
    assert _lib.hip().bs_attention(C.byref(attention_args(q_tokens=0)), None, 0, None) == 0


def test_python_refuses_tensors_off_the_gpu():
    import torch
    from beam_search_collab_amd import embed
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="on a GPU"):
        embed.layer_norm(x)
    with pytest.raises(ValueError, match="on a GPU"):
        embed.linear(x, x)
    with pytest.raises(ValueError, match="on a GPU"):
        embed.attention(x[:, None], x[:, None], x[:, None])
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        embed.linear(x.float(), x.float())
    with pytest.raises(ValueError, match="x must be"):
        embed.layer_norm(x.double())


def test_the_check_of_norms_far_from_zero_rejects_mistakes():
    """planted in a norm in 32 bits on the CPU, at the inputs of the GPU's test"""
    import torch
    from test_gpu_text_encoder import FAR, check_norm_far, far_rows
    for mean, std in FAR:
        x = far_rows(130, 5, 960, mean, std)
        m = x.double().mean(1)
        c = (x.double() - m[:, None]).float()
        r = (1 / torch.sqrt(c.double().square().mean(1) + 1e-5)).float()
        y = c * r[:, None]
        check_norm_far(x, None, None, 1e-5, y, m.float(), r)
        cancelled = (1 / torch.sqrt((x.square().mean(1) - x.mean(1).square()).clamp_min(0) + 1e-5))
        shifted = m.float() + 20 * 2.0 ** -24 * abs(mean)  # as a sum of 20 roundings may be
        for wrong in ((0 * y, m.float(), r), (-y, m.float(), r), (y * 1.001, m.float(), r), (y, m.float(), r * 1.001), (y, m.float(), 0 * r),
                      (c * cancelled[:, None], m.float(), cancelled), ((x - shifted[:, None]) * r[:, None], m.float(), r),
                      (y, shifted, r)):
            with pytest.raises(AssertionError):
                check_norm_far(x, None, None, 1e-5, *wrong)


@pytest.mark.parametrize("rows,inner,cols", [((1 << 31) - 1, 1, 1), ((1 << 31) - 255, 8, 128), ((1 << 30) + 1, 1, 129), (1 << 26, 1, 1 << 13)])
def test_linear_refuses_launches_of_2_to_the_32_threads(rows, inner, cols):
    """a grid of 2^32 threads is cut short without an error"""
    n = C.c_uint64(0)
    refused(_lib.hip().bs_linear_workspace(rows, inner, cols, C.byref(n)), "too large for one launch")
    refused(_lib.hip().bs_linear(PTR, inner, PTR, inner, None, None, 0, PTR, cols, rows, inner, cols, 2, 2, 0, None, 0, None), "too large for one launch")


def test_linear_takes_as_many_rows_as_a_launch_has():
    n = C.c_uint64(1)
    for rows, cols in (((1 << 31) - 256, 1), ((1 << 30) - 256, 256), (32, 1 << 24)):
        assert _lib.hip().bs_linear_workspace(rows, 8, cols, C.byref(n)) == 0


def test_python_refuses_to_lose_a_gradient():
    """autograd does not see these calls: a result without a gradient, from tensors that want one, would be a silent loss"""
    import torch
    from beam_search_collab_amd import embed
    x, w, s = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(32, 32, dtype=torch.bfloat16), torch.zeros(4)
    h = x[:, None]

    def wants(t):
        return t.detach().clone().requires_grad_()
    calls = [lambda: embed.layer_norm(wants(x)), lambda: embed.layer_norm(x, wants(w[0])), lambda: embed.layer_norm(x, None, wants(w[0])),
             lambda: embed.linear(x, wants(w)), lambda: embed.linear(x, w, wants(w[0])), lambda: embed.linear(x, w, residual=wants(x)),
             lambda: embed.attention(wants(h), h, h), lambda: embed.attention(h, h, wants(h)),
             lambda: embed.layer_norm_backward(x, x, s, s, wants(w[0])), lambda: embed.layer_norm_backward(wants(x), x, s, s)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):  # goes on to the next check
            call()
        with torch.inference_mode(), pytest.raises(ValueError, match="on a GPU"):
            call()
