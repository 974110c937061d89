"""The operators that complete an encoder's block, on the GPU against their definitions in 64 bits: norms of heads with the
rotation by their positions, gated products, attention behind a shared prefix.

Tolerances are the sums of the roundings an operator makes, worst case:  U is the unit roundoff of the output type, E =
2^-24 that of the float32 arithmetic; a float32 sum of n terms is off by at most n E times the sum of the magnitudes.
"""
import gc
import math

import pytest
import torch

from beam_search_collab_amd import embed
from test_gpu_text_encoder import BF16, E, F16, F32, TINY, U, near, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_given_back():
    """tests of other files look at the device's free memory"""
    yield
    if torch.cuda.is_available():
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()


# ---------------------------------------------------------------- norm of heads and rotation

def turned(x, angle, layout, magnitude, back=False):
    """pairs of the first 2 n elements turned by angle (tokens x n), in 64 bits"""
    n = angle.shape[1]
    c, s = magnitude * torch.cos(angle)[:, None], magnitude * torch.sin(angle)[:, None] * (-1 if back else 1)
    y = x.clone()
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    y[..., 0:n if layout == "half" else 2 * n:1 if layout == "half" else 2] = a * c - b * s
    y[..., n if layout == "half" else 1:2 * n:1 if layout == "half" else 2] = b * c + a * s
    return y


def partners(x, n, layout):
    """|a| + |b| of a pair in both its places, 0 elsewhere"""
    y = torch.zeros_like(x)
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    both = a.abs() + b.abs()
    if layout == "half":
        y[..., :n], y[..., n:2 * n] = both, both
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = both, both
    return y


def angle_of(positions, frequencies, tokens):
    pos = torch.arange(tokens, device="cuda") if positions is None else positions
    if frequencies is None:
        return torch.zeros(tokens, 0, dtype=torch.float64, device="cuda")
    return pos.double()[:, None] * frequencies


def check_rotary(x, w, eps, angle, layout, magnitude, y):
    x, n = x.double(), angle.shape[1]
    norm = x
    if eps is not None:
        norm = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    want = turned(norm, angle, layout, magnitude)
    # the norm: 24 additions and two roundings, halved by the root, the root, two products.  cos and sin: their argument's
    # and series' roundings and the magnitude's, under 5 E; the angle in float64, 6 units; two roundings of the sum
    far = 6 * 2.0 ** -53 * angle.abs().amax(1)[:, None, None] if n else 0.0
    part = 18 * E if eps is not None else 0.0
    tol = (part + 7 * E + far) * partners(norm, n, layout) * abs(magnitude) + part * norm.abs()
    near(y, want, tol + U[y.dtype] * want.abs() + TINY[y.dtype])


def check_rotary_backward(dy, x, w, eps, angle, layout, magnitude, dx, dw):
    dy, x, n = dy.double(), x.double(), angle.shape[1]
    d = turned(dy, angle, layout, magnitude, back=True)
    ed = (7 * E + (6 * 2.0 ** -53 * angle.abs().amax(1)[:, None, None] if n else 0.0)) * partners(dy, n, layout) * abs(magnitude)
    if eps is None:
        near(dx, d, ed + U[dx.dtype] * d.abs() + TINY[dx.dtype])
        assert dw is None
        return
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    xh = x * r
    wd = torch.ones((), dtype=torch.float64, device="cuda") if w is None else w.double()
    g = d * wd
    along = (g * xh).mean(-1, keepdim=True)
    want = r * (g - xh * along)
    eg = ed * wd.abs() + E * g.abs()
    ea = (eg * xh.abs() + 48 * E * (g * xh).abs()).mean(-1, keepdim=True)  # xh is off by 17 E, the sum by 26
    near(dx, want, r * (eg + xh.abs() * ea + 40 * E * (g.abs() + (xh * along).abs())) + U[dx.dtype] * want.abs() + TINY[dx.dtype])
    if dw is not None:
        rows = x.shape[0] * x.shape[1]
        tol = (rows + 90) * E * (d * xh).abs().sum((0, 1)) + (ed * xh.abs()).sum((0, 1))
        wanted = (d * xh).sum((0, 1))
        near(dw, wanted, tol + U[dw.dtype] * wanted.abs() + TINY[dw.dtype])


HEADS = [  # tokens, heads, kv heads, head_dim, rotary, layout
    (1, 1, 1, 2, 2, "half"), (1, 1, 0, 4, 2, "interleaved"), (3, 2, 1, 6, 4, "half"), (5, 3, 1, 64, 64, "half"), (24, 12, 4, 64, 64, "half"),
    (7, 4, 2, 128, 128, "half"), (7, 4, 2, 128, 128, "interleaved"), (9, 5, 5, 80, 80, "half"), (9, 5, 5, 80, 40, "interleaved"),
    (11, 8, 1, 96, 32, "interleaved"), (13, 3, 3, 100, 50, "half"), (13, 3, 3, 100, 100, "interleaved"), (2, 2, 2, 250, 126, "half"),
    (6, 4, 4, 256, 256, "half"), (6, 4, 4, 256, 64, "interleaved"), (17, 6, 2, 254, 254, "half"), (17, 6, 2, 64, 0, "half"),
    (33, 1, 1, 16, 16, "half"), (33, 1, 1, 8, 8, "interleaved"), (4, 70, 2, 32, 16, "half"), (0, 4, 2, 64, 64, "half"),
    (1100, 2, 1, 32, 32, "half"), (5000, 1, 1, 12, 4, "interleaved"), (2100, 16, 4, 64, 32, "half")]
ODD = (1000, 12345, 1 << 20)  # positions to start from


def head_case(seed, tokens, heads, kv, dim, rotary, dtype, wdtype):
    q, k = ((rand(seed + i, tokens, n, dim) * (1 + 3 * torch.rand(dim, generator=torch.Generator().manual_seed(seed)).cuda())).to(dtype)
            for i, n in enumerate((heads, kv)))
    if kv == 0:
        k = None
    pos = (torch.arange(tokens) % 37 + ODD[seed % 3]).int().cuda() if seed % 4 else None
    f = embed.rotary_frequencies(rotary) if rotary else None
    wq, wk = rand(seed + 2, dim, dtype=wdtype), rand(seed + 3, dim, dtype=wdtype) if kv else None
    return q, k, pos, f, wq, wk


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,layout", HEADS)
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_head_norm_rotary(gpu, tokens, heads, kv, dim, rotary, layout, dtype, wdtype):
    q, k, pos, f, wq, wk = head_case(dim + tokens, tokens, heads, kv, dim, rotary, dtype, wdtype)
    angle = angle_of(pos, f, tokens)
    for eps, magnitude, a, b in ((1e-6, 1.0, wq, wk), (1e-3, 1.25, None, None), (None, 1.0, None, None)):
        y, z = embed.head_norm_rotary(q, k, pos, f, a, b, eps=eps, layout=layout, magnitude=magnitude)
        check_rotary(q, a, eps, angle, layout, magnitude, y)
        if kv:
            check_rotary(k, b, eps, angle, layout, magnitude, z)
        else:
            assert z is None


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,layout", HEADS)
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_head_norm_rotary_backward(gpu, tokens, heads, kv, dim, rotary, layout, dtype, wdtype):
    q, k, pos, f, wq, wk = head_case(dim + tokens, tokens, heads, kv, dim, rotary, dtype, wdtype)
    dq, dk = rand(91, tokens, heads, dim, dtype=dtype), rand(92, tokens, kv, dim, dtype=dtype) if kv else None
    angle = angle_of(pos, f, tokens)
    for eps, magnitude, a, b in ((1e-6, 1.0, wq, wk), (1e-3, 1.25, None, None), (None, 1.0, None, None)):
        args = (dq, dk, q, k, pos, f, a, b)
        got = embed.head_norm_rotary_backward(*args, eps=eps, layout=layout, magnitude=magnitude)
        if eps is not None:
            assert got[2].dtype == (wdtype if a is not None else F32)
        check_rotary_backward(dq, q, a, eps, angle, layout, magnitude, got[0], got[2])
        if kv:
            check_rotary_backward(dk, k, b, eps, angle, layout, magnitude, got[1], got[3])
        again = embed.head_norm_rotary_backward(*args, eps=eps, layout=layout, magnitude=magnitude)
        assert all(x is y is None or torch.equal(x, y) for x, y in zip(got, again))  # no order that changes
        only = embed.head_norm_rotary_backward(*args, eps=eps, layout=layout, magnitude=magnitude, params=False)
        assert torch.equal(only[0], got[0]) and only[2] is None and only[3] is None


def test_rotary_at_far_positions(gpu):
    """positions at both ends of their type, frequencies above 1"""
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 3], dtype=torch.int32, device="cuda")
    q = rand(1, 7, 2, 32)
    f = torch.cat([embed.rotary_frequencies(24), torch.tensor([3.7, 1e-12, 0.0, -0.25], dtype=torch.float64, device="cuda")])
    y, _ = embed.head_norm_rotary(q, None, pos, f, eps=None)
    check_rotary(q, None, None, angle_of(pos, f, 7), "half", 1.0, y)
    assert torch.equal(y[0], q[0])


def test_rotation_turns_back_and_keeps_lengths(gpu):
    """scores depend on the distance of the positions alone"""
    q, k = rand(2, 50, 1, 64), rand(3, 50, 1, 64)
    f = embed.rotary_frequencies(64)
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    scores = []
    for shift in (0, 1000, 1 << 24):
        a, b = embed.head_norm_rotary(q, k, pos + shift, f, eps=None)
        scores.append(a[:, 0].double() @ b[:, 0].double().t().contiguous())
    size = (q[:, 0].double().abs().sum(1)[:, None] * k[:, 0].double().abs().amax(1) * 4)
    for s in scores[1:]:
        assert ((s - scores[0]).abs() <= 60 * E * size).all()
    back = embed.head_norm_rotary_backward(a, b, q, k, pos + shift, f, eps=None)
    near(back[0], q.double(), 30 * E * partners(q.double(), 32, "half"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,shift", [(64, 0), (64, 1), (80, 3), (50, 5)])
def test_head_norm_rotary_of_slices(gpu, dtype, dim, shift):
    """columns of one product, at any element; heads before tokens; in place; what lies between stays"""
    tokens, heads, kv = 21, 4, 2
    f, w = embed.rotary_frequencies(dim // 4 * 2), rand(5, dim)
    big = rand(4, tokens, (heads + 2 * kv) * dim + 8, dtype=dtype)
    was = big.clone()
    cut = big[:, shift:shift + (heads + 2 * kv) * dim].unflatten(1, (heads + 2 * kv, dim))
    q, k = cut[:, :heads], cut[:, heads:heads + kv]
    want = embed.head_norm_rotary(q.contiguous(), k.contiguous(), None, f, w, w)
    got = embed.head_norm_rotary(q, k, None, f, w, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(embed.head_norm_rotary(qt, None, None, f, w)[0], want[0])
    dq, dk = rand(6, tokens, heads, dim + 3, dtype=dtype)[:, :, :dim], rand(7, tokens, kv, dim, dtype=dtype)
    grads = embed.head_norm_rotary_backward(dq, dk, q, k, None, f, w, w)
    whole = embed.head_norm_rotary_backward(dq.contiguous(), dk, q.contiguous(), k.contiguous(), None, f, w, w)
    assert all(torch.equal(a, b) for a, b in zip(grads, whole))
    embed.head_norm_rotary(q, k, None, f, w, w, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    n = shift + (heads + kv) * dim
    assert torch.equal(big[:, :shift], was[:, :shift]) and torch.equal(big[:, n:], was[:, n:])


def test_head_norm_rotary_of_heads_that_are_zero_or_not_finite(gpu):
    q = rand(8, 6, 3, 64, dtype=BF16)
    f = embed.rotary_frequencies(64)
    q[1, 1] = 0
    q[2, 0, 5] = math.nan
    q[3, 2, 63] = math.inf
    y, _ = embed.head_norm_rotary(q, None, None, f)
    assert (y[1, 1] == 0).all() and torch.isnan(y[2, 0]).all()
    assert torch.isnan(y[3, 2, [31, 63]]).all() and (y[3, 2, [0, 1, 30, 32, 62]] == 0).all()
    fine = torch.ones(6, 3, dtype=torch.bool, device="cuda")
    fine[2, 0] = fine[3, 2] = False
    assert torch.isfinite(y[fine]).all()
    d = embed.head_norm_rotary_backward(rand(9, 6, 3, 64, dtype=BF16), None, q, None, None, f, params=False)[0]
    assert torch.isfinite(d[fine]).all() and torch.isnan(d[2, 0]).all()
    z, _ = embed.head_norm_rotary(torch.zeros(2, 1, 8, device="cuda"), eps=0.0)
    assert torch.isnan(z).all()  # 0 / 0


@pytest.mark.parametrize("layout,rotary", [("half", 30), ("interleaved", 16)])
def test_head_norm_rotary_backward_against_differences(gpu, layout, rotary):
    """directional derivatives of the definition in 64 bits"""
    tokens, heads, dim, h = 4, 3, 30, 1e-6
    q, w, dy = rand(10, tokens, heads, dim), rand(11, dim), rand(12, tokens, heads, dim)
    f = embed.rotary_frequencies(rotary)
    angle = angle_of(None, f, tokens)
    dx, _, dw, _ = embed.head_norm_rotary_backward(dy, None, q, None, None, f, w, eps=1e-5, layout=layout, magnitude=0.9)

    def loss(x, w):
        n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w
        return (turned(n, angle, layout, 0.9) * dy.double()).sum().item()
    for t in range(4):
        for i, (p, g) in enumerate(((q, dx), (w, dw))):
            d = rand(20 + t, *p.shape).double()
            args = [q.double(), w.double()]
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + h * d, args[i] - h * d
            slope = (loss(*up) - loss(*down)) / (2 * h)
            assert abs(slope - (g.double() * d).sum().item()) <= 1e-5 * (g.double() * d).abs().sum().item()


def test_head_norm_rotary_refusals(gpu):
    q, k, w, f = rand(1, 4, 2, 64, dtype=BF16), rand(2, 4, 1, 64, dtype=BF16), rand(3, 64), embed.rotary_frequencies(64)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    for call, text in [
        (lambda: embed.head_norm_rotary(q.double()), "q must be"),
        (lambda: embed.head_norm_rotary(q[0]), "q must be tokens"),
        (lambda: embed.head_norm_rotary(q, k[:3]), "k must be"),
        (lambda: embed.head_norm_rotary(q, k.float()), "k must be"),
        (lambda: embed.head_norm_rotary(q[..., ::2]), "elements of a head of q"),
        (lambda: embed.head_norm_rotary(q, k, pos.long(), f), "positions must be"),
        (lambda: embed.head_norm_rotary(q, k, pos[:3], f), "positions must be"),
        (lambda: embed.head_norm_rotary(q, k, pos, f.float()), "frequencies must be"),
        (lambda: embed.head_norm_rotary(q, k, pos, torch.cat([f, f])), "at most head_dim"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, w[:32]), "q_weight must be 64"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, w, w.bfloat16()), "k_weight must be of"),
        (lambda: embed.head_norm_rotary(q, None, pos, f, w, w), "k_weight without k"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, w, w, eps=None), "weights belong to the norm"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, eps=-1.0), "eps must be"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, magnitude=math.inf), "magnitude must be"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, layout="pairs"), "unknown layout"),
        (lambda: embed.head_norm_rotary(q[:, :, :63]), "head_dim must be even"),
        (lambda: embed.head_norm_rotary(rand(4, 2, 2, 258)), "head_dim must be even"),
        (lambda: embed.head_norm_rotary(q, k, pos.cpu(), f), "must be a tensor on"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, out=(q.float(), k)), "out.0. must be"),
        (lambda: embed.head_norm_rotary(q, out=(q[:1].expand(4, 2, 64), None)), "overlap"),
        (lambda: embed.head_norm_rotary(q.expand(4, 2, 64)[:, :1].expand(4, 5, 64)), "overlap"),
        (lambda: embed.head_norm_rotary_backward(q, None, q, k), "given together"),
        (lambda: embed.head_norm_rotary_backward(q[:3], k, q, k), "dq must be"),
        (lambda: embed.head_norm_rotary_backward(q, q, q, k), "dk must be"),
        (lambda: embed.head_norm_rotary(q, k, pos, f, torch.nn.Parameter(w)), "gradient"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


# ---------------------------------------------------------------- gated products

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act_and_slope(z, act):
    f = torch.nn.functional
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        y = {"none": lambda t: t * 1.0, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "silu": f.silu}[act](z)
        slope, = torch.autograd.grad(y.sum(), z)
    return y.detach(), slope


def check_gated(x, wg, wu, act, h, gate=None, up=None):
    k = x.shape[-1]
    xd = x.double()
    (g, eg), (u, eu) = (((xd @ w.double().t().contiguous()), (k + 4) * E * (xd.abs() @ w.double().abs().t().contiguous())) for w in (wg, wu))
    a, _ = act_and_slope(g, act)
    ea = 1.2 * eg  # no activation is steeper than 1.13
    if act != "none":
        ea = ea + 16 * E * g.abs() + 2 * E * g * g  # erf, exp: a few units, exp's argument rounded
    tol = ea * u.abs() + a.abs() * eu + ea * eu + 2 * E * (a * u).abs()
    near(h, a * u, tol + U[h.dtype] * (a * u).abs() + TINY[h.dtype])
    for got, want, e in ((gate, g, eg), (up, u, eu)):
        if got is not None:
            near(got, want, e + U[h.dtype] * want.abs() + TINY[h.dtype])


def check_gated_backward(dh, x, wg, wu, gate, up, act, dx, dwg, dwu):
    t = x.dtype
    dh, x, wg, wu, g, u = (y.double() for y in (dh, x, wg, wu, gate, up))
    a, slope = act_and_slope(g, act)
    dg, du = dh * u * slope, dh * a
    # the slope and the activation in float32: their parts are at most 1.13 and |g|; then the rounding to the type
    eg = (dh * u).abs() * 32 * E + (U[t] + 2 * E) * dg.abs() + TINY[t]
    eu = dh.abs() * 16 * E * g.abs() * (act != "none") + (U[t] + 2 * E) * du.abs() + TINY[t]
    n = 2 * g.shape[1] + 8
    want = dg @ wg + du @ wu
    tol = eg @ wg.abs() + eu @ wu.abs() + n * E * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) * 1.01
    near(dx, want, tol + U[t] * want.abs() + TINY[t])
    for got, d, e in ((dwg, dg, eg), (dwu, du, eu)):
        if got is not None:
            want = d.t().contiguous() @ x
            tol = e.t().contiguous() @ x.abs() + (len(x) + 8) * E * (d.abs().t().contiguous() @ x.abs()) * 1.01
            near(got, want, tol + U[t] * want.abs() + TINY[t])


GATED = [(1, 1, 1), (1, 1024, 128), (2, 100, 3), (5, 63, 65), (16, 64, 128), (17, 4096, 256), (31, 200, 96), (32, 256, 512), (33, 257, 131),
         (64, 1024, 64), (65, 72, 1000), (100, 1000, 300), (127, 128, 127), (128, 128, 128), (129, 192, 257), (200, 1088, 128), (255, 64, 255),
         (256, 512, 256), (257, 520, 264), (300, 768, 2048), (1000, 96, 777), (513, 1024, 1024), (1111, 333, 222), (0, 64, 32), (29, 72, 4109)]


def gated_case(seed, rows, inner, cols, dtype):
    return rand(seed, rows, inner, dtype=dtype), rand(seed + 1, cols, inner, dtype=dtype, std=inner ** -0.5), rand(seed + 2, cols, inner, dtype=dtype, std=inner ** -0.5)


@pytest.mark.parametrize("rows,inner,cols", GATED)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated(gpu, rows, inner, cols, dtype):
    x, wg, wu = gated_case(200, rows, inner, cols, dtype)
    act = ACTS[(rows + cols) % 5]
    h, gate, up = embed.gated(x, wg, wu, activation=act, save=True)
    check_gated(x, wg, wu, act, h, gate, up)
    assert torch.equal(h, embed.gated(x, wg, wu, activation=act))


@pytest.mark.parametrize("rows,inner,cols", GATED)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_backward(gpu, rows, inner, cols, dtype):
    x, wg, wu = gated_case(210, rows, inner, cols, dtype)
    act = ACTS[(rows + cols + 1) % 5]
    gate, up, dh = rand(214, rows, cols, dtype=dtype, std=1.5), rand(215, rows, cols, dtype=dtype), rand(216, rows, cols, dtype=dtype, std=0.3)
    got = embed.gated_backward(dh, x, wg, wu, gate, up, activation=act)
    assert [g.shape for g in got] == [x.shape, wg.shape, wu.shape]
    check_gated_backward(dh, x, wg, wu, gate, up, act, *got)
    assert all(torch.equal(a, b) for a, b in zip(got, embed.gated_backward(dh, x, wg, wu, gate, up, activation=act)))
    only = embed.gated_backward(dh, x, wg, wu, gate, up, activation=act, params=False)  # alone, dx may be cut otherwise
    check_gated_backward(dh, x, wg, wu, gate, up, act, *only)
    assert only[1] is None and only[2] is None


@pytest.mark.parametrize("rows,inner,cols", [(4096, 128, 2048), (4111, 192, 2112), (300, 320, 16500), (8200, 256, 1001), (8000, 72, 512), (2000, 2048, 768)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_of_many_tiles(gpu, rows, inner, cols, dtype):
    """more tiles than compute units, shifted ones at the edges"""
    x, wg, wu = gated_case(220, rows, inner, cols, dtype)
    h, gate, up = embed.gated(x, wg, wu, save=True)
    check_gated(x, wg, wu, "silu", h, gate, up)
    wide = torch.full((rows, cols + 9), 7.0, dtype=dtype, device="cuda")
    embed.gated(x, wg, wu, out=wide[:, 3:cols + 3])
    assert torch.equal(wide[:, 3:cols + 3], h) and (wide[:, :3] == 7).all() and (wide[:, cols + 3:] == 7).all()
    dh = rand(223, rows, cols, dtype=dtype, std=0.3)
    got = embed.gated_backward(dh, x, wg, wu, gate, up)
    check_gated_backward(dh, x, wg, wu, gate, up, "silu", *got)
    assert all(torch.equal(a, b) for a, b in zip(got, embed.gated_backward(dh, x, wg, wu, gate, up)))


@pytest.mark.parametrize("act", ACTS)
def test_gated_activations_far_from_zero(gpu, act):
    """slopes where exponentials overflow, vanish or cancel"""
    z = torch.cat([torch.linspace(-12, 12, 200), torch.tensor([-3e4, -200.0, -90.0, -40.0, 0.0, 40.0, 90.0, 200.0, 3e4, -1e-3, 1e-3, 60.0])])
    for dtype in (F16, BF16):
        gate = z.to(dtype).cuda()[:, None].repeat(1, 64)
        up, dh, x = rand(230, len(z), 64, dtype=dtype), rand(231, len(z), 64, dtype=dtype, std=0.1), rand(232, len(z), 64, dtype=dtype)
        wg, wu = (torch.eye(64, dtype=dtype, device="cuda") for _ in range(2))
        dx, _, _ = embed.gated_backward(dh, x, wg, 0 * wu, gate, up, activation=act)
        check_gated_backward(dh, x, wg, 0 * wu, gate, up, act, dx, None, None)
        dx, _, _ = embed.gated_backward(dh, x, 0 * wg, wu, gate, up, activation=act)
        check_gated_backward(dh, x, 0 * wg, wu, gate, up, act, dx, None, None)


@pytest.mark.parametrize("rows,inner,cols", [(3, 64, 40), (20, 1000, 320), (130, 96, 140), (520, 512, 512)])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_gated_of_slices(gpu, rows, inner, cols, shift):
    """operands inside wider tensors, at any element; the weights are halves of one"""
    x = rand(240, rows, inner + 24, dtype=F16)[:, shift:shift + inner]
    both = rand(241, 2 * cols, inner + 16, dtype=F16, std=inner ** -0.5)[:, shift:shift + inner]
    wg, wu = both[:cols], both[cols:]
    cut = [rand(242 + i, rows, cols + 16, dtype=F16)[:, shift:shift + cols] for i in range(3)]
    plain = [t.contiguous() for t in (x, wg, wu, *cut)]
    h = embed.gated(x, wg, wu, activation="gelu")
    assert torch.equal(h, embed.gated(*plain[:3], activation="gelu")) or shift  # another kernel may take them
    check_gated(x, wg, wu, "gelu", h)
    got = embed.gated_backward(cut[0], x, wg, wu, cut[1], cut[2], activation="gelu")
    check_gated_backward(cut[0], x, wg, wu, cut[1], cut[2], "gelu", *got)
    assert all(t.is_contiguous() for t in got)


def test_gated_leading_dimensions_and_not_finite(gpu):
    x, wg, wu = rand(250, 2, 3, 70, dtype=BF16), rand(251, 50, 70, dtype=BF16), rand(252, 50, 70, dtype=BF16)
    h, gate, up = embed.gated(x, wg, wu, save=True)
    assert h.shape == gate.shape == (2, 3, 50)
    dx, dwg, _ = embed.gated_backward(h, x, wg, wu, gate, up)
    assert dx.shape == x.shape and dwg.shape == wg.shape
    for rows in (6, 200, 700):
        x, wg, wu = gated_case(253, rows, 320, 256, BF16)
        gate, up, dh = (rand(256 + i, rows, 256, dtype=BF16) for i in range(3))
        x[3, 299] = math.nan
        h = embed.gated(x, wg, wu)
        rest = torch.arange(rows, device="cuda") != 3
        assert torch.isnan(h[3]).all() and torch.isfinite(h[rest]).all()
        dh[rows - 1, 5] = math.inf  # of the last row, whose successors do not exist
        dx, dwg, dwu = embed.gated_backward(dh, x, wg, wu, gate, up)
        assert torch.isfinite(dx[:-1]).all() and not torch.isfinite(dx[-1]).any()
        one = torch.arange(256, device="cuda") != 5
        keep = torch.arange(320, device="cuda") != 299
        assert torch.isfinite(dwg[one][:, keep]).all() and torch.isnan(dwg[:, 299]).all() and not torch.isfinite(dwg[5]).any()
        x[3, 299], dh[rows - 1, 5], x[rows - 1, 7] = 0.0, 0.0, math.inf
        _, dwg, _ = embed.gated_backward(dh, x, wg, wu, gate, up)
        want = torch.where(dh[-1] * up[-1] == 0, math.nan, math.inf)  # 0 times infinity
        assert torch.equal(torch.isnan(dwg[:, 7]), torch.isnan(want)) and not torch.isfinite(dwg[:, 7]).any()
        assert torch.isfinite(dwg[:, torch.arange(320, device="cuda") != 7]).all()


def test_gated_backward_against_differences(gpu):
    """directional derivatives of the definition in 64 bits; the gradients' own error is that of the types"""
    rows, inner, cols, h = 40, 24, 56, 1e-6
    x, wg, wu = gated_case(260, rows, inner, cols, F16)
    dh = rand(263, rows, cols, dtype=F16)
    for act in ("gelu", "gelu_tanh", "silu"):
        _, gate, up = embed.gated(x, wg, wu, activation=act, save=True)
        got = embed.gated_backward(dh, x, wg, wu, gate, up, activation=act)

        def loss(x, wg, wu):
            return (act_and_slope(x @ wg.t(), act)[0] * (x @ wu.t()) * dh.double()).sum().item()
        for t in range(3):
            for i, g in enumerate(got):
                d = rand(270 + t, *g.shape).double()
                args = [y.double() for y in (x, wg, wu)]
                up_, down = list(args), list(args)
                up_[i], down[i] = args[i] + h * d, args[i] - h * d
                slope = (loss(*up_) - loss(*down)) / (2 * h)
                # saved values, d and the result are rounded: 5 roundings, none of which moves a term by more than 2^-11 (the
                # second derivatives of the activations are below 1.13)
                assert abs(slope - (g.double() * d).sum().item()) <= 8 * 2.0 ** -11 * (g.double() * d).abs().sum().item()


def test_gated_refusals(gpu):
    x, w = rand(1, 4, 64, dtype=BF16), rand(2, 32, 64, dtype=BF16)
    h = rand(3, 4, 32, dtype=BF16)
    for call, text in [
        (lambda: embed.gated(x.float(), w, w), "x must be"),
        (lambda: embed.gated(x, w[:, :32], w[:, :32]), "x has 64 features"),
        (lambda: embed.gated(x, w, w[:31]), "both of x's type"),
        (lambda: embed.gated(x, w.half(), w), "both of x's type"),
        (lambda: embed.gated(x, w, w, activation="tanh"), "unknown activation"),
        (lambda: embed.gated(x, w, w, out=h.float()), "out must be"),
        (lambda: embed.gated(x, w.cpu(), w), "must be a tensor on"),
        (lambda: embed.gated(x, torch.nn.Parameter(w), w), "gradient"),
        (lambda: embed.gated_backward(h[:3], x, w, w, h, h), "dh must be"),
        (lambda: embed.gated_backward(h, x, w, w, h, h.float()), "up must be"),
        (lambda: embed.gated_backward(h, x, w, w, h[:, :31], h), "gate must be"),
        (lambda: embed.gated_backward(h, x, w, w, h.t().contiguous().t(), h), "features of gate"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


# ---------------------------------------------------------------- attention behind a shared prefix

def prefix_case(seed, nq, nk, prefix, heads, kv, dim, dtype, std=1.0):
    return (rand(seed, sum(nq), heads, dim, dtype=dtype, std=std), rand(seed + 1, sum(nk), kv, dim, dtype=dtype), rand(seed + 2, sum(nk), kv, dim, dtype=dtype),
            rand(seed + 3, prefix, kv, dim, dtype=dtype), rand(seed + 4, prefix, kv, dim, dtype=dtype))


def check_prefix(q, k, v, pk, pv, nq, nk, causal, scale, out, lse):
    """a sequence and a head at a time in 64 bits; tolerances as attention's, whose arithmetic it is: one more joining of parts"""
    heads, kv, dim, t = q.shape[1], k.shape[1], q.shape[2], q.dtype
    a = b = 0
    p = len(pk)
    for m, n in zip(nq, nk):
        if not m:
            b += n
            continue
        for h in range(heads):
            g = h // (heads // kv)
            x = q[a:a + m, h].double()
            y, w = torch.cat([pk[:, g], k[b:b + n, g]]).double(), torch.cat([pv[:, g], v[b:b + n, g]]).double()
            hide = torch.zeros(m, p + n, dtype=torch.bool, device="cuda")
            if causal:
                hide = torch.ones_like(hide).triu(p + n - m + 1)
                hide[:, :p] = False
            z = (x @ y.t().contiguous() * scale).masked_fill(hide, -math.inf)
            s = torch.logsumexp(z, 1)
            none = s == -math.inf
            e = torch.exp(z - torch.where(none, 0.0, s)[:, None])
            spread = (x.abs() @ y.abs().t().contiguous() * abs(scale)).masked_fill(hide, 0).amax(1) if p + n else torch.zeros(m, dtype=torch.float64, device="cuda")
            count = p + n
            d = (dim + 6) * E * spread + 4 * E * (spread + 1)
            want, size, total = e @ w, e @ w.abs(), (~hide).double() @ w.abs()
            tol = (U[t] + 4 * d + (count + 48) * E)[:, None] * size + 2.0 ** -24 * total * (t == F16) + U[t] * want.abs() + TINY[t]
            near(out[a:a + m, h], want, tol)
            if lse is not None:
                near(lse[a:a + m, h], s, 2 * d + (count / 32 + 48) * E + 4 * E * torch.where(none, 0.0, s.abs()))
        a, b = a + m, b + n


def offsets(lengths):
    import numpy as np
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")


def behind_prefix(seed, nq, nk, prefix, heads, kv, dim, dtype, causal=True, scale=None, hints=True):
    q, k, v, pk, pv = prefix_case(seed, nq, nk, prefix, heads, kv, dim, dtype)
    lo = dict(longest_q=max(nq), longest_k=max(nk)) if hints else {}
    out, lse = embed.attention_shared_prefix(q, k, v, pk, pv, offsets(nq), offsets(nk), causal=causal, scale=scale, lse=True, **lo)
    check_prefix(q, k, v, pk, pv, nq, nk, causal, dim ** -0.5 if scale is None else scale, out, lse)
    again = embed.attention_shared_prefix(q, k, v, pk, pv, offsets(nq), offsets(nk), causal=causal, scale=scale, **lo)
    assert torch.equal(again, out)
    return q, k, v, pk, pv, out, lse


PREFIX = [
    ([1], [1], 1), ([1], [0], 3), ([2], [2], 64), ([24], [24], 100), ([1, 1, 1], [5, 700, 64], 65), ([7], [3], 63), ([5, 2], [0, 9], 33),
    ([0, 3, 0, 4], [2, 3, 0, 4], 129), ([1, 40, 3, 130, 17], [1, 40, 3, 130, 17], 200), ([1] * 70, list(range(70)), 300), ([1] * 9, [0] * 9, 1000),
    ([2] * 9, [300 - 31 * i for i in range(9)], 1), ([3], [3], 0), ([1, 2], [900, 40], 2500), ([1] * 40, [20] * 40, 5000)]


@pytest.mark.parametrize("nq,nk,prefix", PREFIX, ids=[str(i) for i in range(len(PREFIX))])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 64, BF16), (3, 1, 128, F16), (2, 2, 32, BF16)])
def test_attention_shared_prefix(gpu, nq, nk, prefix, causal, heads, kv, dim, dtype):
    behind_prefix(300, nq, nk, prefix, heads, kv, dim, dtype, causal)


MANY = [([130, 64, 1, 200, 0, 77] * 4, None, 150, 16, 16), ([300] * 8, None, 64, 16, 8), ([300] * 8, [0] * 8, 1, 16, 8), ([500, 400] * 4, [600, 100] * 4, 1023, 16, 4),
        ([64] * 64, None, 65, 8, 8), ([100] * 40, [37] * 40, 500, 8, 8)]


@pytest.mark.parametrize("nq,nk,prefix,heads,kv", MANY, ids=[str(i) for i in range(len(MANY))])
@pytest.mark.parametrize("dim,dtype,causal", [(32, BF16, True), (64, F16, True), (72, BF16, False), (128, BF16, True)])
def test_attention_shared_prefix_of_full_tiles(gpu, nq, nk, prefix, heads, kv, dim, dtype, causal):
    behind_prefix(310, nq, nq if nk is None else nk, prefix, heads, kv, dim, dtype, causal)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 56, 72, 80, 88, 96, 104, 120])
def test_attention_shared_prefix_head_sizes(gpu, dim):
    behind_prefix(320, [70, 9], [70, 150], 77, 3, 3, dim, BF16)
    behind_prefix(325, [260] * 12, [260] * 12, 77, 16, 16, dim, BF16)


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 1), (8, 8), (12, 4), (16, 1), (40, 2), (64, 1)])
def test_attention_shared_prefix_heads(gpu, heads, kv):
    behind_prefix(330, [19, 1], [19, 77], 140, heads, kv, 64, F16)
    behind_prefix(335, [1] * 5, [3, 0, 7, 200, 64], 140, heads, kv, 64, BF16, hints=False)


def test_attention_shared_prefix_is_attention_over_both(gpu):
    """one sequence: the prefix and its own keys in a row; without offsets; of no prefix"""
    q, k, v, pk, pv = prefix_case(340, [90], [90], 200, 4, 2, 64, BF16)
    out = embed.attention_shared_prefix(q, k, v, pk, pv)
    check_prefix(q, k, v, pk, pv, [90], [90], True, 0.125, out, None)
    whole = embed.attention(q, torch.cat([pk, k]), torch.cat([pv, v]), offsets([90]), offsets([290]))
    assert (out.float() - whole.float()).abs().max() < 0.05
    none = embed.attention_shared_prefix(q, k, v, pk[:0], pv[:0], lse=True)
    assert all(torch.equal(a, b) for a, b in zip(none, embed.attention(q, k, v, lse=True)))
    for scale in (0.0, -0.3, 2.0):
        behind_prefix(341, [90, 1], [90, 3], 200, 4, 2, 64, BF16, scale=scale)
        behind_prefix(342, [300] * 8, [300] * 8, 70, 16, 8, 64, BF16, scale=scale)


@pytest.mark.parametrize("nq,nk,heads,kv", [([70, 20], [70, 20], 4, 2), ([1, 2], [900, 40], 4, 2), ([300] * 8, [300] * 8, 16, 8)])
def test_attention_shared_prefix_of_slices(gpu, nq, nk, heads, kv):
    """all operands as columns of wider tensors, the result inside another; tokens behind the last sequence"""
    dim, more = 64, 5
    q = rand(350, sum(nq) + more, heads * dim + 16, dtype=F16)[:, 8:8 + heads * dim].unflatten(1, (heads, dim))
    own = rand(351, sum(nk) + more, 2 * kv * dim, dtype=F16)
    k, v = own[:, :kv * dim].unflatten(1, (kv, dim)), own[:, kv * dim:].unflatten(1, (kv, dim))
    own[sum(nk):] = math.nan
    q[sum(nq):] = math.nan
    front = rand(352, 300, 2 * kv * dim + 8, dtype=F16)
    pk, pv = front[:, :kv * dim].unflatten(1, (kv, dim)), front[:, kv * dim:2 * kv * dim].unflatten(1, (kv, dim))
    buf = torch.full((sum(nq) + more, heads, dim + 8), 7.0, dtype=F16, device="cuda")
    got, lse = embed.attention_shared_prefix(q, k, v, pk, pv, offsets(nq), offsets(nk), out=buf[:, :, :dim], lse=True)
    assert (buf[:, :, dim:] == 7).all() and (buf[sum(nq):] == 7).all()
    want = embed.attention_shared_prefix(*(t.contiguous() for t in (q, k, v, pk, pv)), offsets(nq), offsets(nk))
    assert torch.equal(buf[:sum(nq), :, :dim], want[:sum(nq)])
    check_prefix(q, k, v, pk, pv, nq, nk, True, 0.125, want, lse)
    pkt, pvt = pk.transpose(0, 1).contiguous().transpose(0, 1), pv.transpose(0, 1).contiguous().transpose(0, 1)  # heads before tokens
    assert torch.equal(embed.attention_shared_prefix(q, k, v, pkt, pvt, offsets(nq), offsets(nk))[:sum(nq)], want[:sum(nq)])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65000.0])
@pytest.mark.parametrize("nq,nk,heads,kv", [([100, 30], [100, 30], 2, 1), ([3, 5], [80, 900], 2, 2), ([1, 4], [1300, 60], 8, 1), ([130] * 20, [130] * 20, 16, 16)])
def test_attention_shared_prefix_never_touches_what_a_query_does_not_see(gpu, bad, nq, nk, heads, kv):
    """the last key and value of every sequence hold `bad`: only the last query's result may change; those of the prefix: all"""
    import numpy as np
    q, k, v, pk, pv = prefix_case(360, nq, nk, 70, heads, kv, 64, BF16)

    def run():
        return embed.attention_shared_prefix(q, k, v, pk, pv, offsets(nq), offsets(nk), lse=True)
    good = run()
    last_q, last_k = (torch.tensor(np.cumsum(n) - 1, device="cuda") for n in (nq, nk))
    keep = torch.ones(sum(nq), dtype=torch.bool, device="cuda")
    keep[last_q] = False
    for which in (k, v):
        was = which.clone()
        which[last_k] = bad
        got = run()
        for a, b in zip(got, good):
            assert torch.equal(a[keep], b[keep])
        if which is v and not math.isfinite(bad):
            assert not torch.isfinite(got[0][last_q]).any()
        which.copy_(was)
    if not math.isfinite(bad):
        for at in (69, 64, 3):
            was = pv.clone()
            pv[at, :, 5] = bad
            got = run()[0]
            assert (torch.isnan(got[..., 5]).all() if math.isnan(bad) else (got[..., 5] == bad).all())
            rest = torch.arange(64, device="cuda") != 5
            assert torch.equal(got[..., rest], good[0][..., rest])
            pv.copy_(was)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("nq,nk,prefix,heads,kv", [([1] * 4, [50] * 4, 2000, 2, 1), ([300] * 8, [300] * 8, 130, 16, 8)])
def test_attention_shared_prefix_of_scores_far_apart(gpu, sign, nq, nk, prefix, heads, kv):
    """the prefix's keys score far more, or far less, than the own ones"""
    q, k, v, pk, pv = prefix_case(370, nq, nk, prefix, heads, kv, 32, BF16)
    q[..., 0] = 8.0
    pk[..., 0] = sign * 30.0
    out, lse = embed.attention_shared_prefix(q, k, v, pk, pv, offsets(nq), offsets(nk), scale=1.0, lse=True)
    check_prefix(q, k, v, pk, pv, nq, nk, True, 1.0, out, lse)


def test_attention_shared_prefix_refusals(gpu):
    q, k = rand(3, 4, 2, 32, dtype=BF16), rand(4, 4, 1, 32, dtype=BF16)
    p, off = rand(5, 9, 1, 32, dtype=BF16), offsets([4])
    for call, text in [
        (lambda: embed.attention_shared_prefix(q, k, k, p, p[:8], off), "one shape"),
        (lambda: embed.attention_shared_prefix(q, k, k, p[..., :16], p[..., :16], off), "one shape"),
        (lambda: embed.attention_shared_prefix(q, k, k, p.half(), p.half(), off), "q's type"),
        (lambda: embed.attention_shared_prefix(q, k, k, rand(6, 9, 1, 64, dtype=BF16)[..., ::2], p, off), "contiguous"),
        (lambda: embed.attention_shared_prefix(q, k, k, p.cpu(), p, off), "must be a tensor on"),
        (lambda: embed.attention_shared_prefix(q, k, k, p, p, None, off), "k_offsets without"),
        (lambda: embed.attention_shared_prefix(q, k, k, torch.nn.Parameter(p), p, off), "gradient"),
        (lambda: embed.attention_shared_prefix(q, k, k, rand(6, 9, 1, 36, dtype=BF16)[..., 4:], p, off), "multiples of 16 bytes|one shape"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


# ---------------------------------------------------------------- on both sides of the rules that choose a kernel

@pytest.mark.parametrize("rows,inner,cols", [
    (32, 300, 8191), (32, 300, 8192), (16, 300, 8192), (17, 260, 8205), (32, 64, 100),       # few rows, by 16 and by 32 columns
    (33, 320, 8192), (33, 320, 8200), (64, 256, 8224), (65, 256, 4096),                      # 256 and 257 narrow tiles
    (256, 96, 8192), (256, 96, 8128), (256, 96, 8256), (128, 100, 16384), (128, 100, 16321), (128, 100, 16385),  # 256 tiles of 128 x 64 and more
    (2816, 128, 1664), (2816, 128, 1537), (2816, 64, 1664), (2816, 192, 1663), (2560, 128, 1792), (300, 256, 9088), (256, 128, 17920),
    (2048, 128, 2048), (2049, 128, 2048), (2304, 128, 1920), (4352, 128, 1984)])  # 128 tiles of 256 x 128 (512 of 128 x 64) and more, 272
def test_gated_on_both_sides_of_the_rules(gpu, rows, inner, cols):
    x, wg, wu = gated_case(400, rows, inner, cols, BF16)
    h, gate, up = embed.gated(x, wg, wu, activation="gelu_tanh", save=True)
    check_gated(x, wg, wu, "gelu_tanh", h, gate, up)
    # weights whose strides differ, so that another kernel takes them
    wide = torch.zeros(cols, inner + 8, dtype=BF16, device="cuda")
    wide[:, :inner] = wu
    other = embed.gated(x, wg, wide[:, :inner], activation="gelu_tanh")
    check_gated(x, wg, wu, "gelu_tanh", other)


@pytest.mark.parametrize("rows,inner,cols", [
    (256, 256, 128), (256, 4096, 2304), (255, 4096, 2304), (3000, 520, 2048), (3008, 520, 2048), (2999, 1024, 1024),  # large tiles, with a tail and without
    (520, 264, 8192), (9000, 256, 192), (16390, 256, 256), (700, 2304, 1088),
    (1000, 512, 2048), (1000, 512, 1984), (600, 600, 1536), (2500, 64, 128), (20000, 64, 64), (70, 64, 8192), (64, 72, 5000)])  # tiles of 128 and 64, pieces of either product
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_backward_on_both_sides_of_the_rules(gpu, rows, inner, cols, dtype):
    x, wg, wu = gated_case(410, rows, inner, cols, dtype)
    gate, up, dh = rand(414, rows, cols, dtype=dtype, std=1.5), rand(415, rows, cols, dtype=dtype), rand(416, rows, cols, dtype=dtype, std=0.3)
    got = embed.gated_backward(dh, x, wg, wu, gate, up)
    check_gated_backward(dh, x, wg, wu, gate, up, "silu", *got)
    assert all(torch.equal(a, b) for a, b in zip(got, embed.gated_backward(dh, x, wg, wu, gate, up)))
    wide = torch.zeros(cols, inner + 8, dtype=dtype, device="cuda")
    wide[:, :inner] = wu
    dx, _, _ = embed.gated_backward(dh, x, wg, wide[:, :inner], gate, up, params=False)
    check_gated_backward(dh, x, wg, wu, gate, up, "silu", dx, None, None)


def test_gated_backward_of_a_tail_beside_a_row_that_is_not_finite(gpu):
    """large tiles: the rows behind the last one are zeros, not repetitions of it"""
    rows, inner, cols = 3001, 512, 2048
    x, wg, wu = gated_case(420, rows, inner, cols, BF16)
    gate, up, dh = (rand(423 + i, rows, cols, dtype=BF16) for i in range(3))
    x[-1, 5] = math.inf
    _, dwg, dwu = embed.gated_backward(dh, x, wg, wu, gate, up, activation="none")
    for dw, d in ((dwg, dh[-1] * up[-1]), (dwu, dh[-1] * gate[-1])):
        want = torch.where(d == 0, math.nan, torch.sign(d.float()) * math.inf)
        assert torch.equal(torch.nan_to_num(dw[:, 5].float(), nan=7.0), torch.nan_to_num(want, nan=7.0))
        assert torch.isfinite(dw[:, :5]).all() and torch.isfinite(dw[:, 6:]).all()


@pytest.mark.parametrize("nq,nk,prefix,heads,kv,dim", [
    ([1] * 8, [40] * 8, 1015, 8, 1, 64), ([1] * 8, [40] * 8, 1017, 8, 1, 64), ([1] * 8, [40] * 8, 700, 8, 8, 128),  # one pass, or the prefix apart
    ([20] * 8, [20] * 8, 900, 32, 8, 128), ([20] * 8, [20] * 8, 2000, 32, 8, 128), ([4] * 3, [4] * 3, 6000, 4, 4, 32),
    ([1], [5000], 100, 4, 1, 64), ([40], [3000], 3000, 4, 4, 96), ([1], [0], 20000, 8, 1, 64), ([1, 1], [3, 900], 9000, 9, 1, 64)])  # own keys in pieces; single tokens
def test_attention_shared_prefix_on_both_sides_of_the_rules(gpu, nq, nk, prefix, heads, kv, dim):
    for causal in (True, False):
        behind_prefix(430, nq, nk, prefix, heads, kv, dim, BF16, causal)


def test_past_32_bit_offsets(gpu):
    """rows and heads 2^31 bytes apart, keys in the last gigabytes of a long prefix"""
    buf = torch.empty((3 << 30) + 4096, dtype=BF16, device="cuda")
    x = buf.as_strided((4, 2, 64), (1 << 30, 128, 1))
    x.copy_(rand(440, 4, 2, 64))
    f, w = embed.rotary_frequencies(64), rand(441, 64)
    want, _ = embed.head_norm_rotary(x.contiguous(), None, None, f, w)
    got, _ = embed.head_norm_rotary(x, None, None, f, w)
    assert torch.equal(got, want)
    heads = buf.as_strided((2, 4, 64), (128, 1 << 30, 1))
    assert torch.equal(embed.head_norm_rotary(heads, None, torch.zeros(2, dtype=torch.int32, device="cuda"), None, w)[0].transpose(0, 1).contiguous(),
                       embed.head_norm_rotary(x, None, torch.zeros(4, dtype=torch.int32, device="cuda"), None, w)[0])
    dy = rand(442, 4, 2, 64, dtype=BF16)
    a, b = embed.head_norm_rotary_backward(dy, None, x, None, None, f, w), embed.head_norm_rotary_backward(dy, None, x.contiguous(), None, None, f, w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    embed.head_norm_rotary(x, None, None, f, w, out=(x, None))
    assert torch.equal(x, want)
    stride = (1 << 22) - 8
    pk, pv = buf.as_strided((700, 1, 64), (stride, 64, 1)), buf.as_strided((700, 1, 64), (stride, 64, 1), 128)
    pk.copy_(rand(443, 700, 1, 64))
    pv.copy_(rand(444, 700, 1, 64))
    for n in (1, 5, 300):
        q, k, v, _, _ = prefix_case(445, [n], [n], 1, 2, 1, 64, BF16)
        out, lse = embed.attention_shared_prefix(q, k, v, pk, pv, lse=True)
        check_prefix(q, k, v, pk.contiguous(), pv.contiguous(), [n], [n], True, 0.125, out, lse)
        back = embed.attention_shared_prefix(q, pk, pv, k, v, offsets([n]), offsets([700]))
        check_prefix(q, pk.contiguous(), pv.contiguous(), k, v, [n], [700], True, 0.125, back, None)
    x = buf.as_strided((4, 512), ((1 << 24) - 8, 1))
    x.copy_(rand(450, 4, 512))
    _, wg, wu = gated_case(451, 4, 512, 96, BF16)
    assert torch.equal(embed.gated(x, wg, wu), embed.gated(x.contiguous(), wg, wu))


# ---------------------------------------------------------------- together

class Block:
    """a block of an encoder as these operators make it"""

    def __init__(self, width=256, heads=8, kv=2, dim=32, hidden=512, dtype=BF16):
        def weight(seed, rows, cols):
            return rand(seed, rows, cols, dtype=dtype, std=cols ** -0.5)
        self.heads, self.kv, self.dim = heads, kv, dim
        self.qkv, self.mix = weight(500, (heads + 2 * kv) * dim, width), weight(501, width, heads * dim)
        self.both, self.down = weight(502, 2 * hidden, width), weight(503, width, hidden)
        self.n1, self.n2 = 1 + 0.1 * rand(504, width), 1 + 0.1 * rand(505, width)
        self.nq, self.nk = 1 + 0.1 * rand(506, dim), 1 + 0.1 * rand(507, dim)
        self.f = embed.rotary_frequencies(dim)

    def heads_of(self, x, positions):
        h, kv = self.heads, self.kv
        t = embed.linear(embed.layer_norm(x, self.n1), self.qkv).unflatten(1, (h + 2 * kv, self.dim))
        q, k = embed.head_norm_rotary(t[:, :h], t[:, h:h + kv], positions, self.f, self.nq, self.nk)
        return q, k, t[:, h + kv:]

    def rest(self, x, o):
        x = embed.linear(o.flatten(1), self.mix, residual=x)
        hidden = self.down.shape[1]
        h, gate, up = embed.gated(embed.layer_norm(x, self.n2), self.both[:hidden], self.both[hidden:], save=True)
        return embed.linear(h, self.down, residual=x), (x, h, gate, up)


def test_a_block_behind_a_prefix_is_the_block_over_all(gpu):
    """sequences encoded behind the cached keys of their prefix, and whole: the same vectors, up to a rounding of every
    operator's on both ways (10 of them, none of which a block of norms and unit weights magnifies in the mean)"""
    b, prefix, lengths = Block(), 70, [5, 40, 1, 23]
    front, tails = rand(510, prefix, 256, dtype=BF16), [rand(511 + i, n, 256, dtype=BF16) for i, n in enumerate(lengths)]
    pos = torch.arange(prefix, dtype=torch.int32, device="cuda")
    _, pk, pv = b.heads_of(front, pos)
    x = torch.cat(tails)
    q, k, v = b.heads_of(x, torch.cat([prefix + torch.arange(n, dtype=torch.int32, device="cuda") for n in lengths]))
    y, _ = b.rest(x, embed.attention_shared_prefix(q, k, v, pk, pv, offsets(lengths)))
    whole = torch.cat([torch.cat([front, t]) for t in tails])
    q, k, v = b.heads_of(whole, torch.cat([torch.arange(prefix + n, dtype=torch.int32, device="cuda") for n in lengths]))
    z, _ = b.rest(whole, embed.attention(q, k, v, offsets([prefix + n for n in lengths])))
    z = torch.cat([t[prefix:] for t in z.split([prefix + n for n in lengths])])
    assert (y.double() - z.double()).square().mean().sqrt() <= 10 * U[BF16] * z.double().square().mean().sqrt()


def test_results_together_on_another_stream_and_in_a_graph(gpu):
    b, lengths = Block(), [200, 1, 60, 39]
    x, off = rand(520, 300, 256, dtype=BF16), offsets(lengths)
    pos = torch.cat([90 + torch.arange(n, dtype=torch.int32, device="cuda") for n in lengths])
    pk, pv = rand(521, 900, 2, 32, dtype=BF16), rand(522, 900, 2, 32, dtype=BF16)
    one = offsets([1, 1, 1, 1])

    def step():
        q, k, v = b.heads_of(x, pos)
        o = embed.attention_shared_prefix(q, k, v, pk, pv, off, longest_q=200, longest_k=200)
        last = embed.attention_shared_prefix(q[:4], k, v, pk, pv, one, off, longest_q=1, longest_k=200)
        y, (mid, h, gate, up) = b.rest(x, o)
        hidden = b.down.shape[1]
        grads = embed.gated_backward(h, mid, b.both[:hidden], b.both[hidden:], gate, up)
        turned_back = embed.head_norm_rotary_backward(o, k, q, k, pos, b.f, b.nq, b.nk)
        return (y, last, *grads, *turned_back)
    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for g in got for a, c in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for t in range(3):
        x.copy_(rand(530 + t, 300, 256))
        pk.copy_(rand(540 + t, 900, 2, 32))
        graph.replay()
        torch.cuda.synchronize()
        copies = [a.clone() for a in captured]
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(copies, want))


def test_two_graphs_with_workspaces_of_their_own(gpu):
    """captured one after the other, replayed in turn on two streams"""
    def case(seed):
        x, wg, wu = gated_case(seed, 300, 256, 512, BF16)
        gate, up, dh = (rand(seed + 3 + i, 300, 512, dtype=BF16) for i in range(3))
        q, k, v, pk, pv = prefix_case(seed + 10, [1] * 30, [5] * 30, 3000, 8, 2, 64, BF16)
        off, one = offsets([5] * 30), offsets([1] * 30)

        def run():
            return (*embed.gated_backward(dh, x, wg, wu, gate, up), embed.attention_shared_prefix(q, k, v, pk, pv, one, off, longest_q=1, longest_k=5))
        return run
    runs = [case(600), case(650)]
    want = [r() for r in runs]
    graphs, outs = [], []
    for r in runs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(r())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


@pytest.mark.parametrize("nq,nk,prefix,heads,kv,dim", [
    ([5] * 3, [2, 3, 1], 13676, 8, 8, 80), ([5] * 40, [1] * 40, 9187, 12, 4, 128), ([2, 97, 40, 1] * 8, [2, 97, 40, 1] * 8, 9000, 8, 8, 32),  # many parts of a row, six and fewer
    ([1] * 16, [3] * 16, 4096, 8, 2, 64), ([1] * 16, [3] * 16, 12000, 8, 2, 64)])
def test_attention_shared_prefix_of_many_parts(gpu, nq, nk, prefix, heads, kv, dim):
    for dtype in (BF16, F16):
        behind_prefix(700, nq, nk, prefix, heads, kv, dim, dtype)


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1), (9, 1), (16, 1), (40, 4)])
@pytest.mark.parametrize("prefix", [0, 100, 1017, 16384])
def test_attention_shared_prefix_of_no_queries(gpu, heads, kv, prefix):
    q, k, p = (rand(440 + i, n, h, 64, dtype=BF16) for i, (n, h) in enumerate([(0, heads), (5, kv), (prefix, kv)]))
    for off in (None, offsets([0]), offsets([0, 0, 0])):
        own = offsets([5] if off is None or len(off) == 2 else [2, 0, 3])
        out, lse = embed.attention_shared_prefix(q, k, k, p, p, off, None if off is None else own, lse=True)
        assert out.shape == q.shape and out.dtype == BF16 and lse.shape == (0, heads)


def every_value(dtype):
    """all 65536 values of a 16-bit type, one row"""
    return torch.arange(1 << 16, device="cuda").to(torch.int16).view(dtype)[None]


def gate_gradients(gate, act):
    """dup and dgate for ones in the other places, as the weights' gradients of one row that is 1"""
    one, w = torch.ones(1, 1, dtype=gate.dtype, device="cuda"), torch.ones(gate.shape[1], 1, dtype=gate.dtype, device="cuda")
    _, slope, value = embed.gated_backward(torch.ones_like(gate), one, w, w, gate, torch.ones_like(gate), activation=act)
    return value[:, 0], slope[:, 0]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_slopes_of_every_finite_gate(gpu, act, dtype):
    gate = every_value(dtype)
    z = gate[0].double()
    # value z s and slope s + z s (1 - s) w' of s = 1 / (1 + exp(-w))
    k = 2 * math.sqrt(2 / math.pi)
    w, bend = (z, 1.0) if act == "silu" else (k * (z + 0.044715 * z ** 3), k * (1 + 3 * 0.044715 * z * z))
    s, rest = torch.sigmoid(w), torch.sigmoid(-w)
    # w in float32, 6 roundings at most, each 1 unit of w in the exponent; the exponential, the sum and the reciprocal, 5, and
    # two products
    part = 6 * E * w.abs() + 8 * E
    # exp(-w) from 2^126 on: 1 / (1 + exp(-w)) is below float32's normal range and may be 0
    lost = torch.where(w <= -126 * math.log(2), 1.0, 0.0)
    floor = 2.0 ** -126 if dtype == BF16 else TINY[dtype]  # bfloat16 below the normal range: matrix products may take it as 0
    value, slope = gate_gradients(gate, act)
    fine = torch.isfinite(z)
    want, whole = z * s, s + (z * s * rest * bend).abs()
    near(value[fine], want[fine], ((part + U[dtype] + lost) * want.abs() + floor)[fine])
    want = s + z * s * rest * bend
    near(slope[fine], want[fine], ((2 * part + 8 * E + lost) * whole + U[dtype] * want.abs() + floor)[fine])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_gradients_of_nan_gates_are_nan(gpu, act, dtype):
    gate = every_value(dtype)
    value, slope = gate_gradients(gate, act)
    assert torch.isnan(value[torch.isnan(gate[0])]).all()
    assert torch.isnan(slope[torch.isnan(gate[0])]).all() if act != "none" else (slope == 1).all()
    if act == "relu":
        fine = ~torch.isnan(gate[0])
        large = fine & ((gate[0].double().abs() >= 2.0 ** -126) | (gate[0] == 0))  # bfloat16 below the normal range
        assert torch.equal(slope[fine], (gate[0] > 0).to(dtype)[fine]) and torch.equal(value[large], torch.relu(gate[0])[large])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gated_gradients_of_infinite_gates_are_the_limits(gpu, act, dtype):
    gate = torch.tensor([[math.inf, -math.inf]], dtype=dtype, device="cuda")
    value, slope = gate_gradients(gate, act)
    assert value.tolist() == [math.inf, -math.inf if act == "none" else 0.0]
    assert slope.tolist() == [1.0, 1.0 if act == "none" else 0.0]


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_gated_gradients_of_products_past_float16(gpu, act):
    """gates that float16 saves as -infinity: the forward call's result and its gradients are 0, not NaN"""
    x, w = torch.full((3, 64), 200.0, dtype=F16, device="cuda"), torch.full((40, 64), 20.0, dtype=F16, device="cuda")
    h, gate, up = embed.gated(x, -w, 0.001 * w, activation=act, save=True)
    assert (gate == -math.inf).all() and (h == 0).all() and torch.isfinite(up).all()
    for g in embed.gated_backward(torch.ones_like(h), x, -w, 0.001 * w, gate, up, activation=act):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gelu_of_every_value_is_near_itself(gpu, dtype):
    """also where it is far below 1: of products with a large factor beside it, of float32 results and of gradients"""
    gate = every_value(dtype)[0]
    gate = gate[gate.abs() < 200]
    z = gate.double()
    lower, density = torch.special.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # the formula is off by 2.7e-6, 45 E, of erfc; its reciprocal, 4 E, weighs 2.3 times, its seven sums and products 1.8 times; the
    # exponent's three roundings, of its square's halves; the exponential, two products
    part = (1.5 * z * z + 45 + 4 * 2.3 + 14 * 1.8 + 6) * E
    lost = torch.where(z <= -13.2, 1.0, 0.0)  # exp(-z^2 / 2) is below float32's normal range
    low = 2.0 ** -126
    want = z * lower
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    got = embed.linear(gate[:, None], one, activation="gelu", out_dtype=F32)[:, 0]
    near(got, want, (part + lost) * want.abs() + low)
    near(embed.linear(gate[:, None], one, activation="gelu")[:, 0], want, (part + U[dtype] + lost) * want.abs() + max(low, TINY[dtype]))
    for factor in (1.0, 2.0 ** 14):  # the latter brings out what float16 has no bits for
        x = torch.stack([gate, torch.full_like(gate, factor)], 1)
        w = torch.eye(2, dtype=dtype, device="cuda")
        fine = (want * factor).abs() < 60000  # float16's largest number
        tol = (part + U[dtype] + 2 * E + lost) * want.abs() * factor + max(low * factor, TINY[dtype])
        near(embed.gated(x, w[:1], w[1:], activation="gelu")[fine, 0], want[fine] * factor, tol[fine])
    value, slope = gate_gradients(gate[None], "gelu")
    near(value, want, (part + U[dtype] + lost) * want.abs() + max(low, TINY[dtype]))
    whole = lower + z.abs() * density
    near(slope, lower + z * density, (part + 6 * E + lost) * whole + U[dtype] * (lower + z * density).abs() + max(low, TINY[dtype]))
