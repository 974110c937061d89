"""The operators that complete an encoder's block without a GPU: refusals before any device call, frequencies."""
import ctypes as C
import math

import pytest

from beam_search_collab_amd import _lib
from test_embed_host import PTR, refused


def rotary_args(**change):
    a = _lib.HeadNormRotaryArgs()
    d = dict(q=PTR, k=PTR, q_out=PTR, k_out=PTR, q_grad=PTR, k_grad=PTR, frequencies=PTR, tokens=5, heads=4, kv_heads=2, head_dim=64,
             rotary=64, norm=1, type=2, wtype=0, eps=1e-6, magnitude=1.0) | change
    for n in ("q", "k", "q_grad", "k_grad", "q_out", "k_out"):
        d.setdefault(n + "_stride", 256)
        d.setdefault(n + "_head_stride", 64)
    for n, x in d.items():
        setattr(a, n, x)
    return a


ROTARY = [
    (dict(type=3), "type must be"), (dict(wtype=1), "wtype must be"), (dict(head_dim=63), "head_dim must be"), (dict(head_dim=0), "head_dim must be"),
    (dict(head_dim=258), "head_dim must be"), (dict(rotary=66), "rotary must be"), (dict(rotary=31), "rotary must be"),
    (dict(heads=0), "heads must be"), (dict(heads=1025), "heads must be"), (dict(kv_heads=1025), "heads must be"),
    (dict(tokens=1 << 31), "tokens must be"), (dict(eps=-1e-9), "eps must be"), (dict(eps=math.nan), "eps must be"), (dict(eps=math.inf), "eps must be"),
    (dict(magnitude=math.nan), "magnitude must be"), (dict(norm=0, q_weight=PTR), "weights belong"), (dict(frequencies=None), "frequencies must be given"),
    (dict(q=None), "q must be given"), (dict(k=None), "k must be given"), (dict(q_out=None), "q_out must be given"),
    (dict(q_stride=63), "heads of q overlap"), (dict(k_head_stride=60), "heads of k overlap"), (dict(q_out_stride=128), "heads of q_out overlap"),
    (dict(k_stride=1 << 41), "too far apart"),
]


@pytest.mark.parametrize("change,text", ROTARY)
def test_head_norm_rotary_refuses(change, text):
    refused(_lib.hip().bs_head_norm_rotary(C.byref(rotary_args(**change)), None), text)
    refused(_lib.hip().bs_head_norm_rotary_backward(C.byref(rotary_args(**change)), PTR, 1 << 30, None), text)


def test_head_norm_rotary_backward_refuses():
    run = _lib.hip().bs_head_norm_rotary_backward
    refused(run(C.byref(rotary_args(q_grad=None)), None, 0, None), "q_grad must be given")
    refused(run(C.byref(rotary_args(k_grad_stride=10)), None, 0, None), "heads of k_grad overlap")
    a, n = rotary_args(q_weight_grad=PTR), C.c_uint64(0)
    assert _lib.hip().bs_head_norm_rotary_backward_workspace(C.byref(a), C.byref(n)) == 0 and n.value > 0
    refused(run(C.byref(a), None, 0, None), "the workspace must hold")
    refused(run(C.byref(a), PTR, n.value - 1, None), "the workspace must hold")
    refused(run(C.byref(a), PTR + 4, n.value, None), "16-byte aligned")
    refused(run(C.byref(rotary_args(norm=0, k_weight_grad=PTR)), PTR, 1 << 20, None), "weights belong")
    refused(run(None, PTR, 1 << 20, None), "args is null")
    refused(_lib.hip().bs_head_norm_rotary_backward_workspace(None, C.byref(n)), "args is null")
    refused(_lib.hip().bs_head_norm_rotary_backward_workspace(C.byref(a), None), "bytes is null")
    assert _lib.hip().bs_head_norm_rotary(C.byref(rotary_args(tokens=0, q=None)), None) == 0
    assert run(C.byref(rotary_args(tokens=0)), None, 0, None) == 0


def test_rotary_frequencies():
    import torch
    from beam_search_collab_amd import embed
    f = embed.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(embed.rotary_frequencies(8, base=100.0, stretch=4.0, device="cpu"), f / 4)
    # turns over the trained length: 1000 f / 2 pi; below 20 stretched, above 100 kept, between them mixed
    g = embed.rotary_frequencies(8, base=100.0, stretch=4.0, trained=1000, low=20.0, high=100.0, device="cpu")
    turns = 1000 * f / (2 * math.pi)
    for i in range(4):
        keep = min(1.0, max(0.0, (turns[i].item() - 20) / 80))
        assert abs(g[i].item() - f[i].item() * (keep + (1 - keep) / 4)) < 1e-15
    assert turns[0] > 100 and g[0] == f[0] and turns[2] < 20 and g[2] == f[2] / 4 and f[1] / 4 < g[1] < f[1]
    assert embed.rotary_frequencies(0, device="cpu").numel() == 0
    for bad in (dict(rotary=7), dict(rotary=-2), dict(rotary=8, base=0.0), dict(rotary=8, stretch=0.0), dict(rotary=8, trained=10, low=3.0, high=3.0)):
        with pytest.raises(ValueError):
            embed.rotary_frequencies(device="cpu", **bad)
