"""Refusals of the decoder operators' C entries and host functions: no GPU, no launch."""
import ctypes

import pytest
import torch

from axs6_b200 import _lib, unified

ARG, ALIGN, DEVICE, WORKSPACE, UNSUPPORTED = -1, -2, -3, -5, -6


def s3(*v):
    return (ctypes.c_int64 * 3)(*v)


def test_rotary_arguments():
    lib = _lib.load()
    ok = dict(q=16, qo=16, qh=2, qs=s3(64, 32, 8), qos=s3(64, 32, 8), k=None, ko=None, kh=0, ks=None, kos=None, dtype=0, batch=1, tokens=4, size=8,
              rotated=8, pos=16, p64=1, pb=0, pt=1, turns=16, gain=1.0, inter=0, inv=0)

    def call(**kw):
        a = ok | kw
        return lib.axs6_rotary(*a.values(), None)
    for bad in (dict(q=None), dict(qo=None), dict(qs=None), dict(dtype=7), dict(rotated=7), dict(rotated=10), dict(size=0), dict(size=5000, rotated=8),
                dict(batch=-1), dict(tokens=-1), dict(qh=-1), dict(pos=None), dict(turns=None), dict(kh=1), dict(rotated=-2)):
        assert call(**bad) == ARG, bad
    assert call(batch=0) == 0 and call(tokens=0) == 0 and call(qh=0) == 0       # nothing to do


def test_distillation_arguments():
    lib = _lib.load()
    fwd = dict(z=16, dt=0, rows=2, vocab=10, ld=10, t=16, tdt=0, ldt=3, ix=16, ldi=3, slots=3, temp=1.0, red=2, loss=16, stats=16, out=16, cnt=16)
    for bad in (dict(z=None), dict(t=None), dict(ix=None), dict(dt=2), dict(tdt=-1), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(slots=0), dict(temp=0.0),
                dict(temp=float("inf")), dict(temp=float("nan")), dict(red=3), dict(loss=None), dict(stats=None), dict(out=None), dict(cnt=None)):
        assert lib.axs6_distill_fwd(*(fwd | bad).values(), None) == ARG, bad
    assert lib.axs6_distill_fwd(*(fwd | dict(slots=1025)).values(), None) == UNSUPPORTED
    assert lib.axs6_distill_fwd(*(fwd | dict(stats=20)).values(), None) == ALIGN
    bwd = dict(z=16, dt=0, rows=2, vocab=10, ld=10, t=16, tdt=0, ldt=3, ix=16, ldi=3, slots=3, temp=1.0, stats=16, up=16, ups=0, cnt=None, grad=16, ldg=10)
    for bad in (dict(stats=None), dict(up=None), dict(grad=None), dict(ldg=-1)):
        assert lib.axs6_distill_bwd(*(bwd | bad).values(), None) == ARG, bad
    assert lib.axs6_distill_bwd(*(bwd | dict(rows=0)).values(), None) == 0


def attn(**kw):
    a = _lib.AttnArgs()
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv", "row_max", "row_sum"):
        setattr(a, n, 256)
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        getattr(a, n + "_strides")[:] = [1024, 512, 64]
    a.batch, a.q_heads, a.k_heads, a.q_len, a.k_len, a.head_size, a.scale = 1, 2, 1, 8, 8, 64, 0.125
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_attention_arguments():
    lib = _lib.load()
    for bad in (dict(q=None), dict(k=None), dict(o=None), dict(row_max=None), dict(dtype=5), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
                dict(scale=float("nan")), dict(batch=-1), dict(q_heads=3, k_heads=2), dict(k_heads=0), dict(head_size=0), dict(window=3), dict(window=-1, causal=1),
                dict(mask_kind=9), dict(mask_kind=1), dict(q_len=1 << 31), dict(batch=1 << 20, q_heads=1 << 12, k_heads=1)):
        assert lib.axs6_attn_fwd(ctypes.byref(attn(**bad)), None) == ARG, bad
    assert lib.axs6_attn_fwd(ctypes.byref(attn(head_size=129)), None) == UNSUPPORTED
    assert lib.axs6_attn_fwd(None, None) == ARG and lib.axs6_attn_bwd(None, None) == ARG
    assert lib.axs6_attn_fwd(ctypes.byref(attn(batch=0)), None) == 0 and lib.axs6_attn_fwd(ctypes.byref(attn(q_len=0)), None) == 0
    for bad in (dict(d_o=None), dict(dq=None), dict(dk=None)):
        assert lib.axs6_attn_bwd(ctypes.byref(attn(**bad)), None) == ARG, bad
    assert lib.axs6_attn_bwd(ctypes.byref(attn()), None) == WORKSPACE
    assert lib.axs6_attn_workspace_bytes(ctypes.byref(attn(dtype=9)), 1) == 0
    need = lib.axs6_attn_workspace_bytes(ctypes.byref(attn()), 1)
    assert need == 2 * 8 * 4
    assert lib.axs6_attn_bwd(ctypes.byref(attn(workspace=264, workspace_bytes=need)), None) == ALIGN
    assert lib.axs6_attn_workspace_bytes(ctypes.byref(attn(dtype=1)), 1) == 2 * 128 * 4 * 2      # whole tiles, two arrays


def test_structure_has_the_size_of_the_header():
    # 8 + 5 + 1 pointers with the workspace's, 24 + 4 strides, 7 sizes, workspace_bytes; scale and four 32-bit numbers padded to 24 bytes
    assert ctypes.sizeof(_lib.AttnArgs) == 8 * (8 + 24 + 6 + 4 + 7 + 2) + 24


def test_host_functions():
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        unified.axs_attention_unified(*(torch.randn(1, 1, 2, 8) for _ in range(3)))
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        unified.axs_distillation_unified(torch.randn(2, 5), torch.randn(2, 1), torch.zeros(2, 1, dtype=torch.int64))
    plan = unified.rotary_frequencies(8, device="cpu")
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        unified.axs_rotary_unified(torch.randn(1, 1, 2, 8), None, torch.arange(2), plan)
    with pytest.raises(ValueError):
        unified.axs_distillation_unified(torch.randn(2, 5), torch.randn(2, 1), torch.zeros(2, 1, dtype=torch.int64), reduction="max")


@pytest.mark.parametrize("rotated,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0)])
def test_fixed_point_turns(rotated, base):
    """Each pair's turns per position, as a 64-bit fraction: off by half a unit and by the rounding of the 64-bit frequency."""
    import math
    plan = unified.rotary_frequencies(rotated, base, device="cpu")
    assert plan.rotated == rotated and plan.gain == 1.0
    for i, t in enumerate(plan.turns.tolist()):
        want = base ** (-2 * i / rotated) / (2 * math.pi)
        assert abs((t % (1 << 64)) / 2.0 ** 64 - want) <= 2.0 ** -51 * want + 2.0 ** -64
