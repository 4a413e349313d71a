"""Rotary positions against the formula in 64 bits, and the gradient against the transposed rotation and against differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from axs6_b200 import unified  # noqa: E402

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}          # half a step, relative


def reference(x, positions, freq, gain, layout, inverse=False):
    """-> (values, bound of the arithmetic's error before the last rounding), 64 bits."""
    R = 2 * len(freq)
    pos = positions.double()
    pos = pos[None] if pos.dim() == 1 else pos
    t = pos[:, None, :, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = gain * t.cos(), gain * t.sin() * (-1 if inverse else 1)
    a, b = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    y, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    u, v = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    # cos and sin: angle, polynomial, gain: at most 4 roundings of 2^-24 relative to 1; two products, a sum: 3 more; the frequencies' fixed
    # point is off by 2^-65 turns a position
    far = 2 * math.pi * float(pos.abs().max() if pos.numel() else 0) * 2.0 ** -64
    e = (u.abs() + v.abs()) * gain * (8 * 2.0 ** -24 + far)
    bound[..., a], bound[..., b] = e, e
    return y, bound


def check(got, x, positions, freq, gain, layout, inverse=False):
    want, bound = reference(x, positions, freq, gain, layout, inverse)
    assert got.shape == x.shape and got.dtype == x.dtype
    err = (got.double() - want).abs()
    assert bool((err <= bound + EPS[x.dtype] * (want.abs() + bound)).all()), float((err - bound).max())


def plain(rotated, base=10000.0):
    return [base ** (-2.0 * i / rotated) for i in range(rotated // 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,R", [(1, 1, 1, 1, 2, 2), (2, 5, 4, 4, 64, 64), (3, 17, 6, 2, 128, 64), (1, 33, 3, 1, 72, 36),
                                            (2, 3, 5, 5, 33, 30), (1, 300, 8, 2, 128, 128), (2, 4, 2, 1, 40, 0), (1, 2, 1, 1, 4096, 4096),
                                            (5, 129, 2, 1, 80, 40)])
def test_forward_and_gradient(dtype, layout, B, S, Hq, Hkv, D, R):
    g = torch.Generator(device="cuda").manual_seed(B * 100 + S)
    q = torch.randn(B, Hq, S, D, generator=g, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(B, S, Hkv, D, generator=g, device="cuda").to(dtype).transpose(1, 2).requires_grad_()
    pos = torch.randint(-50, 200000, (B, S), generator=g, device="cuda")
    f = unified.rotary_frequencies(R)
    assert f.rotated == R
    yq, yk = unified.axs_rotary_unified(q, k, pos, f, layout)
    check(yq.detach(), q.detach(), pos, plain(R), 1.0, layout)
    check(yk.detach(), k.detach(), pos, plain(R), 1.0, layout)
    assert yk.stride() == k.stride()                                   # the operand's layout is kept
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    check(dq, gq, pos, plain(R), 1.0, layout, inverse=True)
    check(dk, gk, pos, plain(R), 1.0, layout, inverse=True)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
def test_scaled_frequencies_far_positions(scaling, factor):
    R, base, n = 64, 10000.0, 4096
    f = unified.rotary_frequencies(R, base, scaling, factor, n)
    freq, gain = plain(R, base), 1.0
    if scaling == "linear":
        freq = [w / factor for w in freq]
    elif scaling == "ntk":
        freq = plain(R, base * factor ** (R / (R - 2)))
        assert math.isclose(freq[-1], plain(R)[-1] / factor, rel_tol=1e-9) and freq[0] == 1.0
    else:
        gain = 0.1 * math.log(factor) + 1
        turns = [n * w / (2 * math.pi) for w in freq]
        got = [t / 2.0 ** 64 * 2 * math.pi for t in f.turns.tolist()]
        for i, (t, w, x) in enumerate(zip(turns, freq, got)):          # the ends are fixed by the definition
            if t > 33 and turns[min(i + 1, R // 2 - 1)] > 32:
                assert math.isclose(x, w, rel_tol=1e-12)
            if t < 1 and turns[max(i - 1, 0)] < 1:
                assert math.isclose(x, w / factor, rel_tol=1e-12)
            assert w / factor * (1 - 1e-12) <= x <= w * (1 + 1e-12)
        freq = got
    x = torch.randn(1, 2, 64, R, device="cuda")
    pos = torch.arange(64, device="cuda") * 33333 + (1 << 21)
    y, none = unified.axs_rotary_unified(x, None, pos, f)
    assert none is None and math.isclose(f.gain, gain)
    check(y, x, pos, freq, f.gain, "half")


def test_int32_positions_large_values_and_shared_positions():
    x = torch.randn(2, 3, 4, 32, device="cuda")
    f = unified.rotary_frequencies(32)
    pos = torch.tensor([0, 1, 2 ** 31 - 1, -2 ** 31], device="cuda")
    a, _ = unified.axs_rotary_unified(x, None, pos, f)
    b, _ = unified.axs_rotary_unified(x, None, pos.to(torch.int32).expand(2, 4), f)
    assert torch.equal(a, b)
    check(a, x, pos, plain(32), 1.0, "half")
    assert torch.equal(a[:, :, 0], x[:, :, 0])                          # position 0 turns nothing


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_views_match_packed_ones(dtype):
    """A slice of a fused projection, rows that start off a 16-byte boundary, and copies of them: the same bits."""
    buf = torch.randn(2, 7, 3 * 4 * 64 + 1, device="cuda").to(dtype)
    f, pos = unified.rotary_frequencies(64), torch.arange(7, device="cuda")
    for off in (0, 1):
        part = buf[..., off:off + 256].unflatten(-1, (4, 64)).transpose(1, 2)
        a, _ = unified.axs_rotary_unified(part, None, pos, f)
        b, _ = unified.axs_rotary_unified(part.contiguous(), None, pos, f)
        assert torch.equal(a, b)
    t = torch.randn(2, 4, 64, 7, device="cuda").to(dtype).transpose(-1, -2)     # inner stride not 1
    a, _ = unified.axs_rotary_unified(t, None, pos, f)
    b, _ = unified.axs_rotary_unified(t.contiguous(), None, pos, f)
    assert torch.equal(a, b)


def test_empty_one_sided_gradient_and_differences():
    f, pos = unified.rotary_frequencies(8), torch.arange(3, device="cuda")
    e, _ = unified.axs_rotary_unified(torch.empty(0, 2, 3, 8, device="cuda"), None, pos, f)
    assert e.shape == (0, 2, 3, 8)
    q = torch.randn(1, 1, 3, 8, device="cuda", requires_grad=True)
    k = torch.randn(1, 1, 3, 8, device="cuda", requires_grad=True)
    yq, yk = unified.axs_rotary_unified(q, k, pos, f)
    dq, dk = torch.autograd.grad(yq.sum(), (q, k), allow_unused=True)
    assert dk is None or not dk.any()
    w = torch.randn_like(yq)
    dq, = torch.autograd.grad((unified.axs_rotary_unified(q, k, pos, f)[0] * w).sum(), q)
    d = torch.randn_like(q)
    # linear in q: the difference quotient has no error of its own; 48 terms of fp32 roundings
    lo, hi = (unified.axs_rotary_unified(q.detach() + s * d, None, pos, f)[0] for s in (-1.0, 1.0))
    assert abs(float((((hi - lo) / 2).double() * w.double()).sum() - (dq.double() * d.double()).sum())) < 48 * 16 * 2.0 ** -22


def test_refusals():
    f, pos = unified.rotary_frequencies(8), torch.arange(3, device="cuda")
    x = torch.randn(1, 1, 3, 8, device="cuda")
    for bad, err in [(dict(q=x.half()), TypeError), (dict(q=x[0]), ValueError), (dict(q=None, k=None), ValueError),
                     (dict(positions=pos.float()), ValueError), (dict(positions=pos[:2]), ValueError), (dict(layout="other"), ValueError),
                     (dict(q=x[..., :6]), ValueError), (dict(k=x.bfloat16()), ValueError), (dict(k=x[:, :, :2]), ValueError),
                     (dict(q=x.cpu()), RuntimeError), (dict(positions=pos.cpu()), ValueError), (dict(frequencies=f.turns), TypeError)]:
        args = dict(q=x, k=None, positions=pos, frequencies=f, layout="half") | bad
        with pytest.raises(err):
            unified.axs_rotary_unified(**args)
    for bad in (dict(rotated=7), dict(rotated=8, base=0.0), dict(rotated=8, scaling="other"), dict(rotated=8, factor=-1.0)):
        with pytest.raises(ValueError):
            unified.rotary_frequencies(**bad)


def test_captured_and_replayed():
    x, f, pos = torch.randn(2, 4, 16, 64, device="cuda").bfloat16(), unified.rotary_frequencies(64), torch.arange(16, device="cuda")
    unified.axs_rotary_unified(x, x, pos, f)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = unified.axs_rotary_unified(x, x, pos, f)
    x.copy_(torch.randn_like(x))
    pos.add_(1000)
    g.replay()
    want, _ = unified.axs_rotary_unified(x, None, pos, f)
    assert torch.equal(a, want) and torch.equal(b, want)
