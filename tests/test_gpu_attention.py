"""Attention forward and backward against the definition in 64 bits, at the sizes, masks and layouts where a kernel can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from attention_reference import check, reference  # noqa: E402
from axs6_b200 import unified  # noqa: E402

# relative 2-norm: fp32 sums; bf16: independent roundings of the probabilities (or the scores' gradients) and of the result, each at most
# half a step (2^-8) and on average less than half of that
NORM = {torch.float32: 4e-6, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]


def tensors(B, Hq, Hkv, Sq, Sk, D, dtype, seed=0, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(S, H):
        t = torch.randn(B, S, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
        return t.contiguous() if packed else t
    return one(Sq, Hq), one(Sk, Hkv), one(Sk, Hkv), one(Sq, Hq)


def compare(q, k, v, g, norm=True, **kw):
    """One call with its backward pass, everything checked -> (o, lse, dq, dk, dv)."""
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o, lse = unified.axs_attention_unified(q, k, v, return_lse=True, **kw)
    assert o.dtype == q.dtype and o.shape == q.shape and lse.dtype == torch.float32
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), g)
    want = reference(q.detach(), k.detach(), v.detach(), g, **kw)
    for name, got in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(name, got.detach(), *want[name], norm=NORM[q.dtype] if norm and name != "lse" else None)
    return o.detach(), lse, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D", [(1, 1, 1, 1, 1, 8), (2, 3, 3, 5, 5, 16), (1, 2, 1, 64, 64, 64), (1, 4, 2, 127, 129, 40),
                                              (2, 2, 2, 128, 128, 128), (1, 8, 1, 130, 257, 64), (1, 6, 2, 300, 300, 96), (3, 2, 2, 33, 700, 72),
                                              (1, 1, 1, 513, 100, 128), (1, 2, 2, 600, 600, 128), (2, 4, 4, 511, 511, 64)])
def test_sizes(dtype, causal, B, Hq, Hkv, Sq, Sk, D):
    compare(*tensors(B, Hq, Hkv, Sq, Sk, D, dtype, Sq + Sk + D), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 7, 33, 65, 100, 127])
def test_odd_head_sizes(dtype, D):
    compare(*tensors(1, 2, 1, 40, 70, D, dtype, D), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq,Sk,window", [(50, 50, 1), (300, 300, 7), (257, 400, 128), (400, 257, 100), (200, 200, 10 ** 9), (1, 900, 300), (700, 700, 256)])
def test_window(dtype, Sq, Sk, window):
    # With one key a row p = 1 and dS = p (dp - p dp) = 0: dq and dk are zeros that only roundings differ from, and a norm relative to them says
    # nothing.  The bounds hold for them as for all.
    compare(*tensors(2, 4, 2, Sq, Sk, 64, dtype, Sq), norm=window > 1, causal=True, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 400, 64), (300, 300, 128), (130, 513, 80)])
def test_lengths_hide_whatever_the_memory_holds(dtype, causal, Sq, Sk, D):
    q, k, v, g = tensors(6, 4, 2, Sq, Sk, D, dtype, 7)
    lengths = torch.tensor([0, 1, Sk, Sk // 2, 128, Sk - 1], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.inf
    o, lse, dq, dk, dv = compare(q, k, v, g, causal=causal, key_lengths=lengths)
    assert not o[0].any() and not dq[0].any() and bool((lse[0] == -math.inf).all())
    for b, n in enumerate(lengths.tolist()):
        assert not dk[b, :, n:].any() and not dv[b, :, n:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["bool", "fp32", "bf16", "lowest"])
@pytest.mark.parametrize("shape", [(2, 4, 90, 200), (2, 1, 90, 200), (1, 1, 1, 200), (90, 200), (4, 1, 200)])
def test_mask_tensors(dtype, kind, shape):
    q, k, v, g = tensors(2, 4, 2, 90, 200, 64, dtype, 11)
    kept = torch.rand(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.6
    if shape[-2] == 90:
        kept[..., 5, :] = False                                    # a row without any key
    kept[..., 100:140] = False
    if kind == "bool":
        mask = kept
    elif kind == "lowest":
        mask = torch.where(kept, 0.0, torch.finfo(torch.float32).min)   # hides nothing by itself: a row of it is uniform
    else:
        mask = torch.where(kept, torch.randn(shape, device="cuda"), -math.inf).to(torch.float32 if kind == "fp32" else torch.bfloat16)
    o, *_ = compare(q, k, v, g, mask=mask)
    if shape[-2] == 90:
        if kind == "lowest":
            assert bool(o[:, :, 5].any())
        else:
            assert not o[:, :, 5].any()
    compare(q, k, v, g, mask=mask, causal=True, key_lengths=torch.tensor([200, 77], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_before_the_first_key_are_empty(dtype):
    """More queries than keys: causal rows that stand before key 0 see nothing."""
    q, k, v, g = tensors(1, 2, 1, 400, 150, 64, dtype, 2)
    o, lse, dq, *_ = compare(q, k, v, g, causal=True)
    assert not o[:, :, :250].any() and not dq[:, :, :250].any() and bool((lse[:, :, :250] == -math.inf).all())
    assert bool(o[:, :, 250:].any(-1).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_growing_scores(dtype):
    """Scores up to a few hundred, and keys whose scores grow along the sequence, so that the running maximum moves in every tile."""
    q, k, v, g = tensors(1, 2, 2, 200, 900, 64, dtype, 5)
    compare((q * 6).to(dtype), (k * 6).to(dtype), v, g, norm=False)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.1, 8.0, 900, device="cuda")[:, None]).to(dtype)
    compare(q, k, v, g, norm=False)
    compare(q, k.flip(2), v, g, norm=False)
    compare(q, -k, v, g, norm=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_scale_and_few_queries_over_long_keys(dtype):
    compare(*tensors(1, 2, 1, 3, 300, 64, dtype, 1), scale=0.3)
    compare(*tensors(1, 8, 2, 1, 5000, 128, dtype, 1))
    compare(*tensors(2, 16, 2, 4, 3001, 64, dtype, 1), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """(batch, tokens, heads, size) views, packed tensors, slices of a fused projection and misaligned views: one result."""
    q, k, v, g = tensors(2, 4, 2, 150, 150, 64, dtype, 8)
    ref = compare(q, k, v, g, causal=True)
    fused = torch.randn(2, 150, 9 * 64, device="cuda").to(dtype)
    off = torch.randn(2, 150, 8 * 64 + 3, device="cuda").to(dtype)
    for part, at, t in ((fused, 64, q), (off, 3, q)):
        part[..., at:at + 256] = t.transpose(1, 2).flatten(2)
    fused[..., 320:448], fused[..., 448:576] = k.transpose(1, 2).flatten(2), v.transpose(1, 2).flatten(2)

    def heads(x, at, n):
        return x[..., at:at + 64 * n].unflatten(-1, (n, 64)).transpose(1, 2)
    qs = [q.contiguous(), heads(fused, 64, 4), heads(off, 3, 4), q.transpose(-1, -2).contiguous().transpose(-1, -2)]
    for qq in qs:
        got = compare(qq, heads(fused, 320, 2), heads(fused, 448, 2), g.contiguous(), causal=True)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    leaf = k[:, :1].detach().requires_grad_()                       # a key head shared through expand: gradients add up
    o = unified.axs_attention_unified(q, leaf.expand(2, 2, 150, 64), v)
    dk, = torch.autograd.grad(o, leaf, g)
    full = k[:, :1].expand(2, 2, 150, 64).contiguous()
    w = reference(q, full, v, g)["dk"]
    check("dk", dk.double(), w[0].sum(1, keepdim=True), w[1].sum(1, keepdim=True) * 1.01 + 2 * 2.0 ** -8 * w[0].abs().sum(1, keepdim=True))
    one = torch.ones((), device="cuda", dtype=dtype)
    o = unified.axs_attention_unified(q.requires_grad_(), k, v)
    dq, = torch.autograd.grad(o, q, one.expand(o.shape))            # an upstream gradient without strides of its own
    want = reference(q.detach(), k, v, torch.ones_like(g))["dq"]
    check("dq", dq, *want)


@pytest.mark.parametrize("dtype", TYPES)
def test_repeatable_and_rows_do_not_depend_on_their_neighbours(dtype):
    q, k, v, g = tensors(2, 4, 2, 333, 333, 64, dtype, 4)
    a, b = compare(q, k, v, g, causal=True), compare(q, k, v, g, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c = compare(q[1:], k[1:], v[1:], g[1:], causal=True)
    assert all(torch.equal(x[1:], y) for x, y in zip(a, c))


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_extents(dtype):
    for B, Hq, Hkv, Sq, Sk in [(0, 2, 2, 4, 4), (1, 2, 2, 0, 4), (1, 2, 1, 4, 0), (1, 0, 0, 4, 4)]:
        q, k, v, g = tensors(B, Hq, Hkv, Sq, Sk, 16, dtype)
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        o = unified.axs_attention_unified(q, k, v)
        assert o.shape == q.shape and not o.any()
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), g)
        assert not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_lies_around_the_outputs_is_left_alone(dtype):
    """Outputs of odd sizes written into the middle of larger tensors."""
    from axs6_b200 import ops
    q, k, v, g = tensors(2, 2, 1, 77, 131, 40, dtype, 6, packed=True)
    mask, scale, window = ops.attention_check(q, k, v, None, None, None, True, None, "test")
    made = []
    real = torch.empty_like

    def guarded(t, **kw):
        if t.dim() != 4:
            return real(t, **kw)
        buf = torch.full((t.shape[0], t.shape[1], t.shape[2] + 2, 48), 7.0, dtype=t.dtype, device=t.device)
        made.append(buf)
        return buf[:, :, 1:-1, :40]
    torch.empty_like = guarded
    try:
        o, stats, lse, q, k, v, low = ops.attention_fwd(q, k, v, None, mask, scale, True, window, True)
        grads = ops.attention_bwd(g, q, k, v, o, low, stats, None, mask, scale, True, window)
    finally:
        torch.empty_like = real
    assert len(made) == 4
    for buf in made:
        assert bool((buf[:, :, 0] == 7).all()) and bool((buf[:, :, -1] == 7).all()) and bool((buf[..., 40:] == 7).all())
    want = reference(q, k, v, g, causal=True)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        check(name, got, *want[name])


def test_gradient_by_differences():
    q, k, v, g = tensors(1, 2, 1, 9, 12, 8, torch.float32, 3)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    grads = torch.autograd.grad(unified.axs_attention_unified(q, k, v, causal=True), (q, k, v), g)
    step = 2.0 ** -8
    for n, t in enumerate((q, k, v)):
        d = torch.randn_like(t)

        def at(s):
            a = [x.detach().double() for x in (q, k, v)]
            a[n] = a[n] + s * d.double()
            return (reference(*a, causal=True)["o"][0] * g.double()).sum()
        quotient = (at(step) - at(-step)) / (2 * step)
        # central difference: step^2 / 6 times a third derivative of a few hundred at most; the kernel's own error is checked elsewhere
        assert abs(float(quotient) - float((grads[n].double() * d.double()).sum())) < step ** 2 * 100 + 1e-4


@pytest.mark.parametrize("dtype", TYPES)
def test_other_streams_and_captures(dtype):
    q, k, v, g = tensors(1, 4, 2, 200, 200, 64, dtype, 9)
    want = compare(q, k, v, g, causal=True)

    def step():
        a = [t.detach().requires_grad_() for t in (q, k, v)]
        o = unified.axs_attention_unified(*a, causal=True)
        return (o.detach(), *torch.autograd.grad(o, a, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [step() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for out in outs:
        assert all(torch.equal(x, y) for x, y in zip(out, (want[0], *want[2:])))
    graphs = []
    for _ in range(2):                                              # two captures alive at once, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for t in (q, k, v):
        t.copy_(t.flip(2))
    want = compare(q, k, v, g, causal=True)
    for graph, out in graphs + graphs[::-1]:
        for t in out:
            t.zero_()
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(out, (want[0], *want[2:])))


def test_refusals():
    q, k, v, _ = tensors(2, 4, 2, 8, 9, 16, torch.float32)
    for bad, err in [(dict(q=q.cpu()), RuntimeError), (dict(q=q.half(), k=k.half(), v=v.half()), TypeError), (dict(q=q.bfloat16()), TypeError),
                     (dict(q=q[:, :3]), ValueError), (dict(q=q[0]), ValueError), (dict(v=v[:, :, :4]), ValueError), (dict(k=k[..., :8], v=v[..., :8]), ValueError),
                     (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.nan), ValueError), (dict(window=4), ValueError),
                     (dict(window=0, causal=True), ValueError), (dict(key_lengths=torch.ones(2, device="cuda")), ValueError),
                     (dict(key_lengths=torch.ones(3, device="cuda", dtype=torch.int32)), ValueError),
                     (dict(key_lengths=torch.ones(2, dtype=torch.int32)), ValueError), (dict(mask=torch.ones(8, 9, device="cuda", dtype=torch.int32)), TypeError),
                     (dict(mask=torch.ones(8, 9, device="cuda", requires_grad=True)), ValueError), (dict(mask=torch.ones(8, 8, device="cuda")), RuntimeError),
                     (dict(q=torch.randn(1, 1, 4, 129, device="cuda"), k=torch.randn(1, 1, 4, 129, device="cuda"), v=torch.randn(1, 1, 4, 129, device="cuda")), ValueError)]:
        with pytest.raises(err):
            unified.axs_attention_unified(**(dict(q=q, k=k, v=v) | bad))


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,causal,window", [(4, 24, 8, 300, 300, 64, True, None), (2, 40, 40, 257, 1100, 128, False, None),
                                                            (3, 32, 8, 1100, 1100, 128, True, None), (5, 130, 1, 1, 900, 64, False, None),
                                                            (2, 48, 16, 700, 700, 80, True, 200), (1, 80, 8, 700, 300, 64, True, None),
                                                            (2, 64, 64, 513, 1025, 64, False, None)])
def test_many_heads(B, Hq, Hkv, Sq, Sk, D, causal, window):
    """Calls that fill the device, one CTA for 256 queries: walks of different and of no length side by side, lengths, masks."""
    q, k, v, g = tensors(B, Hq, Hkv, Sq, Sk, D, torch.bfloat16, Sq + Sk)
    compare(q, k, v, g, causal=causal, window=window)
    compare(q, k, v, g, causal=causal, window=window, mask=torch.rand(B, 1, Sq, Sk, device="cuda") < 0.7)
    lengths = torch.tensor([(Sk * (b + 1) // B if b else 0) for b in range(B)], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
    compare(q, k, v, g, causal=causal, window=window, key_lengths=lengths)


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    from axs6_b200 import _lib
    yield
    assert _lib.load().axs6_attn_status() == 0


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,Sk,D,window", [(1, 1, 1, 1, 70000, 64, None), (3, 8, 2, 1, 2500, 128, None), (2, 12, 4, 7, 1000, 96, None),
                                                     (1, 64, 1, 3, 1500, 64, None), (1, 8, 2, 200, 3000, 128, None), (1, 2, 2, 1000, 1000, 64, None),
                                                     (1, 16, 2, 33, 4000, 64, 500), (1, 4, 1, 400, 300, 72, None), (40, 4, 4, 100, 129, 40, None),
                                                     (2, 4, 2, 1, 1, 64, None), (5, 130, 1, 1, 900, 64, None)])
def test_few_queries_stacked_heads_and_cut_keys(causal, B, Hq, Hkv, Sq, Sk, D, window):
    """One or two tiles of stacked rows, keys in one chunk or many, lengths that leave chunks empty."""
    if window and not causal:
        window = None
    q, k, v, g = tensors(B, Hq, Hkv, Sq, Sk, D, torch.bfloat16, Sq + Sk)
    compare(q, k, v, g, causal=causal, window=window)
    lengths = torch.tensor([(Sk * (b + 1) // B if b else 0) for b in range(B)], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
    compare(q, k, v, g, causal=causal, window=window, key_lengths=lengths)
    mask = torch.rand(1, 1, Sq, Sk, device="cuda") < 0.7
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    compare(q, k, v, g, causal=causal, window=window, mask=mask)
