"""The distillation loss and its gradient against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from axs6_b200 import unified  # noqa: E402

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def reference(z, t, index, tau):
    """-> per row: loss, d loss / d logits, and bounds of their errors before the last rounding; 64 bits."""
    V = z.shape[-1]
    z, t = z.double() / tau, t.double() / tau
    used = (index >= 0) & (index < V) & (t != -math.inf)
    t = t.masked_fill(~used, -math.inf)
    row = used.any(-1)
    p = torch.softmax(t, -1).nan_to_num(0.0)
    ix = index.clamp(0, V - 1)
    log_q = torch.log_softmax(z, -1)
    picked = log_q.gather(-1, ix)
    terms = torch.where(p > 0, p * (p.log() - picked), 0.0)
    loss = terms.sum(-1) * tau * tau
    full = torch.zeros_like(z).scatter_add_(-1, ix, p)
    q = log_q.exp() * row[:, None]
    grad = tau * (q - full)
    # exp2 of (z - max) / tau * log2 e: argument x rounded three times (3 |x| 2^-24 ln 2 < 3 |x| 2^-24), the function itself 2^-22; the row's sum
    # of V / 512 + 16 additions in a thread and across; two more products
    x = (z - z.amax(-1, keepdim=True)).nan_to_num(0.0, neginf=0.0).abs()
    rel = 3 * x * 2.0 ** -24 + 2.0 ** -21 + (V / 512 + 16) * 2.0 ** -24
    tx = (t - t.amax(-1, keepdim=True)).nan_to_num(0.0, neginf=0.0, posinf=0.0).abs()
    prel = 3 * tx * 2.0 ** -24 + 2.0 ** -21 + 64 * 2.0 ** -24
    fullb = torch.zeros_like(z).scatter_add_(-1, ix, p * prel)
    gb = tau * (q * rel + fullb) + 4 * 2.0 ** -24 * tau * (q + full)
    # a term p (log p - log q): both logarithms carry the relative errors above as absolute ones, plus roundings of their parts
    size = tx + x.gather(-1, ix) + 40
    lb = tau * tau * (p * (2 * prel + rel.gather(-1, ix) + 8 * size * 2.0 ** -24) + terms.abs() * prel).sum(-1) + loss.abs() * 64 * 2.0 ** -24
    return loss * row, grad * row[:, None], lb * row, gb, row


def make(T, V, K, zt, tt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(T, V, generator=g, device="cuda") * 3
    t, index = (z + torch.randn(T, V, generator=g, device="cuda")).topk(K, -1)
    return z.to(zt), t.to(tt), index


def run(z, t, index, tau, reduction, up=None):
    z = z.clone().requires_grad_() if z.is_contiguous() else z.detach().requires_grad_()
    loss = unified.axs_distillation_unified(z, t, index, tau, reduction)
    assert loss.dtype == torch.float32
    grad, = torch.autograd.grad(loss, z, up)
    assert grad.dtype == z.dtype and grad.shape == z.shape
    return loss.detach(), grad


def check(z, t, index, tau):
    want, gw, lb, gb, row = reference(z, t, index, tau)
    n = max(1, int(row.sum()))
    h = HALF[z.dtype]
    up = torch.randn(want.shape, device="cuda")
    loss, grad = run(z, t, index, tau, "none", up)
    assert bool(((loss.double() - want).abs() <= lb + 2.0 ** -24 * want.abs()).all())
    u = up.double()[:, None]
    # bf16: also the smallest subnormal step of the type
    assert bool(((grad.double() - gw * u).abs() <= u.abs() * gb + h * (u * gw).abs() + h * u.abs() * gb + 2.0 ** -126).all())
    assert not grad[~row].any() and not loss[~row].any()
    for reduction, d in (("sum", 1), ("mean", n)):
        loss, grad = run(z, t, index, tau, reduction)
        assert loss.dim() == 0
        assert abs(float(loss) - float(want.sum() / d)) <= float(lb.sum() / d) + 2.0 ** -23 * abs(float(want.sum() / d)) + 1e-30
        assert bool(((grad.double() - gw / d).abs() <= (gb / d) * (1 + h) + (h + 2.0 ** -22) * (gw / d).abs() + 2.0 ** -126).all())


@pytest.mark.parametrize("zt,tt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                   (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("T,V,K,tau", [(1, 1, 1, 1.0), (3, 7, 7, 2.0), (5, 200, 20, 1.0), (300, 1000, 64, 2.0), (2, 32000, 64, 1.0),
                                       (7, 50001, 1, 0.5), (4, 131073, 256, 1.0), (2, 2048, 1024, 3.0), (700, 33, 5, 1.0)])
def test_loss_and_gradient(zt, tt, T, V, K, tau):
    check(*make(T, V, K, zt, tt, T + V), tau)


@pytest.mark.parametrize("zt", [torch.float32, torch.bfloat16])
def test_unused_slots_rows_and_repeated_indices(zt):
    z, t, index = make(6, 513, 9, zt, torch.float32, 3)
    index[0] = -1                                                  # nothing used
    index[1, 4:] = -1                                              # some slots used
    index[2, 3] = 513                                              # behind the vocabulary
    index[3] = index[3, 0]                                         # one index nine times
    index[4, 5] = index[4, 1]
    t[4, 7] = -math.inf
    t[5] = -math.inf                                               # no mass at all
    z[0] = math.nan                                                # never read
    z[1, 500] = -math.inf
    want, gw, lb, gb, row = reference(torch.where(z.isnan(), 0.0, z), t, index, 1.0)
    assert row.tolist() == [False, True, True, True, True, False]
    loss, grad = run(z, t, index, 1.0, "none", torch.ones(6, device="cuda"))
    assert bool(((loss.double() - want).abs() <= lb + 2.0 ** -24 * want.abs()).all())
    assert bool(((grad.double() - gw).abs() <= gb * 1.01 + HALF[zt] * gw.abs() + 2.0 ** -126).all())
    assert not grad[0].any() and not grad[5].any()
    loss, _ = run(z, t, index, 1.0, "mean")
    assert abs(float(loss) - float(want.sum() / 4)) <= float(lb.sum() / 4) + 2.0 ** -22 * float(want.sum() / 4)
    index.fill_(-1)
    loss, grad = run(z, t, index, 1.0, "mean")
    assert float(loss) == 0.0 and not grad.any()


def test_large_logits_and_gradient_by_differences():
    z, t, index = make(3, 400, 8, torch.float32, torch.float32, 5)
    check(z * 1000 + 50000, t, index, 1.0)
    z = z / 3
    z.requires_grad_()
    g, = torch.autograd.grad(unified.axs_distillation_unified(z, t, index, 2.0, "sum"), z)
    d = torch.randn_like(z)
    step = 2.0 ** -5

    def at(s):
        return reference((z.detach().double() + s * d.double()), t, index, 2.0)[0].sum()
    # the reference's own central difference: error step^2 / 6 of the third derivative, |d|^3 <= 70 on the mass that counts
    assert abs(float((at(step) - at(-step)) / (2 * step)) - float((g.double() * d.double()).sum())) < step ** 2 / 6 * 70 * 3 + 1e-4


@pytest.mark.parametrize("zt", [torch.float32, torch.bfloat16])
def test_strided_rows_shapes_and_repeatability(zt):
    z, t, index = make(12, 1001, 6, zt, zt, 9)
    want, gw = run(z, t, index, 1.0, "sum")
    wide = torch.randn(12, 1100, device="cuda").to(zt)
    wide[:, 3:1004] = z
    view = wide[:, 3:1004]
    loss, grad = run(view, t, index.to(torch.int32), 1.0, "sum")
    # rows that start elsewhere are split over threads elsewhere: sums of a row differ in the last bits
    assert abs(float(loss - want)) <= 12 * 40 * 2.0 ** -20
    assert bool(((grad.double() - gw.double()).abs() <= (2.0 ** -18 + 2 * HALF[zt]) * gw.double().abs() + 2.0 ** -18).all())
    again, ga = run(z, t, index, 1.0, "sum")
    assert torch.equal(again, want) and torch.equal(ga, gw)
    l3, g3 = run(z.view(3, 4, 1001), t.view(3, 4, 6), index.view(3, 4, 6), 1.0, "none", torch.ones(3, 4, device="cuda"))
    assert l3.shape == (3, 4) and torch.equal(g3.view(12, 1001), gw)
    e, ge = run(torch.empty(0, 10, device="cuda").to(zt), torch.empty(0, 2, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"), 1.0, "mean")
    assert float(e) == 0.0 and ge.shape == (0, 10)


def test_more_rows_than_a_grid():
    check(*make(5000, 65, 3, torch.bfloat16, torch.float32, 2), 1.0)


def test_captured_step_beside_an_eager_one():
    z, t, index = make(40, 1000, 8, torch.bfloat16, torch.float32, 4)
    z.requires_grad_()
    # An eager graph stays alive over the capture.  torch ties a leaf's gradient node to the stream it was first used on, and a capture may not
    # reach it while that graph lives: the captured step has a leaf of its own over the same memory.
    eager = unified.axs_distillation_unified(z, t, index)
    leaf = z.detach().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(unified.axs_distillation_unified(leaf, t, index), leaf)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = unified.axs_distillation_unified(leaf, t, index)
        grad, = torch.autograd.grad(loss, leaf)
    want, = torch.autograd.grad(eager, z)
    g.replay()
    assert torch.equal(grad, want) and torch.equal(loss, eager.detach())


def test_refusals():
    z, t, index = make(4, 50, 3, torch.float32, torch.float32)
    for bad, err in [(dict(temperature=0.0), ValueError), (dict(temperature=math.inf), ValueError), (dict(reduction="other"), ValueError),
                     (dict(teacher_index=index.float()), TypeError), (dict(teacher_index=index[:3]), ValueError),
                     (dict(teacher_logits=t[:, :2]), ValueError), (dict(teacher_logits=t.cpu()), RuntimeError),
                     (dict(logits=z.cpu()), RuntimeError), (dict(logits=z[:, :0]), ValueError),
                     (dict(teacher_logits=t[:, :0], teacher_index=index[:, :0]), ValueError),
                     (dict(teacher_logits=t[:, :1].expand(4, 1025), teacher_index=index[:, :1].expand(4, 1025)), ValueError)]:
        with pytest.raises(err):
            unified.axs_distillation_unified(**(dict(logits=z, teacher_logits=t, teacher_index=index) | bad))
