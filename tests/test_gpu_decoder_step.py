"""Rotary positions, attention and the distillation loss together, as a decoder's training step uses them: the chain's gradients against
plain formulas in 64 bits, and the modules and the pipeline that call them."""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

from axs6_b200 import unified  # noqa: E402


def plain_rotary(x, positions, inv):
    t = positions.double()[..., None] * inv
    c, s = t.cos(), t.sin()
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3 * 2.0 ** -8)])
def test_chain_and_gradients(dtype, tol):
    """q, k, v -> rotary -> causal attention with shared key heads -> a head's product -> distillation, in one backward pass.  Relative 2-norms;
    bf16: three roundings in a row (rotated heads, probabilities, outputs) on the way there and as many back, each at most half a step (2^-8)
    and on average less than half of that; fp32: sums of up to 200 terms on a chain of five products."""
    B, Hq, Hkv, S, D, V, K = 2, 4, 2, 67, 32, 501, 9
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(B, S, h, D, generator=g, device="cuda").to(dtype).transpose(1, 2).requires_grad_() for h in (Hq, Hkv, Hkv))
    w = (torch.randn(V, Hq * D, generator=g, device="cuda") * 0.3).to(dtype)
    pos = torch.arange(S, device="cuda") + torch.tensor([[0], [5000]], device="cuda")
    top, index = torch.randn(B, S, V, generator=g, device="cuda").topk(K, -1)
    index[0, 60:] = -1
    plan = unified.rotary_frequencies(D)
    qr, kr = unified.axs_rotary_unified(q, k, pos, plan)
    o = unified.axs_attention_unified(qr, kr, v, causal=True)
    logits = (o.transpose(1, 2).reshape(B, S, Hq * D).float() @ w.float().T).to(dtype)
    loss = unified.axs_distillation_unified(logits, top, index, temperature=2.0)
    grads = torch.autograd.grad(loss, (q, k, v))

    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    pp = pos[:, None]
    q2, k2 = plain_rotary(leaves[0], pp, inv), plain_rotary(leaves[1], pp, inv).repeat_interleave(Hq // Hkv, 1)
    x = q2 @ k2.mT / math.sqrt(D)
    x = x.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    o2 = torch.softmax(x, -1) @ leaves[2].repeat_interleave(Hq // Hkv, 1)
    log_q = torch.log_softmax(o2.transpose(1, 2).reshape(B, S, Hq * D) @ w.double().T / 2.0, -1)
    p = torch.softmax(top.double() / 2.0, -1)
    used = index[..., 0] >= 0
    want = ((p * (p.log() - log_q.gather(-1, index.clamp_min(0)))).sum(-1) * used).sum() * 4.0 / used.sum()
    want_grads = torch.autograd.grad(want, leaves)
    assert abs(float(loss) - float(want)) <= tol * abs(float(want))
    for a, b in zip(grads, want_grads):
        assert float((a.double() - b).norm() / b.norm()) <= tol


def test_attention_module_without_materialised_weights():
    """quantize_weights=False: the projections as before, the weights exact, masks and rotary positions as in the operators."""
    torch.manual_seed(0)
    E, H, B, S = 96, 4, 2, 50
    plan = unified.rotary_frequencies(E // H)
    m = unified.AXSMultiheadAttentionUnified(E, H, quantize_weights=False, rotary=plan).cuda()
    x = torch.randn(B, S, E, device="cuda")
    mask = torch.zeros(S, S, device="cuda").masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    a, b = m(x, x, x, attn_mask=mask), m(x, x, x, causal=True)
    # the same scores with a mask added and without: fp32 both; then through a quantiser, which may send values next to a border one level apart
    q, k, v = (m._heads(p(x)) for p in (m.q_proj, m.k_proj, m.v_proj))
    q, k = unified.axs_rotary_unified(q, k, torch.arange(S, device="cuda"), plan)
    scores = q.double() @ k.double().mT * m.scale + mask.double()
    ctx = torch.softmax(scores, -1) @ v.double()
    got = unified.axs_attention_unified(q, k, v, causal=True)
    assert float((got.double() - ctx).norm() / ctx.norm()) < 4e-6
    want = m.out_proj(got.transpose(1, 2).reshape(B, S, E))
    assert torch.equal(b, want)
    assert float((a - b).norm() / b.norm()) < 0.02
    lengths = torch.tensor([S, 20], dtype=torch.int32, device="cuda")
    c = m(x, x, x, causal=True, key_lengths=lengths)
    assert torch.equal(c[0], b[0]) and torch.equal(c[1, :20], b[1, :20])
    y = m(x[:, -1:], x, x, positions=torch.arange(S, device="cuda"), causal=True)          # one query over all keys
    assert y.shape == (B, 1, E)
    b.sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any()) for p in (m.q_proj.weight, m.k_proj.weight, m.v_proj.weight))
    old = unified.AXSMultiheadAttentionUnified(E, H).cuda()
    for bad in (dict(causal=True), dict(key_lengths=lengths), dict(positions=torch.arange(S, device="cuda"))):
        with pytest.raises(ValueError):
            old(x, x, x, **bad)
    with pytest.raises(ValueError):
        unified.AXSMultiheadAttentionUnified(E, H, dropout=0.1, quantize_weights=False)
    with pytest.raises(ValueError):
        m(x[:, :3], x, x)


class Student(nn.Module):
    def __init__(self, vocab=300, dim=64, heads=4):
        super().__init__()
        self.tok = unified.AXSEmbeddingUnified(vocab, dim)
        self.attn = unified.AXSMultiheadAttentionUnified(dim, heads, quantize_weights=False, rotary=unified.rotary_frequencies(dim // heads, device="cpu"))
        self.ln = unified.AXSLayerNormUnified(dim)
        self.head = unified.AXSLinearMixedPrecision(dim, vocab, bias=False)

    def forward(self, batch):
        x = self.tok(batch["tokens"])
        h = self.ln(x)
        x = x + self.attn(h, h, h, causal=True, key_lengths=batch["lengths"])
        return self.head(x)


def test_distillation_step_of_the_pipeline():
    torch.manual_seed(3)
    model = Student().cuda()
    tokens = torch.randint(0, 300, (3, 40), device="cuda")
    lengths = torch.tensor([40, 17, 1], dtype=torch.int32, device="cuda")
    top, index = torch.randn(3, 40, 300, device="cuda").topk(8, -1)
    index[torch.arange(40, device="cuda")[None] >= lengths[:, None]] = -1                # padding: no slot used
    batch = {"tokens": tokens, "lengths": lengths}
    pipe = unified.AXSTrainingPipelineUnified(model, torch.optim.AdamW(model.parameters(), lr=1e-3), loss_scale_init=2.0 ** 10)
    before = [p.detach().clone() for p in model.parameters()]
    out = pipe.distillation_step(batch, lambda b: (top, index), temperature=2.0)
    assert not out["overflow"] and math.isfinite(out["loss"]) and math.isfinite(out["grad_norm"]) and out["grad_norm"] > 0
    assert all(bool(p.grad.isfinite().all()) for p in model.parameters())
    assert all(not torch.equal(a, b) for a, b, n in zip(before, model.parameters(), (n for n, _ in model.named_parameters())) if "bias" not in n)
    again = pipe.distillation_step(batch, lambda b: (top, index))
    assert again["step"] == 2


@pytest.mark.parametrize("D", [32, 33])
def test_results_can_be_changed_in_place_and_saved_tensors_are_checked(D):
    """The loss and rotated heads are tensors of their own: in-place changes behind them are differentiated.  Attention's backward pass needs
    its output, and operands are saved: a change of those is reported."""
    x = torch.randn(1, 2, 5, D, device="cuda").bfloat16().requires_grad_()
    o = unified.axs_attention_unified(x, x, x)
    o *= 2
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    top, index = torch.randn(4, 9, device="cuda").topk(3, -1)
    for reduction in ("mean", "sum", "none"):
        loss = unified.axs_distillation_unified(z, top, index, reduction=reduction)
        want, = torch.autograd.grad(loss.sum(), z, retain_graph=True)
        loss /= 4
        got, = torch.autograd.grad(loss.sum(), z)
        assert torch.equal(got, want / 4)
    y, _ = unified.axs_rotary_unified(x.detach().requires_grad_()[..., :32], None, torch.arange(5, device="cuda"), unified.rotary_frequencies(32))
    y += 1
    y.sum().backward()
    top2 = top.clone()
    loss = unified.axs_distillation_unified(z, top2, index)
    top2.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_backward_is_the_first_work_of_its_thread(dtype):
    """A program whose backward thread has not used the device before attention's backward pass: the thread has no context of its own yet."""
    import os
    import subprocess
    import sys
    code = f"""
import torch
from torch.profiler import ProfilerActivity, profile
from axs6_b200 import unified
q, k, v, g = (torch.randn(1, 2, 64, 64, device="cuda").to(torch.{dtype}) for _ in range(4))
leaves = [t.requires_grad_() for t in (q, k, v)]
o = unified.axs_attention_unified(*leaves, causal=True)
torch.cuda.synchronize()
with profile(activities=[ProfilerActivity.CUDA]):
    grads = torch.autograd.grad(o, leaves, g)
    torch.cuda.synchronize()
assert all(bool(t.isfinite().all()) for t in grads)
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-1500:]


def test_second_derivatives_are_refused():
    x = torch.randn(1, 1, 4, 8, device="cuda", requires_grad=True)
    z, top, index = torch.randn(2, 6, device="cuda", requires_grad=True), torch.randn(2, 2, device="cuda"), torch.tensor([[0, 1], [2, 3]], device="cuda")
    plan, pos = unified.rotary_frequencies(8), torch.arange(4, device="cuda")
    for leaf, out in ((x, unified.axs_attention_unified(x, x, x).sum()), (x, unified.axs_rotary_unified(x, None, pos, plan)[0].pow(2).sum()),
                      (z, unified.axs_distillation_unified(z, top, index))):
        g, = torch.autograd.grad(out, leaf, create_graph=True)
        # without a graph behind the gradient, or with one that says so, whichever the upstream gradient leads to
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            g.sum().backward()
