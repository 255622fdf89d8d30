"""The differentiable forms and the drop-ins that use them: gradients stage by
stage against the formulas in 64 bits (bounds as derived in the two modules
they come from), together as a layer, captured, and where nothing is recorded.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from tests.test_gpu_attention_bwd import check as check_attn
from tests.test_gpu_attention_bwd import make as make_attn
from tests.test_gpu_attention_bwd import reference, token_mask
from tests.test_gpu_norm_grad import backward_ref, forward_ref
from tests.test_gpu_norm_grad import check as check_norm
from tests.test_gpu_norm_grad import make as make_norm

pytestmark = pytest.mark.gpu


def test_attention_function_both_results():
    from sinkattn_b200.autograd import block_sparse_attention

    q, k, v, dout, mask = make_attn(2, 3, 400, 500, 0.4, 1)
    dlse = torch.randn(2, 3, 400, device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out, lse = block_sparse_attention(*leaves, mask)
    got = torch.autograd.grad((out, lse), leaves, (dout, dlse))
    keep = token_mask(mask, 2, 3, 400, 500)
    ref, bound = reference(q, k, v, dout, keep, 1 / math.sqrt(128), dlse)
    check_attn(got, ref, bound)
    # through the log-sum-exp alone: dv is 0
    out, lse = block_sparse_attention(*leaves, mask)
    got = torch.autograd.grad(lse, leaves, dlse)
    ref, bound = reference(q, k, v, torch.zeros_like(dout), keep, 1 / math.sqrt(128), dlse)
    check_attn(got, ref, bound)
    with pytest.raises(RuntimeError):
        out, _ = block_sparse_attention(*leaves, mask)
        first = torch.autograd.grad(out.float().sum(), leaves[0], create_graph=True)[0]
        torch.autograd.grad(first.float().sum(), leaves[1])


def test_more_queries_than_the_gradient_takes():
    """The forward pass of a call that records runs as it does unrecorded; the backward refuses."""
    from sinkattn_b200 import ops
    from sinkattn_b200.autograd import block_sparse_attention

    q = torch.randn(1, 1, 131073, 128, device="cuda").bfloat16().requires_grad_()
    k, v = (torch.randn(1, 1, 100, 128, device="cuda").bfloat16() for _ in range(2))
    mask = torch.ones(1, 1, 1025, 1, dtype=torch.bool, device="cuda")
    out, lse = block_sparse_attention(q, k, v, mask)
    want, want_lse = ops.bsattn_fwd(q.detach(), k, v, mask)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    with pytest.raises(RuntimeError, match="at most 131072"):
        out.sum().backward()


def test_broadcast_keys_and_a_broadcast_gradient():
    from sinkattn_b200.autograd import block_sparse_attention

    q, k, v, dout, mask = make_attn(1, 4, 300, 300, 0.6, 2, layout="bhsd")
    k1, v1 = (t[:, :1].detach().clone().requires_grad_() for t in (k, v))
    out, _ = block_sparse_attention(q, k1.expand(-1, 4, -1, -1), v1.expand(-1, 4, -1, -1), mask)
    out.sum().backward()  # a gradient of ones, expanded from one value
    ones = torch.ones_like(dout)
    keep = token_mask(mask, 1, 4, 300, 300)
    ref, bound = reference(q, k[:, :1].expand_as(k), v[:, :1].expand_as(v), ones, keep,
                           1 / math.sqrt(128))
    for got, r, b in ((k1.grad, ref[1], bound[1]), (v1.grad, ref[2], bound[2])):
        # summed over the heads in bf16: three more roundings of partial sums
        b = b.sum(1, keepdim=True) + 3 * 2.0 ** -8 * (r.abs() + b).sum(1, keepdim=True)
        assert ((got.double() - r.sum(1, keepdim=True)).abs() <= b * 1.001 + 2.0 ** -100).all()


@pytest.mark.parametrize("lengths", [[(300, 300), (300, 300)], [(300, 130), (0, 64), (200, 0), (77, 300)]])
def test_varlen_function_is_differentiable(lengths):
    from sinkattn_b200 import block_sparse_attn_func

    H = 2
    cq = torch.tensor([0] + [a for a, _ in lengths], dtype=torch.int32).cumsum(0).int().cuda()
    ck = torch.tensor([0] + [b for _, b in lengths], dtype=torch.int32).cumsum(0).int().cuda()
    g = torch.Generator(device="cuda").manual_seed(4)
    n, m = int(cq[-1]), int(ck[-1])
    q, k, v, dout = (torch.randn(s, H, 128, generator=g, device="cuda").bfloat16()
                     for s in (n, m, m, n))
    Sq, Sk = max(a for a, _ in lengths), max(b for _, b in lengths)
    mask = torch.rand(len(lengths), H, -(-Sq // 128), -(-Sk // 128), generator=g, device="cuda") < 0.6
    args = (cq, ck, torch.ones(H, dtype=torch.int32, device="cuda"), None, mask, Sq, Sk)
    want, lse_want, _ = block_sparse_attn_func(q, k, v, *args, return_attn_probs=True)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out, lse, _ = block_sparse_attn_func(*leaves, *args, return_attn_probs=True)
    assert torch.equal(out, want) and torch.equal(lse, lse_want)
    got = torch.autograd.grad(out, leaves, dout)
    for b, (a, c) in enumerate(lengths):
        qs, ks = slice(int(cq[b]), int(cq[b + 1])), slice(int(ck[b]), int(ck[b + 1]))
        if a == 0 or c == 0:
            for t, s in ((got[0], qs), (got[1], ks), (got[2], ks)):
                assert not t[s].any()
            continue
        view = lambda t, s: t[s].permute(1, 0, 2)[None]
        mb = mask[b:b + 1, :, : -(-a // 128), : -(-c // 128)]
        ref, bound = reference(view(q, qs), view(k, ks), view(v, ks), view(dout, qs),
                               token_mask(mb, 1, H, a, c), 1 / math.sqrt(128))
        check_attn([view(got[0], qs), view(got[1], ks), view(got[2], ks)], ref, bound)


def test_adapter_keeps_its_results_and_records():
    from sinkattn_b200.reference_api import _block_sparse_attn

    q, k, v, dout, mask = make_attn(1, 2, 260, 260, 0.6, 5)
    want, lse_want = _block_sparse_attn(q, k, v, mask)
    assert not want.requires_grad
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    with torch.no_grad():
        assert not _block_sparse_attn(*leaves, mask)[0].requires_grad
    out, lse = _block_sparse_attn(*leaves, mask)
    assert torch.equal(out, want) and torch.equal(lse, lse_want) and lse.dtype == torch.bfloat16
    got = torch.autograd.grad(out, leaves, dout)
    ref, bound = reference(q, k, v, dout, token_mask(mask, 1, 2, 260, 260), 1 / math.sqrt(128))
    check_attn(got, ref, bound)


def test_layer_of_per_head_norm_and_attention():
    """Norm + rotation, attention and a projection-shaped reduction together;
    each stage's gradient against the formulas at the values it was given."""
    from sinkattn_b200 import autograd, ops

    B, S, H = 2, 389, 4
    a, w, cos, sin, pos = make_norm(B, S, H, H, 128, 128, torch.bfloat16, T=900, seed=7)
    v = a["dk"].detach().clone().requires_grad_()
    x = {n: a[n].detach().clone().requires_grad_() for n in ("q", "k")}
    ws = [t.detach().clone().requires_grad_() for t in w]
    nb = -(-S // 128)
    mask = torch.rand(B, H, nb, nb, device="cuda") < 0.5
    mask[..., 0] = True
    q, k = autograd.qk_head_norm_rope(x["q"], x["k"], 1e-6, ws[0], ws[1], cos, sin, positions=pos)
    q.retain_grad(), k.retain_grad()
    out, _ = autograd.block_sparse_attention(*(t.transpose(1, 2) for t in (q, k, v)), mask)
    dout = torch.randn(B, S, H, 128, device="cuda").bfloat16()
    out.transpose(1, 2).backward(dout)
    ops.DeviceStatus.check()
    check_norm("q", q.detach(), *forward_ref(a["q"], w[0], 1e-6, cos, sin, pos, True))
    heads = lambda t: t.detach().transpose(1, 2)
    ref, bound = reference(heads(q), heads(k), heads(v), heads(dout),
                           token_mask(mask, B, H, S, S), 1 / math.sqrt(128))
    check_attn([heads(t) for t in (q.grad, k.grad, v.grad)], ref, bound)
    for n, up, wt, w0 in (("q", q.grad, ws[0], w[0]), ("k", k.grad, ws[1], w[1])):
        dx, bx, dw, bw = backward_ref(up, a[n], w0, 1e-6, cos, sin, pos, True)
        check_norm("d" + n, x[n].grad, dx, bx)
        assert wt.grad.dtype == torch.bfloat16
        check_norm("dw_" + n, wt.grad, dw, bw + 2.0 ** -8 * dw.abs())


def test_hidden_norm_function_and_the_wan_producer():
    from sinkattn_b200 import autograd
    from sinkattn_b200.reference_api import fused_prepare_attention_tensors

    B, S, H, D = 2, 70, 3, 128
    hidden = H * D
    g = torch.Generator(device="cuda").manual_seed(8)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda")
    lin = [torch.nn.Linear(hidden, hidden, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    norms = [SimpleNamespace(weight=torch.nn.Parameter(1 + 0.2 * mk(hidden)), eps=1e-6, bias=None)
             for _ in range(2)]
    attn = SimpleNamespace(to_q=lin[0], to_k=lin[1], to_v=lin[2], norm_q=norms[0], norm_k=norms[1],
                           heads=H)
    h = mk(B, S, hidden).bfloat16()
    ang = torch.rand(S, D // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    with torch.no_grad():
        want = fused_prepare_attention_tensors(attn, h, None, (cos, sin))
    q, k, v, _ = fused_prepare_attention_tensors(attn, h, None, (cos, sin))
    for x, y in zip((q, k, v), want):
        assert torch.equal(x, y)
    dq, dk = mk(B, H, S, D).bfloat16(), mk(B, H, S, D).bfloat16()
    torch.autograd.backward((q, k), (dq, dk))
    with torch.no_grad():
        proj = [lin[0](h), lin[1](h)]
    for up, x, norm, layer in ((dq, proj[0], norms[0], lin[0]), (dk, proj[1], norms[1], lin[1])):
        split = (B, S, H, D)
        dx, bx, dw, bw = backward_ref(up.transpose(1, 2), x.view(split),
                                      norm.weight.detach().view(H, D), 1e-6, cos, sin, None, True,
                                      over=2)
        check_norm("dw", norm.weight.grad.view(H, D), dw, bw)
        # the projection got that gradient: its bias sums it over the tokens (torch's sum,
        # rounded to bf16)
        bias = layer.bias.grad.double()
        tol = bx.sum((0, 1)) + 2.0 ** -8 * (dx.sum((0, 1)).abs() + bx.sum((0, 1)))
        assert ((bias - dx.sum((0, 1)).reshape(-1)).abs() <= tol.reshape(-1) * 1.01).all()
    # the function alone, one input without a gradient
    x = [t.detach().clone() for t in proj]
    x[1].requires_grad_()
    oq, ok = autograd.qk_norm_rope(x[0], x[1], D, 1e-6, norms[0].weight.detach(),
                                   norms[1].weight.detach(), cos, sin)
    ok.backward(dk.transpose(1, 2).reshape(B, S, hidden))
    dx, bx, _, _ = backward_ref(dk.transpose(1, 2), x[1].detach().view(B, S, H, D),
                                norms[1].weight.detach().view(H, D), 1e-6, cos, sin, None, True,
                                over=2)
    check_norm("dk", x[1].grad.view(B, S, H, D), dx, bx)
    assert x[0].grad is None


def test_training_step_captured_and_replayed():
    from sinkattn_b200 import autograd

    B, S, H = 1, 300, 2
    a, w, cos, sin, _ = make_norm(B, S, H, H, 128, 128, torch.bfloat16, seed=9)
    mask = torch.ones(1, H, 3, 3, dtype=torch.bool, device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (a["q"], a["k"], a["dk"], *w)]
    dout = a["dq"].clone()

    def step():
        q, k = autograd.qk_head_norm_rope(leaves[0], leaves[1], 1e-6, leaves[3], leaves[4], cos, sin)
        out, _ = autograd.block_sparse_attention(*(t.transpose(1, 2) for t in (q, k, leaves[2])),
                                                 mask)
        return torch.autograd.grad(out, leaves, dout.transpose(1, 2))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    with torch.no_grad():
        leaves[0].copy_(a["dk"])
        dout.copy_(a["k"])
    graph.replay()
    torch.cuda.synchronize()
    replayed = [t.clone() for t in got]
    for x, y in zip(replayed, step()):
        assert torch.equal(x, y)
    del graph
