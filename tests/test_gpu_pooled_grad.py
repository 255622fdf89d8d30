"""Gradients through the pooled branch (sequence pooling, adaptive mix, the
fused sink + pooled attention) against the formulas in 64 bits, and the
drop-ins that record them; their results stay what they are unrecorded.

Tolerances: U = 2^-8, half a bf16 step, for every rounding of a result to
bf16; E = 2^-16 of the sum of the sizes of what fp32 adds up (at most 128
terms), as in the modules of the other gradients.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from tests.test_gpu_attention_bwd import E_P, token_mask
from tests.test_gpu_attention_bwd import make as make_attn

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
E = 2.0 ** -16
TINY = 2.0 ** -100


def close(name, got, ref, bound):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    over = err - bound * 1.001 - TINY
    i = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name} off by {float(err.reshape(-1)[i]):.3e} where "
                                    f"{float(bound.reshape(-1)[i]):.3e} is allowed")


def randn(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


def pool_matrix(S, pool, prefix):
    """[pooled rows, S] in 64 bits: the prefix as it is, then means of `pool` tokens, the final token
    standing in for those that the last one lacks."""
    rows = prefix + -(-(S - prefix) // pool)
    m = torch.zeros(rows, S, dtype=torch.float64, device="cuda")
    for r in range(rows):
        if r < prefix:
            m[r, r] = 1
        else:
            for i in range(pool):
                m[r, min(prefix + (r - prefix) * pool + i, S - 1)] += 1 / pool
    return m


def pool_grad(d, S, pool, prefix, d_bound=None):
    """Gradient and bound from that of the pooled rows (and its bound)."""
    m = pool_matrix(S, pool, prefix).T
    dx = m @ d.double()
    b = 0 if d_bound is None else m @ d_bound
    return dx, b + U * dx.abs() + E * dx.abs()


@pytest.mark.parametrize("B,H,S,pool,prefix", [
    (2, 3, 90, 30, 0), (1, 2, 257, 30, 77), (2, 2, 5, 8, 0), (1, 1, 9, 4, 8), (1, 4, 1000, 3, 1),
    (2, 2, 64, 2, 64), (1, 2, 64, 1, 0)])
@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
def test_sequence_pooling(B, H, S, pool, prefix, layout):
    from sinkattn_b200 import autograd, ops
    from sinkattn_b200.reference_api import (_mean_pool_sequence,
                                             _mean_pool_sequence_preserve_prefix)

    x = randn(B, H, S, 128, seed=S)
    if layout == "bshd":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    want = ops.mean_pool_seq(x, pool, prefix)
    calls = [lambda t: autograd.mean_pool_seq(t, pool, prefix),
             lambda t: _mean_pool_sequence_preserve_prefix(t, pool, prefix_tokens=prefix)]
    if prefix == 0:
        calls.append(lambda t: _mean_pool_sequence(t, pool))
    for call in calls:
        leaf = x.detach().requires_grad_()
        out = call(leaf)
        assert torch.equal(out, want) and out.stride() == want.stride()
        d = randn(*out.shape, seed=1)
        if out is leaf:  # nothing to pool
            continue
        with torch.no_grad():
            assert not call(leaf).requires_grad
        for up in (d, d[..., :1, :].expand_as(d)):
            (dx,) = torch.autograd.grad(out, leaf, up, retain_graph=True)
            assert dx.dtype == torch.bfloat16
            close("dx", dx, *pool_grad(up, S, pool, prefix))
        out[:, :, 0] = 0  # may be written over, as unrecorded
        (dx,) = torch.autograd.grad(out, leaf, d)
        d[:, :, 0] = 0
        close("dx", dx, *pool_grad(d, S, pool, prefix))


def mix_grads(os, ls, od, ld, gap, d):
    """Gradients and bounds of the adaptive mix, in 64 bits."""
    os, ls, od, ld, d = (t.double() for t in (os, ls, od, ld, d))
    lead = ls - (ld + math.log(gap))
    ws, wd = torch.sigmoid(lead), torch.sigmoid(-lead)
    dl = ws * wd * (d * (os - od)).sum(-1, keepdim=True)
    bl = E * ws * wd * (d.abs() * (os.abs() + od.abs())).sum(-1, keepdim=True)
    out = (d * ws, dl, d * wd, -dl)
    return out, [(E + U) * out[0].abs(), bl, (E + U) * out[2].abs(), bl]


@pytest.mark.parametrize("lse_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,S,gap", [(1, 1, 1, 30), (2, 3, 77, 4), (1, 2, 300, 1)])
def test_adaptive_mix(B, H, S, gap, lse_dtype):
    from sinkattn_b200 import autograd, ops
    from sinkattn_b200.reference_api import _mix_attention_outputs

    os, od, d = (randn(B, H, S, 128, seed=s) for s in (2, 3, 4))
    ls, ld = ((3 * randn(B, H, S, 1, seed=s)).to(lse_dtype) for s in (5, 6))
    ls[:, :, S // 2] = float("-inf")  # a row that keeps no sink block
    os[:, :, S // 2] = 0
    want = ops.mix_outputs(os, ls, od, ld, gap)
    cfg = SimpleNamespace(mixing_mode="adaptive", sample_gap=gap)
    ref, bound = mix_grads(os, ls, od, ld, gap, d)
    for call in (lambda a, b, c, e: autograd.mix_outputs(a, b, c, e, gap),
                 lambda a, b, c, e: _mix_attention_outputs(a, b, c, e, cfg)):
        leaves = [t.detach().clone().requires_grad_() for t in (os, ls, od, ld)]
        out = call(*leaves)
        assert torch.equal(out, want) and out.stride() == want.stride()
        got = torch.autograd.grad(out, leaves, d, retain_graph=True)
        for n, t, g, r, b in zip(("sink", "sink lse", "dynamic", "dynamic lse"), leaves, got, ref,
                                 bound):
            assert g.dtype == t.dtype
            close(n, g, r, b + (U * r.abs() if "lse" in n and lse_dtype != torch.float32 else 0))
        with torch.no_grad():
            assert not call(*leaves).requires_grad
        out.mul_(2)  # may be written over, as unrecorded, and keeps its gradient
        got = torch.autograd.grad(out, leaves[0], d)[0]
        close("sink", got, 2 * ref[0], 2 * bound[0])
        # one of them alone
        out = call(os, leaves[1], od, ld)
        assert torch.equal(out, want) and torch.autograd.grad(out, leaves[1], d)[0].shape == ls.shape


def joint_grads(q, k, v, kp, vp, keep, gap, dout, scale, dlse=None):
    """(dq, dk, dv, dkp, dvp) of one softmax over the kept keys and the pooled ones, whose logits are
    raised by ln(gap), and bounds derived as those of the attention alone; dq is the sum of two
    results rounded before."""
    q, k, v, kp, vp, g = (t.double() for t in (q, k, v, kp, vp, dout))
    n = k.shape[2]
    ka, va = torch.cat([k, kp], 2), torch.cat([v, vp], 2)
    s = scale * q @ ka.transpose(-1, -2)
    s[..., :n] = torch.where(keep, s[..., :n], torch.full_like(s[..., :n], -math.inf))
    s[..., n:] += math.log(gap)
    p = torch.softmax(s, dim=-1)
    out, dp = p @ va, g @ va.transpose(-1, -2)
    delta = (g * out).sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double()[..., None]
    ds = p * (dp - delta)
    dq_parts = [scale * ds[..., :n] @ k, scale * ds[..., n:] @ kp]
    dq, dk, dv = sum(dq_parts), scale * ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ g
    e_d = (g.abs() * (U * (p @ va.abs()) + U * out.abs())).sum(-1, keepdim=True)
    e_ds = (U + E_P) * ds.abs() + p * (e_d + 2.0 ** -15 * (g.abs() @ va.abs().transpose(-1, -2)))
    bq = scale * e_ds @ ka.abs() + U * sum(t.abs() for t in dq_parts)
    bq = bq + U * (dq.abs() + bq)
    bk = scale * e_ds.transpose(-1, -2) @ q.abs() + U * dk.abs()
    bv = (U + E_P) * p.transpose(-1, -2) @ g.abs() + U * dv.abs()
    return ((dq, dk[:, :, :n], dv[:, :, :n], dk[:, :, n:], dv[:, :, n:]),
            (bq, bk[:, :, :n], bv[:, :, :n], bk[:, :, n:], bv[:, :, n:]))


NAMES = ("dq", "dk", "dv", "dk_pool", "dv_pool")


@pytest.mark.parametrize("B,H,Sq,Sk,Skp,gap,p,empty", [
    (1, 1, 1, 1, 1, 30, 1.0, 0.0), (2, 2, 300, 300, 10, 30, 0.5, 0.0),
    (1, 3, 257, 500, 130, 4, 0.4, 0.5), (2, 2, 200, 130, 200, 1, 0.5, 1.0),
    (1, 2, 3000, 3000, 100, 30, 0.2, 0.0), (1, 4, 4096, 4096, 1024, 4, 0.2, 0.0)])
def test_sink_and_pooled_attention(B, H, Sq, Sk, Skp, gap, p, empty):
    from sinkattn_b200 import autograd, ops

    q, k, v, dout, mask = make_attn(B, H, Sq, Sk, p, Sq + Skp, empty=empty)
    kp, vp = (randn(B, Skp, H, 128, seed=s).transpose(1, 2) for s in (7, 8))
    dlse = torch.randn(B, H, Sq, device="cuda")
    want = ops.sink_dynamic_attn(q, k, v, mask, kp, vp, gap, return_lse=True)
    keep = token_mask(mask, B, H, Sq, Sk)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, kp, vp)]

    def call():
        return autograd.sink_dynamic_attention(*leaves[:3], mask, *leaves[3:], gap)

    for up in ((dout, None), (dout, dlse), (None, dlse)):
        out, lse = call()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert out.stride() == want[0].stride()
        got = torch.autograd.grad([t for t, d in zip((out, lse), up) if d is not None], leaves,
                                  [d for d in up if d is not None])
        ref, bound = joint_grads(q, k, v, kp, vp, keep, gap,
                                 torch.zeros_like(dout) if up[0] is None else dout,
                                 1 / math.sqrt(128), up[1])
        for n, g, r, b in zip(NAMES, got, ref, bound):
            close(n, g, r, b)
    ops.DeviceStatus.check()


def test_sink_and_pooled_attention_scale_shared_slices_and_dense_heads():
    from sinkattn_b200 import autograd

    q, k, v, dout, mask = make_attn(2, 3, 300, 400, 0.5, 51, layout="bhsd")
    kp, vp = randn(2, 3, 50, 128, seed=9), randn(2, 3, 50, 128, seed=10)
    hmt = torch.tensor([2, 0, 2], device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, kp, vp)]
    out, _ = autograd.sink_dynamic_attention(*leaves[:3], mask[:, :2], *leaves[3:], 8,
                                             softmax_scale=0.2, head_mask_type=hmt)
    got = torch.autograd.grad(out, leaves, dout)
    keep = token_mask(mask[:, :2], 2, 3, 300, 400, hmt)
    ref, bound = joint_grads(q, k, v, kp, vp, keep, 8, dout, 0.2)
    for n, g, r, b in zip(NAMES, got, ref, bound):
        close(n, g, r, b)


def test_sink_and_pooled_attention_captured():
    from sinkattn_b200 import autograd

    q, k, v, dout, mask = make_attn(1, 2, 700, 700, 0.5, 52)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        kp, vp = (autograd.mean_pool_seq(t, 30, 77) for t in leaves[1:])
        out, _ = autograd.sink_dynamic_attention(*leaves, mask, kp, vp, 30)
        return torch.autograd.grad(out, leaves, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    del graph


@pytest.mark.parametrize("S,prefix", [(1000, 0), (1300, 77)])
def test_wan_inner_attention_records(S, prefix):
    """The fused drop-in of the Wan runtime: same output, and gradients for q, k and v through the
    sink blocks and the pooled branch."""
    from sinkattn_b200 import reference_api as ra

    B, H, gap = 1, 2, 30
    q, k, v, dout, mask = make_attn(B, H, S, S, 0.3, S)
    inner = SimpleNamespace(
        config=SimpleNamespace(mixing_mode="adaptive", dynamic_kernel="auto", text_length=prefix),
        runtime_state=None, sink_mask=mask, _resolve_dynamic_plan=lambda: ("pooled_kv", gap),
        _get_runtime_mask=lambda **kw: mask)
    want = ra.fused_wan_inner_forward(inner, q, k, v)
    assert not want.requires_grad
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    with torch.no_grad():
        assert not ra.fused_wan_inner_forward(inner, *leaves).requires_grad
    out = ra.fused_wan_inner_forward(inner, *leaves)
    assert torch.equal(out, want) and out.stride() == want.stride()
    got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    kp, vp = (ra._mean_pool_sequence_preserve_prefix(t, gap, prefix_tokens=prefix) for t in (k, v))
    ref, bound = joint_grads(q, k, v, kp, vp, token_mask(mask, B, H, S, S), gap, dout,
                             1 / math.sqrt(128))
    close("dq", got[0], ref[0], bound[0])
    for n, g, i in (("dk", got[1], 1), ("dv", got[2], 2)):
        r, b = pool_grad(ref[i + 2], S, gap, prefix, bound[i + 2])
        total, b = ref[i] + r, bound[i] + b
        close(n, g, total, b + U * (total.abs() + b))  # summed in bf16
    out.mul_(2)  # may be written over, as unrecorded
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # values alone, as with frozen projections of q and k
    out = ra.fused_wan_inner_forward(inner, q, k, leaves[2])
    assert torch.equal(torch.autograd.grad(out, leaves[2], dout)[0], got[2])
