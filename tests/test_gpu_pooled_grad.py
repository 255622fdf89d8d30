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
