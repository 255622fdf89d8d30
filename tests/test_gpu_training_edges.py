"""Calls of the training operators at the ends of what they take: magnitudes,
sizes, reports and recorded results, against the formulas in 64 bits with the
bounds derived in the modules they come from.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention_bwd import both as both_attn
from tests.test_gpu_attention_bwd import make as make_attn
from tests.test_gpu_norm_grad import backward_ref, both, check, make

pytestmark = pytest.mark.gpu


# rows of one size: with a mean square of 10^28 to 10^34 or below 10^-26 the cube of its root's
# inverse leaves what fp32 holds, and with it a gradient that is formed from the cube
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,eps", [(1e14, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-13, 0.0),
                                      (1e-17, 0.0)])
@pytest.mark.parametrize("inter", [True, False])
def test_head_norm_of_very_large_and_very_small_rows(size, eps, dtype, inter):
    a, w, cos, sin, pos = make(2, 9, 3, 2, 128, 64, dtype, seed=31)
    for n in ("q", "k"):
        a[n] = (a[n].float() * size).to(dtype)
    both(a, w, cos, sin, pos, inter, eps)


def test_head_norm_gradient_of_zero_rows_beside_a_small_eps():
    a, w, cos, sin, pos = make(1, 5, 2, 2, 64, 64, torch.float32, seed=32)
    a["q"][0, 2] = 0
    a["k"][0, 4, 1] = 0
    both(a, w, cos, sin, pos, True, 1e-28)


@pytest.mark.parametrize("size,eps", [(1e14, 1e-6), (1e15, 1e-6), (1e17, 1e-6), (1e-13, 0.0),
                                      (1e-17, 0.0)])
def test_hidden_norm_gradient_of_very_large_and_very_small_rows(size, eps):
    from sinkattn_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(33)
    B, S, hidden, D = 2, 21, 512, 128

    def t(scale):
        return (torch.randn(B, S, hidden, generator=g, device="cuda") * scale).bfloat16()

    q, k, dq, dk = t(size), t(size), t(1.0), t(1.0)
    w = [(1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")) for _ in range(2)]
    ang = torch.rand(S, D // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    got = ops.qk_norm_rope_bwd(dq, dk, q, k, D, eps, w[0], w[1], cos, sin)
    split = (B, S, hidden // D, D)
    for i, (d, x) in enumerate(((dq, q), (dk, k))):
        dx, bx, dw, bw = backward_ref(d.view(split), x.view(split), w[i].view(hidden // D, D), eps,
                                      cos, sin, None, True, over=2)
        check("dx", got[i].view(split), dx, bx)
        check("dw", got[2 + i].view(hidden // D, D), dw, bw)


def test_sizes_that_no_copy_can_fit_are_refused():
    """Contiguous tensors: the layout is not what is wrong with them."""
    from sinkattn_b200 import ops

    def t(*s, dtype=torch.bfloat16):
        return torch.ones(*s, dtype=dtype, device="cuda")

    for D, dtype in ((100, torch.bfloat16), (12, torch.float16), (12, torch.float32),
                     (6, torch.float32), (264, torch.bfloat16)):
        x = t(2, 5, 3, D, dtype=dtype)
        with pytest.raises(RuntimeError, match="multiple of 8 up to 256"):
            ops.qk_head_norm_rope(x, x, 1e-6)
        with pytest.raises(RuntimeError, match="multiple of 8 up to 256"):
            ops.qk_head_norm_rope_bwd(x, x, x, x, 1e-6)
    x, f = t(2, 5, 3, 128), torch.float32
    for half, inter, match in ((6, True, "multiple of 8 up to"), (0, True, "multiple of 8 up to"),
                               (4, False, "multiple of 16 up to"), (68, True, "multiple of 8 up to")):
        c = t(5, half, dtype=f)
        with pytest.raises(RuntimeError, match=match):
            ops.qk_head_norm_rope(x, x, 1e-6, cos=c, sin=c, interleaved=inter)
        with pytest.raises(RuntimeError, match=match):
            ops.qk_head_norm_rope_bwd(x, x, x, x, 1e-6, cos=c, sin=c, interleaved=inter)
    for hidden, D in ((100, 100), (12, 12), (4104, 8), (256, 96)):
        x = t(2, 5, hidden)
        with pytest.raises(RuntimeError, match="hidden"):
            ops.qk_norm_rope_bwd(x, x, x, x, D, 1e-6)
    lse, mask = torch.zeros(1, 2, 130, device="cuda"), t(1, 2, 2, 2, dtype=torch.bool)
    for D in (100, 64, 136):
        x = t(1, 2, 130, D)
        with pytest.raises(RuntimeError, match="head dim must be 128"):
            ops.bsattn_bwd(x, x, x, x, x, lse, mask)


def test_views_of_nothing():
    from sinkattn_b200 import ops

    bf = torch.bfloat16
    odd = torch.zeros(2, 4, 3, 131, dtype=bf, device="cuda")[:, :0, :, 1:129]
    wide, w = torch.zeros(5, 70, device="cuda")[:0, 2:66], torch.ones(128, device="cuda")
    q, k = ops.qk_head_norm_rope(odd, odd, 1e-6, w, w, wide, wide)
    assert q.shape == k.shape == (2, 0, 3, 128)
    dq, dk, dwq, dwk = ops.qk_head_norm_rope_bwd(odd, odd, odd, odd, 1e-6, w, w, wide, wide)
    assert dq.shape == dk.shape == (2, 0, 3, 128) and not dwq.any() and not dwk.any()
    turned, w = torch.zeros(0, 256, 2, dtype=bf, device="cuda").permute(0, 2, 1), w.repeat(2)
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(turned, turned, turned, turned, 128, 1e-6, w, w)
    assert dq.shape == dk.shape == (0, 2, 256) and not dwq.any() and not dwk.any()
    none = torch.zeros(1, 2, 4, 133, dtype=bf, device="cuda")[:, :, :0, 3:131]
    with pytest.raises(RuntimeError, match="SA_EINVAL"):
        ops.bsattn_bwd(none, none, none, none, none, torch.zeros(1, 2, 0, device="cuda"),
                       torch.zeros(1, 2, 0, 0, dtype=torch.bool, device="cuda"))


def test_the_forward_pass_reports_head_mask_type_past_the_mask():
    """Such a head is dense in both directions; nothing past the mask is read."""
    from sinkattn_b200 import ops
    from sinkattn_b200.autograd import block_sparse_attention

    q, k, v, dout, mask = make_attn(2, 3, 300, 400, 0.5, 41)
    mask = mask[:, :2]
    good = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    for past in (3, 4, 2 ** 31 - 1):
        bad = torch.tensor([1, 2, past], dtype=torch.int32, device="cuda")
        calls = (lambda t: ops.bsattn_fwd(q, k, v, mask, head_mask_type=t),
                 lambda t: ops.sink_dynamic_attn(q, k, v, mask, k[:, :, :90], v[:, :, :90], 4,
                                                 head_mask_type=t, return_lse=True))
        for call in calls:
            want, got = call(good), call(bad)
            with pytest.raises(RuntimeError, match="head_mask_type entry"):
                ops.DeviceStatus.check()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        grads = []
        for t in (good, bad):
            leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
            out, _ = block_sparse_attention(*leaves, mask, head_mask_type=t)
            grads.append(torch.autograd.grad(out, leaves, dout))
        with pytest.raises(RuntimeError, match="head_mask_type entry"):
            ops.DeviceStatus.check()
        for a, b in zip(*grads):
            assert torch.equal(a, b)
    ops.DeviceStatus.check()


def test_results_may_be_written_over():
    """As without a gradient: what was recorded needs the output, so only its backward refuses."""
    from sinkattn_b200.autograd import block_sparse_attention
    from sinkattn_b200.reference_api import _block_sparse_attn

    q, k, v, dout, mask = make_attn(1, 2, 260, 260, 0.6, 5)
    want, want_lse = _block_sparse_attn(q, k, v, mask)
    q.requires_grad_()
    for call in (lambda: block_sparse_attention(q, k, v, mask),
                 lambda: _block_sparse_attn(q, k, v, mask)):
        out, lse = call()
        assert out.requires_grad and out.stride() == want.stride()
        out.mul_(2)
        out[:, :, 3] = 0
        lse.add_(1)
        assert torch.equal(out[:, :, 4:], 2 * want[:, :, 4:]) and not out[:, :, 3].any()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_a_bad_index_does_not_hide_a_wait_that_gave_up():
    """The word says that outputs are not valid until the host has read it."""
    import ctypes

    from sinkattn_b200 import _lib, ops

    x = torch.ones(1, 3, 2, 64, device="cuda")
    table = torch.ones(4, 32, device="cuda")
    bad = torch.tensor([0, 1, 4], device="cuda")
    ops.DeviceStatus.check()
    word = ctypes.c_int32.from_address(ops.DeviceStatus._word(x.device.index)[0])
    word.value = _lib.SA_DEV_WAIT_TIMEOUT
    ops.qk_head_norm_rope(x, x, 1e-6, cos=table, sin=table, positions=bad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bounded wait"):
        ops.DeviceStatus.check()
    ops.qk_head_norm_rope(x, x, 1e-6, cos=table, sin=table, positions=bad)
    with pytest.raises(RuntimeError, match="position outside"):
        ops.DeviceStatus.check()
    ops.DeviceStatus.check()


def test_pieces_at_two_tiles_for_each_processor_beside_another_stream():
    """256 tiles, the first of every head cut: each block of threads claims by the shared counter."""
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make_attn(1, 4, 4096, 4096, 0.2, 26, layout="bhsd")
    want = both_attn(q, k, v, dout, mask)
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        got = ops.bsattn_bwd(dout, q, k, v, out, lse, mask)
        with torch.cuda.stream(side):
            beside = ops.bsattn_bwd(dout, q, k, v, out, lse, mask)
        torch.cuda.synchronize()
        for a, b, c in zip(want, got, beside):
            assert torch.equal(a, b) and torch.equal(a, c)
    ops.DeviceStatus.check()


def test_outputs_in_the_place_of_inputs():
    """By either way into the library: refused where other blocks still read them, else the same."""
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make_attn(1, 2, 300, 300, 0.5, 42)
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    ops.bsattn_bwd(dout, q, k, v, out, lse, mask)
    for kw in (dict(dq=dout), dict(dk=k), dict(dv=out), dict(dq=v, dk=v)):
        with pytest.raises(RuntimeError, match="has the address of"):
            ops.bsattn_bwd(dout, q, k, v, out, lse, mask, **kw)
    # views that interleave in one buffer are apart
    want = ops.bsattn_bwd(dout, q, k, v, out, lse, mask)
    packed = torch.zeros(1, 300, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    dq, dk, dv = (packed[:, :, i].transpose(1, 2) for i in range(3))
    for a, b in zip(ops.bsattn_bwd(dout, q, k, v, out, lse, mask, dq=dq, dk=dk, dv=dv), want):
        assert torch.equal(a, b)
    a, w, cos, sin, _ = make(2, 9, 3, 3, 128, 128, torch.bfloat16, seed=43)
    args = (a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin)
    for kw in (dict(dq=a["dk"]), dict(dk=a["q"])):
        with pytest.raises(RuntimeError, match="has the address of"):
            ops.qk_head_norm_rope_bwd(*args, **kw)
    with pytest.raises(RuntimeError, match="has the address of"):
        ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, out_q=a["k"])
    rows = [a[n].flatten(2) for n in ("dq", "dk", "q", "k")]
    with pytest.raises(RuntimeError, match="has the address of"):
        ops.qk_norm_rope_bwd(*rows, 128, 1e-6, dq=rows[1])
