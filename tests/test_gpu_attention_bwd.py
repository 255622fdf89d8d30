"""Gradients of the block-sparse attention against the formulas in 64 bits.

Tolerances, element by element, from the kernel's roundings (u = 2^-8, half a
bf16 step relative to the value; every sum is fp32):
  * out as the forward kernel stores it is off by u (P|V|) (its bf16 P) plus
    u |out|, so delta = sum dout * out is off by e_d = sum_d |dout| (u P|V| + u |out|);
  * P carries e_p = 2^-13: the exponent is a fp32 difference of terms below 2^9
    (three roundings of 2^-24 * 2^9 * log2 units, 0.7 of it in the result) and
    the fp32 log-sum-exp of the same size;
  * dv = P^T dout rounds P to bf16: (u + e_p) P^T|dout|, then u |dv|;
  * dS = P (dP - delta) rounds to bf16: (u + e_p) |dS| + P (e_d + 2^-15 |dout||v|^T)
    (fp32 dP, 128 terms), and dq, dk sum it against |k|, |q|, then u |dq|, u |dk|.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
E_P = 2.0 ** -13


def token_mask(mask, B, H, Sq, Sk, hmt=None):
    m = mask.expand(B, -1, -1, -1)
    if hmt is not None:
        m = torch.stack([torch.ones_like(m[:, 0]) if t == 0 else m[:, t - 1]
                         for t in hmt.tolist()], dim=1)
    m = m.bool().repeat_interleave(128, dim=2)[:, :, :Sq]
    return m.repeat_interleave(128, dim=3)[..., :Sk]


def reference(q, k, v, dout, keep, scale, dlse=None):
    """(dq, dk, dv), and the bounds above, in 64 bits."""
    q, k, v, g = (t.double() for t in (q, k, v, dout))
    kt, vt = k.transpose(-1, -2), v.transpose(-1, -2)
    s = (q @ kt) * scale
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    p = torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0)
    out = p @ v
    dp = g @ vt
    delta = (g * out).sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double()[..., None]
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ k, scale * ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ g
    e_d = (g.abs() * (U * (p @ v.abs()) + U * out.abs())).sum(-1, keepdim=True)
    e_ds = (U + E_P) * ds.abs() + p * (e_d + 2.0 ** -15 * (g.abs() @ vt.abs()))
    bq = scale * e_ds @ k.abs() + U * dq.abs()
    bk = scale * e_ds.transpose(-1, -2) @ q.abs() + U * dk.abs()
    bv = (U + E_P) * p.transpose(-1, -2) @ g.abs() + U * dv.abs()
    return (dq, dk, dv), (bq, bk, bv)


def check(got, ref, bound):
    for name, a, r, b in zip(("dq", "dk", "dv"), got, ref, bound):
        assert a.shape == r.shape and a.dtype == torch.bfloat16
        err = (a.double() - r).abs()
        assert torch.isfinite(a).all(), f"{name} not finite"
        # 2^-100: nothing smaller is told apart (fp32 sums flush no larger terms)
        over = err - (b * 1.001 + 2.0 ** -100)
        worst = int(over.argmax())
        assert float(over.max()) <= 0, (f"{name} off by {float(err.view(-1)[worst]):.3e} where "
                                        f"{float(b.view(-1)[worst]):.3e} is allowed")


def make(B, H, Sq, Sk, p, seed, scale=1.0, empty=0.0, layout="bshd", Bm=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(S):
        if layout == "bshd":
            x = torch.randn(B, S, H, 128, generator=g, device="cuda").permute(0, 2, 1, 3)
        else:
            x = torch.randn(B, H, S, 128, generator=g, device="cuda")
        return (x * scale).bfloat16()

    q, k, v, dout = t(Sq), t(Sk), t(Sk), t(Sq)
    nq, nk = math.ceil(Sq / 128), math.ceil(Sk / 128)
    mask = torch.rand(Bm or B, H, nq, nk, generator=g, device="cuda") < p
    if empty == 0.0:
        mask[..., 0] = True
    else:
        mask &= torch.rand(Bm or B, H, nq, 1, generator=g, device="cuda") >= empty
    return q, k, v, dout, mask


def run(q, k, v, dout, mask, scale=None, hmt=None, dlse=None, **kw):
    from sinkattn_b200 import ops

    out, lse = ops.bsattn_fwd(q, k, v, mask, softmax_scale=scale, head_mask_type=hmt)
    got = ops.bsattn_bwd(dout, q, k, v, out, lse, mask, softmax_scale=scale, head_mask_type=hmt,
                         dlse=dlse, **kw)
    torch.cuda.synchronize()
    ops.DeviceStatus.check()
    return got


def both(q, k, v, dout, mask, scale=None, hmt=None, dlse=None, **kw):
    B, H, Sq, D = q.shape
    got = run(q, k, v, dout, mask, scale, hmt, dlse, **kw)
    keep = token_mask(mask, B, H, Sq, k.shape[2], hmt)
    ref, bound = reference(q, k, v, dout, keep, scale or 1 / math.sqrt(D), dlse)
    check(got, ref, bound)
    return got


def test_one_block():
    both(*make(1, 1, 128, 128, 1.0, 0))


@pytest.mark.parametrize("B,H,Sq,Sk,p", [
    (1, 1, 1, 1, 1.0), (2, 2, 1, 300, 1.0), (1, 2, 128, 1, 1.0), (2, 3, 257, 129, 0.5),
    (1, 2, 640, 33, 1.0), (2, 2, 1000, 1092, 0.4), (1, 2, 129, 4000, 0.3), (1, 1, 4000, 70, 1.0),
    (1, 3, 2048, 2048, 0.2), (3, 5, 384, 640, 1.0),
])
def test_shapes(B, H, Sq, Sk, p):
    both(*make(B, H, Sq, Sk, p, Sq * 7 + Sk))


@pytest.mark.parametrize("B,H,Sq,Sk", [
    (1, 1, 16384, 100),   # one key tile in sixteen pieces, short query tiles
    (1, 1, 77, 12800),    # the same for one query tile
    (1, 2, 4225, 2049),   # both kinds, tiles of different lengths
    (2, 4, 5120, 5000),   # many tiles: one long column each head
])
def test_tiles_longer_than_a_share_of_the_gpu(B, H, Sq, Sk):
    q, k, v, dout, mask = make(B, H, Sq, Sk, 0.02, 7 + Sq)
    mask[:, -1, 0] = True  # a long query tile too, and every column kept once
    got = both(q, k, v, dout, mask)
    again = run(q, k, v, dout, mask)
    for x, y in zip(got, again):
        assert torch.equal(x, y)


@pytest.mark.parametrize("B,H,Sq,Sk", [(1, 24, 700, 900), (3, 9, 1024, 513), (1, 4, 2500, 2300)])
@pytest.mark.parametrize("empty", [0.0, 0.4])
def test_a_few_tiles_for_each_processor(B, H, Sq, Sk, empty):
    q, k, v, dout, mask = make(B, H, Sq, Sk, 0.4, Sq, empty=empty)
    got = both(q, k, v, dout, mask)
    for x, y in zip(got, run(q, k, v, dout, mask)):
        assert torch.equal(x, y)


def test_long_tiles_of_one_kind_among_many_of_the_other():
    """140 heads of 17 x 16 blocks; all but the first keep nothing: its key tiles may be cut,
    its query tiles are too many to."""
    q, k, v, dout, mask = make(1, 140, 2176, 2048, 0.0, 3, empty=0.5)
    mask[:, 0] = True
    got = run(q, k, v, dout, mask)
    keep = token_mask(mask[:, :1], 1, 1, 2176, 2048)
    ref, bound = reference(q[:, :1], k[:, :1], v[:, :1], dout[:, :1], keep, 1 / math.sqrt(128))
    check([x[:, :1] for x in got], ref, bound)
    assert not any(x[:, 1:].any() for x in got)


@pytest.mark.parametrize("layout", ["bshd", "bhsd"])
@pytest.mark.parametrize("empty", [0.3, 1.0])
def test_rows_and_columns_that_keep_nothing(layout, empty):
    both(*make(2, 3, 900, 700, 0.25, 5, empty=empty, layout=layout))


def test_mask_shared_by_the_batch_and_strided():
    q, k, v, dout, mask = make(3, 2, 500, 600, 0.5, 6, Bm=1)
    both(q, k, v, dout, mask)
    wide = torch.zeros(1, 2, mask.shape[2], 2 * mask.shape[3], dtype=torch.bool, device="cuda")
    wide[..., ::2] = mask
    a = run(q, k, v, dout, mask)
    b = run(q, k, v, dout, wide[..., ::2])
    c = run(q, k, v, dout, mask.transpose(2, 3).contiguous().transpose(2, 3))
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_head_mask_type():
    q, k, v, dout, mask = make(2, 4, 400, 500, 0.4, 7)
    hmt = torch.tensor([2, 0, 1, 1], dtype=torch.int32, device="cuda")
    both(q, k, v, dout, mask[:, :2], hmt=hmt)


@pytest.mark.parametrize("scale", [0.02, 0.3])
def test_scale(scale):
    both(*make(1, 2, 300, 300, 0.7, 8), scale=scale)


def test_gradient_of_the_log_sum_exp():
    q, k, v, dout, mask = make(2, 2, 500, 400, 0.5, 9)
    dlse = torch.randn(2, 2, 500, device="cuda")
    both(q, k, v, dout, mask, dlse=dlse)


def test_statistics_that_overflow_outside_the_lengths():
    """All logits near -280: exp(-lse) overflows for the zero rows behind the
    last key, which must not reach dq."""
    q, k, v, dout, mask = make(1, 2, 200, 150, 1.0, 10)
    q = (q * 0.01 + 5).bfloat16()
    k = (k * 0.01 - 5).bfloat16()
    keep = token_mask(mask, 1, 2, 200, 150)
    got = run(q, k, v, dout, mask)
    ref, bound = reference(q, k, v, dout, keep, 1 / math.sqrt(128))
    check(got, ref, bound)


def test_nan_and_inf_where_nothing_is_kept():
    q, k, v, dout, mask = make(1, 2, 512, 640, 0.5, 11)
    mask[..., 3] = False      # a key block nobody keeps
    mask[:, :, 2] = False     # a query block that keeps nothing
    keep = token_mask(mask, 1, 2, 512, 640)
    ref, bound = reference(q, k, v, dout, keep, 1 / math.sqrt(128))
    k[:, :, 384:512] = float("nan")
    v[:, :, 384:512] = float("inf")
    q[:, :, 256:384] = float("inf")
    dout[:, :, 256:384] = float("nan")
    check(run(q, k, v, dout, mask), ref, bound)


def test_outputs_given_by_the_caller_and_what_lies_behind_them():
    q, k, v, dout, mask = make(2, 2, 300, 200, 0.6, 12)
    plain = run(q, k, v, dout, mask)

    def window(S):  # a strided window of a larger buffer, the rest a marker
        buf = torch.full((2, S + 7, 2, 3, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        return buf, buf[:, :S, :, 1].permute(0, 2, 1, 3)

    bufs = [window(S) for S in (300, 200, 200)]
    got = run(q, k, v, dout, mask, dq=bufs[0][1], dk=bufs[1][1], dv=bufs[2][1])
    for (buf, view), a, b, S in zip(bufs, got, plain, (300, 200, 200)):
        assert a.data_ptr() == view.data_ptr() and torch.equal(a, b)
        rest = buf.clone()
        rest[:, :S, :, 1] = 7.0
        assert (rest == 7.0).all()


def test_layouts_and_misaligned_inputs_agree():
    q, k, v, dout, mask = make(2, 3, 450, 330, 0.5, 13)
    a = run(q, k, v, dout, mask)
    b = run(*(t.contiguous() for t in (q, k, v, dout)), mask)

    def odd(t):  # a view whose base and rows are not 16-byte aligned
        buf = torch.zeros(*t.shape[:-1], 133, dtype=t.dtype, device="cuda")
        buf[..., 3:131] = t
        return buf[..., 3:131]

    c = run(*(odd(t) for t in (q, k, v, dout)), mask)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_keys_shared_by_heads():
    """Keys and values broadcast over the heads by a stride of 0."""
    q, k, v, dout, mask = make(1, 4, 300, 300, 0.6, 14, layout="bhsd")
    ks, vs = k[:, :1].expand(-1, 4, -1, -1), v[:, :1].expand(-1, 4, -1, -1)
    a = run(q, ks, vs, dout, mask)
    b = run(q, ks.contiguous(), vs.contiguous(), dout, mask)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_equal_calls_give_equal_bits():
    args = make(1, 4, 3000, 3000, 0.3, 15)
    first = run(*args)
    for _ in range(5):
        for a, b in zip(first, run(*args)):
            assert torch.equal(a, b)


def test_captured_and_on_two_streams():
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make(1, 3, 700, 700, 0.5, 16)
    q2, k2, v2, dout2, mask2 = make(1, 3, 700, 700, 0.5, 17)
    want = [x.clone() for x in run(q, k, v, dout, mask)]
    want2 = [x.clone() for x in run(q2, k2, v2, dout2, mask2)]
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    out2, lse2 = ops.bsattn_fwd(q2, k2, v2, mask2)
    static = [t.clone() for t in (dout, q, k, v, out, lse, mask)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.bsattn_bwd(*static)
    side = torch.cuda.Stream()
    for _ in range(3):
        graph.replay()  # and, beside it, an eager call on another stream
        with torch.cuda.stream(side):
            beside = ops.bsattn_bwd(dout2, q2, k2, v2, out2, lse2, mask2)
        torch.cuda.synchronize()
        for a, b, c, d in zip(got, want, beside, want2):
            assert torch.equal(a, b) and torch.equal(c, d)
    for s, t in zip(static, (dout2, q2, k2, v2, out2, lse2, mask2)):
        s.copy_(t)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want2):
        assert torch.equal(a, b)
    del graph


def test_gradient_against_differences():
    """The scalar sum(dout * out) along a random direction, by differences of
    the formulas in 64 bits."""
    q, k, v, dout, mask = make(1, 1, 200, 260, 0.7, 18)
    keep = token_mask(mask, 1, 1, 200, 260)
    dirs = [torch.randn(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v)]

    def value(h):
        a, b, c = (t.double() + h * d for t, d in zip((q, k, v), dirs))
        s = (a @ b.transpose(-1, -2)) / math.sqrt(128)
        p = torch.softmax(torch.where(keep, s, torch.full_like(s, -math.inf)), dim=-1)
        return float((dout.double() * (p @ c)).sum())

    h = 1e-4
    want = (value(h) - value(-h)) / (2 * h)
    got = run(q, k, v, dout, mask)
    slope = sum(float((a.double() * d).sum()) for a, d in zip(got, dirs))
    # the sum of n independent roundings of at most `bound` each: 6 standard deviations
    _, bound = reference(q, k, v, dout, keep, 1 / math.sqrt(128))
    tol = 6 * math.sqrt(sum(float((b * d).square().sum()) for b, d in zip(bound, dirs)))
    assert abs(slope - want) <= tol, (slope, want, tol)


def test_refusals():
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make(1, 2, 200, 300, 1.0, 19)
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    ok = (dout, q, k, v, out, lse, mask)

    def refuse(match, **kw):
        names = ("dout", "q", "k", "v", "out", "lse", "block_mask")
        args = {**dict(zip(names, ok)), **kw}
        with pytest.raises(RuntimeError, match=match):
            ops.bsattn_bwd(**args)

    refuse("dout must be bf16", dout=dout.float())
    refuse("v must be bf16", v=v[:, :, :299])
    refuse("out must be bf16", out=out[:, :1])
    refuse("lse must be fp32", lse=lse.bfloat16())
    refuse("dlse must be fp32", dlse=lse[..., :100])
    refuse("block_mask must be", block_mask=mask[..., :1])
    refuse("block_mask must be bool", block_mask=mask.float())
    refuse("head_mask_type must be int32", head_mask_type=torch.ones(2, device="cuda"))
    refuse("dq must", dq=torch.empty(1, 2, 200, 136, device="cuda", dtype=torch.bfloat16)[..., 4:132])
    refuse("dk must be bf16", dk=torch.empty_like(k, dtype=torch.float32))
    refuse("workspace", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    refuse("CUDA tensors only", q=q.cpu())
    refuse("mask has 1 heads", block_mask=mask[:, :1])


def test_expanded_outputs_and_workspaces_are_refused():
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make(2, 2, 200, 300, 1.0, 20)
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    need = 1 << 22
    for name, t in (("dq", q[:, :1].contiguous().expand(-1, 2, -1, -1)),
                    ("dk", k[:1].contiguous().expand(2, -1, -1, -1)),
                    ("dv", v[:, :, :1].contiguous().expand(-1, -1, 300, -1))):
        with pytest.raises(RuntimeError, match=name + " is expanded"):
            ops.bsattn_bwd(dout, q, k, v, out, lse, mask, **{name: t})
    for ws in (torch.empty(1, dtype=torch.uint8, device="cuda").expand(need),
               torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(RuntimeError, match="workspace must be contiguous"):
            ops.bsattn_bwd(dout, q, k, v, out, lse, mask, workspace=ws)
    # inputs may be: keys shared by the heads
    k1 = k[:, :1].expand(-1, 2, -1, -1)
    ops.bsattn_bwd(dout, q, k1, v, out, lse, mask)


def test_from_a_thread_without_a_context():
    """A thread whose first CUDA call is ours (an autograd worker may be one):
    through the C entry point, as torch's own calls would bind the context."""
    import ctypes
    import threading

    from sinkattn_b200 import _lib, ops

    q, k, v, dout, mask = make(1, 2, 300, 300, 0.6, 20)
    want = run(q, k, v, dout, mask)
    out, lse = ops.bsattn_fwd(q, k, v, mask)
    lib = _lib.load()
    size = lib.sa_bsattn_bwd_workspace_size(1, 2, 300, 300)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    got = [torch.empty_like(t) for t in want]
    torch.cuda.synchronize()
    st = [_lib.strides4(t) for t in (dout, q, k, v, out, *got)]
    ms = (ctypes.c_int64 * 4)(*mask.stride())
    rcs = []

    def work():
        rcs.append(lib.sa_bsattn_bwd(
            dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *st[:5],
            lse.data_ptr(), None, 1, 2, 300, 300, 128, mask.data_ptr(), ms, 2, None, -1.0,
            *(t.data_ptr() for t in got), *st[5:], ws.data_ptr(), size, None, None))

    t = threading.Thread(target=work)
    t.start(), t.join()
    torch.cuda.synchronize()
    assert rcs == [_lib.SA_OK]
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_odd_strides_of_dimensions_of_size_one():
    q, k, v, dout, mask = make(1, 1, 1, 300, 1.0, 21, layout="bhsd")
    want = run(q, k, v, dout, mask)

    def odd(t):
        st = [s if n > 1 else 13 for s, n in zip(t.stride(), t.shape)]
        return torch.as_strided(t, t.shape, st)

    from sinkattn_b200 import ops

    out, lse = ops.bsattn_fwd(q, k, v, mask)
    got = ops.bsattn_bwd(odd(dout), odd(q), odd(k), odd(v), odd(out), lse, mask,
                         dq=odd(torch.empty_like(q)))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_head_mask_type_past_the_mask_is_reported():
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make(1, 3, 300, 300, 0.5, 22)
    mask = mask[:, :2]
    good = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    want = run(q, k, v, dout, mask, hmt=good)
    out, lse = ops.bsattn_fwd(q, k, v, mask, head_mask_type=good)
    bad = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    got = ops.bsattn_bwd(dout, q, k, v, out, lse, mask, head_mask_type=bad)
    with pytest.raises(RuntimeError, match="head_mask_type entry"):
        ops.DeviceStatus.check()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_on_a_stream_of_its_own():
    from sinkattn_b200 import ops

    q, k, v, dout, mask = make(1, 2, 900, 900, 0.5, 23)
    want = run(q, k, v, dout, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = ops.bsattn_fwd(q, k, v, mask)
        got = ops.bsattn_bwd(dout, q, k, v, out, lse, mask)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_the_short_way_is_taken_and_agrees_with_the_long_one(monkeypatch):
    from sinkattn_b200 import ops

    assert ops._fast is not None, "the extension module is not built"
    q, k, v, dout, mask = make(2, 3, 500, 400, 0.5, 24)
    hmt = torch.tensor([1, 0, 3], dtype=torch.int32, device="cuda")
    dlse = torch.randn(2, 3, 500, device="cuda")
    out, lse = ops.bsattn_fwd(q, k, v, mask, head_mask_type=hmt)
    args = (dout, q, k, v, out, lse, mask)
    ops.DeviceStatus.pointer(q.device)
    taken = []
    real = ops._short

    def spy(name, *a):
        got = real(name, *a)
        taken.append(got is not None)
        return got

    monkeypatch.setattr(ops, "_short", spy)
    kws = (dict(), dict(head_mask_type=hmt, dlse=dlse, softmax_scale=0.1),
           dict(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v)))
    fast = [ops.bsattn_bwd(*args, **kw) for kw in kws]
    assert taken == [True] * 3
    monkeypatch.setattr(ops, "_short", lambda *a: None)
    for kw, want in zip(kws, fast):
        for x, y in zip(ops.bsattn_bwd(*args, **kw), want):
            assert torch.equal(x, y) and x.stride() == y.stride()
