"""The per-head norm + rotation, its gradient, and the gradient of the
hidden-wide norm + rotation, against the formulas in 64 bits.

Tolerances: u is half a step of the result's type (bf16 2^-8, fp16 2^-11, fp32
2^-24), on the result itself. Before that everything is fp32: the sums run
over at most 512 terms (8 to 64 in a lane, then a tree), so a row's mean square
and dot product are good to 2^-17 of the sum of their terms' sizes, and each
value to 2^-16 of the sum of the sizes of what is added to form it.
dw: n rows of such terms in fp32, at worst (n + 64) 2^-24 more of their sum.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E = 2.0 ** -16
# nothing below fp16's smallest step is told apart in fp16
TINY = {torch.bfloat16: 2.0 ** -100, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -100}


def rotate(y, cos, sin, inter, sizes=False):
    """In 64 bits; with `sizes`, the sum of the sizes of the two products."""
    n = cos.shape[-1]
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if inter else (y[..., :n], y[..., n:2 * n])
    if sizes:
        a, b, cos, sin = a.abs(), b.abs(), cos.abs(), sin.abs()
        first, second = a * cos + b * sin, a * sin + b * cos
    else:
        first, second = a * cos - b * sin, a * sin + b * cos
    out = y.abs() if sizes else y.clone()
    if inter:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = first, second
    else:
        out[..., :n], out[..., n:2 * n] = first, second
    return out


def angles(cos, sin, pos, S):
    if pos is None:
        c, s = cos[None, :S], sin[None, :S]
    else:
        c, s = cos[pos.long()], sin[pos.long()]
        if pos.dim() == 1:
            c, s = c[None], s[None]
    return c.double()[:, :, None], s.double()[:, :, None]


def forward_ref(x, w, eps, cos, sin, pos, inter):
    x64 = x.double()
    y = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps)
    y = y if w is None else y * w.double()
    if cos is None:
        return y, E * y.abs() + U[x.dtype] * y.abs()
    c, s = angles(cos, sin, pos, x.shape[1])
    o = rotate(y, c, s, inter)
    return o, E * rotate(y, c, s, inter, True) + U[x.dtype] * o.abs()


def backward_ref(d, x, w, eps, cos, sin, pos, inter, over=1):
    """Gradients and bounds; the mean is over the last `over` axes of x."""
    axes = tuple(range(-over, 0))
    d64, x64 = d.double(), x.double()
    w64 = torch.ones((), dtype=torch.float64, device=x.device) if w is None else w.double()
    g, ga = d64, d64.abs()
    if cos is not None:
        c, s = angles(cos, sin, pos, x.shape[1])
        g, ga = rotate(d64, c, -s, inter), rotate(d64, c, s, inter, True)
    r = 1 / torch.sqrt(x64.square().mean(axes, keepdim=True) + eps)
    u, ua = g * w64, ga * w64.abs()
    m = (u * x64).mean(axes, keepdim=True)
    ma = (ua * x64.abs()).mean(axes, keepdim=True)
    dx = r * (u - x64 * r * r * m)
    bx = E * r * (ua + x64.abs() * r * r * ma) + U[x.dtype] * dx.abs()
    rows = tuple(range(x.dim() - over))
    n = x[(Ellipsis,) + (0,) * over].numel()
    dw = (g * x64 * r).sum(rows)
    bw = (E + (n + 64) * 2.0 ** -24) * (ga * x64.abs() * r).sum(rows)
    return dx, bx, dw, bw


def check(name, got, ref, bound):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name} not finite"
    if got.numel() == 0:
        return
    err = (got.double() - ref).abs()
    over = err - bound - TINY[got.dtype]
    i = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name} off by {float(err.reshape(-1)[i]):.3e} where "
                                    f"{float(bound.expand_as(err).reshape(-1)[i]):.3e} is allowed")


def make(B, S, Hq, Hk, D, rot, dtype, weights=True, T=0, seed=0, pos_dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = 0.1 + 3 * torch.rand(D, generator=g, device="cuda")

    def t(H, scale):
        return (torch.randn(B, S, H, D, generator=g, device="cuda") * scale).to(dtype)

    a = {"q": t(Hq, spread), "k": t(Hk, spread), "dq": t(Hq, 1.0), "dk": t(Hk, 1.0)}
    w = [None, None]
    if weights:
        w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    pos = cos = sin = None
    if rot:
        rows = T or max(S, 1)
        ang = torch.rand(rows, rot // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
        cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
        if T:
            pos = torch.randint(0, T, (B, S), generator=g, device="cuda").to(pos_dtype)
    return a, w, cos, sin, pos


def both(a, w, cos, sin, pos, inter, eps=1e-6):
    from sinkattn_b200 import ops

    q, k = ops.qk_head_norm_rope(a["q"], a["k"], eps, w[0], w[1], cos, sin, positions=pos,
                                 interleaved=inter)
    grads = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], eps, w[0], w[1], cos, sin,
                                      positions=pos, interleaved=inter)
    torch.cuda.synchronize()
    ops.DeviceStatus.check()
    check("q", q, *forward_ref(a["q"], w[0], eps, cos, sin, pos, inter))
    check("k", k, *forward_ref(a["k"], w[1], eps, cos, sin, pos, inter))
    for i, (x, d) in enumerate((("q", "dq"), ("k", "dk"))):
        dx, bx, dw, bw = backward_ref(a[d], a[x], w[i], eps, cos, sin, pos, inter)
        assert grads[i].dtype == a[x].dtype
        check(d, grads[i], dx, bx)
        if w[i] is None:
            assert grads[2 + i] is None
        else:
            check("dw_" + x, grads[2 + i], dw, bw)
    return (q, k) + grads


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,rot", [(8, 8), (32, 32), (40, 32), (64, 64), (96, 96), (128, 64),
                                   (128, 128), (192, 16), (256, 256), (64, 0)])
def test_head_norm_sizes(D, rot, dtype, inter):
    if not inter and rot % 16:
        rot = 0
    both(*make(2, 37, 5, 2, D, rot, dtype, seed=D + rot), inter)


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (7, 1, 32, 8), (3, 5, 24, 24), (1, 1000, 3, 1),
                                       (2, 2049, 1, 9)])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_head_norm_tokens_and_positions(B, S, Hq, Hk, pos_dtype):
    both(*make(B, S, Hq, Hk, 128, 128, torch.bfloat16, T=5000, seed=S, pos_dtype=pos_dtype), False)


def test_head_norm_without_weights_one_position_row_and_zero_rows():
    a, w, cos, sin, pos = make(3, 9, 4, 4, 64, 64, torch.float32, weights=False, T=50)
    a["q"][1, 3] = 0
    both(a, w, cos, sin, pos[0], True)
    # negative strides do not exist in torch; a step of 2 does
    wide = torch.zeros(3, 18, dtype=torch.int64, device="cuda")
    wide[:, ::2] = pos
    both(a, w, cos, sin, wide[:, ::2], True)


def test_head_norm_of_nothing():
    from sinkattn_b200 import ops

    a, w, cos, sin, _ = make(2, 0, 4, 2, 128, 128, torch.bfloat16)
    q, k, dq, dk, dwq, dwk = both(a, w, cos, sin, None, True)
    assert q.shape == (2, 0, 4, 128) and not dwq.any() and not dwk.any()
    a, w, cos, sin, _ = make(2, 6, 4, 2, 128, 128, torch.bfloat16)
    full = ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin)
    q, k = ops.qk_head_norm_rope(a["q"], None, 1e-6, w[0], None, cos, sin)
    assert k is None and torch.equal(q, full[0])
    g = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin)
    h = ops.qk_head_norm_rope_bwd(a["dq"], None, a["q"], None, 1e-6, w[0], None, cos, sin)
    assert torch.equal(g[0], h[0]) and h[1] is None and h[3] is None
    check("dw_q", h[2], *backward_ref(a["dq"], a["q"], w[0], 1e-6, cos, sin, None, True)[2:])


def test_head_norm_strides_views_and_in_place():
    from sinkattn_b200 import ops

    a, w, cos, sin, pos = make(2, 33, 6, 3, 128, 128, torch.bfloat16, T=99)
    want = ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, positions=pos)
    grads = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin,
                                      positions=pos)
    # one packed projection output [B, S, (q | k | v)], heads-first and misaligned copies
    packed = torch.cat([a["q"].flatten(2), a["k"].flatten(2), a["k"].flatten(2)], dim=-1)
    pq, pk = packed[..., :768].view(2, 33, 6, 128), packed[..., 768:1152].view(2, 33, 3, 128)
    hq, hk = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (a["q"], a["k"]))

    def odd(t):
        buf = torch.zeros(*t.shape[:-1], 131, dtype=t.dtype, device="cuda")
        buf[..., 1:129] = t
        return buf[..., 1:129]

    wide_c, wide_s = (torch.zeros(99, 70, device="cuda") for _ in range(2))
    wide_c[:, 2:66], wide_s[:, 2:66] = cos, sin
    for q, k, c, s in ((pq, pk, cos, sin), (hq, hk, cos, sin), (odd(a["q"]), odd(a["k"]), cos, sin),
                       (a["q"], a["k"], wide_c[:, 2:66], wide_s[:, 2:66])):
        got = ops.qk_head_norm_rope(q, k, 1e-6, *w, c, s, positions=pos)
        back = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], q, k, 1e-6, *w, c, s, positions=pos)
        for x, y in zip(got + back, want + grads):
            assert torch.equal(x, y)
    # into a cache whose other rows stay as they were
    cache = torch.full((2, 50, 3, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, positions=pos,
                          out_k=cache[:, 10:43])
    assert torch.equal(cache[:, 10:43], want[1])
    assert (cache[:, :10] == 7).all() and (cache[:, 43:] == 7).all()
    q, k = a["q"].clone(), a["k"].clone()
    ops.qk_head_norm_rope(q, k, 1e-6, *w, cos, sin, positions=pos, out_q=q, out_k=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    dq, dk = a["dq"].clone(), a["dk"].clone()
    ops.qk_head_norm_rope_bwd(dq, dk, a["q"], a["k"], 1e-6, *w, cos, sin, positions=pos, dq=dq,
                              dk=dk)
    assert torch.equal(dq, grads[0]) and torch.equal(dk, grads[1])


def test_positions_outside_the_table_are_reported_and_nothing_else_changes():
    from sinkattn_b200 import ops

    a, w, cos, sin, pos = make(2, 8, 4, 2, 128, 128, torch.bfloat16, T=40)
    want = ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, positions=pos)
    good = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin,
                                     positions=pos)
    bad = pos.clone()
    bad[0, 3], bad[1, 7] = 40, -1
    hit = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    hit[0, 3] = hit[1, 7] = True
    got = ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, positions=bad)
    with pytest.raises(RuntimeError, match="position outside the rotary"):
        ops.DeviceStatus.check()
    back = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin,
                                     positions=bad)
    with pytest.raises(RuntimeError, match="position outside the rotary"):
        ops.DeviceStatus.check()
    for x, y in zip(got + back[:2], want + good[:2]):
        assert torch.isnan(x[hit]).all() and torch.equal(x[~hit], y[~hit])
    assert torch.isnan(back[2]).all() and torch.isnan(back[3]).all()
    ops.DeviceStatus.check()


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32, None])
@pytest.mark.parametrize("B,S,hidden,D,rope", [
    (1, 1, 8, 8, True), (2, 50, 256, 64, True), (1, 333, 768, 128, True),
    (2, 700, 1536, 128, True), (1, 64, 1544, 8, True), (3, 41, 2048, 128, False),
    (1, 77, 2560, 64, True), (2, 130, 4096, 128, True),
])
def test_hidden_norm_gradient(B, S, hidden, D, rope, w_dtype):
    from sinkattn_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(hidden + S)
    spread = 0.1 + 3 * torch.rand(hidden, generator=gen, device="cuda")

    def t(scale):
        return (torch.randn(B, S, hidden, generator=gen, device="cuda") * scale).bfloat16()

    q, k, dq, dk = t(spread), t(spread), t(1.0), t(1.0)
    w = [None, None]
    if w_dtype is not None:
        w = [(1 + 0.3 * torch.randn(hidden, generator=gen, device="cuda")).to(w_dtype)
             for _ in range(2)]
    cos = sin = None
    if rope:
        ang = torch.rand(S, D // 2, generator=gen, device="cuda", dtype=torch.float64) * 6.3
        cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    got = ops.qk_norm_rope_bwd(dq, dk, q, k, D, 1e-6, w[0], w[1], cos, sin)
    split = (B, S, hidden // D, D)
    for i, (d, x) in enumerate(((dq, q), (dk, k))):
        w4 = None if w[i] is None else w[i].view(hidden // D, D)
        dx, bx, dw, bw = backward_ref(d.view(split), x.view(split), w4, 1e-6, cos, sin, None, True,
                                      over=2)
        check("dx", got[i].view(split), dx, bx)
        if w[i] is None:
            assert got[2 + i] is None
        else:
            check("dw", got[2 + i].view(hidden // D, D), dw, bw)
    again = ops.qk_norm_rope_bwd(dq, dk, q, k, D, 1e-6, w[0], w[1], cos, sin)
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)
    # a strided input, and the gradients written over the upstream ones
    wide = torch.zeros(B, S, hidden + 16, dtype=torch.bfloat16, device="cuda")
    wide[..., 8:hidden + 8] = q
    inq, ink = dq.clone(), dk.clone()
    ops.qk_norm_rope_bwd(inq, ink, wide[..., 8:hidden + 8], k, D, 1e-6, w[0], w[1], cos, sin,
                         dq=inq, dk=ink)
    assert torch.equal(inq, got[0]) and torch.equal(ink, got[1])


def test_hidden_norm_gradient_of_no_rows():
    from sinkattn_b200 import ops

    z = torch.zeros(2, 0, 256, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(256, device="cuda")
    t = torch.zeros(0, 32, device="cuda")
    dq, dk, dwq, dwk = ops.qk_norm_rope_bwd(z, z, z, z, 64, 1e-6, w, w, t, t)
    assert dq.shape == (2, 0, 256) and not dwq.any() and not dwk.any()


def test_captured_beside_an_eager_call():
    from sinkattn_b200 import ops

    a, w, cos, sin, pos = make(2, 300, 6, 3, 128, 128, torch.bfloat16, T=600, seed=1)
    b, w2, _, _, pos2 = make(2, 300, 6, 3, 128, 128, torch.bfloat16, T=600, seed=2)

    def call(x, ws, p):
        y = ops.qk_head_norm_rope(x["q"], x["k"], 1e-6, *ws, cos, sin, positions=p)
        return y + ops.qk_head_norm_rope_bwd(x["dq"], x["dk"], x["q"], x["k"], 1e-6, *ws, cos, sin,
                                             positions=p)

    want, want2 = call(a, w, pos), call(b, w2, pos2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(a, w, pos)
    side = torch.cuda.Stream()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            beside = call(b, w2, pos2)
        torch.cuda.synchronize()
        for x, y in zip(got + beside, want + want2):
            assert torch.equal(x, y)
    for key in a:
        a[key].copy_(b[key])
    for x, y in zip(w + [pos], w2 + [pos2]):
        x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(got, want2):
        assert torch.equal(x, y)
    del graph


def test_gradients_against_differences():
    from sinkattn_b200 import ops

    a, w, cos, sin, pos = make(1, 12, 3, 2, 64, 32, torch.float32, T=30, seed=5)
    q, k, dwq, dwk = ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos,
                                               sin, positions=pos, interleaved=False)
    dirs = {n: torch.randn_like(t).double() for n, t in (("q", a["q"]), ("k", a["k"]),
                                                         ("wq", w[0]), ("wk", w[1]))}

    def value(h):
        total = 0.0
        for x, d, wi, n in (("q", "dq", 0, "wq"), ("k", "dk", 1, "wk")):
            x64 = a[x].double() + h * dirs[x]
            y = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-6)
            y = y * (w[wi].double() + h * dirs[n])
            c, s = angles(cos, sin, pos, 12)
            total += float((rotate(y, c, s, False) * a[d].double()).sum())
        return total

    h = 1e-5
    want = (value(h) - value(-h)) / (2 * h)
    got = sum(float((g.double() * dirs[n]).sum())
              for g, n in ((q, "q"), (k, "k"), (dwq, "wq"), (dwk, "wk")))
    size = sum(float((g.double() * dirs[n]).abs().sum())
               for g, n in ((q, "q"), (k, "k"), (dwq, "wq"), (dwk, "wk")))
    # 2^-16 of every term (above); the difference's own error is h^2 of third derivatives
    assert abs(got - want) <= 2.0 ** -16 * size + 1e-6 * size, (got, want, size)


def test_odd_strides_of_dimensions_of_size_one():
    from sinkattn_b200 import ops

    def odd(t):
        st = [s if n > 1 else 13 for s, n in zip(t.stride(), t.shape)]
        return torch.as_strided(t, t.shape, st)

    a, w, cos, sin, _ = make(1, 1, 1, 1, 128, 128, torch.bfloat16)
    want = ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin)
    want += ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin)
    o = {n: odd(t) for n, t in a.items()}
    got = ops.qk_head_norm_rope(o["q"], o["k"], 1e-6, *w, odd(cos), odd(sin))
    got += ops.qk_head_norm_rope_bwd(o["dq"], o["dk"], o["q"], o["k"], 1e-6, *w, odd(cos), odd(sin))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for B, S in ((1, 1), (3, 1), (1, 5)):
        g = torch.Generator(device="cuda").manual_seed(B + S)
        x = [torch.randn(B, S, 256, generator=g, device="cuda").bfloat16() for _ in range(4)]
        wide = [torch.cat([t, t], dim=-1)[..., 256:] for t in x]
        want = ops.qk_norm_rope_bwd(*x, 128, 1e-6)
        for y in ([odd(t) for t in x], wide, [odd(t) for t in wide]):
            got = ops.qk_norm_rope_bwd(*y, 128, 1e-6)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    from sinkattn_b200 import ops

    a, w, cos, sin, pos = make(2, 5, 4, 2, 128, 128, torch.bfloat16, T=9)

    def refuse(match, fn="qk_head_norm_rope", exc=RuntimeError, **kw):
        args = dict(q=a["q"], k=a["k"], eps=1e-6, w_q=w[0], w_k=w[1], cos=cos, sin=sin,
                    positions=pos)
        if fn.endswith("bwd"):
            args.update(dq_out=a["dq"], dk_out=a["dk"])
        args.update(kw)
        with pytest.raises(exc, match=match):
            getattr(ops, fn)(**args)

    refuse("expects q, k of", q=a["q"][0])
    refuse("k must be", k=a["k"].float())
    refuse("k must be", k=a["k"][:, :4])
    refuse("bf16, fp16 or fp32", q=a["q"].double(), k=a["k"].double())
    refuse("go together", w_k=None)
    refuse("go together", sin=None)
    refuse("128 elements", w_q=w[0][:64])
    refuse("cos and sin must be fp32", cos=cos.double(), sin=sin.double())
    refuse("cos and sin must be fp32", sin=sin[:, :32])
    refuse("positions must be", positions=pos.float())
    refuse("positions must be", positions=pos[:, :4])
    refuse("positions need", cos=None, sin=None)
    refuse("table rows", cos=cos[:4], sin=sin[:4], positions=None)
    refuse("multiple of 16", cos=cos[:, :12], sin=sin[:, :12], interleaved=False)
    refuse("out_q must", out_q=torch.empty(2, 5, 4, 132, dtype=torch.bfloat16, device="cuda")[..., 4:])
    refuse("out_k without k", k=None, w_k=None, out_k=a["k"])
    refuse("CUDA tensors only", cos=cos.cpu(), sin=sin.cpu())
    refuse("multiple of 8 up to 256", q=a["q"][..., :100], k=a["k"][..., :100], w_q=None, w_k=None,
           cos=None, sin=None, positions=None)
    refuse("dk_out is missing", fn="qk_head_norm_rope_bwd", dk_out=None)
    refuse("dq_out must be", fn="qk_head_norm_rope_bwd", dq_out=a["dq"].float())
    refuse("workspace", fn="qk_head_norm_rope_bwd",
           workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    x = torch.zeros(2, 5, 256, dtype=torch.bfloat16, device="cuda")
    h = dict(dq_out=x, dk_out=x, q=x, k=x, head_dim=128, eps=1e-6)
    for match, exc, kw in (("must be bf16", RuntimeError, dict(q=x.float())),
                           ("must be bf16", RuntimeError, dict(dk_out=x[:, :4])),
                           ("256 elements", RuntimeError, dict(w_q=w[0], w_k=w[1])),
                           ("go together", RuntimeError, dict(w_q=x[0, 0])),
                           ("frequency shape", ValueError, dict(cos=cos, sin=sin)),
                           ("uniform rows", RuntimeError, dict(dq=x.transpose(0, 1).contiguous()
                                                               .transpose(0, 1)))):
        with pytest.raises(exc, match=match):
            ops.qk_norm_rope_bwd(**{**h, **kw})


def test_expanded_outputs_workspaces_and_empty_tables_are_refused():
    from sinkattn_b200 import ops

    q = torch.randn(2, 3, 4, 64, device="cuda").bfloat16()
    w = torch.ones(64, device="cuda").bfloat16()
    none = torch.empty(0, 32, device="cuda")
    wide = q[:, :, :1].contiguous().expand(-1, -1, 4, -1)
    small = torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 22)
    with pytest.raises(RuntimeError, match="out_k is expanded"):
        ops.qk_head_norm_rope(q, q, 1e-6, out_k=wide)
    with pytest.raises(RuntimeError, match="dq is expanded"):
        ops.qk_head_norm_rope_bwd(q, q, q, q, 1e-6, dq=wide)
    with pytest.raises(RuntimeError, match="workspace must be contiguous"):
        ops.qk_head_norm_rope_bwd(q, q, q, q, 1e-6, w, w, workspace=small)
    with pytest.raises(RuntimeError, match="have no rows"):
        ops.qk_head_norm_rope(q, q, 1e-6, w, w, none, none)
    with pytest.raises(RuntimeError, match="have no rows"):
        ops.qk_head_norm_rope(q, q, 1e-6, w, w, none, none,
                              positions=torch.zeros(3, dtype=torch.int32, device="cuda"))
    x = torch.randn(2, 3, 256, device="cuda").bfloat16()
    w = torch.ones(256, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="dk is expanded"):
        ops.qk_norm_rope_bwd(x, x, x, x, 64, 1e-6, dk=x[:, :1].contiguous().expand(-1, 3, -1))
    with pytest.raises(RuntimeError, match="workspace must be contiguous"):
        ops.qk_norm_rope_bwd(x, x, x, x, 64, 1e-6, w, w, workspace=small)


def test_the_short_way_is_taken_and_agrees_with_the_long_one(monkeypatch):
    from sinkattn_b200 import ops

    assert ops._fast is not None, "the extension module is not built"
    a, w, cos, sin, pos = make(2, 40, 6, 3, 128, 128, torch.bfloat16, T=99)
    ops.DeviceStatus.pointer(cos.device)
    x = [torch.randn(2, 40, 768, device="cuda").bfloat16() for _ in range(4)]
    wh = torch.randn(768, device="cuda")
    th = [t[:40].contiguous() for t in (cos, sin)]
    packed = torch.cat([a["q"].flatten(2), a["k"].flatten(2)], dim=-1)
    pq, pk = packed[..., :768].unflatten(2, (6, 128)), packed[..., 768:].unflatten(2, (3, 128))
    calls = [
        lambda: ops.qk_head_norm_rope(a["q"], a["k"], 1e-6, *w, cos, sin, positions=pos),
        lambda: ops.qk_head_norm_rope(pq, pk, 1e-6, *w, cos, sin, positions=pos[0].int()),
        lambda: ops.qk_head_norm_rope(a["q"], None, 1e-6, w[0], None, cos, sin, interleaved=False),
        lambda: ops.qk_head_norm_rope(a["q"].float(), a["k"].float(), 1e-6),
        lambda: ops.qk_head_norm_rope_bwd(a["dq"], a["dk"], a["q"], a["k"], 1e-6, *w, cos, sin,
                                          positions=pos),
        lambda: ops.qk_head_norm_rope_bwd(a["dq"], None, pq, None, 1e-6, w[0].float(), None),
        lambda: ops.qk_norm_rope_bwd(*x, 128, 1e-6, wh, wh, *th),
        lambda: ops.qk_norm_rope_bwd(*x, 128, 1e-6, wh.bfloat16(), wh.bfloat16()),
        lambda: ops.qk_norm_rope_bwd(*x, 128, 1e-6, dq=torch.empty_like(x[0])),
    ]
    taken = []
    real = ops._short

    def spy(name, *args):
        got = real(name, *args)
        taken.append(got is not None)
        return got

    monkeypatch.setattr(ops, "_short", spy)
    fast = [c() for c in calls]
    assert taken == [True] * len(calls)
    monkeypatch.setattr(ops, "_short", lambda *args: None)
    for c, want in zip(calls, fast):
        got = c()
        assert len(got) == len(want)
        for p, q in zip(got, want):
            assert (p is None and q is None) or (torch.equal(p, q) and p.stride() == q.stride())


def test_captured_after_a_copy_a_fill_and_another_stream():
    """The launches may start while the one before them ends: whatever that one is, a replay gives
    what an eager run gives."""
    from sinkattn_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(4)
    src = torch.randn(2, 300, 6, 128, generator=g, device="cuda").bfloat16()
    mask = torch.ones(2, 6, 3, 3, dtype=torch.bool, device="cuda")
    w = torch.ones(128, device="cuda")
    x, y, z = (torch.empty_like(src) for _ in range(3))
    side = torch.cuda.Stream()

    def step():
        x.copy_(src)                                       # a copy
        q, _ = ops.qk_head_norm_rope(x, None, 1e-6, w)
        y.zero_()                                          # a fill
        a = ops.qk_head_norm_rope_bwd(q, y, x, y, 1e-6, w, w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                      # another stream's kernel
            z.copy_(a[0])
            z.mul_(2)
        torch.cuda.current_stream().wait_stream(side)
        t = [s.transpose(1, 2) for s in (x, z, q)]
        out, lse = ops.bsattn_fwd(*t, mask)
        y.zero_()
        b = ops.bsattn_bwd(out, *t, out, lse, mask)
        y.copy_(b[0].transpose(1, 2))
        return (q,) + a[:1] + a[2:] + b + ops.qk_norm_rope_bwd(
            y.view(2, 300, 768), x.view(2, 300, 768), z.view(2, 300, 768), y.view(2, 300, 768),
            128, 1e-6)[:2]

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for t in got:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)
    for _ in range(20):  # many calls in a row, each reading what the one before wrote
        eager = step()
    torch.cuda.synchronize()
    for a, b in zip(want, eager):
        assert torch.equal(a, b)
    ops.DeviceStatus.check()
