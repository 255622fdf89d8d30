"""Measured cases of the operators that train a sparse attention layer.

Four operators: the per-head norm + rotation of queries and keys, its gradient,
the gradient of the norm over the hidden dimension + rotation, and the backward
pass of the block-sparse attention. `own` selects the framework's kernels; the
plain forms below are elementary torch operations in 32 bits.
"""
import math

import torch

own = False

BLOCK = 128


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _attn(B, H, Sq, Sk, density, empty=0.0, hmt=False, layout="bshd"):
    return {"op": "bsattn_bwd", "B": B, "H": H, "Sq": Sq, "Sk": Sk, "density": density,
            "empty": empty, "hmt": hmt, "layout": layout}


def _head(op, B, S, Hq, Hk, D, rot, inter, dtype, weights=True, T=0):
    return {"op": op, "B": B, "S": S, "Hq": Hq, "Hk": Hk, "D": D, "rot": rot, "inter": inter,
            "dtype": dtype, "weights": weights, "T": T}


def _hidden(B, S, hidden, D, wdtype):
    return {"op": "qk_norm_rope_bwd", "B": B, "S": S, "hidden": hidden, "D": D, "wdtype": wdtype}


def listed():
    return [
        # one layer of video self-attention over 21x30x52 latent tokens, 12 heads of 128
        dict(_attn(1, 12, 32760, 32760, 0.2), name="attn_bwd_video"),
        # 4096 tokens, 4 heads: an image at low resolution, or one rank's share of heads
        dict(_attn(1, 4, 4096, 4096, 0.2, layout="bhsd"), name="attn_bwd_4k"),
        # video queries against 512 text tokens, every block kept, lengths that end inside a block
        dict(_attn(2, 12, 4680, 500, 1.0, hmt=True), name="attn_bwd_text"),
        # a few hundred tokens, some mask rows empty: latency counts
        dict(_attn(1, 2, 300, 300, 0.5, empty=0.3), name="attn_bwd_short"),
        # image tokens and text tokens of one sample, 30 heads of 128
        dict(_head("qk_head_norm_rope", 1, 16896, 30, 30, 128, 128, True, "bf16"),
             name="head_norm_rope_image"),
        # one new token for each of 8 sequences, fewer key heads, positions far into the table
        dict(_head("qk_head_norm_rope", 8, 1, 32, 8, 128, 128, False, "bf16", T=131072),
             name="head_norm_rope_token"),
        # a ragged length, narrow heads rotated in part, full precision
        dict(_head("qk_head_norm_rope", 2, 1333, 16, 4, 64, 32, False, "fp32", T=4096),
             name="head_norm_rope_fp32"),
        # training the image layer
        dict(_head("qk_head_norm_rope_bwd", 1, 16896, 30, 30, 128, 128, True, "bf16"),
             name="head_norm_rope_bwd_image"),
        # a short ragged batch in fp16, wide heads, split rotation
        dict(_head("qk_head_norm_rope_bwd", 2, 777, 8, 2, 256, 128, False, "fp16", T=1024),
             name="head_norm_rope_bwd_fp16"),
        # training the video layer: 12 heads of 128 normed together
        dict(_hidden(1, 32760, 1536, 128, "fp32"), name="norm_rope_bwd_video"),
        # a short clip
        dict(_hidden(2, 390, 1536, 128, "bf16"), name="norm_rope_bwd_short"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bsattn_bwd", "bsattn_bwd", "qk_head_norm_rope", "qk_head_norm_rope_bwd",
                     "qk_norm_rope_bwd"])
    if op == "bsattn_bwd":
        B, H = rng.choice([1, 1, 2, 3]), rng.choice([1, 2, 3, 4, 6, 12])
        Sq = _log(rng, 1, 16000)
        Sk = Sq if rng.random() < 0.6 else _log(rng, 1, 16000)
        while B * H * Sq * Sk > 12 * 14000 * 14000:
            H = max(1, H // 2)
            B = 1
        return _attn(B, H, Sq, Sk, rng.choice([0.1, 0.2, 0.35, 0.6, 1.0]),
                     empty=rng.choice([0.0, 0.0, 0.25]), hmt=rng.random() < 0.3,
                     layout=rng.choice(["bshd", "bhsd"]))
    if op == "qk_norm_rope_bwd":
        D = rng.choice([64, 128])
        hidden = D * rng.choice([4, 8, 12, 20])
        return _hidden(rng.choice([1, 2]), _log(rng, 1, 8000), hidden, D,
                       rng.choice(["fp32", "bf16"]))
    B = _log(rng, 1, 16)
    S = 1 if rng.random() < 0.25 else _log(rng, 1, 16000 // B)
    D = rng.choice([32, 64, 96, 128, 192, 256])
    Hk = rng.choice([1, 2, 4, 6, 8])
    Hq = Hk * rng.choice([1, 1, 2, 3])
    rot = rng.choice([D, D, D // 2])
    T = rng.choice([0, S, S + _log(rng, 1, 100000)])
    return _head(op, B, S, Hq, Hk, D, rot, rng.random() < 0.5,
                 rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.8, T)


_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _mask(case, gen):
    """Column 0, the diagonal and a random share of the blocks; some rows keep none."""
    B, H = case["B"], case["H"]
    nq, nk = -(-case["Sq"] // BLOCK), -(-case["Sk"] // BLOCK)
    m = torch.rand(B, H, nq, nk, generator=gen, device="cuda") < case["density"]
    m[..., 0] = True
    d = torch.arange(min(nq, nk), device="cuda")
    m[:, :, d, d] = True
    if case["empty"] > 0.0:
        m &= (torch.rand(B, H, nq, 1, generator=gen, device="cuda") >= case["empty"])
    return m


def _kept_pairs(case):
    """Expected number of (query, key) pairs of one head that the mask keeps."""
    Sq, Sk = case["Sq"], case["Sk"]
    nq, nk = -(-Sq // BLOCK), -(-Sk // BLOCK)
    first = float(Sq * min(Sk, BLOCK))
    diag = sum(float(min(BLOCK, Sq - i * BLOCK) * min(BLOCK, Sk - i * BLOCK))
               for i in range(1, min(nq, nk)))
    rest = float(Sq) * Sk - first - diag
    return (first + diag + case["density"] * rest) * (1.0 - case["empty"])


def work(case):
    if case["op"] == "bsattn_bwd":
        B, H, Sq, Sk = case["B"], case["H"], case["Sq"], case["Sk"]
        dense = 0.25 if case["hmt"] else 0.0  # a head in four (rounded down) reads no mask
        pairs = _kept_pairs(case) * (1.0 - dense) + float(Sq) * Sk * dense
        # q, out, dout in and dq out; k, v in and dk, dv out; the row statistics
        return {"bytes": B * H * (4 * Sq * 256 + 4 * Sk * 256 + 4 * Sq),
                "flops": 5.0 * 2.0 * 128.0 * pairs * B * H}
    if case["op"] == "qk_norm_rope_bwd":
        n = 2.0 * case["B"] * case["S"] * case["hidden"]
        return {"bytes": 6.0 * n + 8.0 * case["hidden"] + 4.0 * case["S"] * case["D"],
                "flops": 16.0 * n}
    n = float(case["B"] * case["S"] * (case["Hq"] + case["Hk"]) * case["D"])
    # the rotation of every token: its own row of the tables with positions, else one per index
    tables = 4.0 * case["rot"] * case["S"] * (case["B"] if case["T"] else 1)
    if case["op"] == "qk_head_norm_rope":
        return {"bytes": 2.0 * n * _SIZE[case["dtype"]] + tables, "flops": 8.0 * n}
    return {"bytes": 3.0 * n * _SIZE[case["dtype"]] + tables, "flops": 16.0 * n}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _tables(T, rot):
    ang = (torch.arange(T, dtype=torch.float64, device="cuda")[:, None]
           * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"),
                       -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot))
    return torch.cos(ang).float(), torch.sin(ang).float()


def _prepare_attn(case, gen):
    B, H, Sq, Sk = case["B"], case["H"], case["Sq"], case["Sk"]

    def make(S, shift):
        if case["layout"] == "bshd":
            t = torch.randn(B, S, H, 128, generator=gen, device="cuda").permute(0, 2, 1, 3)
        else:
            t = torch.randn(B, H, S, 128, generator=gen, device="cuda")
        if shift is not None:  # a direction that all tokens share
            t += shift
        return t.bfloat16()

    c = 0.3 * torch.randn(128, generator=gen, device="cuda")
    q, k, v = make(Sq, c), make(Sk, c), make(Sk, None)
    dout = make(Sq, None)
    mask = _mask(case, gen)
    hmt = None
    if case["hmt"]:
        # every fourth head is dense, the others read their own slice
        hmt = torch.arange(1, H + 1, device="cuda", dtype=torch.int32)
        hmt[3::4] = 0
    state = {"q": q, "k": k, "v": v, "dout": dout, "mask": mask, "hmt": hmt,
             "scale": 1.0 / math.sqrt(128.0)}
    # what the forward pass left: the output and the rows' log-sum-exp
    out = torch.empty_like(q)
    lse = torch.empty(B, H, Sq, dtype=torch.float32, device="cuda")
    for b, h, r0, r1, keep in _chunks(state):
        s = (q[b, h, r0:r1].float() @ k[b, h].float().T) * state["scale"]
        s.masked_fill_(~keep, float("-inf"))
        m = s.amax(dim=1, keepdim=True)
        m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
        p = torch.exp(s.sub_(m))
        l = p.sum(dim=1, keepdim=True)
        o = (p @ v[b, h].float()) / l
        out[b, h, r0:r1] = torch.where(l > 0, o, torch.zeros_like(o)).bfloat16()
        lse[b, h, r0:r1] = (torch.log(l) + m)[:, 0]  # log 0 = -inf where no key is kept
    state["out"], state["lse"] = out, lse
    return state


def _chunks(state, rows=4096):
    """(b, h, first row, last row, kept keys of these rows as a truth value per pair)."""
    B, H, Sq, _ = state["q"].shape
    Sk = state["k"].shape[2]
    dense = [] if state["hmt"] is None else list(range(3, H, 4))
    for b in range(B):
        for h in range(H):
            m = state["mask"][b, h]
            if h in dense:
                m = torch.ones_like(m)
            cols = m.repeat_interleave(BLOCK, dim=1)[:, :Sk]
            for r0 in range(0, Sq, rows):
                r1 = min(Sq, r0 + rows)
                keep = cols[r0 // BLOCK:-(-r1 // BLOCK)].repeat_interleave(BLOCK, dim=0)
                yield b, h, r0, r1, keep[:r1 - r0]


def _prepare_head(case, gen):
    B, S, D, dt = case["B"], case["S"], case["D"], _DT[case["dtype"]]

    def make(H, shape_scale):
        t = torch.randn(B, S, H, D, generator=gen, device="cuda")
        return (t * shape_scale).to(dt)

    spread = 0.25 + 3.0 * torch.rand(D, generator=gen, device="cuda")
    st = {"q": make(case["Hq"], spread), "k": make(case["Hk"], spread), "eps": 1e-6,
          "inter": case["inter"], "w_q": None, "w_k": None, "pos": None}
    if case["weights"]:
        st["w_q"] = (1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dt)
        st["w_k"] = (1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dt)
    T = case["T"]
    if T > 0:
        st["pos"] = torch.randint(0, T, (B, S), generator=gen, device="cuda")
    st["cos"], st["sin"] = _tables(T if T > 0 else S, case["rot"])
    if case["op"] == "qk_head_norm_rope_bwd":
        st["dq"], st["dk"] = make(case["Hq"], 1.0), make(case["Hk"], 1.0)
    return st


def _prepare_hidden(case, gen):
    B, S, hidden = case["B"], case["S"], case["hidden"]

    def make(scale):
        return (torch.randn(B, S, hidden, generator=gen, device="cuda") * scale).bfloat16()

    spread = 0.25 + 3.0 * torch.rand(hidden, generator=gen, device="cuda")
    wd = _DT[case["wdtype"]]
    st = {"q": make(spread), "k": make(spread), "dq": make(1.0), "dk": make(1.0), "eps": 1e-6,
          "D": case["D"],
          "w_q": (1.0 + 0.2 * torch.randn(hidden, generator=gen, device="cuda")).to(wd),
          "w_k": (1.0 + 0.2 * torch.randn(hidden, generator=gen, device="cuda")).to(wd)}
    st["cos"], st["sin"] = _tables(S, case["D"])
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "bsattn_bwd":
        st = _prepare_attn(case, gen)
    elif case["op"] == "qk_norm_rope_bwd":
        st = _prepare_hidden(case, gen)
    else:
        st = _prepare_head(case, gen)
    st["op"] = case["op"]
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from sinkattn_b200 import ops

    if st["op"] == "bsattn_bwd":
        return ops.bsattn_bwd(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"],
                              st["mask"], softmax_scale=st["scale"], head_mask_type=st["hmt"])
    if st["op"] == "qk_norm_rope_bwd":
        return ops.qk_norm_rope_bwd(st["dq"], st["dk"], st["q"], st["k"], st["D"], st["eps"],
                                    st["w_q"], st["w_k"], st["cos"], st["sin"])
    if st["op"] == "qk_head_norm_rope":
        return ops.qk_head_norm_rope(st["q"], st["k"], st["eps"], st["w_q"], st["w_k"],
                                     st["cos"], st["sin"], positions=st["pos"],
                                     interleaved=st["inter"])
    out = ops.qk_head_norm_rope_bwd(st["dq"], st["dk"], st["q"], st["k"], st["eps"], st["w_q"],
                                    st["w_k"], st["cos"], st["sin"], positions=st["pos"],
                                    interleaved=st["inter"])
    return [t for t in out if t is not None]


def _rotate(y, cos, sin, inter):
    """Rotates the first 2 * cos.shape[-1] channels; cos, sin broadcast against y's pairs."""
    n = cos.shape[-1]
    head, rest = y[..., :2 * n], y[..., 2 * n:]
    if inter:
        a, b = head[..., 0::2], head[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = head[..., :n], head[..., n:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([r, rest], dim=-1)


def _angles(st):
    cos, sin = st["cos"], st["sin"]
    if st["pos"] is not None:
        cos, sin = cos[st["pos"]], sin[st["pos"]]  # [B, S, n]
    else:
        S = st["q"].shape[1]
        cos, sin = cos[None, :S], sin[None, :S]
    return cos[:, :, None], sin[:, :, None]


def _norm_bwd(g, x, w, eps):
    """Gradients of x / rms(x) * w with respect to x and w, from g; rms over the last axis."""
    r = 1.0 / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps)
    xh = x * r
    u = g if w is None else g * w
    dx = r * (u - xh * (u * xh).mean(dim=-1, keepdim=True))
    dw = None
    if w is not None:
        # one sum over every row: in 64 bits
        dw = (g * xh).reshape(-1, w.numel()).sum(dim=0, dtype=torch.float64).float()
    return dx, dw


def _run_plain(st):
    if st["op"] == "bsattn_bwd":
        return _attn_bwd_plain(st)
    if st["op"] == "qk_head_norm_rope":
        cos, sin = _angles(st)
        outs = []
        for x, w in ((st["q"], st["w_q"]), (st["k"], st["w_k"])):
            xf = x.float()
            y = xf / torch.sqrt((xf * xf).mean(dim=-1, keepdim=True) + st["eps"])
            if w is not None:
                y = y * w.float()
            outs.append(_rotate(y, cos, sin, st["inter"]).to(x.dtype))
        return tuple(outs)
    if st["op"] == "qk_head_norm_rope_bwd":
        cos, sin = _angles(st)
        dxs, dws = [], []
        for d, x, w in ((st["dq"], st["q"], st["w_q"]), (st["dk"], st["k"], st["w_k"])):
            g = _rotate(d.float(), cos, -sin, st["inter"])
            dx, dw = _norm_bwd(g, x.float(), None if w is None else w.float(), st["eps"])
            dxs.append(dx.to(x.dtype))
            if dw is not None:
                dws.append(dw)
        return dxs + dws
    B, S, hidden = st["q"].shape
    D = st["D"]
    dxs, dws = [], []
    cos, sin = st["cos"][None, :, None], st["sin"][None, :, None]
    for d, x, w in ((st["dq"], st["q"], st["w_q"]), (st["dk"], st["k"], st["w_k"])):
        g = _rotate(d.float().view(B, S, hidden // D, D), cos, -sin, True).reshape(B, S, hidden)
        dx, dw = _norm_bwd(g, x.float(), w.float(), st["eps"])
        dxs.append(dx.to(x.dtype))
        dws.append(dw)
    return tuple(dxs + dws)


def _attn_bwd_plain(st):
    q, k, v, dout, scale = st["q"], st["k"], st["v"], st["dout"], st["scale"]
    dq = torch.empty_like(q)
    dk = torch.zeros(k.shape, dtype=torch.float32, device=k.device)
    dv = torch.zeros(v.shape, dtype=torch.float32, device=v.device)
    delta = (dout.float() * st["out"].float()).sum(dim=-1)
    # a row that keeps no key has lse = -inf and no probabilities
    lse = torch.where(torch.isfinite(st["lse"]), st["lse"], torch.zeros_like(st["lse"]))
    for b, h, r0, r1, keep in _chunks(st):
        qf, kf, vf = q[b, h, r0:r1].float(), k[b, h].float(), v[b, h].float()
        df = dout[b, h, r0:r1].float()
        x = (qf @ kf.T) * scale - lse[b, h, r0:r1, None]
        p = torch.exp(x.masked_fill_(~keep, float("-inf")))
        ds = (df @ vf.T - delta[b, h, r0:r1, None]) * p
        dq[b, h, r0:r1] = ((ds @ kf) * scale).to(q.dtype)
        dk[b, h] += (ds.T @ qf) * scale
        dv[b, h] += p.T @ df
    return dq, dk.to(k.dtype), dv.to(v.dtype)


# --------------------------------------------------------------------------
# in 64 bits, from the definition
# --------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "bsattn_bwd":
        return _attn_bwd_exact(st)
    if case["op"] == "qk_norm_rope_bwd":
        B, S, hidden = st["q"].shape
        n = hidden // st["D"]
        split = lambda t: t.double().view(B, S, n, st["D"])
        one = lambda t: t.double().view(1, 1, n, st["D"])
        z = _turn(st["cos"].double().view(1, S, 1, -1), st["sin"].double().view(1, S, 1, -1))
        res = []
        for d, x, w in ((st["dq"], st["q"], st["w_q"]), (st["dk"], st["k"], st["w_k"])):
            res.append(_norm_rope_grad(split(d), split(x), one(w), z, True, st["eps"], (2, 3)))
        return (res[0][0].reshape(B, S, hidden), res[1][0].reshape(B, S, hidden),
                res[0][1].reshape(hidden), res[1][1].reshape(hidden))
    S = st["q"].shape[1]
    rows = st["pos"] if st["pos"] is not None else torch.arange(S, device="cuda")[None]
    z = _turn(st["cos"].double()[rows].unsqueeze(2), st["sin"].double()[rows].unsqueeze(2))
    res = []
    for x, w, d in ((st["q"], st["w_q"], st.get("dq")), (st["k"], st["w_k"], st.get("dk"))):
        w = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
        xd = x.double()
        if d is None:
            y = xd * w * (xd.square().mean(-1, keepdim=True) + st["eps"]).rsqrt()
            res.append(_spin(y, z, st["inter"]))
        else:
            res.append(_norm_rope_grad(d.double(), xd, w, z, st["inter"], st["eps"], (3,)))
    if case["op"] == "qk_head_norm_rope":
        return tuple(res)
    out = [res[0][0], res[1][0]]
    if st["w_q"] is not None:
        out += [r[1].sum(dim=(0, 1, 2)) if r[1].dim() > 1 else r[1] for r in res]
    return out


def _turn(c, s):
    return torch.complex(c, s)


def _spin(y, z, inter):
    """Multiplies the pairs of the first channels, as complex numbers, by z."""
    n = z.shape[-1]
    y = y.clone()
    first = y[..., 0:2 * n:2] if inter else y[..., :n]
    second = y[..., 1:2 * n:2] if inter else y[..., n:2 * n]
    t = torch.complex(first.contiguous(), second.contiguous()) * z
    if inter:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = t.real, t.imag
    else:
        y[..., :n], y[..., n:2 * n] = t.real, t.imag
    return y


def _norm_rope_grad(d, x, w, z, inter, eps, over):
    """d/dx and d/dw of spin(x w / sqrt(mean x^2 + eps)) contracted with d."""
    g = _spin(d, z.conj(), inter)
    count = 1
    for a in over:
        count *= x.shape[a]
    ms = x.square().sum(dim=over, keepdim=True) / count + eps
    dot = (g * w * x).sum(dim=over, keepdim=True) / count
    dx = g * w * ms.pow(-0.5) - x * dot * ms.pow(-1.5)
    keep = (0, 1) if len(over) == 2 else (0, 1, 2)
    return dx, (g * x * ms.pow(-0.5)).sum(dim=keep)


def _attn_bwd_exact(st):
    scale = st["scale"]
    B, H, Sq, _ = st["q"].shape
    Sk = st["k"].shape[2]
    dense = [] if st["hmt"] is None else [h for h in range(H) if int(st["hmt"][h]) == 0]
    dq = torch.zeros(B, H, Sq, 128, dtype=torch.float64, device="cuda")
    dk = torch.zeros(B, H, Sk, 128, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    key_block = torch.arange(Sk, device="cuda") // BLOCK
    step = 2048
    for b in range(B):
        for h in range(H):
            k, v = st["k"][b, h].double(), st["v"][b, h].double()
            for r0 in range(0, Sq, step):
                rows = torch.arange(r0, min(Sq, r0 + step), device="cuda")
                q, g = st["q"][b, h, rows].double(), st["dout"][b, h, rows].double()
                e = scale * (q @ k.T)
                if h not in dense:
                    kept = st["mask"][b, h][rows // BLOCK][:, key_block]
                    e = torch.where(kept, e, torch.full((), -math.inf, dtype=e.dtype, device="cuda"))
                prob = torch.softmax(e, dim=-1)
                prob = torch.nan_to_num(prob, nan=0.0)  # rows that keep no key
                dp = g @ v.T
                de = prob * (dp - (prob * dp).sum(-1, keepdim=True))
                dq[b, h, rows] = scale * (de @ k)
                dk[b, h] += scale * (de.T @ q)
                dv[b, h] += prob.T @ g
    return dq, dk, dv
