"""Host-side refusals of the training operators that need no GPU."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture
def on_device(monkeypatch):
    """ops as it is on a GPU, up to the first look at the device."""
    from sinkattn_b200 import ops

    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: torch.device("cuda", 0))
    monkeypatch.setattr(ops, "_short", lambda *a: None)
    return ops


@pytest.mark.parametrize("D,dtype", [(100, torch.bfloat16), (12, torch.float32), (4, torch.float32),
                                     (264, torch.float16)])
def test_head_sizes_are_refused_whatever_the_layout(on_device, D, dtype):
    x = torch.zeros(2, 5, 3, D, dtype=dtype)
    for call in (lambda: on_device.qk_head_norm_rope(x, x, 1e-6),
                 lambda: on_device.qk_head_norm_rope_bwd(x, x, x, x, 1e-6)):
        with pytest.raises(RuntimeError, match="multiple of 8 up to 256"):
            call()


@pytest.mark.parametrize("half,inter,of", [(6, True, 8), (0, True, 8), (4, False, 16), (36, True, 8)])
def test_rotated_sizes_are_refused_whatever_the_layout(on_device, half, inter, of):
    x, c = torch.zeros(2, 5, 3, 64), torch.zeros(5, half)
    for call in (lambda: on_device.qk_head_norm_rope(x, x, 1e-6, cos=c, sin=c, interleaved=inter),
                 lambda: on_device.qk_head_norm_rope_bwd(x, x, x, x, 1e-6, cos=c, sin=c,
                                                         interleaved=inter)):
        with pytest.raises(RuntimeError, match=f"multiple of {of} up to D"):
            call()


@pytest.mark.parametrize("hidden,D", [(100, 100), (12, 12), (256, 96), (4, 4), (256, 0)])
def test_hidden_sizes_are_refused_whatever_the_layout(on_device, hidden, D):
    x = torch.zeros(2, 5, hidden, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="hidden"):
        on_device.qk_norm_rope_bwd(x, x, x, x, D, 1e-6)


@pytest.mark.parametrize("D", [64, 100, 136])
def test_attention_head_sizes_are_refused_whatever_the_layout(on_device, D):
    x = torch.zeros(1, 2, 130, D, dtype=torch.bfloat16)
    mask = torch.ones(1, 2, 2, 2, dtype=torch.bool)
    with pytest.raises(RuntimeError, match="head dim must be 128"):
        on_device.bsattn_bwd(x, x, x, x, x, torch.zeros(1, 2, 130), mask)


def test_views_of_nothing_need_no_copy(on_device, monkeypatch):
    """An empty tensor's strides may be anything, and contiguous() leaves them."""
    from contextlib import nullcontext

    ops = on_device
    launched = []
    monkeypatch.setattr(ops, "_launch", lambda idx, name, fn, *a: launched.append(name))
    monkeypatch.setattr(ops.DeviceStatus, "pointer", classmethod(lambda cls, dev: 0))
    monkeypatch.setattr(ops, "_check_workspace", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: nullcontext())
    bf = torch.bfloat16
    odd = torch.zeros(2, 4, 3, 131, dtype=bf)[:, :0, :, 1:129]
    turned = torch.zeros(0, 256, 2, dtype=bf).permute(0, 2, 1)
    wide = torch.zeros(5, 70)[:0, 2:66]
    ops.qk_head_norm_rope(odd, odd, 1e-6, cos=wide, sin=wide)
    ops.qk_head_norm_rope_bwd(odd, odd, odd, odd, 1e-6, cos=wide, sin=wide)
    ops.qk_norm_rope_bwd(turned, turned, turned, turned, 128, 1e-6)
    none = torch.zeros(1, 2, 4, 133, dtype=bf)[:, :, :0, 3:131]
    ops.bsattn_bwd(none, none, none, none, none, torch.zeros(1, 2, 0),
                   torch.zeros(1, 2, 0, 0, dtype=torch.bool), workspace=torch.zeros(0))
    assert launched == ["sa_qk_head_norm_rope", "sa_qk_head_norm_rope_bwd", "sa_qk_norm_rope_bwd",
                        "sa_bsattn_bwd"]


def test_head_mask_type_of_another_tensor_is_read_anew():
    """Two tensors at one address, as a freed one and the next of its size: the second's entries
    count."""
    import numpy as np

    from sinkattn_b200.reference_api import _hmt_host

    memory = np.array([1, 0, 2], dtype=np.int32)
    t = torch.from_numpy(memory)
    assert _hmt_host(t) == [1, 0, 2]
    memory[:] = [0, -1, 1]
    u = torch.from_numpy(memory)
    assert u.data_ptr() == t.data_ptr() and u._version == t._version
    assert _hmt_host(u) == [0, -1, 1]
    u[0] = 3
    assert _hmt_host(u) == [3, -1, 1]
    assert _hmt_host(u) is _hmt_host(u)  # the same tensor, unchanged, is not copied again


@pytest.mark.parametrize("mode,heads", [("per_head", 2), ("upstream", 2), ("upstream", 3)])
def test_head_mask_type_past_the_mask_is_refused(monkeypatch, mode, heads):
    from sinkattn_b200 import reference_api

    monkeypatch.setattr(reference_api, "HEAD_MASK_TYPE_MODE", mode)
    q = torch.zeros(200, 3, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 200], dtype=torch.int32)
    mask = torch.ones(1, heads, 2, 2, dtype=torch.bool)
    hmt = torch.tensor([1, 0, heads + 1], dtype=torch.int32)
    for grad in (False, True):
        with pytest.raises(ValueError, match=f"head_mask_type names mask slice {heads + 1} of {heads}"):
            reference_api.block_sparse_attn_func(q.requires_grad_(grad), q, q, cu, cu, hmt, None,
                                                 mask, 200, 200)


def test_sink_dynamic_attention_refuses_what_the_kernel_would_read_past(on_device):
    def t(H=3, S=200, dtype=torch.bfloat16):
        return torch.zeros(2, H, S, 128, dtype=dtype)

    mask, hmt = torch.ones(1, 3, 2, 2, dtype=torch.bool), torch.ones(3, dtype=torch.int64)
    ok = dict(q=t(), k=t(), v=t(), block_mask=mask, k_pool=t(S=20), v_pool=t(S=20), sample_gap=4,
              head_mask_type=hmt)
    for match, kw in (("head_mask_type must be", dict(head_mask_type=hmt[:2])),
                      ("block_mask must be", dict(block_mask=mask.float())),
                      ("block_mask must be", dict(block_mask=mask[..., :1])),
                      ("k and v must be", dict(k=t(H=2))), ("k and v must be", dict(v=t(S=199))),
                      ("k_pool / v_pool must be", dict(k_pool=t(H=2, S=20)))):
        with pytest.raises(RuntimeError, match=match):
            on_device.sink_dynamic_attn(**{**ok, **kw})


def test_kernels_that_start_early_promise_nothing_read_only():
    """A kernel of a dependent launch runs while the one before it still writes, so its inputs are
    not read-only for as long as it runs: no read-only loads, and no __restrict__ that allows them
    (a compiler may move either above the wait)."""
    from pathlib import Path

    import sinkattn_b200

    csrc = Path(sinkattn_b200.__file__).parent / "csrc"
    early = [f for f in csrc.glob("*.cu") if "launch_after(" in f.read_text()]
    assert len(early) == 3
    for f in early + [csrc / "norm_rope.cuh"]:
        text = f.read_text()
        assert "__ldg(" not in text and "__restrict__" not in text, f.name


def test_outputs_in_the_place_of_what_is_still_read_are_refused(on_device):
    """Blocks of threads read one another's inputs, so those may not be written over."""
    ops = on_device

    def t(*s):
        return torch.zeros(*s, dtype=torch.bfloat16)

    dout, q, k, v, out = (t(1, 2, 130, 128) for _ in range(5))
    lse, mask, new = torch.zeros(1, 2, 130), torch.ones(1, 2, 2, 2, dtype=torch.bool), t(1, 2, 130, 128)
    for kw in (dict(dq=dout), dict(dq=q), dict(dk=k), dict(dv=v), dict(dk=out), dict(dv=q),
               dict(dq=new, dk=new), dict(dk=new, dv=new)):
        with pytest.raises(RuntimeError, match="bsattn_bwd: d. has the address of"):
            ops.bsattn_bwd(dout, q, k, v, out, lse, mask, **kw)
    q, k, dq, dk, new = (t(2, 5, 3, 128) for _ in range(5))
    for kw in (dict(out_q=k), dict(out_k=q), dict(out_q=new, out_k=new)):
        with pytest.raises(RuntimeError, match="rope: out_. has the address of"):
            ops.qk_head_norm_rope(q, k, 1e-6, **kw)
    for kw in (dict(dq=k), dict(dq=dk), dict(dk=q), dict(dk=dq), dict(dq=new, dk=new)):
        with pytest.raises(RuntimeError, match="rope_bwd: d. has the address of"):
            ops.qk_head_norm_rope_bwd(dq, dk, q, k, 1e-6, **kw)
    q, k, dq, dk, new = (t(2, 5, 384) for _ in range(5))
    for kw in (dict(dq=k), dict(dq=dk), dict(dk=q), dict(dk=dq), dict(dq=new, dk=new)):
        with pytest.raises(RuntimeError, match="rope_bwd: d. has the address of"):
            ops.qk_norm_rope_bwd(dq, dk, q, k, 128, 1e-6, **kw)
