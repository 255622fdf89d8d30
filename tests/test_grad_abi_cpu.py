"""What the gradient and per-head norm entry points refuse, on the host and
before any CUDA call, and what their Python forms refuse."""
from __future__ import annotations

import ctypes

import pytest
import torch


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _bwd(lib, *, D=128, B=1, H=2, Sq=256, Sk=128, Hm=2, ptr=256, ws=256, ws_bytes=1 << 40,
         st=None, hmt=None, lse=256, dq=256):
    s = st or _i64(H * 512 * 128, 512 * 128, 128, 1)
    m = _i64(0, 1, 1, 1)
    return lib.sa_bsattn_bwd(ptr, ptr, ptr, ptr, ptr, s, s, s, s, s, lse, None, B, H, Sq, Sk, D,
                             ptr, m, Hm, hmt, -1.0, dq, ptr, ptr, s, s, s, ws, ws_bytes, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(D=64), "head dim must be 128"),
    (dict(Sq=0), ">= 1"),
    (dict(Sk=131073), "at most 131072"),
    (dict(B=65536), "too many heads"),
    (dict(Hm=1), "head_mask_type"),
    (dict(ptr=None), "null"),
    (dict(lse=None), "null"),
    (dict(ptr=264), "16-byte aligned"),
    (dict(dq=8), "16-byte aligned"),
    (dict(st=_i64(1 << 20, 1 << 16, 132, 1)), "multiple of 8"),
    (dict(st=_i64(1 << 20, 1 << 16, 128, 2)), "stride(dim)=1"),
    (dict(st=_i64(1 << 20, -128, 128, 1)), "multiple of 8"),
    (dict(ws=None), "workspace"),
    (dict(ws_bytes=255), "workspace"),
    (dict(ws=264), "256-byte aligned"),
])
def test_attention_backward_refuses(lib, kw, text):
    from sinkattn_b200 import _lib

    assert _bwd(lib, **kw) == _lib.SA_EINVAL
    assert text in _lib.last_error(), _lib.last_error()


def test_attention_backward_workspace(lib):
    size = lib.sa_bsattn_bwd_workspace_size
    assert size(0, 1, 1, 1) == 0 and size(1, 1, 0, 1) == 0 and size(1, 1, 131073, 1) == 0
    # many tiles: the counter and two fp32 statistics of every padded query row
    assert size(2, 12, 32760, 32760) == 256 + 2 * 4 * 24 * 32768
    # few long tiles may be cut: room for their pieces' sums, 2 per SM at most
    assert size(1, 1, 4096, 4096) > 256 + 2 * 4 * 4096 + 32 * 2 * 3 * 128 * 128 * 4
    assert size(1, 1, 131072, 131072) < 2 * 4 * 131072 + 256 * 2 * 3 * 128 * 128 * 4 + (1 << 20)


def _head(lib, *, B=1, S=4, Hq=4, Hk=2, D=128, dtype=0, wq=None, wk=None, wd=0, cos=256, sin=256,
          fs=64, rows=16, rot=128, inter=1, pos=None, pst=None, q=256, k=256, qs=None, out=256):
    s = qs or _i64(4 * Hq * D, Hq * D, D, 1)
    return lib.sa_qk_head_norm_rope(q, k, s, s, B, S, Hq, Hk, D, dtype, wq, wk, wd, 1e-6, cos, sin,
                                    fs, rows, rot, inter, pos, 1, pst, out, out, s, s, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(D=100), "multiple of 8 up to 256"),
    (dict(D=264), "multiple of 8 up to 256"),
    (dict(Hq=0), "bad sizes"),
    (dict(Hq=8192), "too many"),
    (dict(dtype=3), "dtype"),
    (dict(wq=256), "weights go together"),
    (dict(wq=8, wk=256), "16-byte aligned"),
    (dict(sin=None), "go together"),
    (dict(rot=12), "multiple of 8"),
    (dict(rot=24, inter=0), "multiple of 16"),
    (dict(rot=256), "up to D"),
    (dict(fs=60), "stride"),
    (dict(fs=66), "stride"),
    (dict(cos=8), "16-byte aligned"),
    (dict(rows=3), "3 table rows for 4 tokens"),
    (dict(rows=0, pos=256, pst=_i64(1, 1)), "table rows"),
    (dict(pos=256), "positions need"),
    (dict(cos=None, sin=None, pos=256, pst=_i64(1, 1)), "positions need"),
    (dict(q=None), "null"),
    (dict(out=None), "null"),
    (dict(q=8), "16-byte aligned"),
    (dict(qs=_i64(512, 512, 100, 1)), "16-byte aligned"),
    (dict(qs=_i64(512, 512, 128, 2)), "stride(dim)=1"),
    (dict(qs=_i64(512, 512, 1 << 31, 1)), "strides"),
])
def test_head_norm_refuses(lib, kw, text):
    from sinkattn_b200 import _lib

    assert _head(lib, **kw) == _lib.SA_EINVAL
    assert text in _lib.last_error(), _lib.last_error()


def test_head_norm_of_nothing_needs_no_device(lib):
    from sinkattn_b200 import _lib

    assert _head(lib, B=0, q=None, k=None, out=None) == _lib.SA_OK
    assert _head(lib, S=0, rows=1, q=None, k=None, out=None) == _lib.SA_OK


def test_gradient_workspaces_and_weights(lib):
    from sinkattn_b200 import _lib

    s = _i64(2048, 512, 128, 1)

    def head(dwq, dwk, wq=256, ws=256, n=1 << 40):
        return lib.sa_qk_head_norm_rope_bwd(256, 256, s, s, 256, 256, s, s, 1, 4, 4, 4, 128, 0, wq,
                                            wq, 0, 1e-6, None, None, 0, 0, 0, 1, None, 0, None,
                                            256, 256, s, s, dwq, dwk, ws, n, None, None)

    assert head(256, None) == _lib.SA_EINVAL and "go together" in _lib.last_error()
    assert head(256, 256, wq=None) == _lib.SA_EINVAL and "need weights" in _lib.last_error()
    assert head(256, 256, n=16) == _lib.SA_EINVAL and "workspace" in _lib.last_error()
    assert head(256, 256, ws=None) == _lib.SA_EINVAL and "workspace" in _lib.last_error()

    def hidden(n=1536, D=128, w=256, dw=256, ws=256, size=1 << 40, stride=1536, q=256, cos=None):
        return lib.sa_qk_norm_rope_bwd(256, 256, stride, stride, q, 256, stride, stride, 8, 8, n, D,
                                       w, w, 1, 1e-6, cos, None, 64, 256, 256, stride, stride, dw,
                                       dw, ws, size, None, None)

    for kw, text in ((dict(n=4104, D=8), "at most 4096"), (dict(n=1540), "multiple"),
                     (dict(D=100), "multiple of 8"), (dict(w=None), "need weights"),
                     (dict(size=64), "workspace"), (dict(stride=1540), "multiples of 8"),
                     (dict(q=8), "16-byte"), (dict(q=None), "null"), (dict(cos=256), "go together")):
        assert hidden(**kw) == _lib.SA_EINVAL
        assert text in _lib.last_error(), _lib.last_error()
    assert lib.sa_qk_norm_rope_bwd_workspace_size(4) == 0
    assert lib.sa_qk_norm_rope_bwd_workspace_size(4104) == 0
    assert lib.sa_qk_head_norm_rope_bwd_workspace_size(4) == 0


def test_python_forms_refuse_cpu_tensors():
    from sinkattn_b200 import ops

    x = torch.zeros(1, 2, 128, 128, dtype=torch.bfloat16)
    m = torch.ones(1, 2, 1, 1, dtype=torch.bool)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.bsattn_bwd(x, x, x, x, x, torch.zeros(1, 2, 128), m)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.qk_head_norm_rope(x, x, 1e-6)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.qk_head_norm_rope_bwd(x, x, x, x, 1e-6)
    y = torch.zeros(1, 4, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.qk_norm_rope_bwd(y, y, y, y, 128, 1e-6)


def test_bad_index_status_is_told_from_a_timeout(lib):
    from sinkattn_b200 import _lib

    word = ctypes.c_int32(_lib.SA_DEV_BAD_INDEX)
    assert lib.sa_check_status(ctypes.addressof(word)) == _lib.SA_EINVAL
    assert "outside the rotary" in _lib.last_error() and word.value == 0
    word.value = _lib.SA_DEV_WAIT_TIMEOUT
    assert lib.sa_check_status(ctypes.addressof(word)) == _lib.SA_ETIMEOUT and word.value == 0
    assert lib.sa_check_status(ctypes.addressof(word)) == _lib.SA_OK


def test_build_without_the_extension_warns_and_leaves_no_stale_one(monkeypatch, tmp_path):
    from sinkattn_b200 import build

    stale = tmp_path / "_fast.so"
    stale.write_bytes(b"")

    def fail(*args):
        raise RuntimeError("no headers")

    monkeypatch.setattr(build, "FAST", stale)
    monkeypatch.setattr(build, "build_fast", fail)
    with pytest.warns(UserWarning, match="no headers"):
        assert build.build() == build.LIB
    assert not stale.exists()
