"""What the attention entry points refuse before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from dgl_amd import _lib

FAKE = 4096                                   # never dereferenced: the checks come first


def struct(**kw):
    a = _lib.Attention()
    a.dtype, a.B, a.Hq, a.Hkv, a.Lq, a.Lk, a.D = _lib.DTYPE_F32, 2, 4, 2, 10, 12, 16
    a.scale, a.cap = 0.25, 0.0
    for n, h, l in (("q", 4, 10), ("k", 2, 12), ("v", 2, 12), ("o", 4, 10)):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(h * l * 16, l * 16, 16))
    a.q = a.k = a.v = a.out = a.lse = FAKE
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,word", [
    ({"dtype": 3}, b"type"), ({"B": 0}, b"B=0"), ({"Hq": 5}, b"heads"), ({"D": 12}, b"head size"), ({"D": 136}, b"head size"),
    ({"Lq": -1}, b"Lq=-1"), ({"Lk": (1 << 24) + 1}, b"length"), ({"cap": -1.0}, b"cap"), ({"cap": float("inf")}, b"cap"),
    ({"scale": float("nan")}, b"scale"), ({"pos_q": FAKE}, b"one side"), ({"pos_q": FAKE, "pos_k": FAKE}, b"slope"),
    ({"doc_k": FAKE}, b"one side"), ({"prefix": FAKE}, b"causal"), ({"q": 0}, b"NULL"), ({"v": 0}, b"NULL"),
    ({"k": FAKE + 4}, b"aligned"), ({"q_stride": (ctypes.c_int64 * 3)(640, 160, 18)}, b"aligned"),
    ({"v_stride": (ctypes.c_int64 * 3)(640, -160, 16)}, b"aligned"), ({"B": 1 << 20, "Lq": 1 << 20}, b"rows"),
])
def test_forward_refuses(kw, word):
    lib = _lib.load()
    a = struct(**kw)
    assert lib.dgl_attention_forward(ctypes.byref(a), None) == -1
    assert word in lib.dgl_last_error_string()
    assert lib.dgl_attention_backward_workspace_floats(ctypes.byref(a)) == -1


def test_backward_refuses():
    lib = _lib.load()
    a, g = struct(), _lib.AttentionGrad()
    assert lib.dgl_attention_forward(None, None) == -1
    assert lib.dgl_attention_backward(ctypes.byref(a), None, FAKE, None) == -1
    assert lib.dgl_attention_backward(ctypes.byref(a), ctypes.byref(g), FAKE, None) == -1
    g.dout = g.dq = g.dk = g.dv = FAKE
    assert lib.dgl_attention_backward(ctypes.byref(a), ctypes.byref(g), None, None) == -1
    g.dslope = FAKE
    assert lib.dgl_attention_backward(ctypes.byref(a), ctypes.byref(g), FAKE, None) == -1 and b"slope" in lib.dgl_last_error_string()
    g.dslope, g.dq = None, FAKE + 8
    assert lib.dgl_attention_backward(ctypes.byref(a), ctypes.byref(g), FAKE, None) == -1 and b"aligned" in lib.dgl_last_error_string()


def test_python_refuses_tensors_off_the_gpu_and_bad_shapes():
    from dgl_amd.attention import attention
    x = torch.zeros(1, 2, 4, 16)
    with pytest.raises(ValueError, match="GPU"):
        attention(x, x, x)
    with pytest.raises(ValueError, match="expected"):
        attention(x[0], x, x)
