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
    assert lib.dgl_attention_forward(ctypes.byref(a), None, None) == -1
    assert word in lib.dgl_last_error_string()
    assert lib.dgl_attention_backward_workspace_floats(ctypes.byref(a)) == -1
    assert lib.dgl_attention_forward_workspace_floats(ctypes.byref(a)) == -1


def test_few_rows_against_many_keys_need_a_workspace():
    lib = _lib.load()
    a = struct(Lk=20000)
    assert lib.dgl_attention_forward_workspace_floats(ctypes.byref(a)) > 0
    assert lib.dgl_attention_forward(ctypes.byref(a), None, None) == -1 and b"workspace" in lib.dgl_last_error_string()
    assert lib.dgl_attention_forward(ctypes.byref(a), FAKE + 4, None) == -1
    a = struct(k_stride=(ctypes.c_int64 * 3)(1 << 30, 1 << 29, 1 << 24))
    assert lib.dgl_attention_forward(ctypes.byref(a), None, None) == -1 and b"64 MiB" in lib.dgl_last_error_string()


def test_backward_refuses():
    lib = _lib.load()
    a, g = struct(), _lib.AttentionGrad()
    assert lib.dgl_attention_forward(None, None, None) == -1
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


def step_struct(cache=(), **kw):
    a = _lib.AttentionStep()
    c = a.cache
    c.dtype, c.B, c.Hkv, c.D, c.page_size, c.max_pages, c.num_pages = _lib.DTYPE_F32, 2, 2, 16, 32, 4, 8
    c.k_stride = c.v_stride = (ctypes.c_int64 * 3)(1024, 512, 16)
    c.table_stride = 4
    c.k_pages = c.v_pages = c.table = c.lengths = FAKE
    a.rows_per_instance, a.Hq, a.scale = 3, 4, 0.25
    a.q_stride = a.o_stride = (ctypes.c_int64 * 2)(64, 16)
    a.q = a.out = FAKE
    for n, v in dict(cache).items():
        setattr(c, n, v)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("cache,kw,word", [
    ({"page_size": 8}, {}, b"page size"), ({"page_size": 48}, {}, b"page size"), ({"num_pages": 0}, {}, b"pages"),
    ({"max_pages": 1 << 26}, {}, b"pages"), ({"D": 20}, {}, b"head size"), ({"table": 0}, {}, b"NULL"),
    ({"k_pages": FAKE + 8}, {}, b"aligned"), ({"v_stride": (ctypes.c_int64 * 3)(1024, 512, 18)}, {}, b"aligned"),
    ({"B": 0}, {}, b"B=0"), ({"dtype": -1}, {}, b"type"), ({}, {"Hq": 3}, b"heads"), ({}, {"rows_per_instance": 0}, b"rows"),
    ({}, {"cap": -2.0}, b"cap"), ({}, {"q": 0}, b"NULL"), ({}, {"out": FAKE + 4}, b"aligned"),
    ({}, {"pos_q": FAKE, "pos_k": FAKE, "pos_rows": 9}, b"slope"), ({}, {"pos_q": FAKE}, b"one side"),
    ({}, {"pos_q": FAKE, "pos_k": FAKE, "slope": FAKE, "pos_rows": 0}, b"rows"),
    ({}, {"pos_q": FAKE, "pos_k": FAKE + 4, "slope": FAKE, "pos_rows": 9}, b"8-byte"),
    ({}, {"blocked": FAKE, "words": -1}, b"words"), ({}, {"rows_per_instance": 1 << 28}, b"many"),
])
def test_step_refuses(cache, kw, word):
    lib = _lib.load()
    a = step_struct(cache, **kw)
    assert lib.dgl_attention_step(ctypes.byref(a), None, None) == -1
    assert word in lib.dgl_last_error_string()
    assert lib.dgl_attention_step_workspace_floats(ctypes.byref(a)) == -1


def test_long_caches_need_their_workspace_and_appends_are_checked():
    lib = _lib.load()
    assert lib.dgl_attention_step(None, None, None) == -1
    a = step_struct({"max_pages": 1 << 14})
    assert lib.dgl_attention_step_workspace_floats(ctypes.byref(a)) > 0
    assert lib.dgl_attention_step(ctypes.byref(a), None, None) == -1 and b"workspace" in lib.dgl_last_error_string()
    s = (ctypes.c_int64 * 3)(32, 16, 16)
    bad = (ctypes.c_int64 * 3)(32, 16, 17)
    c = ctypes.byref(a.cache)
    assert lib.dgl_cache_append(None, FAKE, FAKE, s, s, 1, FAKE, None, None, None) == -1
    assert lib.dgl_cache_append(c, FAKE, FAKE, s, s, -1, FAKE, None, None, None) == -1
    assert lib.dgl_cache_append(c, FAKE, FAKE, s, bad, 1, FAKE, None, None, None) == -1
    assert lib.dgl_cache_append(c, FAKE, FAKE, s, s, 1, None, None, None, None) == -1
    assert lib.dgl_cache_append(c, None, FAKE, s, s, 1, FAKE, None, None, None) == -1


@pytest.mark.parametrize("kw,word", [
    ({"dtype": 7}, b"type"), ({"A": 0}, b"A=0"), ({"R": -1}, b"R=-1"), ({"logits": 0}, b"NULL"), ({"log_probs": 0}, b"NULL"),
    ({"out_stride": 9}, b"overlap"), ({"temperature": 0.0}, b"temperature"), ({"blocked": FAKE, "period": 3}, b"bits"),
    ({"blocked": FAKE, "period": 0}, b"bits"), ({"history": FAKE, "repetition_all": 0.0}, b"repetition"),
    ({"logits_stride": -10}, b"stride"), ({"A": 40000, "out_stride": 40000}, b"workspace"),
])
def test_logits_refuse(kw, word):
    lib = _lib.load()
    a = _lib.Logits()
    a.R, a.A, a.period, a.logits, a.logits_stride, a.temperature, a.log_probs, a.out_stride = 2, 10, 10, FAKE, 10, 1.0, FAKE, 10
    a.repetition_all = 1.0
    for n, v in kw.items():
        setattr(a, n, v)
    assert lib.dgl_logits_process(ctypes.byref(a), None, None) == -1
    assert word in lib.dgl_last_error_string()
