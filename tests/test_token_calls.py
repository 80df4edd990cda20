"""The 4-bit products', the logit rules' and the sampler's argument checks (host only)."""
from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 0x1000
STREAM = type("S", (), {"cuda_stream": 0})()


def q4(ie, rows=16, cols=64, group=32, dtype=1, data=FAKE, scale=FAKE, zero=None):
    return ie.MatrixQ4(data, scale, zero, dtype, group, rows, cols)


def test_structures_are_the_header_s(ie):
    assert ctypes.sizeof(ie.MatrixQ4) == 40 and ctypes.sizeof(ie.LogitRules) == 128


def test_product_checks(ie):
    L = ie.lib()
    ok = q4(ie)
    mm = lambda w, x=FAKE, y=FAKE, T=1, ws=FAKE: L.ie_hip_matmul_q4(y, x, w, None, T, 0, ws, None)
    assert mm(ok, T=0) == ie.OK
    for bad, word in ((q4(ie, group=48), "32, 64 or 128"), (q4(ie, cols=40), "multiple of 32"),
                      (q4(ie, rows=0), "empty"), (q4(ie, data=None), "empty"), (q4(ie, scale=None), "empty"),
                      (q4(ie, dtype=3), "scale_dtype"), (q4(ie, data=FAKE + 8), "16-byte"),
                      (q4(ie, scale=FAKE + 1), "aligned to their type"),
                      (q4(ie, dtype=0, scale=FAKE + 2), "aligned to their type")):
        assert mm(bad) == ie.EINVAL and word in ie.last_error()
    assert mm(ok, T=-1) == ie.EINVAL
    assert mm(ok, x=None) == ie.EINVAL and mm(ok, y=None) == ie.EINVAL
    assert mm(ok, x=FAKE + 4) == ie.EINVAL and "x must be 16-byte" in ie.last_error()
    many = 100000
    if L.ie_hip_matmul_q4_workspace_bytes(many, 64):
        assert mm(ok, T=many, ws=None) == ie.EINVAL and "workspace" in ie.last_error()
        assert mm(ok, T=many, ws=FAKE + 4) == ie.EINVAL and "workspace" in ie.last_error()
    qkv = lambda w, q, kv: L.ie_hip_qkv_proj_q4(FAKE, FAKE, FAKE, FAKE, w, None, 1, q, kv, FAKE, None)
    for q, kv in ((8, 8), (16, 0), (0, 8), (16, 1 << 30), (-(1 << 31), 1 << 30)):
        assert qkv(ok, q, kv) == ie.EINVAL and "q_dim" in ie.last_error()
    assert L.ie_hip_qkv_proj_q4(FAKE, None, FAKE, FAKE, ok, None, 1, 8, 4, FAKE, None) == ie.EINVAL
    gate = lambda a, b: L.ie_hip_gate_up_silu_q4(FAKE, FAKE, a, b, 1, FAKE, None)
    for other in (q4(ie, rows=32), q4(ie, cols=96), q4(ie, group=64), q4(ie, dtype=2)):
        assert gate(ok, other) == ie.EINVAL and "differ" in ie.last_error()
    assert L.ie_hip_matmul_q4_workspace_bytes(0, 64) == L.ie_hip_matmul_q4_workspace_bytes(-5, 64) == 0
    assert L.ie_hip_matmul_q4_workspace_bytes(5, 0) == 0


def test_rules_checks(ie):
    L = ie.lib()
    adj = lambda n=8, R=1, out=FAKE, l=FAKE, **f: L.ie_hip_adjust_logits(out, l, ie.LogitRules(**f), R, n, None)
    assert adj(R=0) == ie.OK
    assert adj(n=0) == ie.EINVAL and adj(R=-1) == ie.EINVAL
    assert adj(out=None) == ie.EINVAL and adj(l=None) == ie.EINVAL
    assert adj(history=FAKE) == ie.EINVAL
    assert adj(history=FAKE, history_start=FAKE, history_len=FAKE, history_size=-1) == ie.EINVAL
    for name in ("repetition", "presence", "frequency", "prompt_len"):
        assert adj(**{name: FAKE}) == ie.EINVAL and "history" in ie.last_error()
    assert adj(bias_token=FAKE) == ie.EINVAL and adj(bias_value=FAKE) == ie.EINVAL
    assert adj(bias_token=FAKE, bias_value=FAKE, bias_start=FAKE) == ie.EINVAL
    assert adj(mask_row=FAKE) == ie.EINVAL and adj(mask=FAKE, mask_rows=-1) == ie.EINVAL
    assert adj(n=2 ** 31 - 1, R=2 ** 31 - 1) == ie.EINVAL and "too many" in ie.last_error()


def test_sample_checks(ie):
    L = ie.lib()
    call = lambda out=FAKE, l=FAKE, t=FAKE, u=FAKE, R=1, n=8, ws=FAKE: L.ie_hip_sample_rows(
        out, l, t, None, None, None, u, R, n, ws, None)
    assert call(R=0) == ie.OK
    assert call(R=-1) == ie.EINVAL and call(n=0) == ie.EINVAL
    for name in ("out", "l", "t", "u"):
        assert call(**{name: None}) == ie.EINVAL and "null" in ie.last_error()
    if L.ie_hip_sample_rows_workspace_bytes(1, 8):
        assert call(ws=None) == ie.EINVAL and "workspace" in ie.last_error()
        assert call(ws=FAKE + 4) == ie.EINVAL and "workspace" in ie.last_error()
    assert L.ie_hip_sample_rows_workspace_bytes(0, 8) == L.ie_hip_sample_rows_workspace_bytes(1, 0) == 0


def test_python_refuses_other_tensors(ie):
    """Tensors of the host, of other types, shapes and strides, before anything is launched."""
    z = torch.zeros
    with pytest.raises(ie.IeHipError, match="contiguous uint8"):
        ie.matrix_q4(z(4, 16, dtype=torch.int8), z(4, 1), 32)
    with pytest.raises(ie.IeHipError, match="contiguous uint8"):
        ie.matrix_q4(z(16, 4, dtype=torch.uint8).t(), z(4, 1), 32)
    u8 = z(4, 32, dtype=torch.uint8)
    with pytest.raises(ie.IeHipError, match="32, 64 or 128"):
        ie.matrix_q4(u8, z(4, 2), 16)
    with pytest.raises(ie.IeHipError, match="shape"):
        ie.matrix_q4(u8, z(4, 1), 32)
    with pytest.raises(ie.IeHipError, match="scales of"):
        ie.matrix_q4(u8, z(4, 2, dtype=torch.float64), 32)
    with pytest.raises(ie.IeHipError, match="zero"):
        ie.matrix_q4(u8, z(4, 2), 32, zero=z(4, 2))
    w = ie.matrix_q4(u8, z(4, 2), 32)
    assert (w.rows, w.cols, w.group, w.scale_dtype) == (4, 64, 32, ie.KV_F32)
    with pytest.raises(ie.IeHipError, match="current GPU"):
        ie.matmul_q4(z(1, 4), z(1, 64), w, stream=STREAM)
    with pytest.raises(ie.IeHipError, match="current GPU"):  # a structure of the caller's own
        ie.matmul_q4(z(1, 4), z(1, 64), q4(ie, rows=4), stream=STREAM)
    with pytest.raises(ie.IeHipError, match="float32"):
        ie.matmul_q4(z(1, 4), z(1, 64, dtype=torch.float16), w, stream=STREAM)
    with pytest.raises(ie.IeHipError, match="contiguous"):
        ie.gate_up_silu_q4(z(2, 4), z(64, 2).t(), w, w, stream=STREAM)
    with pytest.raises(ie.IeHipError, match="current GPU"):
        ie.adjust_logits(z(1, 4), z(1, 4), ie.logit_rules(), stream=STREAM)
    with pytest.raises(ie.IeHipError, match="current GPU"):
        ie.sample_rows(z(1, dtype=torch.int32), z(1, 4), z(1), z(1), stream=STREAM)
    with pytest.raises(ie.IeHipError, match="history"):
        ie.logit_rules(presence=z(2))
    i = lambda *s: z(*s, dtype=torch.int32)
    with pytest.raises(ie.IeHipError, match="shape"):
        ie.logit_rules(history=(i(5), i(2), i(3)))
    with pytest.raises(ie.IeHipError, match="int32"):
        ie.logit_rules(history=(z(5), i(2), i(2)))
    with pytest.raises(ie.IeHipError, match="as many"):
        ie.logit_rules(bias=(i(5), z(4), i(2), i(2)))
    with pytest.raises(ie.IeHipError, match="without a mask"):
        ie.logit_rules(mask_row=i(2))


def test_native_calls_take_their_own_structure(ie):
    calls, z = ie._native(), torch.zeros
    m = ie.matrix(z(16, 32, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="MatrixQ4"):
        calls.ie_hip_matmul_q4(z(1, 16), z(1, 32), m, None, 0, 0, None, 0)
    with pytest.raises(TypeError, match="LogitRules"):
        calls.ie_hip_adjust_logits(z(1, 8), z(1, 8), m, 0, 8, 0)
    with pytest.raises(TypeError, match="Matrix"):
        calls.ie_hip_matmul(z(1, 16), z(1, 64), q4(ie), None, 0, 0, 0)


def test_fits(ie):
    fits, z = ie._native().fits, torch.zeros
    assert fits(z(2, 3), 6, 3, -1) and fits(z(0, 3), 0, 3, -1)
    for t, n, last, dev in ((z(2, 3), 6, 2, -1), (z(2, 3), 5, 3, -1), (z(2, 3), 6, 3, 0), (z(()), 1, 1, -1),
                            (z(2, 3, dtype=torch.float64), 6, 3, -1), (z(3, 2).t(), 6, 3, -1)):
        assert not fits(t, n, last, dev)
    with pytest.raises(AttributeError):
        fits(5, 1, 1, 0)
    with pytest.raises(TypeError):
        fits(z(1), 1, 1)
