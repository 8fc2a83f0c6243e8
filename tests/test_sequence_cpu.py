"""The sequence operators without a GPU: schemas, Meta kernels, refusals of the
C ABI (before any device work) and the structs ctypes passes to it."""
import ctypes
import os
import re

import pytest
import torch

import pla_b200 as P
from pla_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED, TOO_LARGE = 1, 2, 3
BASE = 1 << 20  # never dereferenced: the checks return first


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_meta_kernels_give_shapes_and_dtypes():
    y, s = P.causal_depthwise(meta(2, 9, 24), meta(24, 4), return_state=True)
    assert y.shape == (2, 9, 24) and s.shape == (2, 3, 24) and s.dtype == torch.bfloat16
    cu = meta(6, dtype=torch.int32)
    assert P.causal_depthwise(meta(1, 9, 24), meta(24, 1, 3), cu_seqlens=cu, return_state=True)[1].shape == (5, 2, 24)
    assert P.causal_depthwise_step(meta(3, 24), meta(3, 3, 24), meta(24, 4)).shape == (3, 24)
    q, k = P.qk_norm_rotate(meta(2, 9, 4, 64), meta(2, 9, 2, 64), norm="l2")
    assert q.shape == (2, 9, 4, 64) and k.shape == (2, 9, 2, 64)
    g = meta(2, 9, 4, dtype=torch.float32)
    o, s = P.gated_delta_rule(meta(2, 9, 2, 64), meta(2, 9, 2, 64), meta(2, 9, 4, 32), g, g, return_state=True)
    assert o.shape == (2, 9, 4, 32) and s.shape == (2, 4, 64, 32) and s.dtype == torch.float32
    o = P.gated_delta_rule_step(meta(3, 2, 64), meta(3, 2, 64), meta(3, 4, 32), g[0, :3], g[0, :3],
                                meta(3, 4, 64, 32, dtype=torch.float32))
    assert o.shape == (3, 4, 32)


def test_meta_gradients_have_their_inputs_shapes():
    args = [meta(1, 9, 2, 64).requires_grad_(), meta(1, 9, 2, 64).requires_grad_(), meta(1, 9, 4, 32).requires_grad_(),
            meta(1, 9, 4).requires_grad_(), meta(1, 9, 4).requires_grad_()]
    grads = torch.autograd.grad(P.gated_delta_rule(*args).sum(), args)
    assert [g.shape for g in grads] == [a.shape for a in args]


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    q, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    for call in (lambda: P.causal_depthwise(x, w), lambda: P.causal_depthwise_step(x[0], torch.zeros(4, 3, 8), w),
                 lambda: P.qk_norm_rotate(q, q), lambda: P.gated_delta_rule(q, q, q, g, g),
                 lambda: P.gated_delta_rule_step(q[0], q[0], q[0], g[0], g[0], torch.zeros(4, 2, 8, 8)),
                 lambda: P.causal_depthwise(None, w)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        _lib.ops().gated_delta_rule(q, q, q, g, g, 1.0, None, None, False)


def test_structs_follow_the_header():
    """Field names and order of the ctypes structs are the header's."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "pla_b200.h")).read(), flags=re.S)
    for cls in (_lib.Causal, _lib.CausalGradient, _lib.NormSide, _lib.QkNorm, _lib.Delta, _lib.DeltaGradient, _lib.DeltaStep):
        name = {"Causal": "pla_causal", "CausalGradient": "pla_causal_gradient", "NormSide": "pla_norm_side", "QkNorm": "pla_qk_norm",
                "Delta": "pla_delta", "DeltaGradient": "pla_delta_gradient", "DeltaStep": "pla_delta_step"}[cls.__name__]
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        fields = [re.sub(r"[*\s]", "", re.split(r"\s", part.strip())[-1])
                  for line in body.split(";") for part in line.split(",") if part.strip()]
        assert fields == [f[0] for f in cls._fields_], name


def causal(**kw):
    a = _lib.Causal(x=BASE, x_batch=8 * 16, x_token=16, w=BASE + (1 << 18), y=BASE + (1 << 17), batch=1, tokens=8, channels=16,
                    taps=4, sequences=1, silu=1, dtype=_lib.PLA_BF16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_causal_refusals():
    L = _lib.lib()
    f = lambda a: L.pla_causal_depthwise_forward(ctypes.byref(a), None)  # noqa: E731
    assert L.pla_causal_depthwise_forward(None, None) == INVALID
    for kw in (dict(batch=-1), dict(tokens=-1), dict(channels=-2), dict(sequences=2), dict(x=None), dict(w=None), dict(y=None),
               dict(y=BASE + 32), dict(cu_seqlens=BASE, batch=2), dict(state_in=BASE + (1 << 19), state_out=BASE + (1 << 19) + 32),
               dict(state_out=BASE + 16), dict(state_out=BASE + (1 << 17))):
        assert f(causal(**kw)) == INVALID, kw
    for kw in (dict(taps=1), dict(taps=5), dict(dtype=_lib.PLA_F64), dict(dtype=9)):
        assert f(causal(**kw)) == UNSUPPORTED, kw
    assert f(causal(tokens=(1 << 30) + 1)) == TOO_LARGE
    assert f(causal(channels=0)) == 0 and f(causal(tokens=0)) == 0 and f(causal(batch=0, sequences=0)) == 0
    g = _lib.CausalGradient(dy=BASE + (1 << 16), dy_batch=128, dy_token=16, dx=BASE + (1 << 15), dw=BASE + (1 << 14))
    assert L.pla_causal_depthwise_backward(ctypes.byref(causal()), ctypes.byref(g), None) == INVALID  # no workspace
    g.dw, g.dx = None, BASE + 16
    assert L.pla_causal_depthwise_backward(ctypes.byref(causal()), ctypes.byref(g), None) == INVALID  # dx inside x
    assert L.pla_causal_depthwise_workspace(ctypes.byref(causal())) > 0
    step = lambda **kw: L.pla_causal_depthwise_step(*{**dict(  # noqa: E731
        x=BASE, x_row=16, s=BASE + 4096, s_row=48, w=BASE + 8192, b=None, y=BASE + 16384, n=4, c=16, taps=4, silu=0,
        dtype=_lib.PLA_F32, stream=None), **kw}.values())
    for kw in (dict(n=-1), dict(x=None), dict(s=None), dict(y=None), dict(s_row=47), dict(y=BASE), dict(y=BASE + 4096), dict(s=BASE)):
        assert step(**kw) == INVALID, kw
    assert step(taps=7) == UNSUPPORTED and step(dtype=_lib.PLA_F64) == UNSUPPORTED and step(n=0) == 0


def norm(**kw):
    side = lambda at, heads: _lib.NormSide(x=at, x_batch=8 * heads * 32, x_token=heads * 32, x_head=32, y=at + (1 << 18),  # noqa: E731
                                           heads=heads)
    a = _lib.QkNorm(q=side(BASE, 4), k=side(BASE + (1 << 16), 2), batch=1, tokens=8, dim=32, rot=0, eps=1e-6, dtype=_lib.PLA_F32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_norm_refusals():
    L = _lib.lib()
    f = lambda a: L.pla_qk_norm_rotate_forward(ctypes.byref(a), None)  # noqa: E731
    assert L.pla_qk_norm_rotate_forward(None, None) == INVALID
    for kw in (dict(batch=-1), dict(rot=3), dict(rot=34), dict(rot=8), dict(eps=-1.0), dict(eps=float("nan")), dict(table_rows=-1),
               dict(rot=8, cos_table=BASE, sin_table=BASE, positions=BASE, position_bytes=2)):
        assert f(norm(**kw)) == INVALID, kw
    for kw in (dict(dim=257), dict(dtype=_lib.PLA_F64)):
        assert f(norm(**kw)) == UNSUPPORTED, kw
    a = norm()
    a.k.y = BASE + 64  # inside q
    assert f(a) == INVALID
    assert f(norm(tokens=0)) == 0
    assert f(norm(tokens=(1 << 30) + 1)) == TOO_LARGE
    a = norm()
    a.q.dy = a.k.dy = BASE + (1 << 20)
    a.q.dw = BASE  # a gradient of a weight that is not there
    assert L.pla_qk_norm_rotate_backward(ctypes.byref(a), None, 0, None) == INVALID
    a.q.w = BASE + (1 << 21)
    assert L.pla_qk_norm_rotate_backward(ctypes.byref(a), None, 0, None) == INVALID  # no workspace


def delta(**kw):
    a = _lib.Delta(q=BASE, k=BASE + (1 << 16), v=BASE + (2 << 16), g=BASE + (3 << 16), beta=BASE + (4 << 16), o=BASE + (5 << 16),
                   batch=1, tokens=8, sequences=1, hk=2, hv=4, dk=32, dv=32, dtype=_lib.PLA_BF16, scale=1.0)
    for n, heads in (("q", 2), ("k", 2), ("v", 4)):
        setattr(a, n + "_batch", 8 * heads * 32), setattr(a, n + "_token", heads * 32), setattr(a, n + "_head", 32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_delta_refusals():
    L = _lib.lib()
    f = lambda a: L.pla_gated_delta_rule_forward(ctypes.byref(a), None)  # noqa: E731
    assert L.pla_gated_delta_rule_forward(None, None) == INVALID
    for kw in (dict(batch=-1), dict(sequences=2), dict(hk=0), dict(hk=3), dict(q=None), dict(g=None), dict(o=None), dict(o=BASE + 64),
               dict(state_in=BASE + (6 << 16), state_out=BASE + (6 << 16)), dict(state_out=BASE + (5 << 16)),
               dict(cu_seqlens=BASE, batch=2)):
        assert f(delta(**kw)) == INVALID, kw
    for kw in (dict(dk=129), dict(dk=0), dict(dv=129), dict(dtype=_lib.PLA_F64)):
        assert f(delta(**kw)) == UNSUPPORTED, kw
    assert f(delta(tokens=(1 << 30) + 1)) == TOO_LARGE
    assert L.pla_gated_delta_rule_backward(ctypes.byref(delta()), None, None) == INVALID
    assert L.pla_gated_delta_rule_backward(ctypes.byref(delta()), ctypes.byref(_lib.DeltaGradient()), None) == INVALID
    size = lambda back, **kw: L.pla_gated_delta_rule_workspace(ctypes.byref(delta(**kw)), back)  # noqa: E731
    assert 0 < size(0) < size(1) and size(0, dk=129) == 0
    # a ragged batch may split into one more chunk per sequence
    assert size(0, cu_seqlens=BASE, sequences=7) > size(0)
    s = _lib.DeltaStep(q=BASE, k=BASE + 4096, v=BASE + 8192, g=BASE + 12288, beta=BASE + 12800, state=BASE + (1 << 16),
                       state_row=2 * 32 * 32, o=BASE + (1 << 20), n=2, hk=1, hv=2, dk=32, dv=32, dtype=_lib.PLA_F32, scale=1.0)
    g = lambda **kw: [setattr(s, k, v) for k, v in kw.items()] and L.pla_gated_delta_rule_step(ctypes.byref(s), None)  # noqa: E731
    assert g(n=-1) == INVALID and g(n=2, hk=0) == INVALID and g(hk=1, dk=257) == UNSUPPORTED and g(dk=32, state_row=2047) == INVALID
    assert g(state_row=2048, o=BASE + (1 << 16)) == INVALID and g(o=BASE + (1 << 20), state=None) == INVALID
    assert g(state=BASE + (1 << 16), n=0) == 0


def test_mixer_module_interface():
    m = P.DeltaMixer(32, 2, head_dim=16, value_heads=4, value_dim=8)
    assert set(m.state_dict()) == {"in_proj.weight", "gate_proj.weight", "conv.weight", "conv.bias", "A_log", "dt_bias",
                                   "out_proj.weight"}
    assert m.in_proj.weight.shape == (2 * 32 + 32, 32) and m.conv.weight.shape == (96, 1, 4)
    conv, delta_state = m.new_state(5)
    assert conv.shape == (5, 3, 96) and delta_state.shape == (5, 4, 16, 8) and delta_state.dtype == torch.float32
    with pytest.raises(ValueError):
        P.DeltaMixer(32, 3, value_heads=4)
    with pytest.raises(ValueError):
        m(torch.zeros(1, 4, 32))
