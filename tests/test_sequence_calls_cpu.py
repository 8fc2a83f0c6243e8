"""The sequence operators without a GPU: tangents and states that are refused,
the fault word, and what the kernels' sources have to keep."""
import glob
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import pla_b200 as P
from pla_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def operators():
    """name, call, its differentiable arguments."""
    g, g1 = meta(1, 9, 4), meta(3, 4)
    f32 = torch.float32
    return [
        ("causal_depthwise", lambda x, w, b, s: P.causal_depthwise(x, w, b, state=s),
         [meta(2, 9, 24), meta(24, 4), meta(24), meta(2, 3, 24)]),
        ("causal_depthwise_step", lambda x, w, b, s: P.causal_depthwise_step(x, s, w, b),
         [meta(3, 24), meta(24, 4), meta(24), meta(3, 3, 24)]),
        ("qk_norm_rotate", lambda q, k, wq, wk, c, s: P.qk_norm_rotate(q, k, wq, wk, cos=c, sin=s),
         [meta(1, 9, 4, 64), meta(1, 9, 2, 64), meta(64), meta(64), meta(9, 16, dtype=f32), meta(9, 16, dtype=f32)]),
        ("gated_delta_rule", lambda q, k, v, g, b, s: P.gated_delta_rule(q, k, v, g, b, state=s),
         [meta(1, 9, 2, 64), meta(1, 9, 2, 64), meta(1, 9, 4, 32), g, g.clone(), meta(1, 4, 64, 32, dtype=f32)]),
        ("gated_delta_rule_step", lambda q, k, v, g, b, s: P.gated_delta_rule_step(q, k, v, g, b, s),
         [meta(3, 2, 64), meta(3, 2, 64), meta(3, 4, 32), g1, g1.clone(), meta(3, 4, 64, 32, dtype=f32)]),
    ]


# ---- forward-mode derivatives ----------------------------------------------
@pytest.mark.parametrize("name,call,args", operators(), ids=lambda v: v if isinstance(v, str) else "")
def test_forward_mode_derivatives_raise(name, call, args):
    """There is no forward-mode formula: a tangent is refused, not dropped."""
    call(*args)
    for i in range(len(args)):
        for needs_grad in (False, True):
            with forward_ad.dual_level(), pytest.raises(NotImplementedError):
                dual = forward_ad.make_dual(args[i].detach().clone(), torch.empty_like(args[i]))
                rest = [a.detach().clone().requires_grad_() if needs_grad and j == 0 and i else a for j, a in enumerate(args)]
                call(*[dual if j == i else a for j, a in enumerate(rest)])
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda a: call(a, *args[1:]), (args[0],), (torch.empty_like(args[0]),))


# ---- alignment ---------------------------------------------------------------
def shared_arrays_read_as_vectors(text):
    """Names of __shared__ arrays of scalars that a vector access names and no declaration aligns."""
    bare = set()
    for line in re.findall(r"^\s*__shared__ ([^;]*);", text, re.M):
        if "__align__" in line or "alignas" in line:
            continue
        bare |= set(re.findall(r"(\w+)(?=\s*(?:\[|,|$))", re.sub(r"\[[^\]]*\]", "[", line.split(None, 1)[1])))
    vector = re.findall(r"reinterpret_cast<(?:const )?(?:float[24]|uint[24]|int[24]|Vec<[^>]*>)\s*\*>\(&?(\w+)", text)
    vector += re.findall(r"\b(?:load|store)<\w+, [248]>\(&?(\w+)", text)
    return bare & set(vector)


def test_shared_arrays_that_are_read_as_vectors_are_aligned():
    assert shared_arrays_read_as_vectors("__shared__ float a[4], su[128];\n reinterpret_cast<const float4*>(su + c)") == {"su"}
    assert not shared_arrays_read_as_vectors("__shared__ __align__(16) float su[128];\n reinterpret_cast<const float4*>(su + c)")
    for path in sorted(glob.glob(os.path.join(ROOT, "pla_b200", "csrc", "*.cu*"))):
        # a kernel's declarations reach to its end
        for kernel in open(path).read().split("__global__")[1:]:
            assert not shared_arrays_read_as_vectors(kernel), path


# ---- the block -----------------------------------------------------------------
def test_mixer_states_do_not_follow_the_default_dtype():
    m = P.DeltaMixer(32, 2, head_dim=16, value_heads=4, value_dim=8)
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        conv, delta = m.new_state(3)
    finally:
        torch.set_default_dtype(before)
    assert conv.dtype == m.in_proj.weight.dtype and delta.dtype == torch.float32


def test_mixer_step_refuses_a_state_before_it_changes_any():
    m = P.DeltaMixer(32, 2, head_dim=16, value_heads=4, value_dim=8).to("meta")
    x, (conv, delta) = meta(3, 32, dtype=torch.float32), m.new_state(3)
    version = conv._version
    m.step(x, (conv, delta))
    assert conv._version > version
    version = conv._version
    for bad in (delta.bfloat16(), delta[:2], delta[:, :2], delta.transpose(2, 3), delta[:1].expand(3, -1, -1, -1), delta.requires_grad_()):
        with pytest.raises((ValueError, RuntimeError)):
            m.step(x, (conv, bad))
        assert conv._version == version


# ---- waits that run out ----------------------------------------------------------
def test_check_faults_raises_for_a_set_word(monkeypatch):
    class Library:
        word, status = 0, 0

        def pla_read_device_faults(self, to):
            to._obj.value = self.word
            return self.status

        def __getattr__(self, name):
            return getattr(real, name)

    real, fake = _lib.lib(), Library()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    P.check_faults()
    fake.word = 1
    with pytest.raises(_lib.PlaError, match="0x1"):
        P.check_faults()
    fake.word, fake.status = 0, 4
    with pytest.raises(_lib.PlaError, match="pla_read_device_faults"):
        P.check_faults()


def test_no_wait_of_a_kernel_goes_unread():
    """Every bounded wait's outcome is used, but those that only give copies in flight their time."""
    text = "".join(open(p).read() for p in sorted(glob.glob(os.path.join(ROOT, "pla_b200", "csrc", "delta_*.cuh"))))
    bare = [line.strip() for line in text.splitlines() if re.match(r"\s*(\w+\.)?(barrier_wait|wait)\(", line)]
    drain = re.search(r"void drain\(.*?\n}", text, re.S).group(0)
    assert all(line in drain for line in bare), bare
