"""The sequence operators on a GPU where small calls do not reach: results to
the last bit that their type holds, and the paths that large calls take.

Tolerances.  The error of a vector bounds that of each of its elements, so a
result of a 16-bit type is held element by element to one rounding of the
element, h(t) = finfo(t).eps / 2, and the fp32 error of its token's vector:
tests/test_gpu_sequence.py derives 2.4e-5 of the vector's norm for the delta
rule, 4.8e-5 for its gradients and four times that for the gates'."""
import ctypes

import pytest
import torch

import pla_b200 as P
from pla_b200 import _lib
from tests import sequence_reference as R
from tests import test_gpu_sequence as S
from tests.test_gpu_sequence import BF16, DEV, F16, F32, f64, gpu, half, rand

pytestmark = pytest.mark.gpu


def by_element(got, want, dtype, tol, what):
    """One rounding of each element and ``tol`` of the norm over the last dimension (the average row's if that is larger)."""
    size = want.norm(dim=-1, keepdim=True)
    S.within(got, want, half(dtype) * want.abs() + tol * torch.maximum(size, size.square().mean().sqrt()), what)


# ---- bf16 results are fp32 results, rounded once ----------------------------
ROUNDED = [c[:8] + (None,) for c in S.DELTA if c[1] > 1 and c[4] > 32]


@pytest.mark.parametrize("case", ROUNDED)
def test_delta_bf16_outputs_are_rounded_once(case):
    q, k, v, g, beta, s, cu = S.delta_inputs(case, BF16, seed=101)
    want, _ = R.gated_delta_rule(*(f64(t) for t in (q, k, v, g, beta)), cu=cu, state=f64(s))
    o = P.gated_delta_rule(*(gpu(t) for t in (q, k, v, g, beta)), cu_seqlens=gpu(cu), state=gpu(s))
    by_element(o, want, BF16, S.FORWARD[F32], "o")


@pytest.mark.parametrize("case", ROUNDED)
def test_delta_bf16_gradients_are_rounded_once(case):
    got, want = S.delta_gradients(case, BF16, 102, False)
    for name, a, b in zip("q k v g beta".split(), got, want):
        gate = name in ("g", "beta")
        if gate:  # over a head's tokens, as there
            a, b = a.transpose(1, 2), b.transpose(1, 2)
        by_element(a, b, BF16, S.BACKWARD[F32] * (4 if gate else 1), "d" + name)


# ---- norms of values that overflow, infinities -------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [6, 32, 64, 80, 96, 128, 192, 256])
def test_norm_of_a_head_whose_squares_overflow_is_zero(dim, dtype):
    """1e20^2 is not a float: 1 / sqrt(inf) = 0, times finite values, whatever part of its group a head fills."""
    q = torch.ones(1, 3, 2, dim, device=DEV, dtype=dtype)
    q[0, 1, 1] = 1e20
    k = q.clone()
    w = torch.ones(dim, device=DEV, dtype=dtype)
    leaves = [t.requires_grad_() for t in (q, k, w)]
    out = P.qk_norm_rotate(q, k, w, w)
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out])
    for t in out:
        # 1 / sqrt(1 + eps) is 5e-7 below 1, and a root and two products a few units of 2^-24
        assert not t[0, 1, 1].any() and float((t[0, ::2] - 1).abs().max()) <= 1e-6
    for t in grads[:2]:
        assert not t[0, 1, 1].any() and bool(torch.isfinite(t).all())
    assert bool(torch.isfinite(grads[2]).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 32), (128, 0), (96, 64), (33, 10)])
def test_norm_unrotated_features_do_not_meet(dim, rot, interleaved):
    """An infinity in a feature that is not rotated stays there: in the weight, and for dw in the gradient."""
    g = torch.Generator().manual_seed(111)
    q, k = gpu(rand(g, 1, 5, 2, dim)), gpu(rand(g, 1, 5, 2, dim))
    cos, sin = (torch.ones(5, rot // 2, device=DEV), torch.zeros(5, rot // 2, device=DEV)) if rot else (None, None)
    call = lambda *a: P.qk_norm_rotate(*a, cos=cos, sin=sin, interleaved=interleaved)  # noqa: E731
    w = torch.ones(dim, device=DEV)
    rest = dim - rot
    for bad in (rot, rot + rest // 2, dim - 1):
        others = [i for i in range(dim) if i != bad]
        odd = w.clone()
        odd[bad] = float("inf")
        for got, want in zip(call(q, k, odd, odd), call(q, k, w, w)):
            assert torch.equal(got[..., others], want[..., others]) and not torch.isfinite(got[..., bad]).any()
        leaves = [w.clone().requires_grad_(), w.clone().requires_grad_()]
        dy = torch.ones_like(q)
        want = torch.autograd.grad(call(q, k, *leaves), leaves, (dy, dy))
        dy = dy.clone()
        dy[0, 3, 1, bad] = float("nan")
        for a, b in zip(torch.autograd.grad(call(q, k, *leaves), leaves, (dy, dy)), want):
            assert torch.equal(a[others], b[others]) and bool(torch.isnan(a[bad]))


# ---- C callers ---------------------------------------------------------------
CODE = {F32: _lib.PLA_F32, BF16: _lib.PLA_BF16, F16: _lib.PLA_F16}


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_tensors_that_start_anywhere(dtype):
    """A C caller's tensors are aligned to their elements only: the same bits as from torch's."""
    q, k, v, g, beta, _, _ = (gpu(t) for t in S.delta_inputs((1, 100, 1, 2, 64, 32, False, None, F32), dtype, seed=121))
    d_o = gpu(rand(torch.Generator().manual_seed(122), *v.shape, dtype=dtype))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, g, beta)]
    o = P.gated_delta_rule(*leaves, scale=0.125)
    want = [o.detach(), *torch.autograd.grad(o, leaves, d_o)]

    def odd(t):  # one element behind an aligned address
        return torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)[1:].view(t.shape).copy_(t)

    q, k, v, g, beta, d_o = (odd(t) for t in (q, k, v, g, beta, d_o))
    got = [odd(torch.zeros_like(t)) for t in want]
    a = _lib.Delta(**{n: t.data_ptr() for n, t in zip(("q", "k", "v", "g", "beta", "o"), (q, k, v, g, beta, got[0]))},
                   batch=1, tokens=100, sequences=1, hk=1, hv=2, dk=64, dv=32, gates32=1, dtype=CODE[dtype], scale=0.125)
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta)):
        for part, stride in zip(("batch", "token", "head"), t.stride()):
            setattr(a, f"{name}_{part}", stride)
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    size = max(L.pla_gated_delta_rule_workspace(ctypes.byref(a), back) for back in (0, 1))
    work = torch.empty(size, device=DEV, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = work.data_ptr(), size
    assert L.pla_gated_delta_rule_forward(ctypes.byref(a), stream) == 0
    grad = _lib.DeltaGradient(d_o=d_o.data_ptr(), do_batch=d_o.stride(0), do_token=d_o.stride(1), do_head=d_o.stride(2),
                              **{n: t.data_ptr() for n, t in zip(("dq", "dk", "dv", "dg", "dbeta"), got[1:])})
    assert L.pla_gated_delta_rule_backward(ctypes.byref(a), ctypes.byref(grad), stream) == 0
    for x, y in zip(got, want):
        assert torch.equal(x, y)


# ---- values near the end of the float range ----------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_values_near_the_end_of_the_range(dtype):
    """The planes' scales reach every float: columns of v and of the state of 1e36 give what smaller ones give."""
    q, k, v, g, beta, s, _ = S.delta_inputs((1, 150, 1, 2, 64, 32, True, None, F32), dtype, seed=131)
    v[..., 5] *= 1e36
    v[..., 6] *= 1e-30
    s[..., 5] *= 1e36
    s[..., 7] *= 1e36
    want, last = R.gated_delta_rule(*(f64(t) for t in (q, k, v, g, beta)), cu=None, state=f64(s))
    o, state = P.gated_delta_rule(*(gpu(t) for t in (q, k, v, g, beta)), state=gpu(s), return_state=True)
    for c in range(32):  # columns never meet: each against its own size
        S.token_norms(o[..., c].transpose(1, 2), want[..., c].transpose(1, 2), S.FORWARD[dtype], f"o, column {c}")
        S.token_norms(state[..., c], last[..., c], S.FORWARD[F32], f"state, column {c}")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_gradients_near_the_end_of_the_range(dtype):
    def change(q, k, v, g, beta):
        v[..., 5] *= 4e35

    got, want = S.delta_gradients((1, 30, 1, 2, 64, 32, True, None, F32), dtype, 132, True, change)
    S.check_delta_gradients(got, want, dtype, F32, False)


# ---- the block -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_mixer_under_autocast_is_the_mixer_of_that_dtype(dtype):
    """fp32 weights under autocast: the calls of a block whose products and operators are of that dtype, with the same bits
    (its gates' constants stay fp32)."""
    m = S.make_mixer()
    cast = S.make_mixer().to(dtype)
    cast.A_log.data, cast.dt_bias.data = m.A_log.data.clone(), m.dt_bias.data.clone()
    x = gpu(rand(torch.Generator().manual_seed(141), 2, 70, 48))
    with torch.no_grad():
        want, end = cast(x.to(dtype), return_state=True)
        steps, first = cast.new_state(2), None
        first = cast.step(x[:, 0].to(dtype), steps)
        with torch.autocast("cuda", dtype):
            y, state = m(x, return_state=True)
            held = m.new_state(2)
            one = m.step(x[:, 0], held)
    for a, b in zip((y, *state, one, *held), (want, *end, first, *steps)):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_mixer_trains_under_autocast():
    m = S.make_mixer()
    cast = S.make_mixer().to(BF16)
    cast.A_log.data, cast.dt_bias.data = m.A_log.data.clone(), m.dt_bias.data.clone()
    x = gpu(rand(torch.Generator().manual_seed(142), 2, 70, 48, dtype=BF16))
    with torch.autocast("cuda", BF16):
        y = m(x)
    y.backward(torch.ones_like(y))
    z = cast(x)
    z.backward(torch.ones_like(z))
    assert torch.equal(y, z)
    for (name, a), b in zip(m.named_parameters(), cast.parameters()):
        assert a.grad.dtype == F32 and torch.equal(a.grad.to(b.dtype), b.grad), name


def test_mixer_steps_any_number_of_sequences():
    m, n = S.make_mixer(BF16), 65540
    x = gpu(rand(torch.Generator().manual_seed(151), n, 48, dtype=BF16))
    with torch.no_grad():
        state, part = m.new_state(n), m.new_state(40)
        y, z = m.step(x, state), m.step(x[-40:], part)
    for a, b in ((y[-40:], z), (state[0][-40:], part[0]), (state[1][-40:], part[1])):
        # matrix products of other shapes may sum in another order: a few roundings, as in a prompt and its steps
        assert float((a - b).norm() / b.norm()) <= 16 * half(BF16)


def test_no_wait_ran_out():
    P.check_faults(DEV)


# ---- the kernels and loops that only large calls reach -----------------------
# Compared as in tests/test_gpu_sequence.py, with its tolerances, which do not depend on sizes: sums over tokens there are
# bounded relative to the sum of their terms' magnitudes.  The 64-bit forms run on the GPU.
LONG_CONV = [  # batch, tokens, channels, taps, silu, bias, state, cu
    (1, 1811, 8192, 4, True, True, True, [0, 5, 40, 41, 41, 300, 1000, 1800]),   # strips of 32 forward, 64 back
    (2, 921, 4096, 3, True, False, True, None),                                  # strips of 16 (fp32: 32), 32 back
    (1, 1795, 2049, 2, False, True, False, [0, 700, 1795]),                      # single channels a thread
    (1, 4003, 96, 4, True, True, True, [min(4003, 2 * i - i // 3) for i in range(2402)]),  # thousands of sequences
]


def convolution(x, w, b, silu, cu, state):
    """The definition, a sequence at a time; y and the states after."""
    K, ys, last, at = w.shape[-1], [], [], 0
    for n, (r, a, e) in enumerate(R.spans(x, cu)):
        seen = torch.cat([x.new_zeros(K - 1, x.shape[-1]) if state is None else state[n], x[r, a:e]])
        p = sum(w[:, j] * seen[j:j + e - a] for j in range(K))
        p = p if b is None else p + b
        ys.append(p * torch.sigmoid(p) if silu else p)
        last.append(seen[e - a:])
        at = e
    y = torch.stack(ys) if cu is None else torch.cat(ys + [x.new_zeros(x.shape[1] - at, x.shape[-1])])[None]
    return y, torch.stack(last)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", LONG_CONV, ids=lambda c: "x".join(map(str, c[:4])))
def test_long_convolutions(case, dtype):
    silu = case[4]
    x, w, b, s, cu = S.conv_inputs(case, dtype, seed=161)
    there = [i for i, t in enumerate((x, w, b, s)) if t is not None]
    leaves = [f64(gpu(t), True) for t in (x, w, b, s)]
    y, last = convolution(*leaves[:3], silu, cu, leaves[3])
    gen = torch.Generator().manual_seed(162)
    dy, dlast = rand(gen, *y.shape, dtype=dtype), rand(gen, *last.shape, dtype=dtype)
    grads = torch.autograd.grad((y, last), [leaves[i] for i in there], (f64(gpu(dy)), f64(gpu(dlast))))
    mine = [None if t is None else gpu(t).requires_grad_() for t in (x, w, b, s)]
    out, state = P.causal_depthwise(*mine[:3], silu=silu, cu_seqlens=gpu(cu), state=mine[3], return_state=True)
    got = torch.autograd.grad((out, state), [mine[i] for i in there], (gpu(dy), gpu(dlast)))
    # magnitudes: every term positive, slopes at most 1.1
    pos = [None if t is None else t.detach().abs().requires_grad_() for t in leaves]
    py, pl = convolution(*pos[:3], False, cu, pos[3])
    mags = torch.autograd.grad((py, pl), [pos[i] for i in there], (1.1 * f64(gpu(dy)).abs(), f64(gpu(dlast)).abs()))
    # below 2^-14 an fp16 is a multiple of 2^-24, and its rounding off by up to 2^-25
    step = 2 ** -25 if dtype == F16 else 0
    S.within(out, y.detach().cpu(), (S.conv_bound(dtype, y.detach(), py.detach()) + step).cpu(), "y")
    assert torch.equal(state.detach().double(), last.detach())  # copies
    for i, a, want, mag in zip(there, got, grads, mags):
        S.within(a, want.cpu(), (half(dtype) * want.abs() + 2 ** -15 * mag + step).cpu(), "x w b state".split()[i])


LARGE_NORM = [  # B, T, Hq, Hk, D, rot, l2, weight, interleaved, position bytes
    (1, 4801, 5, 3, 128, 64, False, True, False, 8),     # heads in fours (fp32 twos) and a partial last group of them
    (1, 4801, 6, 3, 96, 96, False, True, True, 4),       # heads that do not fill their lanes
    (2, 5003, 9, 2, 64, 0, True, False, False, 0),       # as a block of this library calls it
    (3, 1601, 7, 1, 256, 128, False, True, False, 8),
    (1, 3001, 6, 5, 250, 100, False, True, False, 8),    # single pairs a lane, a walk over tokens
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", LARGE_NORM, ids=lambda c: "x".join(map(str, c[:6])))
def test_large_norms(case, dtype):
    S.test_norm_forward_and_gradients(case, dtype)


LARGE_DELTA = [  # n, T, Hk, Hv, Dk, Dv, state, cu, gates
    (1, 200, 10, 20, 128, 128, True, None, F32),                       # 32 columns a block
    (2, 150, 10, 20, 64, 128, True, None, None),                       # the same, two blocks an SM (16-bit types)
    (4, 130, 4, 20, 40, 40, False, None, None),                        # a last block of 8 columns
    (1, 300, 5, 20, 64, 100, True, [0, 70, 70, 150, 290], F32),        # a ragged batch, a last block of 4
    (1, 260, 20, 20, 128, 128, False, [0, 3, 260], None),
]
MANY = [[min(2500, 2 * i - i // 3) for i in range(1301)], [min(4003, 2 * i - i // 3) for i in range(2402)]]


def check_delta(case, dtype, with_state):
    inputs = S.delta_inputs(case, dtype, seed=171)
    cu = inputs[6]
    there = [i for i, t in enumerate(inputs[:6]) if t is not None]
    leaves = [f64(gpu(t), True) for t in inputs[:6]]
    o, last = R.gated_delta_rule(*leaves[:5], cu=cu, state=leaves[5])
    gen = torch.Generator().manual_seed(172)
    d_o, ds = rand(gen, *o.shape, dtype=dtype), rand(gen, *last.shape, scale=0.5)
    pick = slice(0, 2 if with_state else 1)
    wants = torch.autograd.grad((o, last)[pick], [leaves[i] for i in there], (f64(gpu(d_o)), f64(gpu(ds)))[pick])
    mine = [None if t is None else gpu(t).requires_grad_() for t in inputs[:6]]
    out, state = P.gated_delta_rule(*mine[:5], cu_seqlens=gpu(cu), state=mine[5], return_state=True)
    got = torch.autograd.grad((out, state)[pick], [mine[i] for i in there], (gpu(d_o), gpu(ds))[pick])
    S.token_norms(out, o.detach().cpu(), half(dtype) + S.FORWARD[F32], "o")
    S.token_norms(state, last.detach().cpu(), S.FORWARD[F32], "state")
    for i, a, want in zip(there, got, wants):
        name, tol = "q k v g beta state".split()[i], S.BACKWARD[F32]
        if name in ("g", "beta"):  # relative to the largest of a head, as there
            a, want, tol = a.transpose(1, 2), want.transpose(1, 2), 4 * tol
        S.token_norms(a, want.cpu(), (half(a.dtype) if a.dtype != F32 else 0) + tol, "d" + name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", LARGE_DELTA, ids=lambda c: "x".join(map(str, c[:6])))
def test_delta_of_many_heads(case, dtype):
    check_delta(case, dtype, True)
    if case[8] is None:
        check_delta(case, dtype, False)


@pytest.mark.parametrize("cu", MANY, ids=lambda c: str(len(c) - 1))
def test_delta_of_many_sequences(cu):
    """More sequences than the plan's threads, and more than it orders by length."""
    check_delta((1, cu[-1] + 9, 1, 2, 16, 16, True, cu, F32), BF16, True)


def test_the_cases_above_reach_the_kernels_of_large_calls():
    from torch.profiler import ProfilerActivity, profile

    def forward_and_back(leaves, f):
        leaves = [None if t is None else gpu(t).requires_grad_(t.is_floating_point()) for t in leaves]
        y = f(*leaves)
        y = y if isinstance(y, tuple) else (y,)
        torch.autograd.grad(y, [t for t in leaves if t is not None and t.requires_grad], y)

    with profile(activities=[ProfilerActivity.CUDA]) as run:
        for case in LARGE_DELTA:
            q, k, v, g, beta, _, cu = S.delta_inputs(case, BF16)
            forward_and_back((q, k, v, g, beta), lambda *a: P.gated_delta_rule(*a, cu_seqlens=gpu(cu)))
        for case, dtype in ((LARGE_NORM[0], BF16), (LARGE_NORM[0], F32), (LARGE_NORM[1], BF16), (LARGE_NORM[2], F16)):
            q, k, wq, wk, cos, sin, pos = S.norm_inputs(case, dtype)
            kw = dict(cos=gpu(cos), sin=gpu(sin), positions=gpu(pos), norm="l2" if case[6] else "rms", interleaved=case[8])
            forward_and_back((q, k, wq, wk), lambda *a: P.qk_norm_rotate(*a, **kw))
        torch.cuda.synchronize()
    names = " ".join({e.key for e in run.key_averages()})
    if "pla::" not in names:
        pytest.skip("the profiler records no kernels here")
    for name in ("delta_sweep<__nv_bfloat16, 128, 32, 2, 1, false>", "delta_sweep<__nv_bfloat16, 64, 32, 1, 2, false>",
                 "delta_sweep<__nv_bfloat16, 64, 32, 3, 1, false>", "delta_sweep<__nv_bfloat16, 64, 32, 1, 2, true>",
                 "delta_sweep_back<__nv_bfloat16, 128, 32, 2, 1>", "delta_sweep_back<__nv_bfloat16, 64, 32, 1, 2>",
                 "qk_norm_forward4<__nv_bfloat16, 16, 4, false>", "qk_norm_forward4<float, 16, 2, false>",
                 "qk_norm_forward4<__nv_bfloat16, 16, 4, true>", "qk_norm_forward4<__half, 8, 4, false>"):
        assert name in names, name


# ---- values that are not finite ------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_delta_values_that_are_not_finite_stay_in_their_place(bad, dtype):
    """They reach their sequence's outputs from the start of their chunk of 64 tokens on: of v its own feature, of k its
    heads; nothing else."""
    cu = torch.tensor([0, 10, 190, 200], dtype=torch.int32, device=DEV)
    q, k, v, g, beta, _, _ = (gpu(t) for t in S.delta_inputs((1, 200, 2, 4, 64, 32, False, None, F32), dtype, seed=181))
    clean, end = P.gated_delta_rule(q, k, v, g, beta, cu_seqlens=cu, return_state=True)
    first = 10 + 64  # chunks of the middle sequence start at 10, 74 and 138
    v2 = v.clone()
    v2[0, 100, 1, 5] = bad
    o, state = P.gated_delta_rule(q, k, v2, g, beta, cu_seqlens=cu, return_state=True)
    assert not torch.isfinite(o[0, 100:190, 1, 5]).any() and not torch.isfinite(state[1, 1, :, 5]).all()
    o[0, first:190, 1, 5], state[1, 1, :, 5] = clean[0, first:190, 1, 5], end[1, 1, :, 5]
    assert torch.equal(o, clean) and torch.equal(state, end)
    k2 = k.clone()
    k2[0, 100, 1, 5] = bad
    o, state = P.gated_delta_rule(q, k2, v, g, beta, cu_seqlens=cu, return_state=True)
    assert not torch.isfinite(o[0, 100:190, 2:]).any()
    o[0, first:190, 2:], state[1, 2:] = clean[0, first:190, 2:], end[1, 2:]
    assert torch.equal(o, clean) and torch.equal(state, end)


# ---- exact zeros ---------------------------------------------------------------
@pytest.mark.parametrize("dtype,gates", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 96), (33, 17)])
def test_delta_decay_of_nothing_has_no_gradient(dtype, gates, dk, dv):
    """A first token's decay acts on no state, or on one of zeros: dg is 0, not a rounding's rest."""
    for n, T, cu, zeros in ((3, 1, None, False), (1, 5, [0, 1, 2, 3, 4, 5], False), (2, 1, None, True)):
        case = (n, T, 2, 4, dk, dv, False, cu, gates)
        q, k, v, g, beta, _, cu = (gpu(t) for t in S.delta_inputs(case, dtype, seed=191))
        leaves = [t.requires_grad_() for t in (q, k, v, g, beta)]
        state = torch.zeros(n, 4, dk, dv, device=DEV) if zeros else None
        o, last = P.gated_delta_rule(*leaves, cu_seqlens=cu, state=state, return_state=True)
        gen = torch.Generator().manual_seed(192)
        d_o, ds = gpu(rand(gen, *o.shape, dtype=dtype)), gpu(rand(gen, *last.shape))
        for outs, grads in (((o,), (d_o,)), ((o, last), (d_o, ds))):
            got = torch.autograd.grad(outs, leaves, grads, retain_graph=True)
            assert not got[3].any(), float(got[3].abs().max())
            assert all(t.any() for t in (got[0], got[1], got[2], got[4]))
