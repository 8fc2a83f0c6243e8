"""The sequence operators (pla_b200.sequence) on a GPU against float64 forms
written token by token (tests/sequence_reference.py).

Tolerances.  h(t) = finfo(t).eps / 2 is the one rounding of a result.

* causal_depthwise sums K + 1 <= 5 terms in fp32 (error <= 5 * 2^-24 of the
  terms' magnitudes, SiLU's slope <= 1.1) and, for 16-bit types, takes a
  sigmoid good to 2^-20: elementwise h |y| + 2^-18 magnitude (16-bit) or
  2^-20 magnitude (fp32: 5 * 1.1 * 2^-24 and about 6 units for sigmoid and the
  products, 2^-20 = 16 units).  Its gradients add one product with a slope
  <= 1.1 and, for w and b, sums over the tokens: fp32 sums in at most n terms
  of one thread (64) and a tree, <= 2^-24 * (64 + 20) = 2^-17.6 of the sum of
  magnitudes (sums of magnitudes of T random terms are up to sqrt(T) times
  their sum, which the magnitude used accounts for).
* qk_norm_rotate: a sum of D <= 256 squares in a tree (relative 2^-24 * 12),
  a root, a division, two products and the rotation: below 2^-19 of the head's
  largest value; gradients twice that, weights as above.
* gated_delta_rule: norms over a token's features, relative to the larger of
  the token's and the average token's.  One product of planes is off by
  3 * 2^-22 of the magnitudes, up to 8 times its result for 64 terms of random
  sign; four are chained (K S, T X, the state's update, the output):
  96 * 2^-22 = 2.3e-5 for fp32 results (states, fp32 outputs).  bf16 outputs
  use one plane in the output's own product: + 8 * 2 * 2^-12.  The backward
  pass chains three products in planes of one for bf16 (8 * 2 * 2^-12 each)
  and doubles the fp32 chain.
"""
import itertools

import pytest
import torch

import pla_b200 as P
from tests import sequence_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rand(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def gpu(t):
    return None if t is None else t.to(DEV)


def f64(t, grad=False):
    return None if t is None else t.detach().double().requires_grad_(grad)


def within(got, want, bound, what):
    got, bound = got.detach().cpu().double(), torch.as_tensor(bound).double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - want).abs() - bound
    if got.numel():
        assert float(over.max()) <= 0, f"{what}: {float((got - want).abs().max()):.3e} off, {float(over.max()):.3e} too far"


# ---- causal depthwise convolution ------------------------------------------
def conv_magnitude(x, w, b, cu, state):
    return R.causal_depthwise(x.abs(), w.abs(), None if b is None else b.abs(), False, cu,
                              None if state is None else state.abs())[0]


CONV = [  # batch, tokens, channels, taps, silu, bias, state, cu
    (1, 1, 8, 4, True, True, False, None),
    (2, 3, 64, 4, True, True, True, None),
    (2, 70, 72, 3, False, True, False, None),
    (3, 33, 40, 2, True, False, True, None),
    (1, 200, 24, 4, True, True, True, [0, 1, 3, 3, 6, 100, 199]),   # empty and short sequences, a tail of one row
    (1, 150, 13, 4, True, True, True, [0, 64, 150]),                # odd channels: single-element loads
    (1, 130, 96, 3, True, True, False, [0, 2, 130]),
    (1, 5, 2048, 4, False, False, False, [0, 5]),
]


def conv_inputs(case, dtype, seed=0):
    B, T, C, K, silu, bias, state, cu = case
    g = torch.Generator().manual_seed(seed)
    n = B if cu is None else len(cu) - 1
    x, w = rand(g, B, T, C, dtype=dtype), rand(g, C, K, dtype=dtype, scale=0.6)
    b = rand(g, C, dtype=dtype, scale=0.3) if bias else None
    s = rand(g, n, K - 1, C, dtype=dtype) if state else None
    return x, w, b, s, None if cu is None else torch.tensor(cu, dtype=torch.int32)


def conv_bound(dtype, y, mag):
    return half(dtype) * y.abs() + (2 ** -20 if dtype == F32 else 2 ** -18) * mag


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", CONV)
def test_causal_forward_and_state(case, dtype):
    x, w, b, s, cu = conv_inputs(case, dtype)
    want, last = R.causal_depthwise(f64(x), f64(w), f64(b), case[4], cu, f64(s))
    y, state = P.causal_depthwise(gpu(x), gpu(w), gpu(b), silu=case[4], cu_seqlens=gpu(cu), state=gpu(s), return_state=True)
    within(y, want, conv_bound(dtype, want, conv_magnitude(f64(x), f64(w), f64(b), cu, f64(s))), "y")
    assert torch.equal(state.cpu().double(), last)  # copies
    again = P.causal_depthwise(gpu(x), gpu(w)[:, None], gpu(b), silu=case[4], cu_seqlens=gpu(cu), state=gpu(s))
    assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", CONV)
def test_causal_gradients(case, dtype):
    x, w, b, s, cu = conv_inputs(case, dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    dy = rand(g, *x.shape, dtype=dtype)
    leaves = [f64(t, True) for t in (x, w, b, s)]
    y, last = R.causal_depthwise(leaves[0], leaves[1], leaves[2], case[4], cu, leaves[3])
    dlast = rand(g, *last.shape, dtype=dtype)
    there = [i for i in range(4) if leaves[i] is not None]
    want = torch.autograd.grad((y, last), [leaves[i] for i in there], (f64(dy), f64(dlast)), allow_unused=True)
    want = [torch.zeros_like(leaves[i]) if v is None else v for v, i in zip(want, there)]
    mine = [None if t is None else gpu(t).requires_grad_() for t in (x, w, b, s)]
    y, last = P.causal_depthwise(mine[0], mine[1], mine[2], silu=case[4], cu_seqlens=gpu(cu), state=mine[3], return_state=True)
    got = torch.autograd.grad((y, last), [mine[i] for i in there], (gpu(dy), gpu(dlast)))
    # magnitudes: the same gradient with every term positive, slopes at most 1.1
    pos = [None if t is None else t.detach().abs().requires_grad_() for t in leaves]
    py, pl = R.causal_depthwise(pos[0], pos[1], pos[2], False, cu, pos[3])
    mag = torch.autograd.grad((py, pl), [pos[i] for i in there], (1.1 * f64(dy).abs(), f64(dlast).abs()), allow_unused=True)
    mag = [torch.zeros_like(pos[i]) if v is None else v for v, i in zip(mag, there)]
    # an error of p reaches dp through act'' <= 0.5: relative to the magnitude of p, at most some tens here
    loose = {0: 2 ** -15, 1: 2 ** -15, 2: 2 ** -15, 3: 2 ** -15}
    for i, a, b_, m in zip(there, got, want, mag):
        within(a, b_, half(dtype) * b_.abs() + loose[i] * m, "x w b state".split()[i])


def test_causal_gradient_against_differences():
    x, w, b, s, cu = conv_inputs((1, 37, 8, 4, True, True, True, [0, 2, 20, 37]), F32, seed=3)
    leaves = [gpu(t).requires_grad_() for t in (x, w, b, s)]
    f = lambda a: P.causal_depthwise(a[0], a[1], a[2], silu=True, cu_seqlens=gpu(cu), state=a[3])  # noqa: E731
    y = f(leaves)
    dy = gpu(rand(torch.Generator().manual_seed(4), *y.shape))
    for i, grad in enumerate(torch.autograd.grad(y, leaves, dy)):
        step = gpu(rand(torch.Generator().manual_seed(5 + i), *leaves[i].shape))
        e = 2 ** -6
        moved = [[t.detach() + sign * e * step if j == i else t.detach() for j, t in enumerate(leaves)] for sign in (1, -1)]
        slope = float(((f(moved[0]).double() - f(moved[1]).double()) / (2 * e) * dy.double()).sum())
        # third derivatives of SiLU < 1: e^2 / 6 of |step|^3 |dy| a term; fp32 values over 2 e
        size = float((dy.abs().double().sum()) * 8)
        assert abs(slope - float((grad.double() * step.double()).sum())) <= size * (e * e + 2 ** -24 / e)


def test_causal_strided_and_streams():
    g = torch.Generator().manual_seed(7)
    wide = gpu(rand(g, 2, 90, 200, dtype=BF16))
    w = gpu(rand(g, 64, 4, dtype=BF16))
    for cut in (wide[..., 8:72], wide[..., 3:67], wide[:, ::2, 16:80], wide.transpose(0, 1)[:, :, :64]):
        want = P.causal_depthwise(cut.contiguous(), w, silu=True)
        assert torch.equal(P.causal_depthwise(cut, w, silu=True), want)
    turned = gpu(rand(g, 2, 64, 90, dtype=BF16)).transpose(1, 2)  # channels not dense: copied
    assert torch.equal(P.causal_depthwise(turned, w), P.causal_depthwise(turned.contiguous(), w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = P.causal_depthwise(wide[..., :64], w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, P.causal_depthwise(wide[..., :64], w))


@pytest.mark.parametrize("dtype,n,c,k", [(BF16, 3, 64, 4), (F32, 1, 20, 3), (F16, 5, 7, 2), (BF16, 33, 1024, 4)])
def test_causal_steps_continue_a_sequence(dtype, n, c, k):
    x, w, b, s, _ = conv_inputs((n, 12, c, k, True, True, True, None), dtype, seed=8)
    x, w, b, s = (gpu(t) for t in (x, w, b, s))
    whole, last = P.causal_depthwise(x, w, b, silu=True, state=s, return_state=True)
    y, state = P.causal_depthwise(x[:, :7], w, b, silu=True, state=s, return_state=True)
    pool = torch.zeros(n, 2, k - 1, c, device=DEV, dtype=dtype)  # one layer's states inside a larger buffer
    pool[:, 1] = state
    state = pool[:, 1]
    for t in range(7, 12):
        out = P.causal_depthwise_step(x[:, t], state, w, b, silu=True)
        assert torch.equal(out, whole[:, t])
    assert torch.equal(state, last) and not pool[:, 0].any()
    assert torch.equal(y, whole[:, :7])


# ---- norms -----------------------------------------------------------------
NORM = [  # B, T, Hq, Hk, D, rot, l2, weight, interleaved, position bytes (0: none)
    (1, 1, 1, 1, 128, 128, False, True, False, 8),
    (2, 5, 4, 2, 64, 32, False, True, False, 4),
    (2, 33, 6, 3, 96, 96, False, True, True, 0),
    (1, 17, 5, 1, 80, 40, True, False, False, 8),
    (3, 9, 2, 2, 256, 64, False, True, True, 4),
    (1, 7, 3, 3, 33, 10, False, True, False, 8),    # odd sizes: single-pair loads, one feature left over
    (1, 11, 2, 1, 6, 6, True, True, True, 0),
    (2, 40, 9, 5, 32, 0, True, False, False, 0),
    (1, 600, 16, 4, 128, 64, False, True, False, 0),
]


def norm_inputs(case, dtype, seed=0):
    B, T, Hq, Hk, D, rot, l2, weight, inter, pos_bytes = case
    g = torch.Generator().manual_seed(seed)
    q, k = rand(g, B, T, Hq, D, dtype=dtype), rand(g, B, T, Hk, D, dtype=dtype, scale=5.0)
    wq, wk = ((1 + rand(g, D, scale=0.3)).to(dtype) if weight else None for _ in "qk")
    cos = sin = pos = None
    if rot:
        turn = torch.arange(2000, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
        cos, sin = turn.cos().float(), turn.sin().float()
        if pos_bytes:
            pos = torch.randint(0, 2000, (B, T), generator=g).to(torch.int32 if pos_bytes == 4 else torch.int64)
    return q, k, wq, wk, cos, sin, pos


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", NORM)
def test_norm_forward_and_gradients(case, dtype):
    l2, inter = case[6], case[8]
    q, k, wq, wk, cos, sin, pos = norm_inputs(case, dtype)
    g = torch.Generator().manual_seed(1)
    dq, dk = rand(g, *q.shape, dtype=dtype), rand(g, *k.shape, dtype=dtype)
    mine = [None if t is None else gpu(t).requires_grad_() for t in (q, k, wq, wk)]
    got = P.qk_norm_rotate(*mine, cos=gpu(cos), sin=gpu(sin), positions=gpu(pos), norm="l2" if l2 else "rms", interleaved=inter)
    leaves = [t for t in mine if t is not None]
    grads = dict(zip([i for i, t in enumerate(mine) if t is not None], torch.autograd.grad(got, leaves, (gpu(dq), gpu(dk)))))
    for i, (x, w, dy) in enumerate([(q, wq, dq), (k, wk, dk)]):
        x64, w64 = f64(x, True), f64(w, True)
        want = R.norm_rotate(x64, w64, cos, sin, pos, l2, 1e-6, inter)
        top = want.detach().abs().amax(-1, keepdim=True)
        within(got[i], want.detach(), half(dtype) * want.detach().abs() + 2 ** -19 * top, "qk"[i])
        need = [x64] + ([] if w64 is None else [w64])
        dx, *dw = torch.autograd.grad(want, need, f64(dy))
        size = (x64.detach().square().sum(-1, keepdim=True) / (1 if l2 else x.shape[-1]) + 1e-6).rsqrt()
        big = size * (f64(dy).abs().amax(-1, keepdim=True) * 2 * (1 if w is None else w64.detach().abs().max()))
        within(grads[i], dx, half(dtype) * dx.abs() + 2 ** -18 * big * (x.shape[-1] ** 0.5 if l2 else 1), "d" + "qk"[i])
        if dw:
            # sum of the terms' magnitudes
            unit = (x64.detach() * size).abs()
            back = f64(dy).abs().amax(-1, keepdim=True) * 1.5
            mag = (unit * back).sum((0, 1, 2))
            within(grads[2 + i], dw[0], half(dtype) * dw[0].abs() + 2 ** -17 * mag, "dw" + "qk"[i])


def test_norm_strided_views_of_one_projection():
    g = torch.Generator().manual_seed(3)
    for dtype, off in itertools.product((BF16, F32), (0, 1)):
        flat = gpu(rand(g, 2, 50, off + (8 + 2 + 2) * 64, dtype=dtype))[..., off:]
        q, k = flat[..., :512].unflatten(-1, (8, 64)), flat[..., 512:640].unflatten(-1, (2, 64))
        *_, cos, sin, _ = norm_inputs((1, 1, 1, 1, 64, 64, False, False, False, 0), dtype)
        cos, sin = gpu(cos), gpu(sin)
        want = P.qk_norm_rotate(q.contiguous(), k.contiguous(), cos=cos, sin=sin)
        for a, b in zip(P.qk_norm_rotate(q, k, cos=cos, sin=sin), want):
            assert float((a.double() - b.double()).abs().max()) <= 4 * half(dtype) * 8  # other lanes, another order of sums


@pytest.mark.parametrize("tokens", [1, 3])
def test_norm_of_many_short_rows_equals_one_long_row(tokens):
    # a row's arithmetic does not depend on how rows are counted: equal bits
    g = torch.Generator().manual_seed(5)
    n = 601 * tokens
    q, k = rand(g, 1, n, 3, 128, dtype=BF16), rand(g, 1, n, 1, 128, dtype=BF16)
    dq, dk = rand(g, *q.shape, dtype=BF16), rand(g, *k.shape, dtype=BF16)
    angle = torch.randn(50, 64, generator=g)
    pos = torch.randint(0, 50, (1, n), generator=g)
    kw = dict(cos=gpu(angle.cos()), sin=gpu(angle.sin()))

    def run(*shape):
        leaves = [gpu(t.reshape(*shape, *t.shape[2:])).requires_grad_() for t in (q, k)]
        out = P.qk_norm_rotate(*leaves, positions=gpu(pos.reshape(shape)), **kw)
        return *out, *torch.autograd.grad(out, leaves, [gpu(t.reshape(*shape, *t.shape[2:])) for t in (dq, dk)])

    for a, b in zip(run(601, tokens), run(1, n)):
        assert torch.equal(a.flatten(0, 1), b.flatten(0, 1))


def test_norm_positions_outside_the_tables_are_nan_and_zero_rows_finite():
    q = torch.zeros(1, 4, 2, 64, device=DEV, dtype=BF16)
    q[:, 2] = 1
    cos, sin = torch.ones(8, 16, device=DEV), torch.zeros(8, 16, device=DEV)
    pos = torch.tensor([0, 8, 7, -1], device=DEV)
    a, b = P.qk_norm_rotate(q, q.clone(), cos=cos, sin=sin, positions=pos)
    for t in (a, b):
        assert torch.isnan(t[0, [1, 3], :, :32]).all() and torch.isfinite(t[0, [1, 3], :, 32:]).all()
        assert torch.equal(t[0, 0], torch.zeros_like(t[0, 0])) and torch.equal(t[0, 2], q[0, 2])


# ---- gated delta rule ------------------------------------------------------
DELTA = [  # n, T, Hk, Hv, Dk, Dv, state, cu, gates
    (1, 1, 1, 1, 128, 128, True, None, F32),
    (2, 63, 1, 2, 64, 64, False, None, None),
    (1, 64, 2, 2, 128, 128, True, None, F32),
    (1, 65, 1, 3, 96, 40, True, None, None),
    (2, 200, 2, 4, 128, 64, True, None, F32),
    (1, 300, 1, 2, 64, 128, True, [0, 1, 1, 64, 129, 280], F32),   # an empty sequence, a tail of 20 rows
    (1, 131, 1, 1, 20, 9, True, [0, 70, 131], None),               # odd head sizes
    (1, 90, 2, 2, 33, 17, False, [3, 60, 90], F32),                # three rows before the first sequence
]


def unit(g, *shape, dtype):
    v = torch.nn.functional.silu(torch.randn(*shape, generator=g))
    return (v / v.norm(dim=-1, keepdim=True)).to(dtype)


def delta_inputs(case, dtype, seed=0, strong=False):
    n, T, Hk, Hv, Dk, Dv, state, cu, gates = case
    g = torch.Generator().manual_seed(seed)
    q, k, v = unit(g, n, T, Hk, Dk, dtype=dtype), unit(g, n, T, Hk, Dk, dtype=dtype), rand(g, n, T, Hv, Dv, dtype=dtype)
    gt = gates or dtype
    rate = torch.linspace(0.01, 3.0 if strong else 0.3, Hv)
    decay = (-rate * torch.nn.functional.softplus(torch.randn(n, T, Hv, generator=g))).to(gt)
    beta = torch.sigmoid(torch.randn(n, T, Hv, generator=g)).to(gt)
    N = n if cu is None else len(cu) - 1
    s = rand(g, N, Hv, Dk, Dv, scale=0.5) if state else None
    return q, k, v, decay, beta, s, None if cu is None else torch.tensor(cu, dtype=torch.int32)


def token_norms(got, want, tol, what):
    """Norms over the last dimension, relative to the larger of the row's and the average row's."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    if not got.numel():
        return
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    floor = size.square().mean().sqrt()
    worst = float((off / torch.maximum(size, floor).clamp_min(1e-30)).max())
    assert worst <= tol, f"{what}: {worst:.3e} > {tol:.3e}"


FORWARD = {F32: 2.4e-5, F16: 2 ** -11 + 2.4e-5, BF16: 2 ** -8 + 16 * 2 ** -12}
BACKWARD = {F32: 4.8e-5, F16: 2 ** -11 + 4.8e-5, BF16: 2 ** -8 + 3 * 16 * 2 ** -12}


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", DELTA)
def test_delta_forward_and_state(case, dtype):
    q, k, v, g, beta, s, cu = delta_inputs(case, dtype)
    want, last = R.gated_delta_rule(*(f64(t) for t in (q, k, v, g, beta)), cu=cu, state=f64(s))
    args = [gpu(t) for t in (q, k, v, g, beta)]
    o, state = P.gated_delta_rule(*args, cu_seqlens=gpu(cu), state=gpu(s), return_state=True)
    token_norms(o, want, FORWARD[dtype], "o")
    token_norms(state, last, FORWARD[F32], "state")
    assert torch.equal(P.gated_delta_rule(*args, cu_seqlens=gpu(cu), state=gpu(s), return_state=True)[0], o)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_strong_decay_resets_and_scales(dtype):
    """Decays of many powers of e, -inf as a reset, beta of 0 and 2, values of very different sizes."""
    case = (1, 150, 1, 2, 64, 32, True, None, F32)
    q, k, v, g, beta, s, _ = delta_inputs(case, dtype, seed=4, strong=True)
    g[0, 40] = -float("inf")
    g[0, 100, 1] = -float("inf")
    beta[0, ::7] = 0
    beta[0, 3::11] = 2
    v[..., 5] *= 1e4
    v[..., 6] *= 1e-4
    s[..., 7] *= 1e4
    want, last = R.gated_delta_rule(*(f64(t) for t in (q, k, v, g, beta)), cu=None, state=f64(s))
    o, state = P.gated_delta_rule(*(gpu(t) for t in (q, k, v, g, beta)), state=gpu(s), return_state=True)
    # columns of v never meet: each against its own size
    token_norms(o.transpose(1, 3), want.transpose(1, 3), FORWARD[dtype], "o by column")
    token_norms(state.transpose(2, 3), last.transpose(2, 3), FORWARD[F32], "state by column")
    # q and k of other sizes: the planes are scaled row by row
    big = P.gated_delta_rule(gpu(q) * 1024, gpu(k) / 4096, gpu(v), gpu(g), gpu(beta), state=gpu(s))
    want, _ = R.gated_delta_rule(f64(q) * 1024, f64(k) / 4096, *(f64(t) for t in (v, g, beta)), cu=None, state=f64(s))
    token_norms(big.transpose(1, 3), want.transpose(1, 3), FORWARD[dtype], "o of scaled q, k")


def test_delta_strided_views_and_graph():
    g = torch.Generator().manual_seed(9)
    q, k, v, gate, beta, s, _ = (gpu(t) for t in delta_inputs((2, 130, 2, 4, 64, 64, True, None, BF16), BF16, seed=9))
    want = P.gated_delta_rule(q, k, v, gate, beta, state=s)
    for off in (0, 3):
        flat = torch.cat([torch.zeros(2, 130, off, device=DEV, dtype=BF16)] + [t.flatten(2) for t in (q, k, v, gate, beta)], -1)
        at, views = off, []
        for t in (q, k, v, gate, beta):
            width = t[0, 0].numel()
            views.append(flat[..., at:at + width].unflatten(-1, t.shape[2:]) if t.dim() == 4 else flat[..., at:at + width])
            at += width
        assert torch.equal(P.gated_delta_rule(*views, state=s), want)
    graph = torch.cuda.CUDAGraph()
    static = [t.clone() for t in (q, k, v, gate, beta)]
    with torch.cuda.graph(graph):
        o, state = P.gated_delta_rule(*static, state=s, return_state=True)
    static[2].copy_(v * 2)
    graph.replay()
    assert torch.equal(o, P.gated_delta_rule(q, k, v * 2, gate, beta, state=s))
    static[2].copy_(v)
    graph.replay()
    assert torch.equal(o, want)


@pytest.mark.parametrize("dtype,n,hk,hv,dk,dv", [(BF16, 1, 1, 1, 128, 128), (F32, 3, 2, 4, 64, 96), (F16, 2, 3, 3, 20, 7),
                                                 (BF16, 2, 1, 2, 256, 200), (F32, 70, 2, 2, 96, 128)])
def test_delta_step(dtype, n, hk, hv, dk, dv):
    q, k, v, g, beta, _, _ = delta_inputs((n, 1, hk, hv, dk, dv, False, None, F32), dtype, seed=11)
    gen = torch.Generator().manual_seed(12)
    s = rand(gen, n, hv, dk, dv, scale=0.5)
    want, last = R.gated_delta_rule(*(f64(t) for t in (q, k, v, g, beta)), cu=None, state=f64(s))
    pool = torch.full((n, 2, hv, dk, dv), 7.0, device=DEV)
    pool[:, 1] = gpu(s)
    o = P.gated_delta_rule_step(*(gpu(t)[:, 0] for t in (q, k, v, g, beta)), pool[:, 1])
    # sums of Dk <= 256 terms in fp32: 2^-24 * 40 in a tree of 8 warps and 32 rows, of magnitudes up to 16 times the result
    token_norms(o, want[:, 0], half(dtype) + 2 ** -14, "o")
    token_norms(pool[:, 1], last, 2 ** -14, "state")
    assert bool((pool[:, 0] == 7).all())


def test_delta_steps_continue_a_prompt():
    q, k, v, g, beta, s, _ = (gpu(t) for t in delta_inputs((2, 80, 2, 4, 64, 64, True, None, F32), F32, seed=13))
    whole, last = P.gated_delta_rule(q, k, v, g, beta, state=s, return_state=True)
    _, state = P.gated_delta_rule(*(t[:, :70] for t in (q, k, v, g, beta)), state=s, return_state=True)
    for t in range(70, 80):
        o = P.gated_delta_rule_step(*(x[:, t] for x in (q, k, v, g, beta)), state)
        token_norms(o, whole[:, t].cpu().double(), 2 * FORWARD[F32], "o")
    token_norms(state, last.cpu().double(), 2 * FORWARD[F32], "state")


def test_sequence_offsets_that_do_not_ascend_stay_in_bounds():
    """Wrong offsets give some result, touch nothing else and leave sane sequences right."""
    q, k, v, g, beta, _, _ = (gpu(t) for t in delta_inputs((1, 100, 1, 1, 64, 16, False, None, F32), F32, seed=14))
    x, w = gpu(rand(torch.Generator().manual_seed(15), 1, 100, 16)), torch.ones(16, 4, device=DEV)
    for cu in ([0, 90, 20, 100], [-5, 50, 1000], [70, 10, 5], [0, 100, 0, 100, 0, 100]):
        cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        o, state = P.gated_delta_rule(q, k, v, g, beta, cu_seqlens=cu, return_state=True)
        y, last = P.causal_depthwise(x, w, cu_seqlens=cu, return_state=True)
        for t in (o, state, y, last):
            assert bool(torch.isfinite(t).all())


# ---- gated delta rule, backward --------------------------------------------
def delta_gradients(case, dtype, seed, with_state, change=None):
    q, k, v, g, beta, s, cu = delta_inputs(case, dtype, seed=seed)
    if change:
        change(q, k, v, g, beta)
    gen = torch.Generator().manual_seed(seed + 1)
    d_o = rand(gen, *v.shape, dtype=dtype)
    leaves = [f64(t, True) for t in (q, k, v, g, beta)]
    s64 = f64(s, True)
    o, last = R.gated_delta_rule(*leaves, cu=cu, state=s64)
    ds = rand(gen, *last.shape, scale=0.5) if with_state else None
    inputs = leaves + ([s64] if s is not None and with_state else [])
    outs = ((o, last), (f64(d_o), f64(ds))) if with_state else ((o,), (f64(d_o),))
    want = torch.autograd.grad(outs[0], inputs, outs[1], allow_unused=True)
    want = [torch.zeros_like(i) if w is None else w for w, i in zip(want, inputs)]
    mine = [gpu(t).requires_grad_() for t in (q, k, v, g, beta)]
    sm = None if s is None else gpu(s).requires_grad_(with_state)
    o, last = P.gated_delta_rule(*mine, cu_seqlens=gpu(cu), state=sm, return_state=True)
    inputs = mine + ([sm] if s is not None and with_state else [])
    outs = ((o, last), (gpu(d_o), gpu(ds))) if with_state else ((o,), (gpu(d_o),))
    got = torch.autograd.grad(outs[0], inputs, outs[1], retain_graph=True)
    again = torch.autograd.grad(outs[0], inputs, outs[1])
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # no atomics in any sum
    return got, want


def check_delta_gradients(got, want, dtype, gates, plain):
    """plain: one plane everywhere (every gradient bf16)."""
    for name, a, b in zip("q k v g beta state".split(), got, want):
        fp32 = name == "state" or (name in ("g", "beta") and gates == F32)
        tol = BACKWARD[F32 if fp32 else dtype if plain or dtype != BF16 else BF16]
        if name in ("g", "beta"):
            # dg sums products over the rest of the sequence and its parts cancel: relative to the largest of a head
            a, b = a.transpose(1, 2), b.transpose(1, 2)
            tol = 4 * tol
        token_norms(a, b, tol, "d" + name)


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", DELTA)
def test_delta_gradients(case, dtype, with_state):
    got, want = delta_gradients(case, dtype, 21, with_state)
    check_delta_gradients(got, want, dtype, case[8] or dtype, not with_state and case[8] is None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_gradients_at_resets_and_zero_gates(dtype):
    def change(q, k, v, g, beta):
        g[0, 40] = -float("inf")
        g[0, 64] = -90.0
        beta[0, ::7] = 0
        beta[0, 3::11] = 2
        q[0, 10], k[0, 11] = 0, 0
        v[..., 5] *= 1e3

    got, want = delta_gradients((1, 150, 1, 2, 64, 32, True, None, F32), dtype, 31, True, change)
    want = [torch.nan_to_num(w, nan=0.0) for w in want]  # exp's slope at -inf times 0
    check_delta_gradients(got, want, dtype, F32, False)


def test_delta_gradient_against_differences():
    q, k, v, g, beta, s, cu = delta_inputs((1, 100, 1, 2, 64, 32, True, [0, 30, 100], F32), F32, seed=41)
    leaves = [gpu(t).requires_grad_() for t in (q, k, v, g, beta, s)]
    f = lambda a: P.gated_delta_rule(*a[:5], cu_seqlens=gpu(cu), state=a[5])  # noqa: E731
    o = f(leaves)
    d_o = gpu(rand(torch.Generator().manual_seed(42), *o.shape))
    for i, grad in enumerate(torch.autograd.grad(o, leaves, d_o)):
        step = gpu(rand(torch.Generator().manual_seed(43 + i), *leaves[i].shape)) * (0.1 if i in (0, 1) else 1)
        e = 2 ** -9
        moved = [[t.detach() + sign * e * step if j == i else t.detach() for j, t in enumerate(leaves)] for sign in (1, -1)]
        up_, down_ = f(moved[0]).double(), f(moved[1]).double()
        slope = float(((up_ - down_) / (2 * e) * d_o.double()).sum())
        want = float((grad.double() * step.double()).sum())
        # o's errors of 2^-16 (see the tolerances) over 2 e, as random terms, and the cubic rest, e^2 of a sum of its size
        noise = 2 ** -16 / e * float(o.detach().double().norm() * d_o.double().norm() / o.numel() ** 0.5)
        cubic = 40 * e * e * float(((up_ - down_) / (2 * e)).norm() * d_o.double().norm())
        assert abs(slope - want) <= noise + cubic, (i, slope, want, noise, cubic)


def test_backward_passes_replay_in_a_graph():
    q, k, v, g, beta, _, _ = (gpu(t) for t in delta_inputs((1, 200, 2, 2, 64, 64, False, None, None), BF16, seed=51))
    x, w, b, _, _ = (gpu(t) for t in conv_inputs((1, 200, 64, 4, True, True, False, None), BF16, seed=52))

    def passes(leaves):
        q, k, v, g, beta, x, w, b = leaves
        y = P.causal_depthwise(x, w, b, silu=True)
        qn, kn = P.qk_norm_rotate(q, k, norm="l2")
        o = P.gated_delta_rule(qn, kn, v, g, beta)
        return [y.detach(), o.detach(), *torch.autograd.grad((y, o), leaves, (x.detach(), v.detach()))]

    fresh = lambda: [t.detach().clone().requires_grad_() for t in (q, k, v, g, beta, x, w, b)]  # noqa: E731
    want = passes(fresh())
    leaves = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes(leaves)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_second_derivatives_raise():
    x = torch.randn(1, 8, 16, device=DEV, requires_grad=True)
    w = torch.randn(16, 4, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(P.causal_depthwise(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_steps_have_no_gradient_and_count_as_changes_of_the_state():
    x, w = torch.randn(2, 16, device=DEV), torch.randn(16, 4, device=DEV, requires_grad=True)
    s = torch.zeros(2, 3, 16, device=DEV)
    before = s._version
    y = P.causal_depthwise_step(x, s, w)
    assert y.requires_grad and s._version > before
    with pytest.raises(RuntimeError, match="no gradient"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="in place"):
        P.causal_depthwise_step(x, s.clone().requires_grad_(), w)
    q, v, g = torch.randn(2, 1, 32, device=DEV, requires_grad=True), torch.randn(2, 1, 32, device=DEV), torch.zeros(2, 1, device=DEV)
    o = P.gated_delta_rule_step(q, q, v, g, g + 1, torch.zeros(2, 1, 32, 32, device=DEV))
    with pytest.raises(RuntimeError, match="no gradient"):
        o.sum().backward()
    with torch.inference_mode():
        assert not P.causal_depthwise_step(x, torch.zeros(2, 3, 16, device=DEV), w).requires_grad


# ---- the block that chains them --------------------------------------------
def mixer_reference(m, x, cu):
    p = {n: t.detach().double().cpu().requires_grad_() for n, t in m.named_parameters()}
    h, conv = R.causal_depthwise(x @ p["in_proj.weight"].T, p["conv.weight"][:, 0], p["conv.bias"], True, cu)
    q, k, v = h.split(m.widths, -1)
    q, k = (R.norm_rotate(t.unflatten(-1, (m.num_heads, m.head_dim)), l2=True) for t in (q, k))
    a, b = (x @ p["gate_proj.weight"].T).chunk(2, -1)
    g = -p["A_log"].exp() * torch.nn.functional.softplus(a + p["dt_bias"])
    o, s = R.gated_delta_rule(q, k, v.unflatten(-1, (m.value_heads, m.value_dim)), g, torch.sigmoid(b), cu=cu)
    return o.flatten(-2) @ p["out_proj.weight"].T, conv, s, p


def make_mixer(dtype=F32):
    torch.manual_seed(71)
    return P.DeltaMixer(48, 2, head_dim=32, value_heads=4, value_dim=16, taps=4).to(DEV, dtype)


@pytest.mark.parametrize("cu", [None, [0, 5, 70, 131]])
def test_mixer_runs_and_its_gradients(cu):
    """fp32 throughout: the operators' tolerances (2.4e-5 forward, 4.8e-5
    backward) and matrix products of 48 to 128 terms (128 * 2^-24 = 2^-17) on
    either side of them: below 1e-4, twice that for gradients, of each
    tensor's norm."""
    m = make_mixer()
    g = torch.Generator().manual_seed(72)
    x = rand(g, 1 if cu else 2, 131, 48)
    dy = rand(g, *x.shape)
    cu = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    x64 = f64(x, True)
    want, conv, s, p = mixer_reference(m, x64, cu)
    xd = gpu(x).requires_grad_()
    y, state = m(xd, cu_seqlens=gpu(cu), return_state=True)
    for a, b in ((y, want), (state[0], conv), (state[1], s)):
        assert float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm()) <= 1e-4
    want = torch.autograd.grad(want, [x64, *p.values()], f64(dy))
    got = torch.autograd.grad(y, [xd, *m.parameters()], gpu(dy))
    for a, b, name in zip(got, want, ["x", *p]):
        assert float((a.cpu().double() - b).norm() / b.norm()) <= 2e-4, name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_mixer_decodes_from_its_prompts_states(dtype):
    m = make_mixer(dtype)
    x = gpu(rand(torch.Generator().manual_seed(73), 3, 40, 48, dtype=dtype))
    with torch.no_grad():
        whole, end = m(x, return_state=True)
        _, state = m(x[:, :30], return_state=True)
        out = torch.stack([m.step(x[:, t], state) for t in range(30, 40)], 1)
        fresh = m.new_state(3)
        first = m.step(x[:, 0], fresh)
    # the same sums in another order, the inputs of each layer rounded to dtype: a few roundings through two products
    tol = 2e-4 if dtype == F32 else 16 * half(BF16)
    assert float((out - whole[:, 30:]).norm() / whole[:, 30:].norm()) <= tol
    assert float((first - whole[:, 0]).norm() / whole[:, 0].norm()) <= tol
    assert float((state[1] - end[1]).norm() / end[1].norm()) <= tol


# ---- refusals and edges ----------------------------------------------------
def test_refusals_name_the_argument():
    x, w = torch.zeros(1, 8, 16, device=DEV), torch.zeros(16, 4, device=DEV)
    bad = [
        lambda: P.causal_depthwise(x[0], w), lambda: P.causal_depthwise(x, w[:, :1]),
        lambda: P.causal_depthwise(x, torch.zeros(16, 5, device=DEV)), lambda: P.causal_depthwise(x, w.half()),
        lambda: P.causal_depthwise(x.double(), w.double()), lambda: P.causal_depthwise(x, w.cpu()),
        lambda: P.causal_depthwise(x, w, state=torch.zeros(2, 3, 16, device=DEV)),
        lambda: P.causal_depthwise(x, w, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=DEV)),
        lambda: P.causal_depthwise(x, w, cu_seqlens=torch.zeros(3, dtype=torch.int64, device=DEV)),
        lambda: P.causal_depthwise(x.expand(2, 8, 16), w, cu_seqlens=torch.zeros(3, dtype=torch.int32, device=DEV)),
        lambda: P.causal_depthwise_step(x[:, 0], torch.zeros(1, 16, 3, device=DEV).mT, w),
        lambda: P.causal_depthwise_step(x[0], torch.zeros(1, 3, 16, device=DEV).expand(8, 3, 16), w),
    ]
    q = torch.zeros(1, 8, 2, 32, device=DEV)
    t = torch.zeros(8, 8, device=DEV)
    bad += [
        lambda: P.qk_norm_rotate(q, q[..., :16]), lambda: P.qk_norm_rotate(q, q, cos=t), lambda: P.qk_norm_rotate(q, q, cos=t.half(), sin=t),
        lambda: P.qk_norm_rotate(q, q, torch.zeros(31, device=DEV)), lambda: P.qk_norm_rotate(q, q, positions=torch.zeros(8, device=DEV)),
        lambda: P.qk_norm_rotate(q, q, cos=torch.zeros(8, 17, device=DEV), sin=torch.zeros(8, 17, device=DEV)),
        lambda: P.qk_norm_rotate(q, q, cos=t, sin=t, positions=torch.zeros(3, dtype=torch.long, device=DEV)),
        lambda: P.qk_norm_rotate(torch.zeros(1, 1, 1, 258, device=DEV), torch.zeros(1, 1, 1, 258, device=DEV)),
        lambda: P.qk_norm_rotate(q, q, eps=-1.0), lambda: P.qk_norm_rotate(q, q, cos=t.clone().requires_grad_(), sin=t),
    ]
    g = torch.zeros(1, 8, 2, device=DEV)
    big = torch.zeros(1, 8, 2, 160, device=DEV)
    bad += [
        lambda: P.gated_delta_rule(q, q, q, g, g[:, :4]), lambda: P.gated_delta_rule(q, q, q, g, g.half()),
        lambda: P.gated_delta_rule(q, q, q[:, :, :1].expand(1, 8, 3, 32), torch.zeros(1, 8, 3, device=DEV), torch.zeros(1, 8, 3, device=DEV)),
        lambda: P.gated_delta_rule(big, big, q, g, g), lambda: P.gated_delta_rule(q, q, big, g, g),
        lambda: P.gated_delta_rule(q, q, q, g, g, state=torch.zeros(1, 2, 32, 32, device=DEV, dtype=BF16)),
        lambda: P.gated_delta_rule_step(q[0], q[0], q[0], g[0], g[0], torch.zeros(8, 2, 32, 32, device=DEV).transpose(2, 3)),
        lambda: P.gated_delta_rule_step(q[0], q[0], q[0], g[0], g[0], torch.zeros(1, 2, 32, 32, device=DEV).expand(8, 2, 32, 32)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(ValueError):
        P.qk_norm_rotate(q, q, norm="batch")


def test_empty_calls():
    w = torch.zeros(16, 4, device=DEV)
    s = torch.randn(2, 3, 16, device=DEV)
    y, last = P.causal_depthwise(torch.zeros(2, 0, 16, device=DEV), w, state=s, return_state=True)
    assert y.shape == (2, 0, 16) and torch.equal(last, s)
    a, b = P.qk_norm_rotate(torch.zeros(0, 3, 2, 32, device=DEV), torch.zeros(0, 3, 1, 32, device=DEV))
    assert a.shape == (0, 3, 2, 32) and b.shape == (0, 3, 1, 32)
    q, g, s = torch.zeros(2, 0, 1, 32, device=DEV), torch.zeros(2, 0, 1, device=DEV), torch.randn(2, 1, 32, 32, device=DEV)
    o, last = P.gated_delta_rule(q, q, q, g, g, state=s, return_state=True)
    assert o.shape == q.shape and torch.equal(last, s)
    x = torch.zeros(0, 16, device=DEV)
    assert P.causal_depthwise_step(x, torch.zeros(0, 3, 16, device=DEV), w).shape == (0, 16)
    wq = torch.ones(32, device=DEV, requires_grad=True)
    q = torch.zeros(1, 0, 1, 32, device=DEV, requires_grad=True)
    yq, yk = P.qk_norm_rotate(q, q, wq, wq)
    assert not torch.autograd.grad((yq, yk), wq, (yq.detach(), yk.detach()))[0].any()
    xg = torch.zeros(1, 0, 16, device=DEV, requires_grad=True)
    wg = w.clone().requires_grad_()
    y = P.causal_depthwise(xg, wg)
    assert not torch.autograd.grad(y, wg, y.detach())[0].any()


def test_compiled_and_fake_tensors_trace():
    q, k, v, g, beta, _, _ = (gpu(t) for t in delta_inputs((1, 70, 1, 1, 32, 32, False, None, None), BF16, seed=91))
    f = lambda *a: P.gated_delta_rule(*P.qk_norm_rotate(a[0], a[1], norm="l2"), *a[2:]) * 2  # noqa: E731
    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    leaves = [t.clone().requires_grad_() for t in (q, k, v, g, beta)]
    again = [t.clone().requires_grad_() for t in (q, k, v, g, beta)]
    a, b = f(*leaves), compiled(*again)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, leaves, v), torch.autograd.grad(b, again, v)):
        assert torch.equal(x, y)
