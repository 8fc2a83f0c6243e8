"""The sequence operators at the sizes they are used at: plain forms, the framework's calls, and the work of each.

Kinds of case (``case["kind"]``):

* ``conv``       causal depthwise convolution over a batch or a ragged batch, with the state after it
* ``conv_train`` the same, forward and backward
* ``conv_step``  one more token for every sequence, state updated in place
* ``norm``       per-head norm of queries and keys with the position rotation
* ``norm_train`` the same, forward and backward
* ``delta``      gated delta rule over a batch or a ragged batch, with the state after it
* ``delta_train`` the same, forward and backward
* ``delta_step`` one more token for every sequence, state updated in place
"""
import math

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64


def listed():
    return [
        # one decoding step of a layer's short convolution over the queries, keys and values of 32 requests
        {"name": "conv step 32", "kind": "conv_step", "dtype": "bf16", "n": 32, "c": 4096, "k": 4, "silu": True},
        # prompts of several requests of odd lengths in one ragged batch, with the state that decoding goes on from
        {"name": "conv ragged 8k", "kind": "conv", "dtype": "bf16", "n": 7, "t": 8191, "c": 8192, "k": 4, "silu": True,
         "ragged": True, "state": True},
        # a training step's convolution, batch of two sequences
        {"name": "conv train 2x4k", "kind": "conv_train", "dtype": "bf16", "n": 2, "t": 4096, "c": 4096, "k": 4,
         "silu": True, "ragged": False, "state": False},
        # decoding: 16 requests, 32 query heads and 8 key heads of 128, half of each head rotated
        {"name": "norm decode 16", "kind": "norm", "dtype": "bf16", "b": 16, "t": 1, "hq": 32, "hk": 8, "d": 128,
         "rot": 64, "mode": "rms", "pairs": False},
        # a prompt of 8192 tokens, whole heads rotated
        {"name": "norm prompt 8k", "kind": "norm", "dtype": "bf16", "b": 1, "t": 8192, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "mode": "rms", "pairs": False},
        # a training step in half precision, odd length, heads of 96
        {"name": "norm train 2x2047", "kind": "norm_train", "dtype": "fp16", "b": 2, "t": 2047, "hq": 16, "hk": 16,
         "d": 96, "rot": 96, "mode": "rms", "pairs": True},
        # decoding, four requests and many requests
        {"name": "delta step 4", "kind": "delta_step", "dtype": "bf16", "n": 4, "hk": 16, "hv": 32, "dk": 128,
         "dv": 128, "gates": "fp32"},
        {"name": "delta step 128", "kind": "delta_step", "dtype": "bf16", "n": 128, "hk": 16, "hv": 32, "dk": 128,
         "dv": 128, "gates": "fp32"},
        # a prompt of odd length in half precision
        {"name": "delta prompt 1001", "kind": "delta", "dtype": "fp16", "n": 1, "t": 1001, "hk": 16, "hv": 16,
         "dk": 64, "dv": 128, "gates": "fp32", "ragged": False, "state": False},
        # long prompts in one ragged batch, going on from states
        {"name": "delta ragged 16k", "kind": "delta", "dtype": "bf16", "n": 3, "t": 16383, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "gates": "fp32", "ragged": True, "state": True},
        # a training step under mixed precision, gates in the activations' type
        {"name": "delta train 4k", "kind": "delta_train", "dtype": "bf16", "n": 1, "t": 4096, "hk": 16, "hv": 32,
         "dk": 128, "dv": 128, "gates": "bf16", "ragged": False, "state": False},
        # a small training step in single precision, odd length, three sequences
        {"name": "delta train fp32", "kind": "delta_train", "dtype": "fp32", "n": 3, "t": 509, "hk": 6, "hv": 6,
         "dk": 64, "dv": 96, "gates": "fp32", "ragged": False, "state": False},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["conv", "conv_train", "conv_step", "norm", "norm_train", "delta", "delta", "delta_train",
                       "delta_train", "delta_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "conv_step":
        return {"kind": kind, "dtype": dtype, "n": log(1, 256), "c": 8 * log(8, 1024), "k": rng.choice([2, 3, 4]),
                "silu": rng.random() < 0.7}
    if kind in ("conv", "conv_train"):
        n = log(1, 12)
        ragged = rng.random() < 0.5
        c = 8 * log(8, 1024) + (rng.choice([0, 0, 0, 1, 3]) if dtype == "fp32" else 0)
        t = log(1, max(2, min(8192, 2 ** 25 // c) // (1 if ragged else n)))
        return {"kind": kind, "dtype": dtype, "n": n, "t": max(t, n) if ragged else t, "c": c,
                "k": rng.choice([2, 3, 4]), "silu": rng.random() < 0.7, "ragged": ragged,
                "state": kind == "conv" and rng.random() < 0.5}
    if kind in ("norm", "norm_train"):
        hk = log(1, 16)
        d = rng.choice([32, 64, 80, 96, 128, 192, 256])
        mode = rng.choice(["rms", "rms", "l2"])
        b = log(1, 16)
        hq = hk * rng.choice([1, 1, 2, 4])
        return {"kind": kind, "dtype": dtype, "b": b, "t": log(1, max(2, min(8192, 2 ** 24 // (b * (hq + hk) * d)))),
                "hq": hq, "hk": hk, "d": d, "rot": rng.choice([0, d // 2, d]), "mode": mode,
                "pairs": rng.random() < 0.5}
    hk = log(1, 16)
    hv = hk * rng.choice([1, 1, 2])
    dk, dv = rng.choice([32, 64, 96, 128, 128]), rng.choice([32, 64, 96, 128, 128])
    if kind == "delta_step":
        return {"kind": kind, "dtype": dtype, "n": log(1, 96), "hk": hk, "hv": hv, "dk": dk, "dv": dv,
                "gates": rng.choice(["fp32", dtype])}
    n = log(1, 4)
    ragged = rng.random() < 0.5
    top = 12000 if kind == "delta" else 2000
    t = log(1, max(2, top // (1 if ragged else n)))
    return {"kind": kind, "dtype": dtype, "n": n, "t": max(t, n) if ragged else t, "hk": hk, "hv": hv, "dk": dk,
            "dv": dv, "gates": "fp32" if kind == "delta" else dtype, "ragged": ragged,
            "state": kind == "delta" and rng.random() < 0.5}


def lengths(case):
    """Token counts of a ragged batch's sequences: uneven, every one at least one token."""
    n, t = case["n"], case["t"]
    parts = [1 + (i * 7919) % 13 for i in range(n)]
    got = [max(1, t * p // sum(parts)) for p in parts]
    got[got.index(max(got))] += t - sum(got)
    return got


def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPE[case["dtype"]]
    kind = case["kind"]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=rng, device="cuda") * scale).to(dtype)

    s = {"case": case, "kind": kind}
    if kind.startswith("conv"):
        n, c, k = case["n"], case["c"], case["k"]
        s["w"], s["b"] = normal(c, k, scale=k ** -0.5), normal(c, scale=0.1)
        if kind == "conv_step":
            s["x"], s["state"] = normal(n, c), normal(n, k - 1, c)
            return s
        s["state"] = normal(n, k - 1, c) if case["state"] else None
        shape = (1, case["t"], c) if case["ragged"] else (n, case["t"], c)
        s["x"] = normal(*shape)
        if kind == "conv_train":
            s["dy"] = normal(*shape)
    elif kind.startswith("norm"):
        b, t, hq, hk, d, rot = (case[k] for k in ("b", "t", "hq", "hk", "d", "rot"))
        s["q"], s["k"] = normal(b, t, hq, d), normal(b, t, hk, d, scale=3.0)
        s["wq"] = s["wk"] = s["cos"] = s["sin"] = s["pos"] = None
        if case["mode"] == "rms":
            s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(d, generator=rng, device="cuda")).to(dtype) for _ in "qk")
        if rot:
            far = 16384
            s["pos"] = torch.arange(t, device="cuda")[None] + torch.randint(0, far - t, (b, 1), generator=rng, device="cuda")
            turn = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * (
                10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))[None]
            s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
        if kind == "norm_train":
            s["dq"], s["dk"] = normal(b, t, hq, d), normal(b, t, hk, d)
    else:
        n, hk, hv, dk, dv = (case[k] for k in ("n", "hk", "hv", "dk", "dv"))
        gates = DTYPE[case["gates"]]
        if kind == "delta_step":
            lead = (n,)
        else:
            lead = (1, case["t"]) if case["ragged"] else (n, case["t"])

        def unit(*shape):  # what a SiLU and an L2 norm leave
            v = torch.nn.functional.silu(torch.randn(*shape, generator=rng, device="cuda"))
            return (v / v.norm(dim=-1, keepdim=True)).to(dtype)

        s["q"], s["k"], s["v"] = unit(*lead, hk, dk), unit(*lead, hk, dk), normal(*lead, hv, dv)
        rate = torch.exp(torch.empty(hv, device="cuda").uniform_(math.log(0.002), math.log(0.2), generator=rng))
        s["g"] = (-rate * torch.nn.functional.softplus(torch.randn(*lead, hv, generator=rng, device="cuda"))).to(gates)
        s["beta"] = torch.sigmoid(torch.randn(*lead, hv, generator=rng, device="cuda")).to(gates)
        s["state"] = None
        if kind == "delta_step" or case["state"]:
            s["state"] = normal(n, hv, dk, dv, scale=0.3, dtype=torch.float32)
        if kind == "delta_train":
            s["do"] = normal(*lead, hv, dv)
    s["cu"], s["most"] = None, case.get("t", 1)
    if case.get("ragged"):
        ends = np.cumsum([0] + lengths(case))
        s["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["most"] = int(np.max(np.diff(ends)))
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import pla_b200 as P

    case, kind = s["case"], s["kind"]
    if kind == "conv_step":
        y = P.causal_depthwise_step(s["x"], s["state"], s["w"], s["b"], silu=case["silu"])
        return {"y": y, "state": s["state"]}
    if kind == "conv":
        y, state = P.causal_depthwise(s["x"], s["w"], s["b"], silu=case["silu"], cu_seqlens=s["cu"], state=s["state"],
                                      return_state=True)
        return {"y": y, "state": state}
    if kind == "conv_train":
        x, w, b = (s[k].detach().requires_grad_() for k in ("x", "w", "b"))
        y = P.causal_depthwise(x, w, b, silu=case["silu"], cu_seqlens=s["cu"])
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if kind.startswith("norm"):
        args = [s[k] for k in ("q", "k", "wq", "wk")]
        if kind == "norm_train":
            args = [None if t is None else t.detach().requires_grad_() for t in args]
        q, k = P.qk_norm_rotate(*args, cos=s["cos"], sin=s["sin"], positions=s["pos"], norm=case["mode"],
                                interleaved=case["pairs"])
        if kind == "norm":
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), [t for t in args if t is not None], (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "grads": list(grads)}
    if kind == "delta_step":
        o = P.gated_delta_rule_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"])
        return {"o": o, "state": s["state"]}
    if kind == "delta":
        o, state = P.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], cu_seqlens=s["cu"], state=s["state"],
                                      return_state=True)
        return {"o": o, "state": state}
    args = [s[k].detach().requires_grad_() for k in ("q", "k", "v", "g", "beta")]
    o = P.gated_delta_rule(*args, cu_seqlens=s["cu"])
    return {"o": o.detach(), "grads": list(torch.autograd.grad(o, args, s["do"]))}


# ---- plain forms: elementary torch operations in 32 bits -------------------
def _places(s):
    """[N, most] row numbers of a ragged batch's tokens, and which of them are there."""
    at = s["cu"][:-1, None].long() + torch.arange(s["most"], device="cuda")[None]
    there = at < s["cu"][1:, None]
    return torch.where(there, at, 0), there


def _spread(s, x):
    """[1, T, ...] to a padded [N, most, ...], zeros in the padding."""
    at, there = s["places"]
    return torch.where(there.reshape(there.shape + (1,) * (x.dim() - 2)), x[0][at], 0)


def _gather(s, y):
    """A padded [N, most, ...] back to [1, T, ...]."""
    at, there = s["places"]
    return y[there][None]


def _plain(s):
    case, kind = s["case"], s["kind"]
    if kind == "conv_step":
        rows = torch.cat([s["state"], s["x"][:, None]], 1)
        p = (rows.float() * s["w"].float().T).sum(1) + s["b"].float()
        s["state"].copy_(rows[:, 1:])
        return {"y": _act(p, case).to(rows.dtype), "state": s["state"]}
    if s["cu"] is not None:
        s = dict(s, places=_places(s))
    if kind == "conv":
        y, state = _conv(s, s["x"], s["w"], s["b"])
        return {"y": y.to(s["x"].dtype), "state": state}
    if kind == "conv_train":
        x, w, b = (s[k].float().requires_grad_() for k in ("x", "w", "b"))
        y, _ = _conv(s, x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), s["dy"].float())
        dx, dw, db = (t.to(s["x"].dtype) for t in grads)
        return {"y": y.detach().to(s["x"].dtype), "dx": dx, "dw": dw, "db": db}
    if kind.startswith("norm"):
        dtype = s["q"].dtype
        args = [None if s[k] is None else s[k].float().requires_grad_(kind == "norm_train") for k in ("q", "k", "wq", "wk")]
        q, k = _norm(s, args[0], args[2]), _norm(s, args[1], args[3])
        if kind == "norm":
            return {"q": q.to(dtype), "k": k.to(dtype)}
        grads = torch.autograd.grad((q, k), [t for t in args if t is not None], (s["dq"].float(), s["dk"].float()))
        return {"q": q.detach().to(dtype), "k": k.detach().to(dtype), "grads": [t.to(dtype) for t in grads]}
    scale = case["dk"] ** -0.5
    if kind == "delta_step":
        q, k = (s[n].float().repeat_interleave(case["hv"] // case["hk"], 1) for n in "qk")
        state = s["state"] * s["g"].float().exp()[..., None, None]
        u = s["beta"].float()[..., None] * (s["v"].float() - (state * k[..., None]).sum(-2))
        state = state + k[..., None] * u[..., None, :]
        o = (state * q[..., None]).sum(-2) * scale
        s["state"].copy_(state)
        return {"o": o.to(s["q"].dtype), "state": s["state"]}
    args = [s[n].float().requires_grad_(kind == "delta_train") for n in ("q", "k", "v", "g", "beta")]
    o, state = _delta(s, *args)
    if kind == "delta":
        return {"o": o.to(s["q"].dtype), "state": state}
    grads = torch.autograd.grad(o, args, s["do"].float())
    return {"o": o.detach().to(s["q"].dtype),
            "grads": [t.to(s[n].dtype) for t, n in zip(grads, ("q", "k", "v", "g", "beta"))]}


def _act(p, case):
    return p * (1 / (1 + torch.exp(-p))) if case["silu"] else p


def _conv(s, x, w, b):
    case, k = s["case"], s["case"]["k"]
    rows = x if s["cu"] is None else _spread(s, x)
    n, most, c = rows.shape
    head = rows.new_zeros(n, k - 1, c) if s["state"] is None else s["state"].to(rows.dtype)
    rows = torch.cat([head, rows], 1)
    wf, p = w.float(), b.float()
    for j in range(k):
        p = p + wf[:, j] * rows[:, j:j + most].float()
    y = _act(p, case)
    if s["cu"] is None:
        return y, rows[:, most:]
    last = (s["cu"][1:] - s["cu"][:-1]).long()[:, None] + torch.arange(k - 1, device="cuda")[None]
    return _gather(s, y), rows[torch.arange(n, device="cuda")[:, None], last]


def _norm(s, x, w):
    case = s["case"]
    square = x * x
    r = 1 / torch.sqrt((square.mean(-1, keepdim=True) if case["mode"] == "rms" else square.sum(-1, keepdim=True)) + 1e-6)
    y = x * r
    if w is not None:
        y = y * w
    rot = case["rot"]
    if not rot:
        return y
    cos, sin = (s[n][s["pos"]][:, :, None] for n in ("cos", "sin"))
    turned, rest = y[..., :rot], y[..., rot:]
    if case["pairs"]:
        one, two = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([one * cos - two * sin, two * cos + one * sin], -1).flatten(-2)
    else:
        one, two = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([one * cos - two * sin, two * cos + one * sin], -1)
    return torch.cat([turned, rest], -1)


def _delta(s, q, k, v, g, beta):
    """The chunked form; the sums of the log decays and the small triangular inverses in 64 bits."""
    case = s["case"]
    if s["cu"] is not None:
        q, k, v, g, beta = (_spread(s, t) for t in (q, k, v, g, beta))
    n, most = q.shape[:2]
    hv, dk, dv = case["hv"], case["dk"], case["dv"]
    chunks = -(-most // CHUNK)

    def parts(t):  # [N, T, H, ...] to [N, H, chunks, CHUNK, ...]
        pad = t.new_zeros(n, chunks * CHUNK - most, *t.shape[2:])
        t = torch.cat([t, pad], 1).unflatten(1, (chunks, CHUNK)).movedim(3, 1)
        return t.repeat_interleave(hv // t.shape[1], 1)

    q, k, v, g, beta = (parts(t) for t in (q, k, v, g, beta))
    total = torch.cumsum(g.double(), -1)
    low = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    decay = torch.exp(torch.where(low, total[..., :, None] - total[..., None, :], -math.inf)).float()
    a = (beta[..., None] * decay * (k @ k.mT)).double().tril(-1)
    eye = torch.eye(CHUNK, device="cuda", dtype=torch.float64)
    inverse, power = eye - a, a @ a
    for _ in range(5):  # (1 - a)(1 + a^2)(1 + a^4)...
        inverse, power = inverse + inverse @ power, power @ power
    inverse = inverse.float()
    within = decay * (q @ k.mT)
    since, until = torch.exp(total).float(), torch.exp(total[..., -1:] - total).float()
    state = torch.zeros(n, hv, dk, dv, device="cuda") if s["state"] is None else s["state"]
    outs = []
    for c in range(chunks):
        x = beta[:, :, c, :, None] * (v[:, :, c] - since[:, :, c, :, None] * (k[:, :, c] @ state))
        u = inverse[:, :, c] @ x
        outs.append(since[:, :, c, :, None] * (q[:, :, c] @ state) + within[:, :, c] @ u)
        state = since[:, :, c, -1, None, None] * state + (until[:, :, c, :, None] * k[:, :, c]).mT @ u
    o = torch.stack(outs, 2).movedim(1, 3).flatten(1, 2)[:, :most] * dk ** -0.5
    return (o if s["cu"] is None else _gather(s, o)), state


# ---- the definitions, in 64 bits -------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    if kind.startswith("conv"):
        return _exact_conv(s)
    if kind.startswith("norm"):
        return _exact_norm(s)
    return _exact_delta(s)


def _spans(s):
    """(batch row, first token, end) of every sequence."""
    case = s["case"]
    if case.get("ragged"):
        ends = np.cumsum([0] + lengths(case))
        return [(0, int(a), int(b)) for a, b in zip(ends[:-1], ends[1:])]
    return [(i, 0, case["t"]) for i in range(case["n"])]


def _exact_conv(s):
    case, k, w = s["case"], s["case"]["k"], s["w"]
    act = torch.nn.functional.silu if case["silu"] else (lambda p: p)
    if s["kind"] == "conv_step":
        y = s["b"] + w[:, -1] * s["x"]
        for j in range(k - 1):
            y = y + w[:, j] * s["state"][:, j]
        return {"y": act(y), "state": torch.cat([s["state"][:, 1:], s["x"][:, None]], 1)}
    x, train = s["x"], s["kind"] == "conv_train"
    y, dx, dw, db = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(s["b"])
    states = []
    for i, (row, a, e) in enumerate(_spans(s)):
        front = x.new_zeros(k - 1, x.shape[-1]) if s["state"] is None else s["state"][i]
        seen = torch.cat([front, x[row, a:e]])
        states.append(seen[e - a:])
        p = torch.nn.functional.conv1d(seen.T[None], w[:, None], s["b"], groups=w.shape[0])[0].T
        y[row, a:e] = act(p)
        if train:
            dp = s["dy"][row, a:e]
            if case["silu"]:
                z = torch.sigmoid(p)
                dp = dp * z * (1 + p * (1 - z))
            db += dp.sum(0)
            for j in range(k):
                back = k - 1 - j
                dw[:, j] += (dp * seen[j:j + e - a]).sum(0)
                if e - a > back:
                    dx[row, a:e - back] += w[:, j] * dp[back:]
    return {"y": y, "dx": dx, "dw": dw, "db": db} if train else {"y": y, "state": torch.stack(states)}


def _exact_norm(s):
    case = s["case"]
    rot = case["rot"]

    def turn(t, way):  # as complex numbers
        if not rot:
            return t
        z = torch.complex(s["cos"][s["pos"]], way * s["sin"][s["pos"]])[:, :, None]
        head = t[..., :rot]
        if case["pairs"]:
            head = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (rot // 2, 2)).contiguous()) * z).flatten(-2)
        else:
            c = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * z
            head = torch.cat([c.real, c.imag], -1)
        return torch.cat([head, t[..., rot:]], -1)

    def one(x, w, dy):
        count = x.shape[-1] if case["mode"] == "rms" else 1
        r = ((x ** 2).sum(-1, keepdim=True) / count + 1e-6) ** -0.5
        unit, w1 = x * r, 1.0 if w is None else w
        y = turn(unit * w1, 1)
        if dy is None:
            return y, None, None
        dn = turn(dy, -1)
        h = dn * w1
        dx = r * (h - unit * (h * unit).sum(-1, keepdim=True) / count)
        return y, dx, None if w is None else (dn * unit).sum((0, 1, 2))

    q, dq, dwq = one(s["q"], s["wq"], s.get("dq"))
    k, dk, dwk = one(s["k"], s["wk"], s.get("dk"))
    if dq is None:
        return {"q": q, "k": k}
    return {"q": q, "k": k, "grads": [dq, dk] + ([] if dwq is None else [dwq, dwk])}


def _exact_delta(s):
    """Token by token."""
    case = s["case"]
    hv, dk, dv = case["hv"], case["dk"], case["dv"]
    scale, group = dk ** -0.5, hv // case["hk"]
    if s["kind"] == "delta_step":
        spans, lead = [(i, 0, 1) for i in range(case["n"])], lambda t: t[:, None]
    else:
        spans, lead = _spans(s), lambda t: t
    q, k, v, g, beta = (lead(s[n]) for n in ("q", "k", "v", "g", "beta"))
    most = max(e - a for _, a, e in spans)
    if 1.5e-4 * most * (4 if s["kind"] == "delta_train" else 1) > 18:
        return None
    at = torch.zeros(len(spans), most, dtype=torch.long, device="cuda")
    there = torch.zeros(len(spans), most, dtype=torch.bool, device="cuda")
    for i, (row, a, e) in enumerate(spans):
        at[i, :e - a] = torch.arange(row * q.shape[1] + a, row * q.shape[1] + e, device="cuda")
        there[i, :e - a] = True

    def pick(t):  # [N, most, ...], nothing in the padding
        t = t.reshape(-1, *t.shape[2:])[at]
        return t * there.reshape(there.shape + (1,) * (t.dim() - 2))

    def back(t):
        out = t.new_zeros(q.shape[0] * q.shape[1], *t.shape[2:])
        out[at[there]] = t[there]
        return out.reshape(*q.shape[:2], *t.shape[2:])

    qs, ks = (pick(t).repeat_interleave(group, 2) for t in (q, k))
    vs, bs, al = pick(v), pick(beta), torch.exp(pick(g))
    state = torch.zeros(len(spans), hv, dk, dv, dtype=torch.float64, device="cuda") if s["state"] is None else s["state"]
    train = s["kind"] == "delta_train"
    o, held, us, ds = torch.zeros_like(vs), [], [], []
    for t in range(most):
        held.append(state if train else None)
        state = state * al[:, t, :, None, None]
        d = vs[:, t] - torch.einsum("nhkv,nhk->nhv", state, ks[:, t])
        u = bs[:, t, :, None] * d
        state = state + ks[:, t, :, :, None] * u[:, :, None]
        o[:, t] = scale * torch.einsum("nhkv,nhk->nhv", state, qs[:, t])
        if train:
            us.append(u)
            ds.append(d)
    if s["kind"] == "delta_step":
        return {"o": o[:, 0], "state": state}
    if not train:
        return {"o": back(o), "state": state}
    do = pick(s["do"]) * scale
    gq, gk, gv, gg, gb = (torch.zeros_like(t) for t in (qs, ks, vs, al, bs))
    grad = torch.zeros_like(state)
    for t in reversed(range(most)):
        a, b, kt, s0 = al[:, t, :, None], bs[:, t, :, None], ks[:, t], held[t]
        s1 = a[..., None] * s0 + kt[..., None] * us[t][:, :, None]
        gq[:, t] = torch.einsum("nhkv,nhv->nhk", s1, do[:, t])
        grad = grad + qs[:, t, :, :, None] * do[:, t, :, None]
        du = torch.einsum("nhkv,nhk->nhv", grad, kt)
        gv[:, t] = b * du
        gb[:, t] = (du * ds[t]).sum(-1)
        gk[:, t] = torch.einsum("nhkv,nhv->nhk", grad, us[t]) - a * b * torch.einsum("nhkv,nhv->nhk", s0, du)
        grad = grad - b[..., None] * kt[..., None] * du[:, :, None]
        gg[:, t] = a[..., 0] * (grad * s0).sum((-2, -1))
        grad = a[..., None] * grad
    gq, gk = (t.unflatten(2, (-1, group)).sum(3) for t in (gq, gk))
    return {"o": back(o), "grads": [back(t) for t in (gq, gk, gv, gg, gb)]}


def work(case):
    e = DTYPE[case["dtype"]].itemsize
    kind = case["kind"]
    if kind.startswith("conv"):
        n, c, k = case["n"], case["c"], case["k"]
        if kind == "conv_step":
            return {"bytes": n * c * e * (2 + 2 * (k - 1)) + c * (k + 1) * e, "flops": 2 * n * c * k}
        tokens = case["t"] if case["ragged"] else n * case["t"]
        fixed = c * (k + 1) * e
        if kind == "conv":
            return {"bytes": 2 * tokens * c * e + fixed + n * (k - 1) * c * e * (2 if case["state"] else 1),
                    "flops": 2 * tokens * c * k}
        return {"bytes": 4 * tokens * c * e + 2 * fixed, "flops": 6 * tokens * c * k}
    if kind.startswith("norm"):
        values = case["b"] * case["t"] * (case["hq"] + case["hk"]) * case["d"]
        small = (2 * case["d"] * e if case["mode"] == "rms" else 0) + case["b"] * case["t"] * case["rot"] * 4
        if kind == "norm":
            return {"bytes": 2 * values * e + small, "flops": 8 * values}
        return {"bytes": 4 * values * e + 2 * small, "flops": 24 * values}
    n, hk, hv, dk, dv = (case[k] for k in ("n", "hk", "hv", "dk", "dv"))
    tokens = n if kind == "delta_step" else case["t"] if case["ragged"] else n * case["t"]
    each = 2 * hk * dk * e + 2 * hv * dv * e + 2 * hv * DTYPE[case["gates"]].itemsize
    state = n * hv * dk * dv * 4
    flops = 6 * tokens * hv * dk * dv
    if kind == "delta_step":
        return {"bytes": tokens * each + 2 * state, "flops": flops}
    if kind == "delta":
        return {"bytes": tokens * each + state * (2 if case["state"] else 1), "flops": flops}
    return {"bytes": 2 * tokens * each, "flops": 4 * flops}
