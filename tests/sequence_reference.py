"""Plain float64 forms of the sequence operators, token by token, for the
tests: differentiable torch code written from the operators' definitions."""
import torch


def spans(x, cu):
    """(batch row, first token, end) of every sequence."""
    if cu is None:
        return [(b, 0, x.shape[1]) for b in range(x.shape[0])]
    ends = [int(v) for v in cu]
    return [(0, a, e) for a, e in zip(ends[:-1], ends[1:])]


def causal_depthwise(x, w, b=None, silu=False, cu=None, state=None):
    K = w.shape[-1]
    rows = [[None] * x.shape[1] for _ in range(x.shape[0])]
    last = []
    zero = x.new_zeros(x.shape[-1])
    for n, (r, a, e) in enumerate(spans(x, cu)):
        seen = [zero] * (K - 1) if state is None else list(state[n])
        for t in range(a, e):
            seen.append(x[r, t])
            p = sum(w[:, j] * seen[len(seen) - K + j] for j in range(K))
            if b is not None:
                p = p + b
            rows[r][t] = p * torch.sigmoid(p) if silu else p
        last.append(torch.stack(seen[len(seen) - (K - 1):]))
    y = torch.stack([torch.stack([zero if v is None else v for v in row]) if row else x.new_zeros(0, x.shape[-1])
                     for row in rows])
    return y, torch.stack(last)


def norm_rotate(x, w=None, cos=None, sin=None, positions=None, l2=False, eps=1e-6, interleaved=False):
    B, T, H, D = x.shape
    count = 1 if l2 else D
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / count + eps)
    if w is not None:
        y = y * w
    if cos is None:
        return y
    half = cos.shape[1]
    if positions is None:
        positions = torch.arange(T)
    c, s = (t.to(x.dtype)[positions.reshape(-1, T).long()][:, :, None] for t in (cos, sin))
    if interleaved:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
    else:
        a, b = y[..., :half], y[..., half:2 * half]
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def gated_delta_rule(q, k, v, g, beta, scale=None, cu=None, state=None):
    Hk, Dk, Hv, Dv = q.shape[2], q.shape[3], v.shape[2], v.shape[3]
    scale = Dk ** -0.5 if scale is None else scale
    q, k = (t.repeat_interleave(Hv // Hk, 2) for t in (q, k))
    rows = [[None] * v.shape[1] for _ in range(v.shape[0])]
    last = []
    for n, (r, a, e) in enumerate(spans(v, cu)):
        S = v.new_zeros(Hv, Dk, Dv) if state is None else state[n]
        for t in range(a, e):
            S = torch.exp(g[r, t])[:, None, None] * S
            u = beta[r, t][:, None] * (v[r, t] - torch.einsum("hkv,hk->hv", S, k[r, t]))
            S = S + k[r, t][:, :, None] * u[:, None, :]
            rows[r][t] = scale * torch.einsum("hkv,hk->hv", S, q[r, t])
        last.append(S)
    zero = v.new_zeros(Hv, Dv)
    o = torch.stack([torch.stack([zero if x is None else x for x in row]) if row else v.new_zeros(0, Hv, Dv)
                     for row in rows])
    return o, torch.stack(last)
