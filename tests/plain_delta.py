"""The gated delta rule, its convolution and gates in 64 bits, token by token from the formulas."""
import torch

F64 = torch.float64


def rule(q, k, v, log_decay, beta, state, scale, eps):
    """One request: q, k [n, heads, dim], v [n, heads, vdim], log_decay and beta [n, heads], state [heads, dim, vdim];
    returns o [n, heads, vdim] and the state behind the last token."""
    q, k, v, a, b, s = (x.to(F64) for x in (q, k, v, log_decay.to(F64).exp(), beta, state))
    q = q / (q.square().sum(-1, keepdim=True) + eps).sqrt() * scale
    k = k / (k.square().sum(-1, keepdim=True) + eps).sqrt()
    out = torch.zeros(v.shape, dtype=F64, device=v.device)
    for t in range(len(q)):
        s = s * a[t][:, None, None]
        u = b[t][:, None] * (v[t] - (s * k[t][:, :, None]).sum(1))
        s = s + k[t][:, :, None] * u[:, None]
        out[t] = (s * q[t][:, :, None]).sum(1)
    return out, s


def convolved(inputs, before, weights):
    """inputs [n, channels] behind `before` [taps - 1, channels], weights [taps, channels]: silu of the causal convolution, and
    the inputs that the next token looks back on."""
    u, w = torch.cat([before.to(F64), inputs.to(F64)]), weights.to(F64)
    n, taps = len(inputs), len(w)
    c = sum(w[j] * u[j:j + n] for j in range(taps))
    return c / (1 + (-c).exp()), u[n:]


def gates(a, b, a_log, dt_bias):
    a, b = a.to(F64) + dt_bias.to(F64), b.to(F64)
    return -a_log.to(F64).exp() * torch.where(a > 30, a, torch.log1p(a.clamp(max=30).exp())), 1 / (1 + (-b).exp())
