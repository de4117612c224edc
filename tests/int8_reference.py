"""The 8-bit integer linears in 64 bits on the CPU, with what the device's 32-bit arithmetic may change.

A code may come out one step off only where the 64-bit quotient 127 v / m lies within `loose` (relative) of a tie; `slack` adds up
what such codes could change in an output.  Codes of 16-bit activations have no such place: they are determined."""
import torch

FLOOR = 2.0 ** -40


def half_step(dt):
    return torch.finfo(dt).eps / 2


def quantise(v, loose=0.0):
    """Rows of v (fp64) -> codes, scales, mask of the codes that may come out a step off."""
    m = v.abs().amax(1, keepdim=True).clamp_min(FLOOR)
    t = 127.0 * v / m
    near = ((t.abs() - t.abs().floor() - 0.5).abs() <= loose * t.abs()) if loose else torch.zeros_like(t, dtype=torch.bool)
    return torch.round(t), (m / 127.0).squeeze(1), near


def product(q, s, near, w, ws):
    """-> (q @ w^T) s ws in fp64 and the slack of codes that may be a step off."""
    factor = torch.outer(s, ws.double())
    out = (q @ w.double().t()) * factor
    slack = (near.double() @ w.double().abs().t()) * factor if bool(near.any()) else torch.zeros_like(out)
    return out, slack


def silu_mul(rows):
    g, u = rows.chunk(2, dim=1)
    return g / (1.0 + torch.exp(-g)) * u


def norm(x, residual, weight, eps):
    a = x.double() + residual.double()
    return a, a / torch.sqrt((a * a).mean(1, keepdim=True) + eps) * weight.double()


def within(got, ref, slack, dt, rel, parts=None):
    """got (16-bit) against ref: one rounding, `rel` of the summands for the 32-bit steps in front of it, the codes' slack, and the
    spacing of subnormal numbers."""
    size = ref.abs() if parts is None else parts
    tol = half_step(dt) * (ref.abs() + rel * size + slack) + rel * size + slack + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ~((got.double() - ref).abs() <= tol)
    return not bool(bad.any()), float(((got.double() - ref).abs() / tol.clamp_min(1e-300)).max()) if got.numel() else 0.0


def codes_like_weights(g, *shape):
    return (torch.randn(*shape, generator=g) * 34).round().clamp(-127, 127).to(torch.int8)


def scales(g, *shape):
    return 0.02 / 34 * (0.5 + torch.rand(*shape, generator=g))
