"""The int8 operators in 64 bits (and where a result is a matter of fp32 roundings, in fp32 as it is defined)."""
import torch

LEAST = 1e-10


def quant_rows(v):
    """Codes and scales of rows by the definition.  16-bit rows: 127 v / a, ties to even (127 v is exact in 64 bits, so a tie's quotient is);
    32-bit rows: v times the least fp32 number that is no less than 127 / a, unrounded (64 bits hold the product)."""
    wide = v.dtype == torch.float32
    v = v.float().cpu()
    amax = v.abs().amax(dim=-1) if v.shape[-1] else v.new_zeros(v.shape[:-1])
    amax = torch.maximum(amax, torch.tensor(LEAST))
    if wide:
        inv = torch.tensor(127.0) / amax
        inv = torch.where(inv.double() * amax.double() < 127.0, torch.nextafter(inv, torch.full_like(inv, float("inf"))), inv)
        q = v.double() * inv.double()[..., None]
    else:
        q = 127.0 * v.double() / amax.double()[..., None]
    return torch.round(q).to(torch.int8), amax / torch.tensor(127.0)


def linear(q, qs, w, ws, bias=None):
    """(exact result, the product before the bias), float64."""
    p = q.double() @ w.double().t() * torch.outer(qs.double(), ws.double())
    return (p if bias is None else p + bias.double()), p


def linear_tolerance(y, p, dtype):
    """fp32: the sum to 24 bits, two products and the bias's addition, a rounding of 2^-24 each (to second order); then the output's
    rounding, half a step of its type, or of its subnormal numbers."""
    f = 2.0 ** -24
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return (3.01 * f * p.abs() + f * y.abs()) * (1 + half) + half * y.abs() * (1 + 2 ** -10) + least


def silu(g):
    return g / (1.0 + torch.exp(-g))


def weights(n, k, gen, experts=None, device="cuda"):
    shape = (n, k) if experts is None else (experts, n, k)
    w = torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8)
    s = (torch.rand(shape[:-1], generator=gen) + 0.5) * 0.01
    return w.to(device), s.to(device)
