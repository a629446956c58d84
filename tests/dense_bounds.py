"""The dense products beside the packed experts from their definition in 64 bits, each with a bound on what a kernel with fp32 sums and
16-bit inputs and outputs may be off by.

Roundings that the bounds count: ``half_step`` of the output's type; the same once more for the value between the two products of an
MLP, which has to be 16 bits wide for the tensor cores; and sums in fp32, of which every one of K additions may lose 2^-23 of the sum
of magnitudes (2^-24 where it rounds, twice that where it truncates)."""
import torch

EXP_REL = 2.0 ** -18        # silu: fp32 exponential (argument up to 100: 2 + 100 ulp), division, products


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def sum_loss(k):
    return (k + 8) * 2.0 ** -23


def linear(x, w):
    """x [.., K] . w [N, K]^T -> (value, bound on an fp32 sum), float64."""
    x, w = x.double(), w.double()
    return x @ w.T, sum_loss(x.shape[-1]) * (x.abs() @ w.abs().T)


def rounded(value, err, dtype):
    """Bound once the fp32 result has been rounded to ``dtype``."""
    return err + half_step(dtype) * (value.abs() + err) + tiny(dtype)


def silu(v):
    return v * torch.sigmoid(v)


def swiglu(x, gate, up, down, dtype):
    """(value, bound before the output's rounding) of down . (silu(gate . x) * (up . x)) with the product held in ``dtype``."""
    (g, ge), (u, ue) = linear(x, gate), linear(x, up)
    z = silu(g) * u
    ze = 1.1 * ge * (u.abs() + ue) + silu(g).abs() * ue + EXP_REL * z.abs()        # |silu'| < 1.1
    ze = rounded(z, ze, dtype)
    d, de = linear(z, down)
    return d, de + ze @ down.double().abs().T * (1 + sum_loss(z.shape[-1]))


def check(got, value, err, what):
    got, value, err = got.detach().double().cpu(), value.cpu(), err.cpu()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - value).abs() - err
    if over.numel():
        i = int(over.argmax())
        assert float(over.reshape(-1)[i]) <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} outside, worst at {i}: got "
                                                 f"{float(got.reshape(-1)[i]):.6g}, expected {float(value.reshape(-1)[i]):.6g}, "
                                                 f"allowed {float(err.reshape(-1)[i]):.3g}")
