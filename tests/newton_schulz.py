"""Newton-Schulz steps in 64 bits, and how far a result may be from them.

`inner` is what rounding every operand (X, A and B of each step) to some number of bits does to the 64-bit result, found by doing
it.  A result is that far off before it is rounded to its own type, which adds to it in squares what the 64-bit result's rounding
is off by.  Where `inner` is small beside a unit u of the type, more can be said: an element that is off by d before it is rounded
becomes a neighbour of the right one for a share d / u of the places between two of them, so the squares of what separates the
result from the rounded 64-bit one add up to d u on average.

Bits.  Pairs of half-precision parts are good for 22 (2^-23 of a value at most, half of that as a root mean square).  Their float32
sums lose as much again and more: the tensor core cuts what does not fit, for four to eight additions of 16 products by half
a unit of 2^-23 each, all to the same side, of partial sums that grow evenly: 2^-23 to 2^-22.  Together less than operands of
20 bits, whose rounding is 2^-21 at most and 2^-22 as a root mean square; twice their effect is allowed.  One part is good for
11 bits, and float32 sums are small beside that: twice the effect of 11 bits is allowed.  On float64 matrices (a shorter side
of up to 32) it is 2^-52 by the matrices' size and by what the steps make of it.
"""
import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def rounded(x, bits):
    """float64 values to `bits` significant bits."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** bits) * 2.0 ** -bits, e)


def steps_of(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, bits=None):
    """The formula in 64 bits; with `bits` every operand is rounded to that many."""
    a, b, c = coefficients
    near = (lambda x: x) if bits is None else (lambda x: rounded(x, bits))
    x = g.double()
    norm = torch.linalg.matrix_norm(x, keepdim=True) + eps
    flip = x.shape[-2] > x.shape[-1]
    x = near((x.mT if flip else x) / norm)
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for i in range(steps):
        gram = near(x @ x.mT)
        x = near(a * eye + b * gram + c * (gram @ gram)) @ x
        if i < steps - 1:
            x = near(x)
    return x.mT if flip else x


def inner_error(g, want, operand_bits, **kwargs):
    """Relative to the result (2-norm over all matrices), see above.  operand_bits: 22, 11, or 64 for float64 matrices."""
    if operand_bits == 64:
        # what is off grows by at most the largest slope of x (a + b x^2 + c x^4) in each step (up to 1.21, which no step here exceeds)
        a, b, c = kwargs.get("coefficients", COEFFICIENTS)
        t = torch.linspace(0, 1.21, 1001, dtype=torch.float64)
        slope = float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max())
        return 2.0 ** -52 * 32 * max(slope, 1.0) ** kwargs.get("steps", 5)
    off = steps_of(g, bits={22: 20, 11: 11}[operand_bits], **kwargs) - want
    return 2.0 * float(off.norm() / want.norm())


def allowed(dtype, inner):
    """Of |result - want rounded to dtype| / |want|.  Four times the mean of the squares: they are few and large where the
    error is small beside a unit."""
    unit = torch.finfo(dtype).eps
    return (4 * inner * unit) ** 0.5 + inner


def check(got, g, operand_bits, **kwargs):
    """Over the whole result, and by blocks of 32 x 32, of which none may be off by more than four times its share (and a unit
    of its own size: few elements make no mean)."""
    want = steps_of(g, **kwargs)
    assert got.shape == g.shape and got.dtype == g.dtype
    size, unit = float(want.norm()), torch.finfo(got.dtype).eps
    nearest = want.to(got.dtype).double()
    inner = inner_error(g, want, operand_bits, **kwargs)
    off = float((got.double() - want).norm()) / size
    tol = (1.1 * (float((nearest - want).norm()) / size) ** 2 + inner ** 2) ** 0.5
    single = unit * float(want.abs().max()) / size                    # one element's neighbour
    assert off <= max(tol, single), (off, tol)
    apart = float((got.double() - nearest).norm()) / size
    assert apart <= max(allowed(got.dtype, inner), single), (apart, allowed(got.dtype, inner))
    blocks = lambda x: torch.nn.functional.pad(x, (0, -x.shape[-1] % 32, 0, -x.shape[-2] % 32)).unflatten(-2, (-1, 32)).unflatten(-1, (-1, 32))
    squares = lambda x: blocks(x).square().sum(dim=(-3, -1)).sqrt()
    share = squares(torch.ones_like(want)) / want.numel() ** 0.5
    limit = 4 * tol * size * share + unit * squares(want)
    over = squares(got.double() - want) / limit.clamp_min(1e-300)
    assert float(over.max()) <= 1.0, float(over.max())
    return off


def update(shape, seed, dtype=torch.float32, rank=None):
    """A momentum: a few strong directions over noise; with `rank` only that many directions."""
    g = torch.Generator().manual_seed(seed)
    r, c = shape[-2:]
    k = rank or max(1, min(r, c) // 8)
    u, v = torch.randn(shape[:-1] + (k,), generator=g, dtype=torch.float64), torch.randn(shape[:-2] + (k, c), generator=g, dtype=torch.float64)
    noise = 0.0 if rank else torch.randn(shape, generator=g, dtype=torch.float64)
    return (1e-3 * (u @ v / k ** 0.5 + noise)).to(dtype)
