"""How precise cross attention is as a whole, rather than at its worst element (plain torch on the CPU).

A bound that holds for every element has to add up the worst of every rounding, and lets pass what errs eight
times, or at f32 precision a hundred times, as much as it should.  The norm of all errors together does not: roundings
are as often up as down, and their root mean square is known.

16-bit products: the output's own rounding, whose norm follows from the exact result, is most of the error.  Beside it
stand probabilities of 11 bits or more, on 1-byte pages keys and values of 11 bits, each off by 2^-12.2 of itself
(root mean square; 2^-9.2 with 8 bits).  Outputs are sums of n terms p v of random signs, so that relative errors of the
terms are those of the norm: sqrt(3) 2^-12.2 = 3.7e-4, beside the rounding's 2^-9.2 = 1.7e-3 a factor of 1.024.  One of 8 bits
gives sqrt(2).  WITHIN lies between.

f32 precision: products of three-part values leave out parts of about 2^-23 of them (2^-21 at most), sums, exponentials
and the scale round by 2^-24: a score of 1 to 4 errs by about 2^-22, and so do probabilities and outputs.  Two parts, 16 bits,
err by 2^-18 to 2^-16.  F32 lies between."""
import torch

WITHIN = 1.1
F32 = 2.0 ** -20


def off(out, want):
    """The norm of the error, relative to the result's (where that is all zeros, the error's)."""
    return float((out.double() - want).norm() / (want.norm() if want.any() else 1.0))


def floor(want, dtype):
    """The same of the exact result, rounded to dtype."""
    return off(want.to(dtype), want)
