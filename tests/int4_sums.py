"""How far sums of a product with 4-bit weights may be off when they are held in 32 bits, for any device.

E = 2^-24 is half a unit in the last place of 32 bits.  Terms are of either sign and about independent, so errors are held in their root mean
square, relative to sigma = sqrt(sum of (w x)^2) of an element, which a typical result is as large as.

A step on the tensor cores adds 16 products, which are exact, to a sum.  Each of the 17 is cut at 2^-23 of the power of two of the largest:
off by up to 2 E of it, 1.2 E in the root mean square, sqrt(17) = 4.1 of those are 5 E of the largest, and that is taken as twice the
group's sigma.  Cutting is biased, so steps add up: 10 E for each of a group's group / 16.  Groups are about independent.  Adding a
group, scaled, to the result rounds once, E of a sum of sigma at most; so do shares of a tile (up to 8) and the parts of a 32-bit value:
2 sqrt(groups + 8) + 2.  Results are rounded to their type at the end, by up to ``U`` of themselves.
"""
import math

import torch

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def of_sigma(columns, group):
    return E * (10 * group / 16 + 2 * math.sqrt(-(-columns // group) + 8) + 2)


def far(y, x, w, group):
    """(root mean square, largest) error of ``y``, in units of what it may be in the root mean square, against x w^T in 64 bits."""
    x, w = x.double(), w.double()
    want, sigma = x @ w.T, (x.square() @ w.square().T).sqrt()
    r = (y.double() - want) / (of_sigma(w.shape[1], group) * sigma + U[y.dtype] * want.abs() + TINY[y.dtype] + 1e-30)
    return float(r.square().mean().sqrt()), float(r.abs().max())


def near(y, x, w, group):
    """Whether sums can have been held in 32 bits: the root mean square over a few hundred elements and more, and no element six times that."""
    rms, most = far(y, x, w, group)
    return rms <= 1 and most <= 6


# rows, outputs, columns, group, zeros: both kernels, long sums, tiles whose columns several CTAs share, evenly and not
SHAPES = [
    (1, 960, 9000, 128, False), (2, 1000, 1001, 64, True), (8, 130, 2570, 32, True),
    (40, 96, 9000, 128, False), (33, 160, 2500, 64, True), (40, 30, 5001, 64, True), (12, 300, 300, 32, True), (100, 130, 1400, 64, False),
    (20, 128, 4096, 64, True), (200, 64, 520, 128, True), (64, 128, 1088, 128, True), (17, 66, 640, 32, False),
]
