"""Plain float64 forms of the 8-bit operators, on the CPU, for the tests of the kernels."""
import numpy as np
import torch

BLOCK = 128
U = 2.0 ** -24                      # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # finfo(t).eps / 2
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half the smallest subnormal


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def exponent(largest):
    """smallest e >= -127 with largest <= 448 * 2^e"""
    e = np.full(largest.shape, -127.0)
    pos = largest > 0
    f, x = np.frexp(largest[pos] / 448.0)
    e[pos] = np.maximum(x - (f == 0.5), -127)
    return e


def spacing(y):
    """distance of the e4m3 codes around y"""
    return np.exp2(np.frexp(np.maximum(np.abs(y), 2.0 ** -6))[1] - 4.0)


def cast(a, tile):
    """(codes, scale exponents) of a float64 matrix; NaN codes where it is not finite"""
    rows, cols = a.shape
    high = BLOCK if tile else 1
    x = np.pad(a, ((0, -rows % high), (0, -cols % BLOCK)))
    x = x.reshape(-1, high, x.shape[1] // BLOCK, BLOCK)
    e = exponent(np.where(np.isfinite(x), np.abs(x), 0.0).max(axis=(1, 3)))
    with np.errstate(invalid="ignore"):
        y = x / np.exp2(e)[:, None, :, None]
        q = np.where(np.isfinite(y), np.rint(y / spacing(np.where(np.isfinite(y), y, 0.0))) * spacing(np.where(np.isfinite(y), y, 0.0)), np.nan)
    return q.reshape(x.shape[0] * high, -1)[:rows, :cols], e


def values(q):
    """what a BlockScaled stands for, in float64"""
    v, s = q.values.float().cpu().double().numpy(), q.scales.float().cpu().double().numpy()
    if s.shape[0] != v.shape[0]:
        s = np.repeat(s, BLOCK, 0)[:v.shape[0]]
    return v * np.repeat(s, BLOCK, 1)[:, :v.shape[1]]


def dither(n, step, seed, offset=0):
    """32 bits an element, see csrc/adamw.hip"""
    i = np.arange(offset, offset + n, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    x = ((i & low) * np.uint64(0x9E3779B9)) & low
    x ^= x >> np.uint64(16)
    x = ((x * np.uint64(0x6A09E667) & low) + np.uint64((step * 0x3C6EF373 + seed * 0x6A09E667) & 0xFFFFFFFF)
         + ((i >> np.uint64(32)) * np.uint64(0xBB67AE85) & low)) & low
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & low
    return x ^ (x >> np.uint64(16))


def dithered(x, u, least):
    """codes and scale exponents of the blocks of 128 of x (float64, flat), rounded up with probability = part of the distance"""
    b = x.reshape(-1, BLOCK)
    e = exponent(np.abs(b).max(axis=1))
    y = b / np.exp2(e)[:, None]
    d = spacing(y)
    code = np.floor(np.abs(y) / d + u.reshape(-1, BLOCK) / 65536.0) * d
    if least:
        code = np.where(y != 0, np.maximum(code, 2.0 ** -9), code)
    return (code * np.sign(y)).reshape(-1), e


def adamw(p, g, m, v, t, lr, b1, b2, eps, decay, coef=1.0):
    """one step in float64 from arrays; (p, m, v, error bounds of the float32 arithmetic for each)"""
    g = g * coef
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    size, rs = lr / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    den = np.sqrt(v2) * rs + eps
    p2 = p * (1 - lr * decay) - size * m2 / den
    # roundings of u each: m: the constants, both products, the sum, g's own; v: the same and the square
    em = U * (4 * np.abs(b1 * m) + 5 * np.abs((1 - b1) * g)) * 1.01
    ev = U * 7 * v2 * 1.01
    # in units of u: root: half of v's 7 and 2 of its own (one unit in the last place); denominator: root, the constant, product, sum;
    # reciprocal 2, product, constant, product: 13.5 in all; p: constant's three, product, sum of both terms
    ep = (5 * U * np.abs(p) + size * (em + 13.5 * U * np.abs(m2)) / den + 2 * U * np.abs(size * m2 / den)) * 1.01
    return p2, m2, v2, ep, em, ev
