"""The feed-forward operators in float64 numpy, and the error bounds of the library's results.

Roundings that the bounds count: u16 = 2^-8 (bf16, half a step relative to the value), u32 = 2^-24 (fp32).  The tensor
core adds products of bf16 into its fp32 accumulator without rounding to nearest: each addition may lose up to one unit
in the last place of the running sum, which ``sum_slack`` bounds by 2^-23 for each 16-element step, relative to the sum
of magnitudes."""
import math

import numpy as np

U16, U32 = 2.0 ** -8, 2.0 ** -24
TINY16 = 2.0 ** -133  # the step of bf16's subnormals
SILU, GELU, GELU_TANH = 0, 1, 2
_erf = np.vectorize(math.erf, otypes=[np.float64])


def normal_cdf(g):
    return 0.5 * (1.0 + _erf(g * math.sqrt(0.5)))


def logistic(x):
    return 0.5 * (1.0 + np.tanh(0.5 * x))


def gate(g, act):
    """(act(g), act'(g))"""
    if act == SILU:
        p = logistic(g)
        return g * p, p + g * p * (1 - p)
    if act == GELU:
        p = normal_cdf(g)
        return g * p, p + g * np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    p = logistic(2 * c * (g + 0.044715 * g ** 3))
    return g * p, p + g * p * (1 - p) * 2 * c * (1 + 3 * 0.044715 * g ** 2)


def quantize_rows(x):
    """(q, scale) of a float32 array (bf16 widened): the fp32 quotients, the exact product to the nearest integer."""
    x = np.asarray(x, np.float32)
    bits = np.abs(x).max(axis=1).view(np.uint32)
    bits = np.maximum(bits, np.abs(x).view(np.uint32).max(axis=1))  # a NaN counts as the largest
    finite = bits < 0x7F800000
    top = np.where(finite, bits, 0).astype(np.uint32).view(np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        lift = np.where(top < np.float32(2.0 ** -100), np.float32(2.0 ** 100), np.float32(1))
        inverse = np.where(top > 0, np.float32(127) / (top * lift), np.float32(0))
        q = np.rint(np.where(finite[:, None], x, 0).astype(np.float64) * lift[:, None].astype(np.float64)
                    * inverse[:, None].astype(np.float64))
    return q.astype(np.int8), np.where(finite, top / np.float32(127), np.float32(np.nan)).astype(np.float32)


def scaled_product(a, b, row, col, bias):
    """(value, bound on the fp32 result): int32 sums are exact; the conversion to fp32, the two products and the
    addition of the bias each round once."""
    s = a.astype(np.float64) @ b.astype(np.float64).T * row.astype(np.float64)[:, None] * col.astype(np.float64)
    y = s + (0 if bias is None else bias.astype(np.float64))
    return y, 4 * U32 * (np.abs(s) + np.abs(y)) + 2.0 ** -149


def to_bf16_bound(y, fp32_bound):
    """The bound after one more rounding, to bf16."""
    return fp32_bound * (1 + U16) + U16 * np.abs(y) + TINY16


def sum_slack(k):
    return 2.0 ** -23 * (k / 16 + 2)


def products(x, w):
    """x w^T and the sum of magnitudes |x| |w|^T."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    return x @ w.T, np.abs(x) @ np.abs(w).T


def gated(g, u, eg, eu, act):
    """(h, bound) from exact pre-activations and bounds on their fp32 values.  |act'| <= 1.2 for all three; the fast
    exponential and division, or erfc, leave act(g) within 2^-19 relative and 2^-20 of |g| absolute."""
    a, _ = gate(g, act)
    ea = 1.2 * eg + 2.0 ** -19 * np.abs(a) + 2.0 ** -20 * np.minimum(np.abs(g), 1.0)
    h = a * u
    eh = ea * np.abs(u) + np.abs(a) * eu + ea * eu + 2 * U32 * np.abs(h)
    return h, to_bf16_bound(h, eh)


def gate_backward(g, u, dh, act):
    """(dg, du, bound dg, bound du): elementwise in fp32, rounded once to bf16."""
    a, slope = gate(g, act)
    dg, du = dh * u * slope, dh * a
    # slope: the fast functions' error against terms of size up to 1 + |g p (1 - p)|
    e_slope = 2.0 ** -18 * (1.0 + np.abs(slope))
    return (dg, du, to_bf16_bound(dg, np.abs(dh * u) * e_slope),
            to_bf16_bound(du, np.abs(dh) * (2.0 ** -19 * np.abs(a) + 2.0 ** -20 * np.minimum(np.abs(g), 1.0))))
