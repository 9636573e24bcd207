"""Feed-forward operators: int8 products with token and channel scales, gated projections, their backward pass.
Plain float64 oracle in tests/ffn_oracle.py; the bounds are derived there."""
import os
import subprocess
import sys

import numpy as np
import pytest

from tests import ffn_oracle as fo
from tests import inputs
from tests.guard import Guarded

bf16_bits, widen = inputs.f32_to_bf16_bits, inputs.bf16_bits_to_f32


@pytest.fixture(scope="module")
def lib():
    from exo_b200 import build

    build.build()
    import exo_b200

    return exo_b200.library()


def normal(seed, shape, std=1.0):
    """float32 values that are bf16 values"""
    return widen(inputs.normal_bf16(seed, shape, std))


def int8_operand(seed, rows, k):
    return inputs.int8(seed, (rows, k), -127, 127), np.exp(inputs.uniform_f32(seed + 1, (rows,))) * np.float32(0.01)


def close(got, want, bound):
    got = np.asarray(got, np.float64)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], np.broadcast_to(bound, want.shape)[bad][:4])


# ------------------------------------------------------------------ refusals (no GPU needed)
def operands(name, sizes, change=None):
    """Host operands of the right types and shapes for an entry point."""
    from exo_b200 import _lib

    dtypes = {"bf16": np.uint16, "i8": np.int8, "f32": np.float32}
    return [np.ones([sizes[d] for d in dims], dtypes[kind]) for kind, _, dims in _lib.SIGNATURES[name][1]]


SIZES = {"quantize_rows_bf16_exo": [3, 5], "quantize_rows_f32_exo": [3, 5], "gemm_i8_scaled_bf16_exo": [3, 4, 5],
         "gemm_i8_scaled_f32_exo": [3, 4, 5], "linear_i8_bf16_exo": [3, 4, 5], "linear_i8_f32_exo": [3, 4, 5],
         "gated_bf16_exo": [0, 3, 4, 5], "gated_bf16_backward_exo": [0, 3, 4, 5], "gated_i8_bf16_exo": [0, 3, 4, 5]}


@pytest.mark.parametrize("name", SIZES)
def test_sizes_and_missing_operands_are_refused(lib, name):
    import exo_b200
    from exo_b200 import _lib

    sizes = SIZES[name]
    ops = operands(name, sizes)
    before = [o.copy() for o in ops]
    first = 1 if name.startswith("gated") else 0
    for i in range(first, len(sizes)):
        for wrong in (0, -1):
            bad = sizes[:i] + [wrong] + sizes[i + 1:]
            with pytest.raises((exo_b200.ExoB200Error, ValueError)):
                getattr(lib, name)(None, *bad, *ops)
            # the C entry point itself, without the wrapper's check of the element counts
            getattr(lib.dll, name)(None, *bad, *[o.ctypes.data for o in ops])
            assert lib.dll.exo_b200_last_error() == exo_b200.ERR_INVALID_ARGUMENT
    for i, (_, optional, _) in enumerate(_lib.SIGNATURES[name][1]):
        if optional:
            continue
        with pytest.raises(exo_b200.ExoB200Error) as e:
            getattr(lib, name)(None, *sizes, *ops[:i], None, *ops[i + 1:])
        assert e.value.code == exo_b200.ERR_INVALID_ARGUMENT
    assert all(np.array_equal(a, b) for a, b in zip(ops, before))


@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_wrong_types_and_counts(lib, name):
    import torch

    sizes = SIZES[name]
    ops = operands(name, sizes)
    for i, o in enumerate(ops):
        for wrong in (o.astype(np.float64), np.ones(o.size + 1, o.dtype), torch.ones(o.size, dtype=torch.float64), 3):
            with pytest.raises(ValueError):
                getattr(lib, name)(None, *sizes, *ops[:i], wrong, *ops[i + 1:])
        if o.ndim == 2:
            with pytest.raises(ValueError):  # not dense
                getattr(lib, name)(None, *sizes, *ops[:i], np.ones(o.shape[::-1], o.dtype).T, *ops[i + 1:])


def test_other_refusals(lib):
    import exo_b200

    def code(name, *args):
        with pytest.raises(exo_b200.ExoB200Error) as e:
            getattr(lib, name)(None, *args)
        return e.value.code

    for name in ("gated_bf16_exo", "gated_bf16_backward_exo", "gated_i8_bf16_exo"):
        for act in (-1, 3):
            assert code(name, act, 3, 4, 5, *operands(name, SIZES[name])) == exo_b200.ERR_INVALID_ARGUMENT
    ops = operands("gated_bf16_exo", SIZES["gated_bf16_exo"])
    assert code("gated_bf16_exo", 0, 3, 4, 5, *ops[:5], None) == exo_b200.ERR_INVALID_ARGUMENT  # G without U
    ops = operands("gated_bf16_backward_exo", SIZES["gated_bf16_backward_exo"])
    assert code("gated_bf16_backward_exo", 0, 3, 4, 5, *ops[:10], None) == exo_b200.ERR_INVALID_ARGUMENT
    # int32 sums
    K = 131072
    a, s = np.zeros((1, K), np.int8), np.ones(1, np.float32)
    assert code("gemm_i8_scaled_f32_exo", 1, 1, K, a, a, s, s, None, s.copy()) == exo_b200.ERR_UNSUPPORTED
    assert code("gated_i8_bf16_exo", 0, 1, 1, K, a, a, a, s, s, s, np.zeros(1, np.uint16)) == exo_b200.ERR_UNSUPPORTED
    assert code("linear_i8_f32_exo", 1, 1, K, np.ones((1, K), np.float32), a, s, None, a.copy(), s.copy(), s.copy()) \
        == exo_b200.ERR_UNSUPPORTED
    # an address that is not a multiple of the element
    raw = np.zeros(64, np.uint8)
    x = raw[1:1 + 4 * 8].view(np.float32).reshape(2, 4)
    assert code("quantize_rows_f32_exo", 2, 4, x, np.zeros((2, 4), np.int8), np.zeros(2, np.float32)) \
        == exo_b200.ERR_INVALID_ARGUMENT


def test_a_valid_call_without_a_device_is_an_error(lib):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    import exo_b200

    for name, sizes in SIZES.items():
        ops = operands(name, sizes)
        before = [o.copy() for o in ops]
        with pytest.raises(exo_b200.ExoB200Error) as e:
            getattr(lib, name)(None, *sizes, *ops)
        assert e.value.code in (exo_b200.ERR_CUDA, exo_b200.ERR_UNSUPPORTED)
        assert all(np.array_equal(a, b) for a, b in zip(ops, before))


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("act", [fo.SILU, fo.GELU, fo.GELU_TANH])
def test_oracle_slopes_are_the_differences(act):
    g = np.linspace(-9, 9, 301)
    h = 1e-5
    numeric = (fo.gate(g + h, act)[0] - fo.gate(g - h, act)[0]) / (2 * h)
    assert np.abs(numeric - fo.gate(g, act)[1]).max() < 1e-8


# ------------------------------------------------------------------ on the GPU
def dev(a):
    import torch

    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def dev_shifted(a, elements=1):
    """On the device, `elements` off a 16-byte boundary."""
    import torch

    t = dev(a)
    room = torch.empty(t.numel() + 16, dtype=t.dtype, device="cuda")
    view = room[elements:elements + t.numel()].view(t.shape)
    view.copy_(t)
    return view


def out(shape, kind, offset=0):
    import torch

    return Guarded(torch, shape, {"bf16": torch.int16, "f32": torch.float32, "i8": torch.int8}[kind], offset=offset)


def values(g):
    assert g.bands_intact()
    a = g.view.cpu().numpy()
    return widen(a.view(np.uint16)) if a.dtype == np.int16 else a


QUANT_SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 33), (130, 1000), (7, 4099), (2, 40000), (300, 128), (4, 16384), (5, 8200),
                (3, 32768), (1300, 512), (1301, 1000), (1200, 2040), (1250, 77), (3, 2056)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M,K", QUANT_SHAPES)
def test_quantize_rows(lib, M, K, kind):
    x = normal(M + K, (M, K), 3.0) if kind == "bf16" else inputs.uniform_f32(M + K, (M, K)) * np.float32(5)
    if M >= 3:
        x[1] = 0
        x[2] *= np.float32(1e-30)
    if kind == "bf16":
        x = widen(bf16_bits(x))  # what the kernel is given
    want_q, want_s = fo.quantize_rows(x)
    q, s = out((M, K), "i8"), out((M,), "f32")
    fn = lib.quantize_rows_bf16_exo if kind == "bf16" else lib.quantize_rows_f32_exo
    fn(None, M, K, dev(bf16_bits(x) if kind == "bf16" else x), q.view, s.view)
    assert np.array_equal(values(q), want_q)
    assert np.array_equal(values(s), want_s)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [8, 100, 4096, 9000])
def test_quantize_rows_extremes(lib, K):
    """Ties, subnormal rows, the largest values, infinities, NaN, a largest magnitude that is negative."""
    x = inputs.uniform_f32(K, (10, K))
    x[0] = np.float32(127) * np.float32(0.5)
    x[0, :4] = [127, 0.5, 1.5, -2.5]          # exact ties go to even
    x[1] = np.float32(1e-45)                  # the smallest subnormal: its scale underflows to zero
    x[2] = np.float32(1e-41) * x[2]
    x[3, 0] = np.finfo(np.float32).max
    x[4, K // 2] = np.inf
    x[5, K - 1] = np.nan
    x[6, 0], x[6, 1] = -np.inf, np.nan
    x[7, 3] = -8
    x[8] = 0
    x[9] = -np.float32(2.0 ** -100)
    want_q, want_s = fo.quantize_rows(x)
    assert want_q[0, :4].tolist() == [127, 0, 2, -2] and not want_q[4:7].any()
    q, s = out((10, K), "i8"), out((10,), "f32")
    lib.quantize_rows_f32_exo(None, 10, K, dev(x), q.view, s.view)
    assert np.array_equal(values(q), want_q)
    assert np.array_equal(values(s), want_s, equal_nan=True)


# sizes around the tiles and vectors of the kernels, one token to many, long and short reductions
PRODUCT_SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 1024), (2, 300, 17), (7, 129, 255), (16, 512, 2048), (17, 4099, 513),
                  (33, 64, 4096), (64, 200, 96), (100, 1000, 1000), (128, 128, 64), (129, 257, 1040), (257, 513, 384),
                  (300, 2048, 512), (1024, 1024, 256), (1500, 777, 131), (2048, 2304, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", PRODUCT_SHAPES)
def test_gemm_i8_scaled(lib, M, N, K, kind, bias):
    a, row = int8_operand(M + K, M, K)
    b, col = int8_operand(N + K + 7, N, K)
    add = inputs.uniform_f32(3, (N,)) if bias else None
    want, bound = fo.scaled_product(a, b, row, col, add)
    c = out((M, N), kind)
    fn = lib.gemm_i8_scaled_bf16_exo if kind == "bf16" else lib.gemm_i8_scaled_f32_exo
    fn(None, M, N, K, dev(a), dev(b), dev(row), dev(col), None if add is None else dev(add), c.view)
    close(values(c), want, bound if kind == "f32" else fo.to_bf16_bound(want, bound))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 40), (130, 300)])
def test_gemm_i8_scaled_largest_sums(lib, M, N):
    """-128 * -128 over the longest reduction stays below 2^31."""
    K = 131071
    a, b = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    one_m, one_n = np.ones(M, np.float32), np.ones(N, np.float32)
    c = out((M, N), "f32")
    lib.gemm_i8_scaled_f32_exo(None, M, N, K, dev(a), dev(b), dev(one_m), dev(one_n), None, c.view)
    assert (values(c) == np.float32(131071 * 16384)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (5, 130, 100), (17, 4099, 513), (200, 384, 1024), (1000, 640, 77)])
def test_linear_i8_is_the_two_calls(lib, M, N, K, kind):
    x = normal(M, (M, K)) if kind == "bf16" else inputs.uniform_f32(M, (M, K))
    x = x.copy()
    if M > 4:
        x[2] = 0
        x[3, K // 2] = np.nan
    dx = dev(bf16_bits(x) if kind == "bf16" else x)
    b, col = int8_operand(N + K, N, K)
    add = dev(inputs.uniform_f32(4, (N,)))
    db, dcol = dev(b), dev(col)
    q, s, y = out((M, K), "i8"), out((M,), "f32"), out((M, N), kind)
    q2, s2, y2 = out((M, K), "i8"), out((M,), "f32"), out((M, N), kind)
    getattr(lib, f"linear_i8_{kind}_exo")(None, M, N, K, dx, db, dcol, add, q.view, s.view, y.view)
    getattr(lib, f"quantize_rows_{kind}_exo")(None, M, K, dx, q2.view, s2.view)
    getattr(lib, f"gemm_i8_scaled_{kind}_exo")(None, M, N, K, q2.view, db, s2.view, dcol, add, y2.view)
    assert np.array_equal(values(q), values(q2)) and np.array_equal(values(s), values(s2), equal_nan=True)
    assert np.array_equal(values(y), values(y2), equal_nan=True)
    want_q, want_s = fo.quantize_rows(x)
    assert np.array_equal(values(q), want_q)
    got = values(y)
    if M > 4:
        assert np.isnan(got[3]).all() and np.array_equal(got[2], got[2]) and np.isfinite(np.delete(got, 3, 0)).all()
    fine = np.isfinite(want_s)
    want, bound = fo.scaled_product(want_q[fine], b, want_s[fine], col, inputs.uniform_f32(4, (N,)))
    close(got[fine], want, bound if kind == "f32" else fo.to_bf16_bound(want, bound))


GATED_SHAPES = [(1, 1, 1), (1, 256, 512), (1, 4100, 1024), (3, 65, 31), (16, 512, 1000), (17, 1025, 513), (64, 64, 64),
                (100, 300, 130), (128, 1024, 256), (129, 127, 264), (300, 513, 96), (1000, 1030, 513), (512, 640, 2048),
                (2048, 1216, 192)]


def gated_inputs(M, F, K):
    """float32 (x, wg, wu) that are bf16 values; pre-activations of a few units"""
    std = 1.5 / np.sqrt(K)
    return normal(M + 1, (M, K)), normal(F + 2, (F, K), std), normal(F + K + 3, (F, K), std)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("M,F,K", GATED_SHAPES)
def test_gated_bf16(lib, M, F, K, keep):
    act = (M + F + K) % 3
    x, wg, wu = gated_inputs(M, F, K)
    (g, gm), (u, um) = fo.products(x, wg), fo.products(x, wu)
    eg, eu = fo.sum_slack(K) * gm, fo.sum_slack(K) * um
    want, bound = fo.gated(g, u, eg, eu, act)
    h = out((M, F), "bf16")
    kept = [out((M, F), "bf16"), out((M, F), "bf16")] if keep else [None, None]
    lib.gated_bf16_exo(None, act, M, F, K, dev(bf16_bits(x)), dev(bf16_bits(wg)), dev(bf16_bits(wu)), h.view,
                       *[k and k.view for k in kept])
    close(values(h), want, bound)
    if keep:
        close(values(kept[0]), g, fo.to_bf16_bound(g, eg))
        close(values(kept[1]), u, fo.to_bf16_bound(u, eu))


@pytest.mark.gpu
@pytest.mark.parametrize("act", [fo.SILU, fo.GELU, fo.GELU_TANH])
def test_gated_bf16_range_of_gates(lib, act):
    """Gates from -1e30 to 1e30, through a reduction of length one."""
    g = np.concatenate([np.linspace(-12, 12, 180), [1e30, -1e30, 88, -88, 104, -104, 1e-30, -1e-30, 0, 30, -30, 1e13]])
    g = widen(bf16_bits(g.astype(np.float32)))
    F = g.size
    h = out((1, F), "bf16")
    one = bf16_bits(np.ones((1, 1), np.float32))
    up = bf16_bits(np.full((F, 1), 2, np.float32))
    lib.gated_bf16_exo(None, act, 1, F, 1, dev(one), dev(bf16_bits(g[:, None])), dev(up), h.view, None, None)
    with np.errstate(over="ignore"):
        g64 = np.clip(g.astype(np.float64), -1e3, 1e3) if act == fo.GELU_TANH else g.astype(np.float64)
        p = fo.gate(g64, act)[0] / np.where(g64 == 0, 1, g64)
    want = 2 * g.astype(np.float64) * p
    close(values(h)[0], want, fo.to_bf16_bound(want, 2.0 ** -18 * np.abs(want) + 2.0 ** -19 * np.minimum(np.abs(g), 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", GATED_SHAPES)
def test_gated_i8(lib, M, F, K):
    act = (M + F + K) % 3
    a, row = int8_operand(M + K, M, K)
    bg, sg = int8_operand(F + 5, F, K)
    bu, su = int8_operand(F + 9, F, K)
    row = row / np.float32(K ** 0.5 / 4)
    g, eg = fo.scaled_product(a, bg, row, sg, None)
    u, eu = fo.scaled_product(a, bu, row, su, None)
    want, bound = fo.gated(g, u, eg, eu, act)
    h = out((M, F), "bf16")
    lib.gated_i8_bf16_exo(None, act, M, F, K, dev(a), dev(bg), dev(bu), dev(row), dev(sg), dev(su), h.view)
    close(values(h), want, bound)


BACKWARD_SHAPES = [(1, 1, 1), (1, 256, 128), (3, 65, 31), (17, 1025, 513), (64, 64, 64), (100, 300, 130), (129, 127, 264),
                   (128, 1024, 256), (300, 513, 96), (512, 640, 1024), (1000, 520, 777), (2048, 1216, 192)]


def backward_oracle(x, wg, wu, g, u, dh, act):
    """Outputs and bounds.  The products take dG and dU as the library rounded them, so the bound of each carries the
    elementwise bound through the sum."""
    dg, du, eg, eu = fo.gate_backward(*(t.astype(np.float64) for t in (g, u, dh)), act)
    x, wg, wu = (t.astype(np.float64) for t in (x, wg, wu))
    M, F = dg.shape
    want = {"dg": dg, "du": du, "dx": dg @ wg + du @ wu, "dwg": dg.T @ x, "dwu": du.T @ x}
    ax, ag, au = np.abs(x), np.abs(wg), np.abs(wu)
    mg, mu = np.abs(dg) + eg, np.abs(du) + eu
    raw = {"dx": eg @ ag + eu @ au + fo.sum_slack(2 * F) * (mg @ ag + mu @ au),
           "dwg": eg.T @ ax + fo.sum_slack(M) * (mg.T @ ax), "dwu": eu.T @ ax + fo.sum_slack(M) * (mu.T @ ax)}
    bound = {"dg": eg, "du": eu} | {k: fo.to_bf16_bound(want[k], raw[k]) for k in raw}
    return want, bound


def run_backward(lib, M, F, K, act, x, wg, wu, g, u, dh, skip=()):
    shapes = {"dg": (M, F), "du": (M, F), "dx": (M, K), "dwg": (F, K), "dwu": (F, K)}
    outs = {k: None if k in skip else out(s, "bf16") for k, s in shapes.items()}
    lib.gated_bf16_backward_exo(None, act, M, F, K, *(dev(bf16_bits(t)) for t in (x, wg, wu, g, u, dh)),
                                *[o and o.view for o in outs.values()])
    return {k: values(o) for k, o in outs.items() if o}


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", BACKWARD_SHAPES)
def test_gated_backward(lib, M, F, K):
    act = (M + F + K) % 3
    x, wg, wu = gated_inputs(M, F, K)
    g, u, dh = normal(5, (M, F), 2.0), normal(6, (M, F)), normal(7, (M, F), 0.01)
    want, bound = backward_oracle(x, wg, wu, g, u, dh, act)
    got = run_backward(lib, M, F, K, act, x, wg, wu, g, u, dh)
    for k in want:
        close(got[k], want[k], bound[k])
    # what is not asked for is not computed, the rest is the same
    for skip in (("dx",), ("dwg", "dwu"), ("dx", "dwg", "dwu")):
        part = run_backward(lib, M, F, K, act, x, wg, wu, g, u, dh, skip)
        assert set(part) == set(want) - set(skip)
        assert all(np.array_equal(part[k], got[k]) for k in part)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [fo.SILU, fo.GELU, fo.GELU_TANH])
def test_gated_backward_against_differences(lib, act):
    """The derivative of sum(dH * H) along random directions of X, Wg, Wu against central differences of the float64
    forward pass (step 2^-12: truncation and the gradients' bf16 roundings stay below 3 * 2^-8 of the sum of
    magnitudes)."""
    M, F, K = 24, 40, 32
    x, wg, wu = gated_inputs(M, F, K)
    dh = normal(7, (M, F))
    f64 = lambda *t: [v.astype(np.float64) for v in t]
    xs, gs, us, ds = f64(x, wg, wu, dh)
    g, u = xs @ gs.T, xs @ us.T
    # the kept pre-activations are bf16: the gradient is taken at those
    got = run_backward(lib, M, F, K, act, x, wg, wu, widen(bf16_bits(g.astype(np.float32))),
                       widen(bf16_bits(u.astype(np.float32))), dh)
    loss = lambda x, wg, wu: float((ds * fo.gate(x @ wg.T, act)[0] * (x @ wu.T)).sum())
    for name, at in (("dx", 0), ("dwg", 1), ("dwu", 2)):
        d = inputs.uniform_f32(at + 1, (xs, gs, us)[at].shape).astype(np.float64)
        step, point = 2.0 ** -12, [xs, gs, us]
        hi, lo = list(point), list(point)
        hi[at], lo[at] = point[at] + step * d, point[at] - step * d
        numeric = (loss(*hi) - loss(*lo)) / (2 * step)
        terms = got[name].astype(np.float64) * d
        assert abs(terms.sum() - numeric) <= 3 * fo.U16 * np.abs(terms).sum(), (name, terms.sum(), numeric)


@pytest.mark.gpu
def test_unaligned_operands(lib):
    """Bases one element off a 16-byte boundary, outputs too: the same values as aligned ones."""
    M, F, K = 70, 200, 136
    a, row = int8_operand(1, M, K)
    b, col = int8_operand(2, F, K)
    b2, col2 = int8_operand(3, F, K)
    x, wg, wu = gated_inputs(M, F, K)
    g, u, dh = normal(5, (M, F)), normal(6, (M, F)), normal(7, (M, F), 0.01)
    results = []
    for put, off in ((dev, 0), (dev_shifted, 1)):
        res = {}
        for kind, e in (("bf16", 2), ("f32", 4)):
            c = out((M, F), kind, offset=off * e)
            getattr(lib, f"gemm_i8_scaled_{kind}_exo")(None, M, F, K, put(a), put(b), put(row), put(col), None, c.view)
            res["c" + kind] = values(c)
            q, s = out((M, K), "i8", offset=off), out((M,), "f32", offset=4 * off)
            xs = put(bf16_bits(x)) if kind == "bf16" else put(x)
            getattr(lib, f"quantize_rows_{kind}_exo")(None, M, K, xs, q.view, s.view)
            res["q" + kind], res["s" + kind] = values(q), values(s)
        h = out((M, F), "bf16", offset=2 * off)
        lib.gated_i8_bf16_exo(None, 0, M, F, K, put(a), put(b), put(b2), put(row), put(col), put(col2), h.view)
        res["h8"] = values(h)
        h, kg, ku = (out((M, F), "bf16", offset=2 * off) for _ in range(3))
        bits = [put(bf16_bits(t)) for t in (x, wg, wu, g, u, dh)]
        lib.gated_bf16_exo(None, 0, M, F, K, *bits[:3], h.view, kg.view, ku.view)
        res |= {"h": values(h), "g": values(kg), "u": values(ku)}
        outs = [out(s, "bf16", offset=2 * off) for s in ((M, F), (M, F), (M, K), (F, K), (F, K))]
        lib.gated_bf16_backward_exo(None, 0, M, F, K, *bits, *[o.view for o in outs])
        res |= {f"b{i}": values(o) for i, o in enumerate(outs)}
        results.append(res)
    for k in results[0]:
        assert np.array_equal(results[0][k], results[1][k]), k


@pytest.mark.gpu
def test_host_operands(lib):
    """numpy arrays in and out give what device tensors give; so does a mixture."""
    M, F, K = 33, 100, 64
    a, row = int8_operand(1, M, K)
    b, col = int8_operand(2, F, K)
    bias = inputs.uniform_f32(3, (F,))
    c = out((M, F), "f32")
    lib.gemm_i8_scaled_f32_exo(None, M, F, K, dev(a), dev(b), dev(row), dev(col), dev(bias), c.view)
    host = np.full((M, F), 7, np.float32)
    lib.gemm_i8_scaled_f32_exo(None, M, F, K, a, b, row, col, bias, host)
    assert np.array_equal(host, values(c))
    host[:] = 7
    lib.gemm_i8_scaled_f32_exo(None, M, F, K, a, dev(b), row, dev(col), bias, host)
    assert np.array_equal(host, values(c))
    x, wg, wu = gated_inputs(M, F, K)
    g, u, dh = normal(5, (M, F)), normal(6, (M, F)), normal(7, (M, F), 0.01)
    bits = [bf16_bits(t) for t in (x, wg, wu, g, u, dh)]
    outs = [np.full(s, 7, np.uint16) for s in ((M, F), (M, F), (M, K), (F, K), (F, K))]
    lib.gated_bf16_backward_exo(None, 1, M, F, K, *bits, *outs)
    want = run_backward(lib, M, F, K, 1, x, wg, wu, g, u, dh)
    for got, k in zip(outs, ("dg", "du", "dx", "dwg", "dwu")):
        assert np.array_equal(widen(got), want[k])


@pytest.mark.gpu
def test_feed_forward_block(lib):
    """The operators together, as a block runs them: trained in bf16 (gated projections, down projection, backward),
    served in int8 (quantise, gated, linear), against the block in float64."""
    import torch

    M, F, K = 96, 512, 256
    x, wg, wu = gated_inputs(M, F, K)
    wd = normal(9, (K, F), 1 / np.sqrt(F))
    bits = [dev(bf16_bits(t)) for t in (x, wg, wu)]
    h, g, u, y = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((M, F), (M, F), (M, F), (M, K)))
    lib.gated_bf16_exo(None, fo.SILU, M, F, K, *bits, h, g, u)
    lib.gemm_bf16_exo(None, M, K, F, h, dev(bf16_bits(wd)), y)
    f64 = [t.astype(np.float64) for t in (x, wg, wu, wd)]
    g64, u64 = f64[0] @ f64[1].T, f64[0] @ f64[2].T
    h64 = fo.gate(g64, fo.SILU)[0] * u64
    y64 = h64 @ f64[3].T
    mag = np.abs(h64) @ np.abs(f64[3]).T
    # H is rounded once (2^-8) before the down projection, Y once more
    close(y.float().cpu().numpy(), y64, 1.1 * fo.U16 * mag + fo.U16 * np.abs(y64))
    # backward from dY: dH = dY Wd, with its weight transposed for the library's column-major product
    dy = normal(11, (M, K), 0.1)
    dh, dg, du = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    lib.gemm_bf16_exo(None, M, F, K, dev(bf16_bits(dy)), dev(np.ascontiguousarray(bf16_bits(wd).T)), dh)
    dx = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    dwg, dwu = (torch.empty(F, K, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lib.gated_bf16_backward_exo(None, fo.SILU, M, F, K, *bits, g, u, dh, dg, du, dx, dwg, dwu)
    k = lambda t: t.float().cpu().numpy()
    want, bound = backward_oracle(x, wg, wu, k(g), k(u), k(dh), fo.SILU)
    for name, t in (("dg", dg), ("du", du), ("dx", dx), ("dwg", dwg), ("dwu", dwu)):
        close(k(t), want[name], bound[name])
    # int8
    qw = [fo.quantize_rows(t) for t in (wg, wu, wd)]
    dq = [(dev(a), dev(s)) for a, s in qw]
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    q2, s2 = torch.empty(M, F, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    lib.quantize_rows_bf16_exo(None, M, K, bits[0], q, s)
    lib.gated_i8_bf16_exo(None, fo.SILU, M, F, K, q, dq[0][0], dq[1][0], s, dq[0][1], dq[1][1], h)
    lib.linear_i8_bf16_exo(None, M, K, F, h, dq[2][0], dq[2][1], None, q2, s2, y)
    wide = lambda a, s: a.astype(np.float64) * s.astype(np.float64)[:, None]
    x8, (g8, u8, d8) = wide(*fo.quantize_rows(x)), [wide(*t) for t in qw]
    pre = x8 @ g8.T
    want_h = fo.gate(pre, fo.SILU)[0] * (x8 @ u8.T)
    close(k(h), want_h, fo.to_bf16_bound(want_h, 2.0 ** -16 * (np.abs(want_h) + np.abs(x8 @ u8.T))))
    h8 = wide(*fo.quantize_rows(k(h)))
    close(k(y), h8 @ d8.T, fo.to_bf16_bound(h8 @ d8.T, 2.0 ** -20 * (np.abs(h8) @ np.abs(d8).T)))


def graph_of(calls, stream):
    import torch

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        for f in calls:
            f()
    return g


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", [(4, 256, 512), (40, 77, 129)])
def test_captured_calls_replay_on_new_inputs(lib, M, F, K):
    """Every entry point captured into a graph, replayed after its inputs change (an unaligned pitch included), with an
    eager call of larger sizes in between; two graphs alive at once keep apart."""
    import torch

    stream = torch.cuda.Stream()
    x, wg, wu = (dev(bf16_bits(t)) for t in gated_inputs(M, F, K))
    g, u, dh = (dev(bf16_bits(normal(s, (M, F)))) for s in (5, 6, 7))
    b, col = (dev(t) for t in int8_operand(2, F, K))
    b2, col2 = (dev(t) for t in int8_operand(3, F, K))

    def buffers():
        e = lambda t, *s: torch.zeros(s, dtype=t, device="cuda")
        h, i = torch.int16, torch.int8
        return [e(i, M, K), e(torch.float32, M), e(h, M, F), e(h, M, F), e(h, M, F), e(h, M, F), e(h, M, F), e(h, M, F),
                e(h, M, F), e(h, M, K), e(h, F, K), e(h, F, K)]

    def calls(o):
        return [lambda: lib.linear_i8_bf16_exo(None, M, F, K, x, b, col, None, o[0], o[1], o[2]),
                lambda: lib.gated_i8_bf16_exo(None, 0, M, F, K, o[0], b, b2, o[1], col, col2, o[3]),
                lambda: lib.gated_bf16_exo(None, 1, M, F, K, x, wg, wu, o[4], o[5], o[6]),
                lambda: lib.gated_bf16_backward_exo(None, 2, M, F, K, x, wg, wu, g, u, dh, *o[7:12])]

    one, two, eager = buffers(), buffers(), buffers()
    with torch.cuda.stream(stream):
        for f in calls(eager):
            f()
    stream.synchronize()
    g1, g2 = graph_of(calls(one), stream), graph_of(calls(two), stream)
    for seed in (21, 22):
        x.copy_(dev(bf16_bits(normal(seed, (M, K)))))
        dh.copy_(dev(bf16_bits(normal(seed + 1, (M, F)))))
        torch.cuda.synchronize()
        g1.replay()
        big = [torch.zeros(s, dtype=torch.int16, device="cuda") for s in ((131, 515), (777, 515), (777, 515), (131, 777))]
        lib.gated_bf16_exo(None, 0, 131, 777, 515, *big, None, None)
        g2.replay()
        for f in calls(eager):
            f()
        torch.cuda.synchronize()
        for a, c, d in zip(one, two, eager):
            assert torch.equal(a, d) and torch.equal(c, d)


FIRST_CALL = """
import sys, torch
sys.path.insert(0, {root!r})
import exo_b200
lib = exo_b200.library()
M, F, K = 40, 77, 129  # copies of operands, too
x, w, v = (torch.randn(s, device="cuda").bfloat16() for s in ((M, K), (F, K), (F, K)))
h, g, u = (torch.zeros(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(3))
eager = torch.zeros_like(h)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    lib.gated_bf16_exo(None, 0, M, F, K, x, w, v, h, g, u)
graph.replay()
torch.cuda.synchronize()
lib.gated_bf16_exo(None, 0, M, F, K, x, w, v, eager, None, None)
torch.cuda.synchronize()
assert torch.equal(h, eager) and float(h.float().abs().sum()) > 0
print("captured")
"""


@pytest.mark.gpu
def test_the_first_call_of_a_process_may_be_captured(lib):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_threads_share_the_default_context(lib):
    """Two host threads, each on its own stream with its own operands (copies among them), through the one default
    context."""
    import threading

    import torch

    M, F, K = 50, 333, 257
    x = [dev(bf16_bits(normal(s, (M, K)))) for s in (1, 2)]
    _, wg, wu = (dev(bf16_bits(t)) for t in gated_inputs(M, F, K))
    want, got, failed = [], [], []
    for xi in x:
        want.append(torch.zeros(M, F, dtype=torch.int16, device="cuda"))
        got.append([torch.zeros(M, F, dtype=torch.int16, device="cuda") for _ in range(50)])
        lib.gated_bf16_exo(None, 0, M, F, K, xi, wg, wu, want[-1], None, None)
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for o in got[i]:
                    lib.gated_bf16_exo(None, 0, M, F, K, x[i], wg, wu, o, None, None)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.gpu
def test_infinities_and_nans_stay_in_their_rows(lib):
    """A token, a channel or a gradient that is not finite spoils its own row or column of the products and no other,
    at sizes that end inside tiles and vectors."""
    import torch

    for M, F, K in ((3, 77, 129), (20, 100, 136), (40, 131, 75), (300, 520, 264)):
        x, wg, wu = (t.copy() for t in gated_inputs(M, F, K))
        x[1, K - 1] = np.inf
        wg[F - 1, K - 1] = np.nan
        h = out((M, F), "bf16")
        lib.gated_bf16_exo(None, 0, M, F, K, dev(bf16_bits(x)), dev(bf16_bits(wg)), dev(bf16_bits(wu)), h.view, None, None)
        got = values(h)
        fine = np.ones((M, F), bool)
        fine[1] = fine[:, F - 1] = False
        assert np.isfinite(got[fine]).all() and np.isnan(got[:, F - 1]).all(), (M, F, K)
        g, u, dh = normal(5, (M, F)), normal(6, (M, F)), normal(7, (M, F), 0.01)
        dh[M - 1, F - 1] = np.inf
        x, wg, wu = gated_inputs(M, F, K)
        res = run_backward(lib, M, F, K, 0, x, wg, wu, g, u, dh)
        for name, row in (("dx", M - 1), ("dwg", F - 1), ("dwu", F - 1)):
            ok = np.isfinite(res[name]).all(axis=1)
            assert not ok[row] and np.delete(ok, row).all(), (name, M, F, K)


@pytest.mark.gpu
def test_host_operands_are_refused_while_capturing(lib):
    import torch

    import exo_b200

    stream = torch.cuda.Stream()
    x, q, s = np.ones((2, 8), np.float32), torch.zeros(2, 8, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda")
    keep = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        keep += 1
        with pytest.raises(exo_b200.ExoB200Error) as e:
            lib.quantize_rows_f32_exo(None, 2, 8, x, q, s)
    assert e.value.code == exo_b200.ERR_UNSUPPORTED
    graph.replay()
    torch.cuda.synchronize()
    assert float(keep) == 1.0


@pytest.mark.gpu
def test_streams_and_contexts(lib):
    """Calls on two streams and through two contexts at once, operands with odd pitches: each gets its own result."""
    import torch

    import exo_b200

    M, F, K = 50, 333, 257
    x, wg, wu = (dev(bf16_bits(t)) for t in gated_inputs(M, F, K))
    x2 = dev(bf16_bits(normal(99, (M, K))))
    want = [torch.zeros(M, F, dtype=torch.int16, device="cuda") for _ in range(2)]
    for xi, w in zip((x, x2), want):
        lib.gated_bf16_exo(None, 0, M, F, K, xi, wg, wu, w, None, None)
    torch.cuda.synchronize()
    for contexts in ((None, None), (exo_b200.Context(), exo_b200.Context())):
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [torch.zeros(M, F, dtype=torch.int16, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(20):
            for c, s, xi, o in zip(contexts, streams, (x, x2), got):
                with torch.cuda.stream(s):
                    lib.gated_bf16_exo(c, 0, M, F, K, xi, wg, wu, o, None, None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", SIZES)
def test_wrapper_refuses_wrong_device_tensors(lib, name):
    """The compiled path hands what it does not take to the Python path, which says what is wrong; errors of the entry
    point itself come back through it."""
    import torch

    import exo_b200

    sizes = SIZES[name]
    types = {"uint16": torch.bfloat16, "int8": torch.int8, "float32": torch.float32}
    ops = [torch.ones(o.shape, dtype=types[str(o.dtype)], device="cuda") for o in operands(name, sizes)]
    for i, o in enumerate(ops):
        wrong = [o.double(), torch.cat([o.flatten(), o.flatten()[:1]]), 3, "x"]
        if o.dim() == 2:
            wrong.append(torch.ones(o.shape[::-1], dtype=o.dtype, device="cuda").T)
        for w in wrong:
            with pytest.raises(ValueError):
                getattr(lib, name)(None, *sizes, *ops[:i], w, *ops[i + 1:])
    with pytest.raises(exo_b200.ExoB200Error) as e:
        getattr(lib, name)(None, *sizes, None, *ops[1:])
    assert e.value.code == exo_b200.ERR_INVALID_ARGUMENT
    with pytest.raises((exo_b200.ExoB200Error, ValueError)):
        getattr(lib, name)(None, *[0] * len(sizes), *ops)
    with pytest.raises(TypeError):
        getattr(lib, name)(None, *sizes, *ops[1:])
    with pytest.raises(ValueError):
        getattr(lib, name)(None, *sizes, *ops, stream=1)
    getattr(lib, name)(None, *sizes, *ops)
    getattr(lib, name)(None, *(np.int64(n) for n in sizes), *ops)  # through the Python path


@pytest.mark.gpu
def test_entry_points_of_both_wrappers_agree_on_the_stream(lib):
    """A checked and an unchecked entry point called in turn on two streams: each enqueues on its caller's."""
    import torch

    n = 256
    w = torch.nn.Parameter(torch.randn(n, n, device="cuda").bfloat16(), requires_grad=False)
    x, h, y = (torch.randn(n, n, device="cuda").bfloat16() for _ in range(3))
    want = {}
    streams = [torch.cuda.Stream(), torch.cuda.current_stream(), torch.cuda.Stream()]
    for rep in range(4):
        for s in streams:
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                h.zero_(), y.zero_()
                lib.gated_bf16_exo(None, 0, n, n, n, x, w, w, h, None, None)
                lib.gemm_bf16_exo(None, n, n, n, h, w.data, y)
                got = y.float().sum()
            s.synchronize()
            want.setdefault("y", float(got))
            assert float(got) == want["y"] != 0.0


# ------------------------------------------------------------------ sizes of the large kernels, oracle on the GPU in float64
def gpu_close(got, want, bound):
    import torch

    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], want[bad][:4])


def gpu_normal(seed, *shape, std=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()


def gpu_int8(seed, rows, k):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int8),
            torch.rand(rows, generator=g, device="cuda") * 0.02 + 0.001)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,kind", [(4096, 4096, 8192, "bf16"), (4100, 3990, 8208, "bf16"), (4099, 4001, 8191, "bf16"),
                                        (3000, 2600, 6400, "f32"), (512, 4096, 4096, "bf16"), (520, 4000, 4000, "f32"),
                                        (300, 700, 20000, "bf16"), (20, 100, 65536, "f32")])
def test_gemm_i8_scaled_large(lib, M, N, K, kind):
    import torch

    (a, row), (b, col) = gpu_int8(1, M, K), gpu_int8(2, N, K)
    bias = torch.randn(N, device="cuda")
    c = torch.empty(M, N, dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
    getattr(lib, f"gemm_i8_scaled_{kind}_exo")(None, M, N, K, a, b, row, col, bias, c)
    s = a.double() @ b.double().T * row.double()[:, None] * col.double()
    want = s + bias.double()
    bound = 4 * fo.U32 * (s.abs() + want.abs())
    gpu_close(c, want, bound if kind == "f32" else bound * (1 + fo.U16) + fo.U16 * want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", [(4096, 4096, 2048), (4100, 4104, 1000), (3500, 4097, 2001), (5, 9000, 200), (4200, 300, 260)])
def test_gated_backward_large(lib, M, F, K):
    """The bounds of backward_oracle, with the products of magnitudes on the GPU."""
    import torch

    x, wg, wu = gpu_normal(1, M, K), gpu_normal(2, F, K, std=0.02), gpu_normal(3, F, K, std=0.02)
    g, u, dh = gpu_normal(4, M, F), gpu_normal(5, M, F), gpu_normal(6, M, F, std=0.01)
    e = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
    dg, du, dx, dwg, dwu = e(M, F), e(M, F), e(M, K), e(F, K), e(F, K)
    lib.gated_bf16_backward_exo(None, fo.SILU, M, F, K, x, wg, wu, g, u, dh, dg, du, dx, dwg, dwu)
    g, u, dh, x, wg, wu = (t.double() for t in (g, u, dh, x, wg, wu))
    p = torch.sigmoid(g)
    a, slope = g * p, p + g * p * (1 - p)
    wdg, wdu = dh * u * slope, dh * a
    half = lambda y, err: err * (1 + fo.U16) + fo.U16 * y.abs() + fo.TINY16
    eg = half(wdg, (dh * u).abs() * 2.0 ** -18 * (1 + slope.abs()))
    eu = half(wdu, dh.abs() * (2.0 ** -19 * a.abs() + 2.0 ** -20 * g.abs().clamp_max(1)))
    gpu_close(dg, wdg, eg)
    gpu_close(du, wdu, eu)
    mg, mu = wdg.abs() + eg, wdu.abs() + eu
    want = wdg @ wg + wdu @ wu
    gpu_close(dx, want, half(want, eg @ wg.abs() + eu @ wu.abs() + fo.sum_slack(2 * F) * (mg @ wg.abs() + mu @ wu.abs())))
    for got, d, ed, md in ((dwg, wdg, eg, mg), (dwu, wdu, eu, mu)):
        want = d.T @ x
        gpu_close(got, want, half(want, ed.T @ x.abs() + fo.sum_slack(M) * (md.T @ x.abs())))


@pytest.mark.gpu
@pytest.mark.parametrize("M,F,K", [(4096, 4096, 1024), (4099, 4103, 520), (1024, 1024, 4096), (1, 16384, 4095), (20, 6000, 3001)])
def test_gated_large(lib, M, F, K):
    import torch

    x, wg, wu = gpu_normal(1, M, K), gpu_normal(2, F, K, std=0.02), gpu_normal(3, F, K, std=0.02)
    h, g, u = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    lib.gated_bf16_exo(None, fo.SILU, M, F, K, x, wg, wu, h, g, u)
    x, wg, wu = (t.double() for t in (x, wg, wu))
    wantg, wantu = x @ wg.T, x @ wu.T
    eg, eu = (fo.sum_slack(K) * (x.abs() @ w.abs().T) for w in (wg, wu))
    half = lambda y, err: err * (1 + fo.U16) + fo.U16 * y.abs() + fo.TINY16
    gpu_close(g, wantg, half(wantg, eg))
    gpu_close(u, wantu, half(wantu, eu))
    a = wantg * torch.sigmoid(wantg)
    ea = 1.2 * eg + 2.0 ** -19 * a.abs() + 2.0 ** -20 * wantg.abs().clamp_max(1)
    want = a * wantu
    gpu_close(h, want, half(want, ea * wantu.abs() + a.abs() * eu + ea * eu + 2 * fo.U32 * want.abs()))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(lib):
    """More than 2^31 elements in an output, an input and a weight; rows at both ends and around the border."""
    import torch

    M, N, K = 70000, 33000, 16
    (a, row), (b, col) = gpu_int8(1, M, K), gpu_int8(2, N, K)
    c = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    lib.gemm_i8_scaled_bf16_exo(None, M, N, K, a, b, row, col, None, c)
    rows = torch.tensor([0, 1, 2 ** 31 // N - 1, 2 ** 31 // N, 2 ** 31 // N + 1, M - 1], device="cuda")
    s = a[rows].double() @ b.double().T * row[rows].double()[:, None] * col.double()
    gpu_close(c[rows], s, 8 * fo.U32 * s.abs() * 2 + fo.U16 * s.abs())
    del c
    M, K = 40000, 60000  # X and Q
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda").normal_()
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    lib.quantize_rows_bf16_exo(None, M, K, x, q, s)
    rows = [0, 2 ** 31 // K, 2 ** 31 // K + 1, M - 1]
    want_q, want_s = fo.quantize_rows(x[rows].float().cpu().numpy())
    assert np.array_equal(q[rows].cpu().numpy(), want_q) and np.array_equal(s[rows].cpu().numpy(), want_s)
    del x
    # Q as the weight of a few tokens: the last channels lie beyond 2^31
    for m in (2, 24):
        t, ts = gpu_int8(5, m, K)
        y = torch.empty(m, M, device="cuda")
        lib.gemm_i8_scaled_f32_exo(None, m, M, K, t, q, ts, s, None, y)
        want = t.double() @ q[rows].double().T * ts.double()[:, None] * s[rows].double()
        gpu_close(y[:, rows], want, 8 * fo.U32 * want.abs() * 2)


VARIANTS = {
    "split kernel": {"EXOB200_FFN_PAIR": "0", "EXOB200_FFN_ROWS": "0"},
    "pairs": {"EXOB200_FFN_PAIR": "1", "EXOB200_FFN_TALL": "0", "EXOB200_FFN_ROWS": "0"},
    "tall tiles": {"EXOB200_FFN_PAIR": "1", "EXOB200_FFN_TALL": "1", "EXOB200_FFN_ROWS": "0"},
    "two pairs a tile": {"EXOB200_FFN_PAIR": "2", "EXOB200_FFN_ROWS": "0"},
    "copied operands, plain launches": {"EXOB200_FFN_GATHER": "0", "EXOB200_FFN_ROWS": "0", "EXOB200_PDL": "0"},
}


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
def test_every_kernel_at_every_size(variant):
    """The sizes above with each kernel forced (in a process of its own: the switches are read once)."""
    names = "test_gemm_i8_scaled or test_linear or test_gated or unaligned or captured or block"
    r = subprocess.run([sys.executable, "-m", "pytest", __file__, "-x", "-q", "-m", "gpu", "-k",
                        f"({names}) and not large and not every_kernel"], capture_output=True, text=True,
                       env={**os.environ, **VARIANTS[variant]}, timeout=600)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]
