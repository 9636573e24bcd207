"""Feed-forward operators: values that are not finite, and gates far out in the activations' tails.  Oracle and bounds
as in tests/ffn_oracle.py where nothing else is said."""
import math

import numpy as np
import pytest

from tests import ffn_oracle as fo
from tests import inputs

bf16_bits, widen = inputs.f32_to_bf16_bits, inputs.bf16_bits_to_f32
ACTS = {"silu": fo.SILU, "gelu": fo.GELU, "gelu_tanh": fo.GELU_TANH}


@pytest.fixture(scope="module")
def lib():
    from exo_b200 import build

    build.build()
    import exo_b200

    return exo_b200.library()


def normal(seed, shape, std=1.0):
    """float32 values that are bf16 values"""
    return widen(inputs.normal_bf16(seed, shape, std))


def dev(x):
    import torch

    return torch.from_numpy(bf16_bits(np.asarray(x, np.float32)).view(np.int16)).cuda()


def backward(lib, act, x, wg, wu, g, u, dh):
    import torch

    (M, K), F = x.shape, wg.shape[0]
    outs = {k: torch.zeros(s, dtype=torch.int16, device="cuda")
            for k, s in (("dg", (M, F)), ("du", (M, F)), ("dx", (M, K)), ("dwg", (F, K)), ("dwu", (F, K)))}
    lib.gated_bf16_backward_exo(None, act, M, F, K, *(dev(t) for t in (x, wg, wu, g, u, dh)), *outs.values())
    return {k: widen(o.cpu().numpy().view(np.uint16)) for k, o in outs.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,F,K", [(20, 104, 136), (41, 131, 75)])  # elements by eights, and one by one
def test_what_is_not_finite_reaches_its_own_gradients(lib, M, F, K, act, value):
    """One element (m, f) of G, U or dH is NaN or an infinity.  dG and dU follow their formulas there, row m of dX and row
    f of the weight gradients are spoilt where a spoilt dG or dU enters them, and everything else is bit for bit what it
    is without."""
    x, wg, wu = normal(1, (M, K)), normal(2, (F, K), 0.1), normal(3, (F, K), 0.1)
    clean = {"g": normal(4, (M, F)), "u": normal(5, (M, F)), "dh": normal(6, (M, F), 0.01)}
    m, f = M - 3, F - 2
    for k in clean:
        clean[k][m, f] = 1.0  # so that no factor of the formulas is zero there
    args = lambda t: (x, wg, wu, t["g"], t["u"], t["dh"])
    base = backward(lib, ACTS[act], *args(clean))
    assert all(np.isfinite(t).all() for t in base.values())
    for where in clean:
        t = {k: v.copy() for k, v in clean.items()}
        t[where][m, f] = value
        got = backward(lib, ACTS[act], *args(t))
        dg, du = got["dg"][m, f], got["du"][m, f]
        if where == "g" and not np.isnan(value):
            # g p(g) and its slope at an infinity: the limit, or NaN where the formula is inf * 0 (torch's are NaN, too)
            limit = 1.0 if value > 0 else 0.0
            assert np.isnan(dg) or dg == limit, dg
            assert np.isnan(du) or du == (np.inf if value > 0 else 0.0), du
        elif np.isnan(value):
            assert np.isnan(dg) and (where == "u" or np.isnan(du)), (where, dg, du)
        else:  # the other factors are positive
            assert dg == value and (where == "u" or du == value), (where, dg, du)
        if where == "u":
            assert du == base["du"][m, f]
        spoilt = {"dx": (m, not (np.isfinite(dg) and np.isfinite(du))), "dwg": (f, not np.isfinite(dg)),
                  "dwu": (f, not np.isfinite(du))}
        for k, (row, bad) in spoilt.items():
            assert not bad or not np.isfinite(got[k][row]).any(), (where, k)
            assert np.array_equal(np.delete(got[k], row, 0), np.delete(base[k], row, 0)), (where, k)
            if np.isnan(value) and bad:
                assert np.isnan(got[k][row]).all(), (where, k)
        if where == "u":
            assert np.array_equal(got["dwu"], base["dwu"])
        rest = np.ones((M, F), bool)
        rest[m, f] = False
        assert all(np.array_equal(got[k][rest], base[k][rest]) for k in ("dg", "du")), where


# ------------------------------------------------------------------ tails
def tail_of(act):
    """Negative gates (bf16 values) out to where p(g) leaves fp32's normal range, and p there, from functions that keep
    their relative accuracy."""
    end = {"silu": -86.0, "gelu": -12.75, "gelu_tanh": -9.5}[act]
    g = np.unique(widen(bf16_bits(np.linspace(end, -0.015625, 700).astype(np.float32)))).astype(np.float64)
    if act == "gelu":
        p = np.array([0.5 * math.erfc(-v / math.sqrt(2)) for v in g])
        density = g * np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        z = g if act == "silu" else 2 * c * (g + 0.044715 * g ** 3)
        p = np.exp(z) / (1 + np.exp(z))
        density = g * p / (1 + np.exp(z)) * (1.0 if act == "silu" else 2 * c * (1 + 3 * 0.044715 * g ** 2))
    return g, p, density  # act'(g) = p + density


# Relative error of p in fp32: the argument of the exponential is at most 88, each of its up to four roundings costs
# 88 * 2^-24, and so does the product with log2(e) inside; the fast exponential and division 2^-22 each; the fitted
# coefficients of the normal distribution 2.6e-5.  Together below 6e-5 < 2^-14; the slope adds terms of the same kind.
TAIL = 2.0 ** -13


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("act", ACTS)
def test_activations_are_relatively_close_in_their_tails(lib, act, rows):
    """H = act(g) for gates through a reduction of length one, in the few-row kernel and in the tiles: one bf16 rounding
    and TAIL, relative to the value itself."""
    import torch

    g, p, _ = tail_of(act)
    h = torch.zeros(rows, g.size, dtype=torch.int16, device="cuda")
    one = np.ones((rows, 1), np.float32)
    lib.gated_bf16_exo(None, ACTS[act], rows, g.size, 1, dev(one), dev(g[:, None]), dev(np.ones((g.size, 1))), h, None, None)
    got = widen(h.cpu().numpy().view(np.uint16)).astype(np.float64)
    want = g * p
    bad = ~(np.abs(got - want) <= (fo.U16 * (1 + TAIL) + TAIL) * np.abs(want) + fo.TINY16)
    assert not bad.any(), (g[bad[0]][:4], got[0][bad[0]][:4], want[bad[0]][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_slopes_are_relatively_close_in_their_tails(lib, act):
    """dG = act'(g) and dU = act(g) (dH and U are one): relative to the magnitudes of the two terms of the slope."""
    g, p, density = tail_of(act)
    ones = np.ones((1, g.size), np.float32)
    x, w = np.ones((1, 1), np.float32), np.ones((g.size, 1), np.float32)
    got = backward(lib, ACTS[act], x, w, w, g[None], ones, ones)
    for k, want, size in (("dg", p + density, p + np.abs(density)), ("du", g * p, np.abs(g * p))):
        bad = ~(np.abs(got[k][0] - want) <= fo.U16 * (np.abs(want) + TAIL * size) + TAIL * size + fo.TINY16)
        assert not bad.any(), (k, g[bad][:4], got[k][0][bad][:4], want[bad][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
def test_gates_that_are_not_finite(lib, act):
    """A NaN token spoils its row of H, an infinite one gives what g p(g) u gives: inf for +inf, NaN or zero for -inf."""
    import torch

    x = np.array([[np.nan], [np.inf], [-np.inf], [1.0]], np.float32)
    for rows in (4, 64):
        a = np.concatenate([x, np.ones((rows - 4, 1), np.float32)])
        h = torch.zeros(rows, 40, dtype=torch.int16, device="cuda")
        # the up projection takes a second, finite channel: u = 0 * x would be NaN
        xs = np.concatenate([a, np.ones((rows, 1), np.float32)], 1)
        wg, wu = np.tile([[1.0, 0.0]], (40, 1)), np.tile([[1.0, 0.0]], (40, 1))
        lib.gated_bf16_exo(None, ACTS[act], rows, 40, 2, dev(xs), dev(wg), dev(wu), h, None, None)
        got = widen(h.cpu().numpy().view(np.uint16))
        assert np.isnan(got[0]).all() and (got[1] == np.inf).all() and np.isfinite(got[3:]).all()
        assert (np.isnan(got[2]) | (got[2] == 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [3, 20, 300])
def test_gated_i8_with_scales_that_are_not_finite(lib, act, M):
    """A row that could not be quantised has scale NaN: its row of H is NaN and no other; so is the column of a channel
    whose scale is NaN, and a gate that overflows to infinity gives what infinity gives."""
    import torch

    F, K = 200, 96
    one = torch.ones(M, K, dtype=torch.int8, device="cuda")
    w = torch.ones(F, K, dtype=torch.int8, device="cuda")
    row, gate, up = torch.full((M,), 0.01, device="cuda"), torch.ones(F, device="cuda"), torch.ones(F, device="cuda")
    row[1], gate[5], up[7], gate[9] = math.nan, math.nan, math.nan, math.inf
    h = torch.zeros(M, F, dtype=torch.bfloat16, device="cuda")
    lib.gated_i8_bf16_exo(None, ACTS[act], M, F, K, one, w, w, row, gate, up, h)
    got = h.float().cpu().numpy()
    bad = np.zeros((M, F), bool)
    bad[1] = bad[:, 5] = bad[:, 7] = True
    inf = np.zeros((M, F), bool)
    inf[:, 9] = ~bad[:, 9]
    assert np.isnan(got[bad]).all() and (got[inf] == np.inf).all() and np.isfinite(got[~bad & ~inf]).all()


# ------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("F", [33000, 33001])  # rows that TMA reads and stores, and rows that are copied and stored singly
def test_gated_tensors_beyond_32_bits(lib, F):
    """More than 2^31 elements in H, G, U and their gradients; rows at both ends and around the border, in float64."""
    import torch

    M, K = 66000, 24
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    g = torch.Generator(device="cuda").manual_seed(F)
    make = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda").mul_(std).bfloat16()
    x, wg, wu = make(M, K), make(F, K, std=0.2), make(F, K, std=0.2)
    h, pre, up = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    lib.gated_bf16_exo(None, fo.SILU, M, F, K, x, wg, wu, h, pre, up)
    border = 2 ** 31 // F
    rows = torch.tensor([0, 1, border - 1, border, border + 1, M - 1], device="cuda")
    half = lambda y, err: err * (1 + fo.U16) + fo.U16 * y.abs() + fo.TINY16

    def near(got, want, bound):
        bad = ~((got.double() - want).abs() <= bound)
        assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], want[bad][:4])

    xr, wgd, wud = x[rows].double(), wg.double(), wu.double()
    wantg, wantu = xr @ wgd.T, xr @ wud.T
    eg, eu = (fo.sum_slack(K) * (xr.abs() @ w.abs().T) for w in (wgd, wud))
    near(pre[rows], wantg, half(wantg, eg))
    near(up[rows], wantu, half(wantu, eu))
    a = wantg * torch.sigmoid(wantg)
    ea = 1.2 * eg + TAIL * a.abs()
    near(h[rows], a * wantu, half(a * wantu, ea * wantu.abs() + a.abs() * eu + ea * eu + 2 * fo.U32 * (a * wantu).abs()))
    # the backward pass, with H as the gradient of itself
    dg, du = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dx, dwg, dwu = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((M, K), (F, K), (F, K)))
    lib.gated_bf16_backward_exo(None, fo.SILU, M, F, K, x, wg, wu, pre, up, h, dg, du, dx, dwg, dwu)
    gr, ur, hr = (t[rows].double() for t in (pre, up, h))
    p = torch.sigmoid(gr)
    slope = p + gr * p * (1 - p)
    near(dg[rows], hr * ur * slope, half(hr * ur * slope, (hr * ur).abs() * TAIL * p * (1 + gr.abs())))
    near(du[rows], hr * gr * p, half(hr * gr * p, TAIL * (hr * gr * p).abs()))
    # the products take dG and dU as the library rounded them
    dgr, dur = dg[rows].double(), du[rows].double()
    want = dgr @ wgd + dur @ wud
    near(dx[rows], want, half(want, fo.sum_slack(2 * F) * (dgr.abs() @ wgd.abs() + dur.abs() @ wud.abs())))
    cols, xd = torch.tensor([0, 1, F // 2, F - 1], device="cuda"), x.double()
    for got, d in ((dwg, dg), (dwu, du)):
        d = d[:, cols].double().T
        near(got[cols], d @ xd, half(d @ xd, fo.sum_slack(M) * (d.abs() @ xd.abs())))
    del h, pre, up, dg, du
    lib.trim()
    torch.cuda.empty_cache()
