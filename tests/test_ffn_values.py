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
