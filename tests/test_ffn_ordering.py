"""Ordering between the lanes of a warp in the feed-forward kernels.  What these rules prevent shows on a GPU by chance
or not at all, so they are held against the source; the results of the paths concerned are compared on the GPU beside
them."""
import os
import re

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "exo_b200", "csrc")


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def body(text, start):
    """The braces that open after `start`, with what is between them."""
    at = text.index("{", text.index(start))
    depth = 0
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end + 1]
    raise AssertionError(start)


def test_gathered_rows_are_read_behind_a_warp_barrier():
    """cp.async.wait_group makes a lane's own copies visible to that lane.  place() also reads the vector that the next
    lane copied: between the two stands a barrier of the warp, which orders memory (a vote does not), and another one
    stands before the slot is filled again."""
    loop = body(source("ffn_tc.cu"), "for (int i = 0; i < n_kb; i++) {\n    fetch(")
    wait, place = loop.index("cp_async_wait<G_DEPTH - 1>()"), loop.index(".place(")
    assert "__syncwarp()" in loop[wait:place]
    assert "__syncwarp()" in loop[loop.rindex(".place("):]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(7, 300, 1003), (32, 1000, 4099), (17, 4099, 513)])
def test_gathered_products_repeat_exactly(M, N, K):
    """int8 sums are whole numbers, so each of many calls on new operands has one right answer."""
    import torch

    import exo_b200

    lib = exo_b200.library()
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    c = torch.empty(M, N, device="cuda")
    for _ in range(40):
        a, b = (torch.randint(-11, 12, (r, K), generator=g, device="cuda", dtype=torch.int8) for r in (M, N))
        lib.gemm_i8_scaled_f32_exo(None, M, N, K, a, b, one_m, one_n, None, c)
        # sums of at most 4099 * 121 are exact in fp32, too
        assert np.array_equal(c.double().cpu().numpy(), (a.double() @ b.double().T).cpu().numpy())
