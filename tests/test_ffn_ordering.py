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


def test_warps_come_together_before_aligned_instructions():
    """Cluster barriers and the allocation, release and loads of tensor memory are .sync.aligned: all lanes of a warp
    execute them together.  Behind code in which lanes go different ways (rows past M, columns past N, one lane that
    stores or reports) a barrier of the warp brings them back."""
    for name, functions in (("umma.cuh", ("tmem_alloc", "tmem_dealloc")),
                            ("umma_pair.cuh", ("cluster_sync_all", "tmem_alloc2", "tmem_dealloc2"))):
        for f in functions:
            inside = body(source(name), f"void {f}(")
            assert "__syncwarp();" in inside[:inside.index("asm")], f
    text = source("ffn_tc.cu")
    put = body(text, "void put(const uint32_t (&w)[WORDS]")
    assert re.search(r"__syncwarp\(\);\s*}$", put)
    # (the one return in front is the whole warp's: the block's first row and column)
    assert put.count("return;") == 1 and "if (row0 >= p.M || col >= p.N) return;" in put
    drain = body(text, "for (int ch = 0; ch < 4; ch++)")
    assert re.search(r"__syncwarp\(\);\s*}$", drain) and "if (m0 + row < p.M)" in drain


@pytest.mark.gpu
@pytest.mark.parametrize("K", [64, 640, 4096])
@pytest.mark.parametrize("N", [5, 66, 300, 2312])
@pytest.mark.parametrize("M", [33, 97, 129, 515])
def test_products_that_end_inside_a_warp(M, N, K):
    """Lanes of one warp inside and outside the output, with one CTA and several CTAs to a tile."""
    import torch

    import exo_b200

    lib = exo_b200.library()
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, b = (torch.randint(-11, 12, (r, K), generator=g, device="cuda", dtype=torch.int8) for r in (M, N))
    c = torch.empty(M, N, device="cuda")
    lib.gemm_i8_scaled_f32_exo(None, M, N, K, a, b, torch.ones(M, device="cuda"), torch.ones(N, device="cuda"), None, c)
    assert torch.equal(c.double(), a.double() @ b.double().T)


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
