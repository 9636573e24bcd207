"""How the feed-forward entry points are called: memory that calls leave, what the wrapper refuses, the binding's
build."""
import numpy as np
import pytest

from tests.test_ffn import SIZES, operands


@pytest.fixture(scope="module")
def lib():
    from exo_b200 import build

    build.build()
    import exo_b200

    return exo_b200.library()


# ------------------------------------------------------------------ memory of operand copies
def test_trim_without_a_device_is_an_error(lib):
    import torch

    import exo_b200

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(exo_b200.ExoB200Error) as e:
        lib.trim()
    assert e.value.code in (exo_b200.ERR_CUDA, exo_b200.ERR_UNSUPPORTED)


@pytest.mark.gpu
def test_trim_gives_the_copies_memory_back(lib):
    """Weights of an odd pitch are copied into the context's pool, which keeps the memory for the next call until it is
    trimmed; what calls in a context of its own leave is that context's.  Results do not depend on it."""
    import torch

    import exo_b200

    M, F, K = 64, 16384, 4095  # 2 * 134 MB of copies
    x, wg, wu = (torch.randn(s, device="cuda").bfloat16() * 0.02 for s in ((M, K), (F, K), (F, K)))
    h, again = (torch.empty(M, F, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ctx = exo_b200.Context()

    def free():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[0]

    for c in (None, ctx):
        lib.trim(c)
        before = free()
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, h, None, None)
        kept = before - free()
        assert kept >= 2 * F * K * 2
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, again, None, None)
        assert before - free() == kept and torch.equal(h, again)
        lib.trim(c)
        # (a first call of a kernel may have loaded its code: some MB at most)
        assert before - free() < 64 << 20
        again.zero_()
        lib.gated_bf16_exo(c, 0, M, F, K, x, wg, wu, again, None, None)
        torch.cuda.synchronize()
        assert torch.equal(h, again)
        lib.trim(c)
    # trimmed while work is enqueued: its copies stay
    for _ in range(20):
        lib.gated_bf16_exo(None, 0, M, F, K, x, wg, wu, again, None, None)
        lib.trim()
    torch.cuda.synchronize()
    assert torch.equal(h, again)
    lib.trim()
