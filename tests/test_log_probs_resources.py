"""What the compiler makes of the kernels for log-probabilities: registers, scratch memory, and the requests of the product with a score's or a
gradient's epilogue, which obey what the other products' do."""
import re

import pytest
from test_kernel_resources import compiled, csrc, resources


def test_row_kernels_keep_out_of_scratch():
    kernels = resources("log_probs.hip")
    assert len(kernels) > 30
    for name, r in kernels.items():
        assert r["ScratchSize"] == 0 and r["VGPRs Spill"] == 0, (name, r)


def test_products_with_an_epilogue_of_their_own():
    """No scratch and no LDS of their own, two waves per SIMD; every kernel with requests in its code is one that the build looks at."""
    from picotron_amd import build
    kernels, assembly = compiled(csrc("linear_log_probs.hip"))
    looked_at = {name for name in kernels if re.search(build.REQUESTING["linear_log_probs.hip"], name)}
    assert len(looked_at) == 14
    for name, r in kernels.items():
        body = assembly[assembly.index(f"\n{name}:"):]
        assert (" lds\n" in body[:body.index(".Lfunc_end")]) == (name in looked_at), name
        assert r["ScratchSize"] == 0 and r["VGPRs Spill"] == 0, (name, r)
        if name in looked_at:
            assert r["LDS Size"] == 0 and r["Occupancy"] >= 2, (name, r)


def test_requests_find_their_aim_in_m0():
    import test_kernel_resources
    test_kernel_resources.test_requests_find_their_aim_in_m0("linear_log_probs.hip")
