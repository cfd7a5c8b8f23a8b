"""Rules of the sampler that its source or its plan show: what goes wrong without them takes a timing, or a row, that
no ordinary test makes."""
import ctypes as C

import pytest

from starter_b200._lib import check, lib
from tests.test_kernel_waits import between, source


def test_the_count_of_listed_values_is_cleared_after_every_thread_has_read_it():
    """collect() copies as many entries as sh.found says: a warp that reads it after thread 0 has cleared it would
    leave its entries out of a list that counts them. Cleared again before the cluster meets, since the next values
    are pushed behind that."""
    collect = between(source("sampling.cu"), "auto collect = [&]", "\n  };\n")
    read, cleared = collect.index("found = sh.found;"), collect.index("sh.found = 0;")
    assert collect.count("sh.found") == 2
    assert "__syncthreads();" in collect[:read], "the pushes are not complete"
    assert "__syncthreads();" in collect[read:cleared], "other warps may not have read the count yet"
    assert "cluster_sync();" in collect[cleared:], "the next push could come first"


@pytest.mark.parametrize("aligned", [0, 1])
@pytest.mark.parametrize("fp32", [0, 1])
def test_the_values_of_a_cta_fit_their_sums(fp32, aligned):
    """A histogram's masses are kept in pieces of 15 bits that add up in 32: 2^17 values of the largest piece do, a few
    more do not. Stretches are rounded up to whole vectors, so that a row of 2^17, 2^18 or 2^19 values leaves a CTA more
    than its share."""
    ctas, values = C.c_int(), C.c_int()
    for vocab in [1, 2 ** 17 - 9, 2 ** 17, 2 ** 17 + 1, 151936, 2 ** 18 - 1, 2 ** 18, 2 ** 18 + 3, 400001, 2 ** 19 - 5, 2 ** 19]:
        for rows in (1, 17, 33, 64, 130, 1000):
            check(lib.q_sample_tokens_plan(fp32, rows, vocab, aligned, C.byref(ctas), C.byref(values)))
            assert ctas.value in (1, 2, 4, 8)
            assert ctas.value * values.value >= vocab
            assert values.value * (2 ** 15 - 1) < 2 ** 32, (rows, vocab, ctas.value, values.value)
            if aligned and rows == 64 and vocab == 2 ** 18:
                assert (ctas.value, values.value) == (2, 2 ** 17)               # (and no more CTAs than it takes)


def test_the_plan_refuses_what_the_call_refuses():
    n = C.c_int()
    for fp32, rows, vocab in ((0, 0, 10), (1, 1, 0), (0, 1, 2 ** 19 + 1), (0, 2 ** 24 + 1, 10)):
        with pytest.raises(ValueError):
            check(lib.q_sample_tokens_plan(fp32, rows, vocab, 0, C.byref(n), C.byref(n)))
    with pytest.raises(ValueError):
        check(lib.q_sample_tokens_plan(0, 1, 10, 0, None, C.byref(n)))
