"""Rules of the sampler that its source or its plan show: what goes wrong without them takes a timing, or a row, that
no ordinary test makes."""
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
