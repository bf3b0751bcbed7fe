"""CPU: objects of the operators for requests that branch that no call would take are refused when they are made."""

import pytest


def test_more_rows_or_tokens_than_a_selection_takes(hm):
    for args in ((65536, 1, 1, 10), (16384, 4, 4, 10), (256, 256, 4, 10), (1, 1, 1, 2 ** 24 + 1)):
        with pytest.raises(ValueError, match="BeamStep: at most"):
            hm.BeamStep(*args, "cpu")
    assert hm.BeamStep(65535, 1, 1, 10, "cpu").tokens.shape == (65535, 1)
    hm.BeamStep(1, 4, 4, 2 ** 24, "cpu")


def test_more_requests_than_a_fork_takes(hm):
    with pytest.raises(ValueError, match="4096 requests"):
        hm.PageFork(4097, 4, 16, "cpu")
    hm.PageFork(4096, 4, 16, "cpu")


@pytest.mark.parametrize("page_size", [0, 1, 8, 17, 48, -16, 2 ** 31])
def test_page_sizes(hm, page_size):
    for make in (lambda p: hm.PageFork(3, 4, p, "cpu"), lambda p: hm.PageCompact(9, p, "cpu"), lambda p: hm.SharePlan(3, p, 8, 2, "cpu")):
        with pytest.raises(ValueError, match="page_size"):
            make(page_size)
        make(16)
