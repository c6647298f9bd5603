"""Limits of the products whose weights a row chooses (no GPU: the arguments are checked before the context)."""
import pytest

from test_rows import ADAPTER, GROUPED, ROUTE, call, lib, message


@pytest.mark.parametrize("sizes", [(5, 8, 9), (5, 64, 17), (5, 1024, 17), (5, 1025, 1), (2 ** 30, 8, 2), (5, 8, -1), (-5, 8, 1)], ids=str)
def test_no_router_workspace_for_sizes_that_are_refused(sizes):
    rows, experts, k = sizes
    assert call("sb_route_topk", ROUTE, rows=rows, experts=experts, ld=2000, k=k) == 11 and message() == "bad router shape"
    assert lib().sb_route_topk_workspace(*sizes) == 0


def test_a_router_workspace_for_every_size_that_is_taken():
    for rows in (1, 127, 129, 5000, 10 ** 6):
        for experts in (1, 2, 15, 16, 17, 1024):
            for k in {1, min(experts, 16)}:
                size = lib().sb_route_topk_workspace(rows, experts, k)
                assert size >= 16
                assert call("sb_route_topk", ROUTE, rows=rows, experts=experts, ld=experts, k=k, size=size) == 11 and message() == "ctx is null"


@pytest.mark.parametrize("M,rank", [(5, 12), (5, 4), (5, 127), (5, 136), (5, 0), (5, -8), (2 ** 31, 16)])
def test_no_adapter_workspace_for_sizes_that_are_refused(M, rank):
    assert call("sb_adapter_gemm", ADAPTER, M=M, rank=rank, N=1, ldo=8) == 11 and message() != "ctx is null"
    assert lib().sb_adapter_gemm_workspace(M, rank) == 0


@pytest.mark.parametrize("groups", [2 ** 31 - 1, 2 ** 31 - 127, 2 ** 31 - 512])
def test_groups_whose_walk_would_pass_32_bits_are_refused(groups):
    """The kernel steps through the groups 128 at a time in 32 bits: from 2^31 - 128 on the next step is negative, and an offset before the
    first one would be read."""
    assert call("sb_grouped_gemm", GROUPED, groups=groups, N=1, ldo=1) == 11 and message() == "bad product shape"


def test_the_most_groups():
    assert call("sb_grouped_gemm", GROUPED, groups=2 ** 31 - 513, N=1, ldo=1) == 11 and message() == "ctx is null"
