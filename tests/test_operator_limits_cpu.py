"""Sizes at the ends of the integers that the checkpoint entry points take: refused before anything is launched."""
import pytest

from pacednegatives_amd import _lib

A = 4096            # a 16-byte aligned address that is never followed


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("T", [2 ** 31 - 63, 2 ** 31 - 33, 2 ** 31 - 1])
def test_token_counts_that_do_not_round_up_to_whole_blocks_within_an_int(lib, T):
    assert lib.paced_act8_quantize(A, 16, A, A, T, 16, None) == -1 and "2147483584" in lib.paced_last_error().decode()
    assert lib.paced_act8_dequantize(A, A, A, 16, T, 16, None) == -1 and "2147483584" in lib.paced_last_error().decode()
    assert lib.paced_act8_dweight(A, 8, 0, A, A, A, 16, T, 8, 16, 0, A, 1 << 60, None) == -1 and "2147483584" in lib.paced_last_error().decode()
    assert lib.paced_act8_dweight_workspace_bytes(T, 8, 16) == 0


def test_the_largest_token_count_has_a_plan(lib):
    need = lib.paced_act8_dweight_workspace_bytes(2 ** 31 - 64, 8, 16)
    assert 0 < need <= 64 * 8 * 16 * 4


def test_the_loss_asks_for_the_statistics_that_it_writes(lib):
    """A float pair for a row and 64 columns, 32 only where 64x64 tiles take the product; a float a row for the label."""
    up = lambda b: (b + 255) // 256 * 256  # noqa: E731
    for R, V, d, width in ((8192, 50001, 1024, 64), (131072, 50001, 1024, 64), (1088, 32128, 768, 64), (16, 32128, 768, 32), (64, 32128, 768, 32), (100, 300, 64, 32)):
        assert lib.paced_linear_ce_fwd_workspace_bytes_for(R, V, d) == up(-(-V // width) * R * 8) + up(R * 4), (R, V, d)
        assert lib.paced_linear_ce_fwd_workspace_bytes_for(R, V, d) <= lib.paced_linear_ce_fwd_workspace_bytes(R, V)
    assert lib.paced_linear_ce_fwd_workspace_bytes_for(0, 5, 64) == lib.paced_linear_ce_fwd_workspace_bytes_for(5, 0, 64) == lib.paced_linear_ce_fwd_workspace_bytes_for(5, 5, 0) == 0
    lib.paced_gemm_set_tile(64)
    try:
        assert lib.paced_linear_ce_fwd_workspace_bytes_for(8192, 50001, 1024) == lib.paced_linear_ce_fwd_workspace_bytes(8192, 50001)
    finally:
        lib.paced_gemm_set_tile(0)
