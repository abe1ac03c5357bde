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
