"""Workspaces of a serving step's calls for counts that 32 bits do not hold."""
import pytest

from qwen35_amd import adapters, sampling


@pytest.mark.parametrize("big", [2**31, 2**32, 2**32 + 4, 2**40 + 8, -2**32 + 8])
def test_counts_beyond_32_bits_are_refused(big):
    for rows, vocab in ((big, 100), (4, big)):
        with pytest.raises(ValueError, match="unsupported"):
            sampling.sample_workspace(rows, vocab, device="cpu")
    for tokens, rank in ((big, 16), (4, big)):
        with pytest.raises(ValueError, match="unsupported"):
            adapters.adapters_workspace(tokens, rank, device="cpu")


def test_counts_that_are_taken():
    assert sampling.sample_workspace(4, 100, device="cpu").numel() > 0
    assert adapters.adapters_workspace(5, 16, device="cpu").numel() > 0
