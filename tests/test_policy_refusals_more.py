"""More arguments of the token-policy operators that are refused before anything is launched.  Runs without a GPU."""
import struct

import pytest

from test_policy_refusals import L, P, refused, rules, shape


@pytest.mark.parametrize("least", [2.0 ** -149, 2.0 ** -130, 2.0 ** -128, 2.0 ** -127, 1e-50])
def test_divisors_without_a_finite_reciprocal(least):
    refused(shape(r=rules(repetition=least)), "repetition")
    refused(shape(r=rules(temperature=least)), "temperature")


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_more_work_items_than_a_dispatch_counts(dtype):
    """2^32 work items or more would wrap round: the least refused numbers of rows, and some far beyond."""
    stats = lambda rows, vocab: L.ppo_xp_action_stats(0, None, dtype, P, vocab, P, P, P, rows, vocab, P, 1 << 60)  # noqa: E731
    batch = struct.pack("6Q", *(P,) * 6)
    loss = lambda rows, vocab: L.ppo_xp_policy_loss(0, None, dtype, P, vocab, batch, 0.2, 0.01, 0.5, 1.0, P, vocab, P, P, P, P, rows, vocab,  # noqa: E731
                                                    P, 1 << 60)
    back = lambda rows, vocab: L.ppo_xp_shape_logits_backward(0, None, dtype, P, vocab, P, vocab, P, vocab, rows, vocab, rules())  # noqa: E731
    for rows in (1 << 24, (1 << 24) + 8, 1 << 31, 1 << 40, (1 << 64) - 1):
        refused(stats(rows, 2056), "too many")                     # a workgroup of 256 a row
        refused(shape(dtype=dtype, rows=rows, vocab=16384, ls=16384, os_=16384), "too many")
        refused(back(rows, 16384), "too many")
        refused(loss(rows, 150000), "too many")                    # 1024 threads a row
    refused(loss(1 << 22, 150000 if dtype else 70000), "too many")
    refused(stats(1 << 31, 100), "too many")
    refused(stats(1 << 31, 2), "too many")
    refused(shape(dtype=dtype, rows=1 << 16, vocab=1 << 30, ls=1 << 30, os_=1 << 30), "too many")


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_more_stored_rows_than_a_dispatch_counts(dtype):
    for n in (1 << 34, 1 << 62, (1 << 64) - 1):
        refused(L.ppo_xp_quantize_rows(0, None, dtype, P, 64, n, 64, 1, 64, P, 64, P, 1, (1 << 64) - 1, 0), "too many")
        refused(L.ppo_xp_dequantize_rows(0, None, dtype, P, 64, P, 1, 8, 64, 1, 64, P, 32, 0, n, P, 64), "too many")
    # 2^33 units of 8 elements, two a lane; 2^34 of 16 bytes, four a lane
    refused(L.ppo_xp_quantize_rows(0, None, dtype, P, 64, 1 << 30, 64, 1, 64, P, 64, P, 1, 1 << 40, 0), "too many")
    n = (1 << 34) // (16 if dtype == 0 else 8)
    refused(L.ppo_xp_dequantize_rows(0, None, dtype, P, 64, P, 1, 8, 64, 1, 64, P, 32, 0, n, P, 64), "too many")


def test_denominators_without_a_finite_reciprocal():
    batch = struct.pack("6Q", *(P,) * 6)
    for denom in (2.0 ** -128, 1e-39, 1e-300, 5e-324):
        refused(L.ppo_xp_policy_loss(0, None, 0, P, 100, batch, 0.2, 0.01, 0.5, denom, P, 100, P, P, P, P, 4, 100, P, 1 << 40), "denom")
