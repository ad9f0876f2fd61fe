"""More arguments of the token-policy operators that are refused before anything is launched.  Runs without a GPU."""
import pytest

from test_policy_refusals import refused, rules, shape


@pytest.mark.parametrize("least", [2.0 ** -149, 2.0 ** -130, 2.0 ** -128, 2.0 ** -127, 1e-50])
def test_divisors_without_a_finite_reciprocal(least):
    refused(shape(r=rules(repetition=least)), "repetition")
    refused(shape(r=rules(temperature=least)), "temperature")
