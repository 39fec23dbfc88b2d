"""Refusals of the microscaled calls' settings that need no GPU."""


def test_wait_limit_refusals(b200):
    limit = b200.lib().b200_mx_wait_limit
    assert limit(0, 3) == b200.ERR_INVALID_ARG
    assert limit(0, -1) == b200.ERR_INVALID_ARG
    assert limit(5_000_000, 0) == 0
    assert limit(0, 0) == 0
