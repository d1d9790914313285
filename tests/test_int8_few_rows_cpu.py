"""Which few rows of 8-bit integers go to the CUDA cores (csrc/rules.h), at sizes on both sides of what was measured."""
import pytest

from test_int8_rules_cpu import rules  # noqa: F401 (the fixture)


@pytest.mark.parametrize("m,n,k,of_8,of_16", [
    # two rows: from K = 513 on, up to 8 M elements of W, 16 M of rows up to 1024; below, tiles, as the weight-streaming planner starts at 511
    (2, 4096, 64, False, True), (2, 1024, 255, False, True), (2, 1024, 256, False, True), (2, 8192, 384, False, True), (2, 4096, 510, False, True),
    (2, 4096, 512, False, True), (2, 4096, 513, True, True), (2, 512, 768, True, True), (2, 16384, 768, True, True), (2, 16384, 1024, True, True),
    (2, 32768, 1024, False, True), (2, 4096, 2048, True, True), (2, 8192, 2048, False, True), (2, 1024, 8192, True, True), (2, 100, 81920, True, True),
    (2, 100, 81921, False, False), (2, 127, 512, True, True), (1, 16384, 256, True, True),
    # three and four in 16 bits: as long as W is small, and not in steps of one vector a lane
    (3, 4096, 256, False, False), (4, 1024, 512, False, False), (4, 1024, 513, False, True), (4, 1024, 4096, False, True), (4, 1025, 4096, False, False),
    (3, 4096, 1024, False, True), (5, 1024, 1024, False, False),
])
def test_which_rows_go_to_the_cuda_cores(rules, m, n, k, of_8, of_16):  # noqa: F811
    assert rules(m, n, k, False) == of_8 and rules(m, n, k, True) == of_16
