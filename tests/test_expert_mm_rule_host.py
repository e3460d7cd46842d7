"""The rule of expert_mm_rule.h on a device of 256 CUs: which calls the kernel of few rows takes."""
import pytest

from tests.mm_kernel_choice import FORWARD, ROWS, SWIGLU, WEIGHTS, takes_few


@pytest.mark.parametrize("kind,experts,rows,n,k,few", [
    # one token's experts, a decode step, a few rows an expert however many tiles they are
    (SWIGLU, 8, 8, 4096, 7168, True), (FORWARD, 32, 256, 7168, 2048, True), (FORWARD, 32, 257, 7168, 2048, False),
    # little to multiply
    (SWIGLU, 8, 256, 4096, 7168, True), (SWIGLU, 1, 512, 4096, 7168, True), (FORWARD, 8, 200, 720, 520, True),
    # a prompt, a training step
    (SWIGLU, 32, 8192, 4096, 7168, False), (FORWARD, 32, 16384, 4096, 2048, False), (SWIGLU, 1, 1024, 4096, 7168, False),
    # the rows' gradient: only where tiles are not enough for the CUs
    (ROWS, 8, 512, 4096, 2048, True), (ROWS, 1, 512, 4096, 4096, True), (ROWS, 32, 512, 4096, 2048, False), (ROWS, 32, 16384, 4096, 2048, False),
    # the weights' gradient: tiles for half the CUs at most, or rows that are few for the weights
    (WEIGHTS, 8, 400, 720, 520, True), (WEIGHTS, 1, 4096, 1024, 1024, True), (WEIGHTS, 3, 1500, 2048, 2048, False),
    (WEIGHTS, 32, 32, 4096, 2048, True), (WEIGHTS, 32, 512, 4096, 2048, True), (WEIGHTS, 32, 2048, 4096, 2048, False),
])
def test_which_kernel(kind, experts, rows, n, k, few):
    assert takes_few(kind, experts, rows, n, k, 256) == few


@pytest.mark.parametrize("kind", [FORWARD, SWIGLU, ROWS, WEIGHTS])
def test_the_ends_of_the_range(kind):
    """The smallest call goes to the kernel of few rows and the largest to the other; products of the sizes do not pass 64 bits."""
    assert takes_few(kind, 1, 1, 16, 8, 256)
    most = (1 << 31) - 1
    assert not takes_few(kind, 1024, most, 1 << 20, 1 << 20, 256)
    assert takes_few(kind, 1, most, 16, 8, 256) == (kind == WEIGHTS)
