"""Dropout of more elements than the counter's first word reaches."""
import pytest
import torch

from ivae_amd import ops
from tests.test_philox_cpu import words

pytestmark = pytest.mark.gpu


def test_the_counters_second_word():
    n = 2 ** 34 + 1003
    if torch.cuda.mem_get_info()[0] < 6 * n:
        pytest.skip("needs 100 GB of device memory")
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, .5, 3, 5)
    del x
    for first in (0, 2 ** 31 - 8, 2 ** 32 - 8, 2 ** 34 - 8, n - 100 - n % 4):
        got = (y[first:first + 100] != 0).cpu().tolist()
        draws = [v for q in range(first // 4, first // 4 + 25) for v in words((q % 2 ** 32, q >> 32, 5, 0), (3, 0))]
        assert got == [v >= 2 ** 31 for v in draws], first
    assert bool(y[-1] == 0) == (words((n // 4 % 2 ** 32, n // 4 >> 32, 5, 0), (3, 0))[(n - 1) % 4] < 2 ** 31)
    del y
    torch.cuda.empty_cache()
