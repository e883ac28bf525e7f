"""Column sums of the norms' gradients where a workgroup takes several turns of rows (more rows than 512 workgroups have at once), at every
number of lanes that a row has: widths to 512, 1024, 2048, 4096 and 8192, multiples of eight and others. Bounds of
test_gpu_norm.py, against float64."""
import pytest
import torch

from test_gpu_norm import TYPES, check, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stream,branch", TYPES)
@pytest.mark.parametrize("width", [505, 512, 513, 645, 1024, 1032, 2050, 2048, 3001, 4096, 4104])
def test_sums_over_several_turns(width, stream, branch):
    rows = 5003 if width <= 512 else 1541 if width > 4096 else 2563
    v = lambda s: rand(s, width, gain=0.3, shift=1.0)  # noqa: E731
    x, y = rand(1, rows, width, dtype=stream, gain=2, shift=0.5), rand(2, rows, width, dtype=branch)
    check(x, y, v(3), v(4), v(5), v(6), v(7), "layer", 0.7, 0.1)
    check(x, y, v(3), None, v(5), None, v(7), "rms", 1.0, 0.0)
    check(x, y, v(3), None, None, None, rand(8, rows, width, dtype=branch), "rms", 1.0, 0.0)
