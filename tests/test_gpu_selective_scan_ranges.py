"""The selective scan where magnitudes differ: between channels, between tokens, between a state and what enters it, and at the ends of the types' ranges."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from scan_reference import check_scan  # noqa: E402
from test_gpu_selective_scan import make, scan  # noqa: E402


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("least", [1e-39, 2.0 ** -126, 1e-30])
@pytest.mark.parametrize("seq", [20, 150, 1500])
def test_steps_of_next_to_nothing(ops, dtype, least, seq):
    # steps that are no normal float: nothing enters the state, and the logarithm of such a step is not to be taken for a number
    args = make(dtype, 1, 2, 64, 1, 64, seq)
    args["dt"] = args["dt"].clone()
    args["dt"][:, :, 3:17] = torch.finfo(args["dt"].dtype).min
    args["dt"][:, 1] = torch.finfo(args["dt"].dtype).min
    y, state = scan(ops, args, dt_limit=(least, math.inf))
    check_scan(y, state, {**args, "limit": (least, math.inf)})
