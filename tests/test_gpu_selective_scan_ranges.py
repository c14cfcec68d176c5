"""The selective scan where magnitudes differ: between channels, between tokens, between a state and what enters it, and at the ends of the types' ranges."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from scan_reference import check_scan, magnitudes, selective_scan  # noqa: E402
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


@pytest.mark.parametrize("dtype,much", [("f32", 1e5), ("f32", 1e12), ("f32", 1e25), ("f32", 1e37), ("f16", 1e5), ("f16", 1e25), ("f16", 5e35)])
@pytest.mark.parametrize("seq", [9, 70, 1500])
def test_a_large_state_beside_small_operands(ops, dtype, much, seq):
    # what brings small products to the top of a half's range is not to meet the state: some channels are zeros, some next to nothing
    args = make(dtype, 1, 2, 64, 1, 64, seq)
    for key in ("x", "b"):
        args[key] = args[key] * 1e-4
    args["x"][:, :, 7] = 0.0
    args["x"][:, :, 20:24] *= 1e-3
    args["bias"] = torch.full((2,), -12.0, device="cuda")
    args["dt"] = torch.zeros_like(args["dt"])
    # (results of halves cannot take such a state: nobody reads it there)
    args["c"] = args["c"] * (1e-4 if dtype == "f32" else 0.0)
    args["state"] = args["state"].clamp(-2.0, 2.0) * much
    y, state = scan(ops, args)
    check_scan(y, state, args)


@pytest.mark.parametrize("dtype,much", [("f32", 1.0), ("f32", 1e5), ("f32", 1e12), ("f32", 1e30), ("f16", 1.0), ("f16", 500.0)])
def test_tokens_without_weights(ops, dtype, much):
    # B and C that do not meet for every other token: all that it sees is the state in front
    args = make(dtype, 1, 2, 64, 1, 64, 70)
    args["skip"] = None
    args["x"], args["b"], args["c"] = args["x"] * 1e-4, args["b"] * 1e-4, args["c"].clone()
    args["b"][:, :, 32:] = 0.0
    args["c"][:, :, :32, ::2] = 0.0
    args["state"] = args["state"] * much
    y, state = scan(ops, args)
    if dtype == "f16":
        check_scan(y, state, args)
        return
    # The bounds of check_scan, and besides: a decay since the chunk's start (70 tokens: since the first or the 65th) that is no normal float counts as none.  The state
    # in front decays on from there, so such a result is off by less than 2^-126 of what the first token's state would have given it without any decay.
    want, want_state = selective_scan(**args)
    mag, mag_state = magnitudes(**args)
    undecayed = (args["state"].double().abs()[:, :, :, :, None] * args["c"].double().abs()[:, :, None]).sum(3).permute(0, 3, 1, 2)
    f32 = (4 * 70 + 64 + 16) * 2.0 ** -24
    assert float(((y.double() - want).abs() / (f32 * mag + 2.0 ** -126 * undecayed + 2.0 ** -149)).max()) <= 1.0
    assert float(((state.double() - want_state).abs() / (f32 * mag_state + 2.0 ** -126 * args["state"].double().abs() + 1e-37)).max()) <= 1.0
