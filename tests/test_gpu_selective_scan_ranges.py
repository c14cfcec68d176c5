"""The selective scan where magnitudes differ: between channels, between tokens, between a state and what enters it, and at the ends of the types' ranges."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from scan_reference import check_scan, magnitudes, relative, selective_scan  # noqa: E402
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


def rows_apart(t, dim, low):
    """t times factors from 1 down to `low` along the axis, every sixteenth row the same"""
    n = t.shape[dim]
    shape = [1] * t.dim()
    shape[dim] = n
    return t * torch.logspace(0.0, math.log10(low), 16, device="cuda").repeat(-(-n // 16))[:n].reshape(shape)


# Two halves leave 2^-22 of an operand at most, and a product of two pairs leaves out 2^-22: of a term (B C) weight x eight such errors at most (three operands, the
# weight, three products, exponential and step together).  They are spread evenly and are no one's fault together: eight of 2^-22 / sqrt(3) each add up to 1.7 * 2^-22 in
# the 2-norm, of results whose 2-norm is that of their terms, for these have no sign in common.  2^-20 leaves a factor of two.
F32 = 2.0 ** -20


@pytest.mark.parametrize("largest", [0.02, 0.1, 1.0, 30.0, 1e4])
@pytest.mark.parametrize("low", [1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("size,seq", [(64, 20), (64, 130), (128, 70), (64, 1500)])
def test_quiet_channels_in_float32(ops, largest, low, size, seq):
    args = make("f32", 1, 2, 64, 1, size, seq, carried=False)
    args["x"] = rows_apart(args["x"] / args["x"].abs().max(), 2, low) * largest
    args["state"] = torch.zeros(1, 2, 64, size, device="cuda")
    y, state = scan(ops, args)
    check_scan(y, state, args)
    want, want_state = selective_scan(**args)
    for p in range(64):
        assert relative(y[..., p], want[..., p]) <= F32, p
        assert relative(state[:, :, p], want_state[:, :, p]) <= F32, p


@pytest.mark.parametrize("key", ["b", "c"])
@pytest.mark.parametrize("largest", [0.02, 0.1, 1.0, 30.0])
@pytest.mark.parametrize("low", [1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("seq", [20, 130])
def test_quiet_elements_of_the_state_in_float32(ops, key, largest, low, seq):
    args = make("f32", 1, 2, 64, 1, 64, seq, carried=False)
    args[key] = rows_apart(args[key] / args[key].abs().max(), 2, low) * largest
    # (the other one makes up for it, so that every element counts in a result)
    other = "c" if key == "b" else "b"
    args[other] = rows_apart(args[other], 2, 1.0 / low)
    args["state"] = torch.zeros(1, 2, 64, 64, device="cuda")
    y, state = scan(ops, args)
    check_scan(y, state, args)
    want, want_state = selective_scan(**args)
    assert relative(y, want) <= F32
    for n in range(64):
        assert relative(state[..., n], want_state[..., n]) <= F32, n


@pytest.mark.parametrize("key", ["x", "b", "c"])
@pytest.mark.parametrize("much", [1e4, 1e6, 1e8])
@pytest.mark.parametrize("size", [64, 128, 200])
def test_a_loud_token_in_float32(ops, key, much, size):
    # the tokens in front of it know nothing of it
    args = make("f32", 1, 2, 64, 1, size, 100)
    args[key] = args[key].clone()
    args[key][..., 50] *= much
    y, state = scan(ops, args)
    check_scan(y, state, args)
    want, _ = selective_scan(**args)
    mag, _ = magnitudes(**args)
    # (against the terms' magnitudes: all channels of a token share its weights, whose own sums over the state may cancel for all of them alike)
    for t in range(50):
        assert float((y[:, t].double() - want[:, t]).norm() / mag[:, t].norm()) <= F32, t


@pytest.mark.parametrize("scale_x,scale_b,scale_c", [(1e-30, 1.0, 1.0), (1e30, 1.0, 1.0), (1e37, 1e-20, 1.0), (1e-18, 1e-15, 1e20), (1e25, 1e-20, 1e20), (1.0, 1e-17, 1e17), (1e35, 1e-10, 1e-10),
                                                    (1.0, 1e30, 1e-30), (1e-5, 1e-20, 1e30)])
@pytest.mark.parametrize("seq", [100, 1500])
def test_the_whole_range_of_float32(ops, scale_x, scale_b, scale_c, seq):
    args = make("f32", 1, 2, 64, 1, 64, seq, carried=False)
    args.update(x=args["x"] * scale_x, b=args["b"] * scale_b, c=args["c"] * scale_c, state=torch.zeros(1, 2, 64, 64, device="cuda"))
    if scale_x * scale_b * scale_c > 1e-3 * scale_x:
        args["skip"] = None
    y, state = scan(ops, args)
    want, want_state = selective_scan(**args)
    assert relative(y, want) <= F32 and relative(state, want_state) <= F32
    check_scan(y, state, args)


@pytest.mark.parametrize("dtype,much", [("f32", 1e10), ("f32", 1e16), ("f32", 1e30), ("f16", 1e6), ("f16", 1e10), ("f16", 1e30)])
def test_a_loud_state_stays_in_its_row(ops, dtype, much):
    # an element of a row of the state that nobody reads, far above everything else
    args = make(dtype, 1, 2, 64, 1, 64, 100)
    args["c"] = args["c"].clone()
    args["c"][:, :, 0] = 0.0
    args["state"][:, :, 3] = 0.0
    args["state"][:, :, 3, 0] = much
    args["x"] = args["x"].clone()
    args["x"][:, :, 3] = 0.0
    y, state = scan(ops, args)
    check_scan(y, state, args)
    assert not y[..., 3].any()
    want, _ = selective_scan(**args)
    for p in (0, 2, 4, 15):
        assert relative(y[..., p], want[..., p]) <= (2.0 ** -10.5 if dtype == "f16" else 2.0 ** -20), p


@pytest.mark.parametrize("low", [1e-3, 1e-5, 1e-7])
def test_quiet_rows_of_the_state_in_float32(ops, low):
    args = make("f32", 1, 2, 64, 1, 64, 100)
    args["state"], args["x"] = rows_apart(args["state"], 2, low), rows_apart(args["x"], 2, low)
    y, state = scan(ops, args)
    check_scan(y, state, args)
    want, want_state = selective_scan(**args)
    # (beside a largest element between 1 and 2^7, as here, an operand is good to 2^-44 at least, which is 2^-44 / low of a row whose values are `low`)
    for p in range(64):
        assert relative(y[..., p], want[..., p]) <= F32 + 2.0 ** -44 / low, p
        assert relative(state[:, :, p], want_state[:, :, p]) <= F32 + 2.0 ** -44 / low, p


@pytest.mark.parametrize("step,much", [(1e-6, 100.0), (1e-5, 30.0), (1e-6, 1.0), (1e-4, 1000.0)])
@pytest.mark.parametrize("seq", [16, 64, 100])
def test_weights_far_below_the_skip_term_in_half_precision(ops, step, much, seq):
    # D of one on a token's own place, weights of a millionth for the others, and channels where the token itself has nothing: those see only the small weights
    args = make("f16", 1, 2, 64, 1, 64, seq, carried=False)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seq)
    x = torch.empty(1, 2, 64, seq, device="cuda").normal_(generator=gen) * much
    x[..., 1::2] *= (torch.rand(1, 2, 64, x[..., 1::2].shape[-1], device="cuda", generator=gen) < 0.5)
    x[:, :, :32, seq // 2:] = 0.0
    args.update(x=x.half(), skip=torch.ones(2, device="cuda"), bias=torch.full((2,), math.log(math.expm1(step)), device="cuda"), dt=torch.zeros_like(args["dt"]),
                b=(args["b"].float().abs() * 0.3 + 0.3).half(), c=(args["c"].float().abs() * 0.3 + 0.3).half(), state=torch.zeros(1, 2, 64, 64, device="cuda"))
    y, state = scan(ops, args)
    check_scan(y, state, args)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("key,value", [("b", math.inf), ("b", math.nan), ("c", -math.inf), ("c", math.nan), ("dt", math.nan), ("dt", math.inf)])
@pytest.mark.parametrize("seq", [70, 1500])
def test_what_is_not_finite_in_b_c_and_dt_stays_behind_its_token(ops, dtype, key, value, seq):
    at = seq - 30
    args = make(dtype, 1, 4, 64, 2, 64, seq)
    want, want_state = selective_scan(**args)
    odd = {**args, key: args[key].clone()}
    if key == "dt":
        odd["dt"][0, 1, at] = value
    else:
        odd[key][0, 0, 5, at] = value
    y, state = scan(ops, odd)
    # heads 0 and 1 share the first group, head 1 has the step
    hit = [1] if key == "dt" else [0, 1]
    assert not torch.isfinite(y[0, at, hit]).any()
    if key != "c":
        assert not torch.isfinite(y[0, at:, hit]).any()
        assert not torch.isfinite(state[0, hit] if key == "dt" else state[0, hit, :, 5]).any()
    # all else is what it is without it: put that in where it belongs, and compare everything
    for h in hit:
        y[0, at if key == "c" else slice(at, None), h] = want[0, at if key == "c" else slice(at, None), h].to(y)
        if key == "dt":
            state[0, h] = want_state[0, h].to(state)
        elif key == "b":
            state[0, h, :, 5] = want_state[0, h, :, 5].to(state)
    check_scan(y, state, args)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("quiet", [1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("seq", [40, 64, 150])
def test_a_loud_token_beside_quiet_ones_in_a_row_of_the_state(ops, dtype, quiet, seq):
    # the loud one meets B in one half of the state, the quiet ones in the other: each half has its own errors, but the products are made with one scale
    args = make(dtype, 1, 2, 64, 1, 64, seq, carried=False)
    args["x"], args["b"] = args["x"] * quiet, args["b"].clone()
    args["x"][..., 9] *= 1.0 / quiet
    args["b"][:, :, :32] = 0.0
    args["b"][:, :, :, 9] = 0.0
    args["b"][:, :, :32, 9] = 1.0
    args.update(a=torch.full((2,), -1e-3, device="cuda"), bias=torch.full((2,), -4.0, device="cuda"), dt=torch.zeros_like(args["dt"]), state=torch.zeros(1, 2, 64, 64, device="cuda"))
    _, state = scan(ops, args)
    _, want = selective_scan(**args)
    _, mag = magnitudes(**args)
    # as in check_scan; and what is lost of step times x below the largest of a row: 2^-21 of it, in float32 2^-51, for every token (decays are next to one)
    step = math.log1p(math.exp(-4.0))
    lost = (2.0 ** -21 if dtype == "f16" else 2.0 ** -51) * step * args["x"].double().abs().amax(dim=3)[..., None] * args["b"].double().abs().sum(3)[:, :, None]
    assert float(((state.double() - want).abs() / ((4 * seq + 64 + 16) * 2.0 ** -24 * mag + lost + 1e-37)).max()) <= 1.0
    assert relative(state[..., :32], want[..., :32]) <= 2.0 ** -20
    if dtype == "f32":
        assert relative(state[..., 32:], want[..., 32:]) <= 2.0 ** -20


@pytest.mark.parametrize("size", [64, 128, 200])
def test_a_state_whose_products_with_c_are_floats_only_once_it_has_decayed(ops, size):
    args = make("f32", 1, 2, 64, 1, size, 70)
    args["state"], args["c"] = args["state"].clamp(-2.0, 2.0) * 1e37, args["c"] * 1e4
    args["a"], args["bias"], args["dt"] = torch.full((2,), -8.0, device="cuda"), torch.full((2,), 1.0, device="cuda"), torch.zeros_like(args["dt"])
    y, state = scan(ops, args)
    want, want_state = selective_scan(**args)
    mag, mag_state = magnitudes(**args)
    assert float(mag.max()) < 3e38 and torch.isfinite(y).all()
    # (decays below 2^-126 since the chunk's start count as none: see above)
    undecayed = (args["state"].double().abs()[:, :, :, :, None] * args["c"].double().abs()[:, :, None]).sum(3).permute(0, 3, 1, 2)
    f32 = (4 * 70 + size + 16) * 2.0 ** -24
    assert float(((y.double() - want).abs() / (f32 * mag + 2.0 ** -126 * undecayed)).max()) <= 1.0
    assert float(((state.double() - want_state).abs() / (f32 * mag_state + 2.0 ** -126 * args["state"].double().abs())).max()) <= 1.0


@pytest.mark.parametrize("step", [1e-20, 1e-30, 1e-33, 1e25])
@pytest.mark.parametrize("size", [64, 128])
def test_steps_far_from_one_in_float32(ops, step, size):
    # nothing but what such steps bring in: no state, no D (and next to no decay)
    args = make("f32", 1, 2, 64, 1, size, 130, carried=False)
    args.update(skip=None, state=torch.zeros(1, 2, 64, size, device="cuda"), a=torch.full((2,), -1e-3 / max(step, 1.0), device="cuda"), limit=(step, step))
    y, state = scan(ops, {k: v for k, v in args.items() if k != "limit"}, dt_limit=(step, step))
    want, want_state = selective_scan(**args)
    assert relative(y, want) <= F32 and relative(state, want_state) <= F32


@pytest.mark.parametrize("step", [1e-20, 1e-27, 1e-30, 1e-33])
@pytest.mark.parametrize("size,seq", [(64, 130), (128, 40), (250, 70), (64, 1500)])
def test_small_steps_reach_the_state_in_half_precision(ops, step, size, seq):
    args = make("f16", 1, 2, 64, 1, size, seq, carried=False)
    args.update(state=torch.zeros(1, 2, 64, size, device="cuda"), a=torch.full((2,), -1e-3, device="cuda"), limit=(step, step))
    y, state = scan(ops, {k: v for k, v in args.items() if k != "limit"}, dt_limit=(step, step))
    check_scan(y, None, args)
    _, want = selective_scan(**args)
    assert relative(state, want) <= 2.0 ** -20
