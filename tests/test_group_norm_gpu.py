"""Channels-last group norm with its activation, through the public operator, against torch in 64 bits."""
import numpy as np
import pytest
import torch

from glow_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": ops.NORM_ACT_NONE, "relu": ops.NORM_ACT_RELU, "swish": ops.NORM_ACT_SWISH}


def case(seed, shape, dtype, mean=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    C = shape[-1]
    x = torch.randn(shape, device=DEV, generator=g) * (0.2 + torch.rand(C, device=DEV, generator=g))
    x = (x + mean * torch.randn(C, device=DEV, generator=g)).to(TYPES[dtype])
    return x, 1 + 0.3 * torch.randn(C, device=DEV, generator=g), 0.3 * torch.randn(C, device=DEV, generator=g)


def wanted(x, G, gamma, beta, eps, act, half):
    """(the result in 64 bits, how far a correct kernel may be off)"""
    n, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, G, C // G)
    mean, count = v.mean((1, 3), keepdim=True), v.shape[1] * v.shape[3]
    d = v - mean
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + eps)
    ga = (gamma if gamma is not None else torch.ones(C, device=DEV)).double().view(G, C // G)
    be = (beta if beta is not None else torch.zeros(C, device=DEV)).double().view(G, C // G)
    y = d * rstd * ga + be
    # A sum of `count` numbers by a block of 128 threads or more: count / 128 additions one after the other in a thread, then
    # trees (some 32 more), 2^-24 each, relative to the sum of magnitudes.  The mean is off by that; the variance by as
    # much of itself and by the mean's error squared, half of which goes into its root; a few roundings behind it.
    steps = (min(1024, count // 128) + 32) * 2.0 ** -24
    off_mean = steps * v.abs().mean((1, 3), keepdim=True)
    off = ((rstd * (off_mean + 2.0 ** -24 * v.abs()) + (d * rstd).abs() * (steps + (off_mean * rstd) ** 2 + 8 * 2.0 ** -24)) * ga.abs()
           + 4 * 2.0 ** -24 * be.abs())
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "swish":  # slope at most 1.1; exp's and the quotient's roundings, |y| 2^-24 each a few times over
        off = 1.1 * off + 16 * 2.0 ** -24 * (1 + y.abs()) * y.abs()
        y = y * torch.sigmoid(y)
    return y.reshape(x.shape), (off * (1 + half) + half * y.abs() + 1e-30).reshape(x.shape)


SHAPES = [((1, 1, 1, 1), 1), ((1, 1, 1, 8), 8), ((2, 1, 1, 64), 4), ((1, 7, 7, 30), 5), ((3, 5, 4, 6), 2), ((1, 14, 14, 1024), 32),
          ((2, 56, 56, 64), 32), ((5, 9, 11, 90), 9), ((4, 28, 28, 512), 1), ((2, 200, 128), 16), ((3, 70, 90), 3), ((2, 33, 31, 96), 32),
          ((70, 3, 3, 48), 8), ((1, 100, 100, 40), 8), ((2, 64, 64, 320), 32), ((1, 4097, 24), 24), ((2, 17, 2056), 257), ((1, 160, 160, 64), 8),
          ((1, 256, 256, 128), 32), ((2, 5), 1), ((1, 3, 16384), 2)]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_group_norm(shape, G, dtype):
    act = ["none", "relu", "swish"][(len(shape) + shape[-1] + G) % 3]
    x, gamma, beta = case(shape[-1] + G, shape, dtype)
    got = ops.group_norm(x, G, gamma, beta, activation=ACTS[act])
    y, off = wanted(x, G, gamma, beta, 1e-5, act, torch.finfo(x.dtype).eps / 2)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # half a step of subnormal results
    assert got.dtype == x.dtype and ((got.double() - y).abs() <= off + tiny).all()


@pytest.mark.parametrize("act", ["none", "relu", "swish"])
@pytest.mark.parametrize("dtype,out", [("fp16", torch.float32), ("fp32", torch.bfloat16), ("bf16", torch.float16)])
def test_other_result_types_and_no_parameters(dtype, out, act):
    x, _, _ = case(5, (2, 12, 12, 64), dtype)
    got = ops.group_norm(x, 8, eps=1e-3, activation=ACTS[act], out_dtype=out)
    y, off = wanted(x, 8, None, None, 1e-3, act, torch.finfo(out).eps / 2)
    assert got.dtype == out and ((got.double() - y).abs() <= off + torch.finfo(out).smallest_normal * torch.finfo(out).eps).all()


@pytest.mark.parametrize("shape,G", [((2, 30, 30, 32), 4), ((1, 96, 96, 64), 4)])
def test_a_mean_far_from_zero(shape, G):
    """Numbers around 4096 with a spread of one: a variance from the difference of two sums of squares has no digit left."""
    x, gamma, beta = case(7, shape, "fp32", mean=0.0)
    x = x + 4096
    got = ops.group_norm(x, G, gamma, beta)
    y, off = wanted(x, G, gamma, beta, 1e-5, "none", 2.0 ** -24)
    assert ((got.double() - y).abs() <= off).all()


def test_constant_groups_give_beta():
    x = torch.full((2, 9, 9, 64), 3.25, dtype=torch.float16, device=DEV)
    beta = torch.randn(64, device=DEV)
    assert torch.equal(ops.group_norm(x, 8, torch.ones(64, device=DEV), beta), beta.half().expand_as(x))


def test_nan_and_infinity_stay_in_their_group():
    x, gamma, beta = case(9, (2, 10, 10, 64), "fp32")
    x[0, 3, 3, 17] = float("nan")
    x[1, 0, 0, 63] = float("inf")
    for act in ACTS.values():
        got = ops.group_norm(x, 8, gamma, beta, activation=act).view(2, 100, 8, 8)
        bad = got.isnan().all(1).all(2)
        want = torch.zeros(2, 8, dtype=torch.bool, device=DEV)
        want[0, 2] = True
        assert torch.equal(bad[0], want[0]) and torch.equal(got[1].isnan().any(0).any(1), torch.arange(8, device=DEV) == 7)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,G", [((2, 15, 15, 64), 16), ((1, 7, 7, 30), 5), ((1, 192, 192, 96), 32), ((3, 50, 8), 2)])
def test_int8_result_is_the_quantize_node_behind_it(shape, G, dtype):
    x, gamma, beta = case(11, shape, dtype)
    q = ops.group_norm(x, G, gamma, beta, activation=ops.NORM_ACT_RELU, quant=(0.02, -100))
    y = ops.group_norm(x, G, gamma, beta, activation=ops.NORM_ACT_RELU, out_dtype=torch.float32)
    assert q.dtype == torch.int8 and torch.equal(q, ops.element_quantize_i8(y, 0.02, -100))


def test_given_result_workspace_and_refusals():
    x, gamma, beta = case(14, (1, 300, 300, 64), "fp16")
    need = int(_lib.lib().glowb200_group_norm_workspace_bytes(1, 90000, 64, 8))
    room = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
    assert torch.equal(ops.group_norm(x, 8, gamma, beta, workspace=room), ops.group_norm(x, 8, gamma, beta))
    with pytest.raises(_lib.GlowB200Error, match="workspace"):
        ops.group_norm(x, 8, gamma, beta, workspace=room[:need - 1])
    x, gamma, beta = case(13, (2, 8, 8, 32), "fp16")
    need = int(_lib.lib().glowb200_group_norm_workspace_bytes(2, 64, 32, 4))
    room = torch.full((max(need, 8),), 0xFF, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(x)
    assert ops.group_norm(x, 4, gamma, beta, out=out, workspace=room) is out
    assert torch.equal(out, ops.group_norm(x, 4, gamma, beta))
    assert torch.equal(ops.group_norm(out, 4, gamma, beta, out=out), ops.group_norm(ops.group_norm(x, 4, gamma, beta), 4, gamma, beta))  # in place
    assert ops.group_norm(x[:0], 4, gamma, beta).shape == (0, 8, 8, 32)
    assert ops.group_norm(x[:, :0], 4, gamma, beta).shape == (2, 0, 8, 32)
    with pytest.raises(_lib.GlowB200Error, match="groups"):
        ops.group_norm(x, 5, gamma, beta)
    with pytest.raises(ValueError, match="gamma"):
        ops.group_norm(x, 4, gamma[:31], beta)
    with pytest.raises(TypeError):
        ops.group_norm(x.double(), 4)
    with pytest.raises(TypeError):
        ops.group_norm(x, 4, gamma.half())
    with pytest.raises(ValueError, match="contiguous"):
        ops.group_norm(x.transpose(1, 3), 4)
    with pytest.raises(ValueError, match="shape"):
        ops.group_norm(x, 4, out=torch.empty(2, 8, 8, 16, dtype=torch.float16, device=DEV))
    with pytest.raises(TypeError):
        ops.group_norm(x, 4, quant=(0.1, 0), out=out)
    with pytest.raises(_lib.GlowB200Error, match="activation"):
        ops.group_norm(x, 4, activation=7)


@pytest.mark.parametrize("shape,G", [((1, 20, 20, 64), 8), ((2, 90, 90, 64), 8), ((2, 9, 9, 6), 3)])
def test_tensors_off_16_byte_boundaries(shape, G):
    """Such tensors are taken in smaller pieces, so sums have another order: both are held to the definition."""
    x, gamma, beta = case(15, shape, "fp16")
    odd, out = (torch.empty(x.numel() + 1, dtype=torch.float16, device=DEV)[1:].view(x.shape) for _ in range(2))
    odd.copy_(x)
    y, off = wanted(x, G, gamma, beta, 1e-5, "none", 2.0 ** -11)
    for got in (ops.group_norm(odd, G, gamma, beta), ops.group_norm(x, G, gamma, beta, out=out), ops.group_norm(odd, G, gamma, beta, out=out)):
        assert ((got.double() - y).abs() <= off + 2.0 ** -25).all()


@pytest.mark.parametrize("shape", [(2, 14, 14, 64), (1, 224, 224, 96)])
def test_captured_and_replayed_and_on_two_streams(shape):
    x, gamma, beta = case(17, shape, "bf16")
    room = torch.empty(int(_lib.lib().glowb200_group_norm_workspace_bytes(shape[0], shape[1] * shape[2], shape[3], 8)) + 8, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(x)
    ops.group_norm(x, 8, gamma, beta, out=out, workspace=room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.group_norm(x, 8, gamma, beta, out=out, workspace=room)
    new, _, _ = case(18, shape, "bf16")
    x.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    want = ops.group_norm(new, 8, gamma, beta)
    assert torch.equal(out, want)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(ops.group_norm(new, 8, gamma, beta))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_block_of_layers(oracle):
    """Norm and activation into int8 for a channelwise convolution, and into the 4-bit pointwise layer over the pixels."""
    n, h, w, C, OC = 2, 13, 11, 64, 48
    x, gamma, beta = case(19, (n, h, w, C), "fp16")
    scale, offset = 0.03, -128
    q = ops.group_norm(x, 8, gamma, beta, activation=ops.NORM_ACT_RELU, quant=(scale, offset))
    rng = np.random.default_rng(3)
    filt = rng.normal(0, 0.1, (OC, 3, 3, C)).astype(np.float32)
    c = ops.channelwise_conv_prepare(filt, rng.normal(0, 1, OC).astype(np.float32), scale)
    out_scale = 0.05
    trip = ops.rowwise_requant_params(c["filter_scales"], scale, c["bias_scales"], out_scale)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    got = ops.channelwise_quantized_conv2d(q, d(c["filter"]), d(c["bias"]), (3, 3), (1, 1), (1, 1, 1, 1), 1, (1, 1), 3, offset, d(c["filter_offsets"]),
                                           d(c["bias_offsets"]), tuple(d(v) for v in trip[:3]), tuple(d(v) for v in trip[3:]))
    # the same in 64 bits from the int8 numbers: the requantisation is off by a unit at most
    qf = (q.cpu().double() - offset) * scale
    wf = torch.from_numpy(c["filter"].astype(np.float64) * c["filter_scales"][:, None, None, None].astype(np.float64))
    bf = torch.from_numpy(c["bias"].astype(np.float64) * c["bias_scales"].astype(np.float64))
    y = torch.nn.functional.conv2d(qf.permute(0, 3, 1, 2), wf.permute(0, 3, 1, 2), bf, padding=1).permute(0, 2, 3, 1)
    want = torch.clamp(torch.round(y / out_scale) + 3, -128, 127)
    assert ((got.cpu().double() - want).abs() <= 1).all()
    # the pointwise layer: pixels are rows
    a = ops.group_norm(x, 8, gamma, beta, activation=ops.NORM_ACT_SWISH)
    wq, ws = ops.microscaled_fp4_quantize(torch.randn(OC, C, device=DEV))
    bias = torch.randn(OC, device=DEV)
    got = ops.dynamic_microscaled_fp4_fc(a.view(-1, C), wq, ws, bias, flags=ops.FC_FUSE_RELU).view(n, h, w, OC)
    aq, asc = ops.microscaled_fp4_quantize(a.view(-1, C))
    va, vb = (ops.microscaled_fp4_dequantize(p, s, C).double() for p, s in ((aq, asc), (wq, ws)))
    y, size = va @ vb.T + bias.double(), va.abs() @ vb.abs().T + bias.abs().double()
    off = (got.view(-1, OC).double() - y.clamp(min=0)).abs()
    assert (off <= (C + 2) * 2.0 ** -23 * size * (1 + 2.0 ** -11) + 2.0 ** -11 * y.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,G", [((1, 14, 14, 608), 32), ((2, 17, 17, 104), 8), ((1, 17, 17, 416), 32), ((3, 14, 14, 152), 1), ((1, 12, 12, 208), 1),
                                     ((2, 8, 10, 384), 1), ((2, 8, 10, 192), 1), ((1, 13, 12, 1536), 4), ((1, 34, 34, 104), 8), ((1, 24, 24, 52), 4)])
def test_slices_whose_pieces_do_not_divide_a_block(shape, G, dtype):
    """Slices of 13, 19, 26, 48 and more pieces of 16 bytes over clusters, in shared memory that another norm has filled with
    large numbers: a pixel that is not copied there would count with one of those."""
    ops.group_norm(torch.full((64, 56, 56, 256), 6e4, dtype=torch.float16, device=DEV), 32)
    x, gamma, beta = case(shape[-1] + 2 * G, shape, dtype)
    got = ops.group_norm(x, G, gamma, beta)
    y, off = wanted(x, G, gamma, beta, 1e-5, "none", torch.finfo(x.dtype).eps / 2)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((got.double() - y).abs() <= off + tiny).all()


@pytest.mark.parametrize("value", [1000.03, 3.3])
@pytest.mark.parametrize("shape,G", [((1184, 128, 513), 1), ((37, 1000, 4096), 32), ((1, 3000, 513), 27)])
def test_a_constant_far_from_zero_with_a_block_to_a_group(shape, G, value):
    """Pixels of more pieces than a block has threads: one block adds up a whole group.  Whatever its sum of equal numbers is off by,
    the sum of their exact differences from the quotient takes it out again, up to a few times (the sums' depth * 2^-24)^2, so the
    mean is off by its own rounding alone, less than a unit in its last place (2^-23), and nothing is left of the variance."""
    x = torch.full(shape, value, device=DEV)
    got = ops.group_norm(x, G)
    assert float(got.abs().max()) <= 2.0 ** -23 * value / 1e-5 ** 0.5
