"""The microscaled 4-bit format and the layers over it, through the public operators, against numpy in 64 bits."""
import numpy as np
import pytest
import torch

import microscaled_reference as ref
from glow_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def same(a, b):
    """Equal numbers of one type, NaNs in the same places (rows_of reaches beyond fp16: infinities are part of the inputs)."""
    return a.dtype == b.dtype and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def rounded_from(got, exact, off):
    """Whether every number is what its type's rounding makes of one within `off` of the exact one (beyond the type's range:
    infinity); rounding is monotonic.  NaN where the exact one is."""
    low, high = (torch.from_numpy(exact + d * off).to(got.dtype) for d in (-1, 1))
    nan = torch.from_numpy(np.isnan(exact))
    return torch.equal(got.isnan(), nan) and bool((nan | (low <= got) & (got <= high)).all())


def rows_of(seed, rows, cols, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    x[:, ::7] *= 20
    if cols > 40:
        x[rows // 2, 3:40] = 0
    # numbers on the midpoints between neighbouring codes, of both signs
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7])
    k = min(cols, 16)
    x[0, :k] = torch.cat([mids, -mids])[:k]
    if k == 16:
        x[0, 16:32] = 0
    return x.to(TYPES[dtype])


def check_format(x, data, scales):
    codes, sc = ref.quantize(x.float().cpu().numpy())
    np.testing.assert_array_equal(data.cpu().numpy(), ref.pack(codes))
    np.testing.assert_array_equal(scales.cpu().numpy(), ref.tiles(sc))
    return codes, sc


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (128, 128), (129, 136), (260, 479), (4, 4096), (33, 1000),
                                       (300, 72)])
def test_quantize_and_back(rows, cols, dtype):
    x = rows_of(rows + cols, rows, cols, dtype)
    data, scales = ops.microscaled_fp4_quantize(x.to(DEV))
    codes, sc = check_format(x, data, scales)
    want = torch.from_numpy(ref.values(codes, sc)[:, :cols])
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = ops.microscaled_fp4_dequantize(data, scales, cols, out_dtype=out_dtype).cpu()
        # one rounding of the exact number (none at all for fp32 and bf16)
        assert same(got, want.float().to(out_dtype))


def test_quantize_leaves_no_byte_of_the_buffers_unwritten():
    x = rows_of(1, 130, 200, "fp16").to(DEV)
    data = torch.full((130, 112), 0xAA, dtype=torch.uint8, device=DEV)
    scales = torch.full((2, 2, 512), 0xAA, dtype=torch.uint8, device=DEV)
    a, b = ops.microscaled_fp4_quantize(x, out=data, scales=scales)
    assert a is data and b is scales
    check_format(x, data, scales)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("cols,start,stride", [(96, 0, 101), (96, 3, 128), (64, 8, 80), (31, 1, 33)])
def test_quantize_rows_that_are_apart(cols, start, stride, dtype):
    whole = rows_of(cols + start, 40, stride, dtype).to(DEV)
    x = whole[:, start:start + cols]
    data, scales = ops.microscaled_fp4_quantize(x)
    check_format(x, data, scales)


def test_results_between_rows_that_are_apart():
    """A result may lie where the input's rows leave room."""
    buf = torch.randn(3, 4096, device=DEV)
    x, want = buf[:, :64], ops.microscaled_fp4_quantize(buf[:, :64].contiguous())
    data, scales = buf[0, 64:].view(torch.uint8)[:96].view(3, 32), buf[1, 64:].view(torch.uint8)[:512].view(1, 1, 512)
    ops.microscaled_fp4_quantize(x, out=data, scales=scales)
    assert torch.equal(data, want[0]) and torch.equal(scales, want[1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_extreme_numbers(dtype):
    fi = torch.finfo(TYPES[dtype])
    x = torch.zeros(10, 64)
    x[0, :32] = fi.max
    x[1, :32] = -fi.max
    x[2, :32] = fi.tiny
    x[3, :32] = fi.smallest_normal * fi.eps          # the smallest subnormal
    x[4, 5] = fi.smallest_normal * fi.eps * 3
    x[5, 7] = float("inf")
    x[6, 9] = float("-inf")
    x[7, 31] = float("nan")
    x[8, :32] = -0.0
    x[9, 32] = 1.0
    x = x.to(TYPES[dtype])
    data, scales = ops.microscaled_fp4_quantize(x.to(DEV))
    codes, sc = check_format(x, data, scales)
    got = ops.microscaled_fp4_dequantize(data, scales, 64).cpu().double().numpy()
    np.testing.assert_array_equal(got, ref.values(codes, sc))
    assert np.isnan(got[5:8, :32]).all() and not np.isnan(got[5:8, 32:]).any()


# ---- products ----
def operand(seed, rows, cols, spread):
    """Random codes under scales of 2^-spread .. 2^spread, packed, with zeros behind the last column."""
    rng = np.random.default_rng(seed)
    blocks = -(-cols // 32)
    codes = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    codes[:, cols:] = 0
    sc = rng.integers(127 - spread, 128 + spread, (rows, blocks)).astype(np.uint8)
    return t(ref.pack(codes)), t(ref.tiles(sc)), ref.values(codes, sc)


def rounded(exact_sum, bias, relu, dtype):
    """What the layer gives for sums that fp32 holds exactly: bias added in fp32, one rounding to the result's type."""
    y = torch.from_numpy(exact_sum).float()
    assert (y.double().numpy() == exact_sum).all()
    if bias is not None:
        y = y + bias.cpu()
    return (y.clamp(min=0) if relu else y).to(dtype)


SHAPES = [(1, 32, 1), (1, 64, 8), (1, 4096, 256), (2, 480, 100), (3, 100, 130), (7, 1024, 64), (8, 512, 4096), (16, 256, 512),
          (17, 4096, 96), (33, 96, 33), (64, 2048, 320), (65, 32, 1000), (100, 479, 1000), (127, 544, 129), (128, 256, 256),
          (129, 288, 257), (200, 31, 500), (256, 4096, 512), (257, 800, 512), (300, 1, 300), (400, 479, 1000), (512, 1056, 768),
          (1025, 160, 640)]


@pytest.mark.parametrize("out", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_fc_is_exact_where_fp32_is(M, K, N, out):
    # products are multiples of 2^-2 * 2^-2; every partial sum of fewer than 2^24 of them is an fp32 number
    a, sa, va = operand(M + K, M, K, 1)
    b, sb, vb = operand(N + K + 1, N, K, 1)
    assert (np.abs(va) @ np.abs(vb).T).max() * 16 < 2 ** 24
    g = torch.Generator().manual_seed(N)
    bias = torch.randn(N, generator=g).to(DEV) if (M + N) % 3 else None
    relu = (M + N) % 2 == 0
    st = ops.new_status(DEV)
    got = ops.microscaled_fp4_fc(a, sa, b, sb, bias, flags=ops.FC_FUSE_RELU if relu else 0, out_dtype=TYPES[out], status=st)
    assert torch.equal(got.cpu(), rounded(va @ vb.T, bias, relu, TYPES[out]))
    assert int(st.item()) == 0


@pytest.mark.parametrize("M,K,N", [(1, 2048, 500), (40, 1000, 136), (300, 4096, 260)])
def test_fc_over_a_wide_range_of_scales(M, K, N):
    a, sa, va = operand(M, M, K, 20)
    b, sb, vb = operand(N, N, K, 20)
    got = ops.microscaled_fp4_fc(a, sa, b, sb, out_dtype=torch.float32).cpu().double().numpy()
    want, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
    # K additions, each off by at most one unit in the last place (2^-23, as truncation is) of a number below the sum of magnitudes
    assert (np.abs(got - want) <= (K + 1) * 2.0 ** -23 * size).all()


def test_fc_of_scales_at_both_ends_and_nan():
    a, sa, va = operand(1, 4, 64, 0)
    b, sb, vb = operand(2, 5, 64, 0)
    tiles = sa.clone()
    for r, byte in ((0, 0), (1, 254 - 20), (2, 255)):  # 2^-127, 2^107, NaN, in the first of two blocks
        tiles[0, 0, r % 32 * 16] = byte
    want = va.copy()
    want[0, :32] *= 2.0 ** -127
    want[1, :32] *= 2.0 ** 107
    want[2, :32] = np.nan
    got = ops.microscaled_fp4_fc(a, tiles, b, sb, out_dtype=torch.float32).cpu().double().numpy()
    full = want @ vb.T
    assert np.isnan(got[2]).all()
    size = np.abs(want) @ np.abs(vb).T
    ok = [0, 1, 3]
    assert (np.abs(got - full)[ok] <= 65 * 2.0 ** -23 * size[ok]).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 64, 40), (1, 4096, 512), (5, 479, 100), (8, 4096, 4096), (16, 1024, 130), (40, 33, 70), (130, 256, 300),
                                   (257, 1000, 512)])
def test_dynamic_fc_is_quantize_and_fc(M, K, N, dtype):
    x = rows_of(M + K, M, K, dtype).to(DEV)
    w, ws = ops.microscaled_fp4_quantize(rows_of(N, N, K, "fp32").to(DEV))
    bias = torch.randn(N, device=DEV)
    st = ops.new_status(DEV)
    got = ops.dynamic_microscaled_fp4_fc(x, w, ws, bias, status=st)
    assert got.dtype == x.dtype
    data, scales = ops.microscaled_fp4_quantize(x)
    want = ops.microscaled_fp4_fc(data, scales, w, ws, bias, out_dtype=x.dtype)
    assert same(got, want)
    # ... and the numbers are those of the format
    va, vb = ref.values(*ref.quantize(x.float().cpu().numpy())), ref.values(*ref.quantize(rows_of(N, N, K, "fp32").numpy()))
    exact, size = va @ vb.T + bias.cpu().double().numpy(), np.abs(va) @ np.abs(vb).T + bias.abs().cpu().double().numpy()
    assert rounded_from(got.cpu(), exact, (K + 2) * 2.0 ** -23 * size)
    assert int(st.item()) == 0


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 16500), (1, 9000, 2500), (1, 20000, 300), (2, 9000, 2500), (3, 8200, 9600), (5, 6000, 9600), (7, 9000, 2500),
                                   (16, 12000, 700), (20, 5000, 5000), (32, 20000, 300)])
def test_dynamic_fc_of_long_rows(M, K, N, dtype):
    """More k-blocks to a block than its ring holds, twice over and more, for every way of dealing rows to warps."""
    g = torch.Generator(device=DEV).manual_seed(M + K)
    x = torch.randn(M, K, device=DEV, generator=g).to(TYPES[dtype])
    w, ws = ops.microscaled_fp4_quantize(torch.randn(N, K, device=DEV, generator=g))
    st = ops.new_status(DEV)
    got = ops.dynamic_microscaled_fp4_fc(x, w, ws, out_dtype=torch.float32, status=st)
    va, vb = (ops.microscaled_fp4_dequantize(d, s, K).double() for d, s in (ops.microscaled_fp4_quantize(x), (w, ws)))
    assert ((got.double() - va @ vb.T).abs() <= (K + 1) * 2.0 ** -23 * (va.abs() @ vb.abs().T)).all()
    # rows of ones: sums of the weights, multiples of 2^-8 below 2^16 here, exact in fp32 whatever their order
    assert torch.equal(ops.dynamic_microscaled_fp4_fc(torch.ones_like(x), w, ws, out_dtype=torch.float32).double()[-1], vb.sum(1))
    assert int(st.item()) == 0


def test_dynamic_fc_with_rows_apart_and_a_given_workspace():
    whole = rows_of(3, 20, 300, "fp16").to(DEV)
    x = whole[:, 10:266]
    w, ws = ops.microscaled_fp4_quantize(rows_of(4, 96, 256, "fp32").to(DEV))
    need = int(_lib.lib().glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(20, 256, 96))
    room = torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)
    out = torch.empty(20, 96, dtype=torch.float32, device=DEV)
    got = ops.dynamic_microscaled_fp4_fc(x, w, ws, out=out, workspace=room)
    assert got is out
    assert same(out, ops.dynamic_microscaled_fp4_fc(x.contiguous(), w, ws, out_dtype=torch.float32))
    with pytest.raises(_lib.GlowB200Error, match="workspace"):
        ops.dynamic_microscaled_fp4_fc(x, w, ws, out=out, workspace=room[:need - 1])


def test_rows_of_one_product_do_not_depend_on_the_others():
    """A token alone and among others: the same bits (sums of one order whatever kernel takes the rows)."""
    w, ws = ops.microscaled_fp4_quantize(rows_of(5, 512, 1024, "fp32").to(DEV))
    x = rows_of(6, 300, 1024, "bf16").to(DEV)
    x[0] = x[5]
    all_rows = ops.dynamic_microscaled_fp4_fc(x, w, ws, out_dtype=torch.float32)
    size = torch.from_numpy(np.abs(ref.values(*ref.quantize(x.float().cpu().numpy()))) @ np.abs(ref.values(*ref.quantize(rows_of(5, 512, 1024, "fp32").numpy()))).T)
    for n in (1, 2, 9, 30, 100):
        some = ops.dynamic_microscaled_fp4_fc(x[:n], w, ws, out_dtype=torch.float32)
        assert ((some - all_rows[:n]).abs().cpu().double() <= 2 * 1025 * 2.0 ** -23 * size[:n]).all()
    assert same(all_rows[0], all_rows[5])


@pytest.mark.parametrize("M,N", [(4, 96), (300, 96), (300, 256)])
def test_results_off_16_byte_boundaries(M, N):
    """Into a view two bytes behind a boundary: the same bits, and nothing beside them."""
    w, ws = ops.microscaled_fp4_quantize(rows_of(31, N, 320, "fp32").to(DEV))
    x = rows_of(32, M, 320, "bf16").to(DEV)
    whole = torch.full((M * N + 9,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = whole[1:1 + M * N].view(M, N)
    assert ops.dynamic_microscaled_fp4_fc(x, w, ws, out=out) is out
    assert same(out, ops.dynamic_microscaled_fp4_fc(x, w, ws)) and (whole[0] == 7) and (whole[1 + M * N:] == 7).all()


@pytest.mark.parametrize("M", [1, 20, 129, 300])
def test_nothing_is_written_beside_the_result(M):
    """Rows and columns of a tile that are not the matrix's leave what lies behind it alone."""
    w, ws = ops.microscaled_fp4_quantize(rows_of(33, 72, 96, "fp32").to(DEV))
    a, sa = ops.microscaled_fp4_quantize(rows_of(34, M, 96, "fp32").to(DEV))
    whole = torch.full((M * 72 + 4096,), 7.0, dtype=torch.float32, device=DEV)
    ops.microscaled_fp4_fc(a, sa, w, ws, out=whole[:M * 72].view(M, 72))
    assert (whole[M * 72:] == 7).all()


def test_empty_results():
    w, ws = ops.microscaled_fp4_quantize(torch.randn(40, 64, device=DEV))
    assert ops.dynamic_microscaled_fp4_fc(torch.empty(0, 64, device=DEV), w, ws).shape == (0, 40)
    d, s = ops.microscaled_fp4_quantize(torch.empty(0, 64, device=DEV))
    assert d.shape == (0, 32) and s.numel() == 0 and ops.microscaled_fp4_dequantize(d, s, 64).shape == (0, 64)
    assert ops.microscaled_fp4_fc(d, s, w, ws).shape == (0, 40)
    assert ops.microscaled_fp4_fc(w, ws, d, s).shape == (40, 0)


@pytest.mark.parametrize("M", [4, 300])
def test_captured_and_replayed(M):
    w, ws = ops.microscaled_fp4_quantize(rows_of(8, 256, 512, "fp32").to(DEV))
    bias = torch.randn(256, device=DEV)
    x = rows_of(9, M, 512, "fp16").to(DEV)
    out = torch.empty(M, 256, dtype=torch.float16, device=DEV)
    room = torch.empty(int(_lib.lib().glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(M, 512, 256)), dtype=torch.uint8, device=DEV)
    ops.dynamic_microscaled_fp4_fc(x, w, ws, bias, out=out, workspace=room)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.dynamic_microscaled_fp4_fc(x, w, ws, bias, out=out, workspace=room)
    for seed in (10, 11):
        new = rows_of(seed, M, 512, "fp16").to(DEV)
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, ops.dynamic_microscaled_fp4_fc(new, w, ws, bias))


def test_two_streams_at_once():
    w, ws = ops.microscaled_fp4_quantize(rows_of(12, 640, 1024, "fp32").to(DEV))
    xs = [rows_of(20 + i, 200 if i % 2 else 6, 1024, "bf16").to(DEV) for i in range(8)]
    want = [ops.dynamic_microscaled_fp4_fc(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None] * 8
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = ops.dynamic_microscaled_fp4_fc(x, w, ws)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))


def test_refusals():
    x = torch.randn(8, 64, device=DEV)
    d, s = ops.microscaled_fp4_quantize(x)
    w, ws = ops.microscaled_fp4_quantize(torch.randn(16, 64, device=DEV))
    with pytest.raises(TypeError):
        ops.microscaled_fp4_quantize(x.double())
    with pytest.raises(TypeError):
        ops.microscaled_fp4_quantize(x.cpu())
    with pytest.raises(ValueError, match="side by side"):
        ops.microscaled_fp4_quantize(x.t())
    with pytest.raises(ValueError, match="matrix"):
        ops.microscaled_fp4_quantize(x[0])
    with pytest.raises(ValueError, match="shape"):
        ops.microscaled_fp4_quantize(x, out=torch.empty(8, 16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="scale tiles"):
        ops.microscaled_fp4_quantize(x, scales=torch.empty(511, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="columns"):
        ops.microscaled_fp4_dequantize(d, s, 65)
    with pytest.raises(TypeError):
        ops.microscaled_fp4_dequantize(d, s, 64, out_dtype=torch.int8)
    with pytest.raises(ValueError, match="scale tiles"):
        ops.microscaled_fp4_fc(d, s[:, :0], w, ws)
    with pytest.raises(ValueError, match="columns"):
        ops.microscaled_fp4_fc(d, s, *ops.microscaled_fp4_quantize(torch.randn(16, 96, device=DEV)))
    with pytest.raises(ValueError, match="bias"):
        ops.microscaled_fp4_fc(d, s, w, ws, torch.zeros(15, device=DEV))
    with pytest.raises(_lib.GlowB200Error, match="flags"):
        ops.microscaled_fp4_fc(d, s, w, ws, flags=ops.FC_FORCE_ANY_SHAPE_KERNEL)
    with pytest.raises(ValueError, match="shape"):
        ops.microscaled_fp4_fc(d, s, w, ws, out=torch.empty(8, 15, device=DEV))
    with pytest.raises(ValueError, match="columns"):
        ops.dynamic_microscaled_fp4_fc(torch.randn(8, 65, device=DEV), w, ws)
    off = torch.empty(8 * 32 + 8, dtype=torch.uint8, device=DEV)[8:].view(8, 32)
    with pytest.raises(_lib.GlowB200Error, match="16-byte"):
        ops.microscaled_fp4_fc(off, s, w, ws)


@pytest.mark.parametrize("M,K,N", [(16, 4096, 4096), (20, 2048, 512), (16, 1024, 8320), (8, 4096, 16384), (24, 4096, 6000), (32, 1024, 1024)])
def test_dynamic_fc_where_the_two_layers_add_in_another_order(M, K, N):
    """The depth in another number of parts, or another kernel than for the packed input: equal where fp32 holds all sums, and
    within the roundings of K additions and of one number more a part (at most one unit in the last place each) elsewhere."""
    a, sa, _ = operand(M + K, M, K, 1)
    b, sb, _ = operand(N + K, N, K, 1)
    x, w = ops.microscaled_fp4_dequantize(a, sa, K), ops.microscaled_fp4_dequantize(b, sb, K).double()
    assert K * 12 * 12 * 16 < 2 ** 24  # products are multiples of 1 / 16, of numbers up to 12
    got = ops.dynamic_microscaled_fp4_fc(x, b, sb, out_dtype=torch.float32)
    assert torch.equal(got, ops.microscaled_fp4_fc(a, sa, b, sb, out_dtype=torch.float32)) and torch.equal(got.double(), x.double() @ w.T)
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, K, device=DEV, generator=g) * torch.exp(4 * torch.randn(M, K, device=DEV, generator=g))
    a, sa = ops.microscaled_fp4_quantize(x)
    x = ops.microscaled_fp4_dequantize(a, sa, K).double()
    want, size = x @ w.T, x.abs() @ w.abs().T
    for got in (ops.dynamic_microscaled_fp4_fc(x.float(), b, sb, out_dtype=torch.float32), ops.microscaled_fp4_fc(a, sa, b, sb, out_dtype=torch.float32)):
        assert ((got.double() - want).abs() <= (K + 8) * 2.0 ** -23 * size).all()
