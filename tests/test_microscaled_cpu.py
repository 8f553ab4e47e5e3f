"""The microscaled 4-bit entry points and group norm turn down on the host what they cannot take; no GPU is needed."""
import ctypes as C
import time

import numpy as np
import pytest

import microscaled_reference as ref


@pytest.fixture(scope="module")
def l():
    from glow_b200 import _lib, build
    build.build()
    return _lib.lib()


FAKE, ODD = C.c_void_p(4096), C.c_void_p(4096 + 8)


def test_sizes(l):
    assert l.glowb200_microscaled_fp4_scales_bytes(1, 1) == 512
    assert l.glowb200_microscaled_fp4_scales_bytes(129, 129) == 4 * 512
    assert l.glowb200_microscaled_fp4_scales_bytes(0, 64) == 0 and l.glowb200_microscaled_fp4_scales_bytes(-1, 64) == 0
    assert l.glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(5, 100, 7) >= 5 * 64 + 512
    assert l.glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(-5, 100, 7) == 0
    assert l.glowb200_group_norm_workspace_bytes(0, 9, 8, 2) == 0 and l.glowb200_group_norm_workspace_bytes(3, 1 << 20, 64, 8) > 0


@pytest.mark.parametrize("args", [(FAKE, 3, 4, 64, 64, FAKE, FAKE), (FAKE, 0, -1, 64, 64, FAKE, FAKE), (FAKE, 0, 4, 0, 64, FAKE, FAKE),
                                  (FAKE, 0, 4, 64, 63, FAKE, FAKE), (None, 0, 4, 64, 64, FAKE, FAKE), (FAKE, 0, 4, 64, 64, ODD, FAKE),
                                  (FAKE, 0, 4, 64, 64, FAKE, ODD), (C.c_void_p(4098), 0, 4, 64, 64, FAKE, FAKE)])
def test_quantize_refuses(l, args):
    assert l.glowb200_microscaled_fp4_quantize(*args, None) == 1
    assert l.glowb200_last_error()


def test_nothing_to_do_needs_no_gpu(l):
    assert l.glowb200_microscaled_fp4_quantize(None, 0, 0, 64, 64, None, None, None) == 0
    assert l.glowb200_microscaled_fp4_dequantize(None, None, 0, 64, None, 0, None) == 0
    assert l.glowb200_microscaled_fp4_fc(None, 0, None, None, None, None, None, 0, 64, 8, 0, None, None) == 0
    assert l.glowb200_dynamic_microscaled_fp4_fc(None, 0, None, 0, 64, None, None, None, 8, 64, 0, 0, None, 0, None, None) == 0
    assert l.glowb200_group_norm(None, 0, None, 1.0, 0, None, 0, None, None, 0, 9, 8, 2, 1e-5, 0, None, 0, None, None) == 0


@pytest.mark.parametrize("change", [dict(out_type=3), dict(K=0), dict(M=-1), dict(N=1 << 31), dict(flags=2), dict(out=None), dict(a=None),
                                    dict(sa=None), dict(b=None), dict(sb=None), dict(a=ODD), dict(sa=ODD), dict(b=ODD), dict(sb=ODD),
                                    dict(out=C.c_void_p(4098))])
def test_fc_refuses(l, change):
    v = dict(out=FAKE, out_type=0, a=FAKE, sa=FAKE, b=FAKE, sb=FAKE, bias=None, M=4, K=64, N=8, flags=0)
    v.update(change)
    assert l.glowb200_microscaled_fp4_fc(*v.values(), None, None) == 1
    assert l.glowb200_last_error()


def test_dynamic_fc_refuses(l):
    def call(in_type=0, stride=64, ws=FAKE, size=1 << 20, inp=FAKE):
        return l.glowb200_dynamic_microscaled_fp4_fc(FAKE, 0, inp, in_type, stride, FAKE, FAKE, None, 4, 64, 8, 0, ws, size, None, None)
    assert call(in_type=5) == 1 and call(stride=63) == 1 and call(inp=C.c_void_p(4097)) == 1 and call(inp=None) == 1
    assert call(ws=None) == 3 and call(size=10) == 3 and b"needed" in l.glowb200_last_error()
    assert call(ws=C.c_void_p(4096 + 16)) == 1


@pytest.mark.parametrize("change,code", [(dict(groups=3), 1), (dict(groups=0), 1), (dict(channels=0), 1), (dict(images=-1), 1), (dict(act=3), 1),
                                         (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(in_type=4), 1), (dict(out_type=4), 1),
                                         (dict(out_i8=FAKE), 1), (dict(out=None), 1), (dict(inp=None), 1), (dict(inp=C.c_void_p(4097)), 1),
                                         (dict(pixels=1 << 20, ws=None), 3), (dict(pixels=1 << 20, size=7), 3),
                                         (dict(pixels=1 << 20, ws=C.c_void_p(4096 + 64)), 1)])
def test_group_norm_refuses(l, change, code):
    v = dict(out=FAKE, out_type=0, out_i8=None, scale=1.0, offset=0, inp=FAKE, in_type=1, gamma=None, beta=None, images=2, pixels=9, channels=8,
             groups=2, eps=1e-5, act=0, ws=FAKE, size=1 << 20)
    v.update(change)
    assert l.glowb200_group_norm(*v.values(), None, None) == code
    assert l.glowb200_last_error()


def at(n):
    return C.c_void_p(1 << 20 | n)


def over(l, code):
    return code == 1 and b" over " in l.glowb200_last_error()


def test_results_over_operands_are_refused(l):
    """Addresses are never read: these calls end on the host."""
    far, q = C.c_void_p(1 << 24), l.glowb200_microscaled_fp4_quantize
    # 4 rows of 64 floats (256 bytes), 512 bytes apart: bytes 0-255, 512-767, ...; data 128 bytes, scales 512
    for data in (0, 255 // 16 * 16, 512, 1536, 464, 1776):  # (464: its last bytes reach row 1; 1776: the last row's last ones)
        assert over(l, q(at(0), 0, 4, 64, 128, at(data), far, None)), data
    assert over(l, q(at(4096), 0, 4, 64, 64, at(4096 - 112), far, None)) and over(l, q(at(0), 0, 4, 64, 128, far, at(256), None))
    assert over(l, q(at(0), 0, 4, 64, 64, far, C.c_void_p((1 << 24) + 112), None))
    assert over(l, l.glowb200_microscaled_fp4_dequantize(at(0), far, 4, 64, at(64), 0, None))
    assert over(l, l.glowb200_microscaled_fp4_dequantize(far, at(0), 4, 64, at(508), 0, None))
    for k in range(2, 7):  # the result (128 bytes) at each operand's last bytes in turn
        args = [at(0), 0] + [C.c_void_p((1 << 24) + 4096 * i) for i in range(5)] + [4, 64, 8, 0, None, None]
        args[0] = C.c_void_p(args[k].value + 28)
        assert over(l, l.glowb200_microscaled_fp4_fc(*args)), k
    d = l.glowb200_dynamic_microscaled_fp4_fc
    far2, far3 = C.c_void_p(1 << 25), C.c_void_p(1 << 26)
    assert over(l, d(at(0), 0, at(0), 0, 64, far, far2, None, 4, 64, 64, 0, far3, 1 << 20, None, None))
    assert over(l, d(at(0), 0, far3, 0, 64, far, far2, None, 4, 64, 64, 0, at(512), 1 << 20, None, None))
    assert over(l, d(at(0), 0, far3, 0, 64, far, far2, None, 4, 64, 64, 0, far3, 1 << 20, None, None))
    assert over(l, d(far2, 0, far3, 0, 64, far, far2, None, 4, 64, 64, 0, at(0), 1 << 20, None, None))

    def norm(out, inp, out_type=1, out_i8=None, gamma=None, ws=None, pixels=9):
        return l.glowb200_group_norm(out, out_type, out_i8, 1.0, 0, inp, 1, gamma, None, 2, pixels, 8, 2, 1e-5, 0, ws, 1 << 20, None, None)
    assert over(l, norm(at(2), at(0))) and over(l, norm(at(0), at(2))) and over(l, norm(at(0), at(0), out_type=0))
    assert over(l, norm(None, at(0), out_i8=at(0))) and over(l, norm(at(0), at(0), gamma=at(4)))
    assert over(l, norm(far, at(0), ws=at(0), pixels=1 << 20)) and over(l, norm(far, far2, ws=far, pixels=1 << 16))


def test_group_norm_plans_any_number_of_groups_at_once(l):
    """A prime number of groups has no whole number of groups in a slice: the search for one ends early (2^31 steps take seconds)."""
    prime = 2**31 - 1
    start = time.perf_counter()
    assert l.glowb200_group_norm_workspace_bytes(1, 1, prime, prime) > 8 * prime
    assert time.perf_counter() - start < 1


def test_the_reference_itself():
    """The tests' own quantizer on numbers worked out by hand."""
    x = np.zeros((1, 64), np.float32)
    x[0, :10] = [7.9, 5, 2.5, -3.5, 0.25, 0.75, -0.2, 1.25, 1.75, 6.1]  # e = 0: 7.9 and 6.1 saturate, ties go to even codes
    x[0, 32:34] = [8, -3]                                               # e = 1: 4, -1.5
    codes, sc = ref.quantize(x)
    assert list(ref.values(codes, sc)[0, :10]) == [6, 4, 2, -4, 0, 1, 0, 1, 2, 6]
    assert list(ref.values(codes, sc)[0, 32:34]) == [8, -3] and list(sc[0]) == [127, 128]
    assert codes[0, 6] == 8  # -0.2 becomes -0


@pytest.mark.parametrize("rows", [4, 40, 200])
def test_a_workspace_over_weights_or_bias_is_refused(l, rows):
    """The quantized input goes through the workspace: over the weights it would be multiplied with itself, and they would be gone."""
    names, size = ("out", "inp", "weights", "weights_scales", "bias", "ws"), 1 << 22
    need = l.glowb200_dynamic_microscaled_fp4_fc_workspace_bytes(rows, 64, 512)
    for name, last in (("weights", 512 * 32), ("weights_scales", 4 * 512), ("bias", 2048)):
        # on the operand, on its last bytes, and with its own last bytes on the operand's first
        for move in (0, last - 256, -((need - 1) // 256 * 256)):
            v = {n: size * (i + 1) for i, n in enumerate(names)}
            v["ws"] = v[name] + move
            a = {n: C.c_void_p(p) for n, p in v.items()}
            rc = l.glowb200_dynamic_microscaled_fp4_fc(a["out"], 0, a["inp"], 0, 64, a["weights"], a["weights_scales"], a["bias"], rows, 64, 512, 0,
                                                       a["ws"], 1 << 20, None, None)
            assert over(l, rc), (name, move)


def test_a_workspace_over_gamma_or_beta_is_refused(l):
    pixels, far, far2 = 1 << 20, C.c_void_p(1 << 30), C.c_void_p(1 << 40)
    need = l.glowb200_group_norm_workspace_bytes(2, pixels, 64, 8)
    for gamma, beta in ((1 << 20, None), (None, 1 << 20), (1 << 28, 1 << 20)):
        g, b = (None if v is None else C.c_void_p(v) for v in (gamma, beta))
        for ws in (1 << 20, (1 << 20) - (need - 1) // 256 * 256):
            rc = l.glowb200_group_norm(far, 1, None, 1.0, 0, far2, 1, g, b, 2, pixels, 64, 8, 1e-5, 0, C.c_void_p(ws), 1 << 20, None, None)
            assert over(l, rc), (gamma, beta, ws)
