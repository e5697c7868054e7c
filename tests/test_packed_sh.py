"""CPU: the packed-SH record format and the dropout generator as restated in fp64, and what the Python entry points
refuse before anything is launched."""
import types

import numpy as np
import pytest
import torch

import gsplat_amd as gs
from oracle import packed_ref


class _NoLaunch:
    """Library stand-in: a call that gets this far is a refusal that did not happen."""

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(name + " was launched")
        return call


def _ctx():
    c = types.SimpleNamespace(lib=_NoLaunch(), handle=None, device=torch.device("cpu"), sync_stream=lambda: None)
    c.clone = c.new_stream = lambda: None
    return c


def _packed(n):
    return gs.PackedSH(torch.zeros((n, 8), dtype=torch.int32), ctx=_ctx())


def test_philox_published_vectors():
    """Known answers of Philox4x32-10 (counter and key all zero, all ones, digits of pi)."""
    assert packed_ref.philox((0,) * 4, (0,) * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert packed_ref.philox((0xffffffff,) * 4, (0xffffffff,) * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert packed_ref.philox((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_records_of_representable_coefficients_are_lossless():
    rng = np.random.default_rng(0)
    code = rng.integers(0, 8, (40, 3, 15))
    code[:, :, 0] = 7                                          # a 6 fixes the scale
    sh = np.zeros((40, 3, 16))
    sh[:, :, 1:] = packed_ref.E2M1[code] * rng.choice([-1, 1], code.shape) * 2.0 ** rng.integers(-40, 40, (40, 3, 1))
    sh[:, :, 0] = rng.integers(-2048, 2049, (40, 3)) / 1024
    np.testing.assert_array_equal(packed_ref.dequantize(packed_ref.quantize(sh)), sh)


def test_rounding_error_is_within_half_a_step():
    rng = np.random.default_rng(1)
    sh = rng.normal(size=(50, 3, 16)).astype(np.float32)
    err = np.abs(packed_ref.dequantize(packed_ref.quantize(sh)) - sh)[:, :, 1:]
    amax = np.abs(sh[:, :, 1:]).max(axis=2, keepdims=True)
    # the largest step below 6 scales is 2 scales, and saturation (6..7 scales) costs at most 1: 1 scale <= amax / 3.5
    assert (err <= amax / 3.5 + 1e-12).all()


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9])
def test_mask_rate_and_independence_of_the_batch(p):
    n, views = 2000, [0, 1, 2, 3, 9, 2 ** 40 + 1, 2 ** 64 - 1]
    m = packed_ref.keep_mask(n, p, 12345, views)
    # 14 000 Bernoulli draws: six standard deviations
    assert abs((~m).mean() - p) <= 6 * np.sqrt(p * (1 - p) / m.size)
    np.testing.assert_array_equal(m[4], packed_ref.keep_mask(n, p, 12345, [9])[0])
    if 0 < p:
        assert (m[0] != m[1]).any() and (m[0] != packed_ref.keep_mask(n, p, 12346, [0])[0]).any()


def test_camera_position_is_rotation_transposed_times_translation():
    rng = np.random.default_rng(2)
    r, t = rng.normal(size=(3, 3)), rng.normal(size=3)
    np.testing.assert_allclose(gs.camera_position(r, t), r.T @ t, rtol=0, atol=1e-15 * 10)
    np.testing.assert_array_equal(gs.camera_position(torch.from_numpy(r), torch.from_numpy(t)), gs.camera_position(r, t))


def test_refused_before_a_launch():
    c = _ctx()
    with pytest.raises(ValueError, match=r"\[N,3,16\]"):
        gs.quantize_sh(np.zeros((4, 16, 3)), ctx=c)
    with pytest.raises(ValueError, match=r"\[N,3,16\]"):
        gs.quantize_sh(torch.zeros(4, 48), ctx=c)
    with pytest.raises(ValueError, match="int32"):
        gs.PackedSH(torch.zeros((4, 8), dtype=torch.int64), ctx=c)
    with pytest.raises(ValueError, match="int32"):
        gs.PackedSH(torch.zeros((4, 7), dtype=torch.int32), ctx=c)
    with pytest.raises(ValueError, match="32-bit"):
        gs.PackedSH(np.zeros((4, 8)), ctx=c)
    packed = _packed(5)
    assert packed.shape == (5, 3, 16) and len(packed[1:3]) == 2 and packed.nbytes == 160
    with pytest.raises(TypeError, match="packed already"):
        gs.quantize_sh(packed, ctx=c)
    with pytest.raises(IndexError, match="slice"):
        packed[2]
    with pytest.raises(TypeError, match="quantize_sh"):
        gs.sh_color(torch.zeros(5, 3, 16), torch.zeros(5, 3), np.zeros((1, 3)), ctx=c)
    with pytest.raises(ValueError, match="means"):
        gs.sh_color(packed, torch.zeros(4, 3), np.zeros((1, 3)), ctx=c)
    with pytest.raises(ValueError, match="cam_pos"):
        gs.sh_color(packed, torch.zeros(5, 3), np.zeros((3, 4)), ctx=c)
    means, cam = torch.zeros(5, 3), np.zeros((2, 3))
    good = torch.zeros(2, 5, 3)
    with pytest.raises(ValueError, match="clamped"):
        gs.sh_color_backward(packed, means, cam, good[:1], good, ctx=c)
    with pytest.raises(ValueError, match="d_colors"):
        gs.sh_color_backward(packed, means, cam, good, good[:, :4], ctx=c)
    with pytest.raises(ValueError, match="accumulate"):
        gs.sh_color_backward(packed, means, cam, good, good, accumulate=True, ctx=c)
    with pytest.raises(ValueError, match="d_sh"):
        gs.sh_color_backward(packed, means, cam, good, good, out=(torch.zeros(5, 16, 3), torch.zeros(5, 3)), ctx=c)
    with pytest.raises(ValueError, match="d_means"):
        gs.sh_color_backward(packed, means, cam, good, good, out=(torch.zeros(5, 3, 16), torch.zeros(3, 5).t()), ctx=c)
    op = torch.zeros(5)
    with pytest.raises(ValueError, match="opacity"):
        gs.dropout_opacity(torch.zeros(5, 2), .1, 0, [0], ctx=c)
    with pytest.raises(ValueError, match="seed"):
        gs.dropout_opacity(op, .1, -1, [0], ctx=c)
    for bad in (-1, 2 ** 64):
        with pytest.raises(ValueError, match="view numbers"):
            gs.dropout_opacity(op, .1, 0, [bad], ctx=c)
    with pytest.raises(ValueError, match="d_opacities"):
        gs.dropout_opacity_backward(torch.zeros(1, 5), op, .1, 0, [0, 1], ctx=c)
    with pytest.raises(ValueError, match="accumulate"):
        gs.dropout_opacity_backward(torch.zeros(1, 5), op, .1, 0, [0], accumulate=True, ctx=c)
    with pytest.raises(ValueError, match="out"):
        gs.dropout_opacity_backward(torch.zeros(1, 5), op, .1, 0, [0], out=torch.zeros(4), ctx=c)


def test_library_refuses_a_missing_context():
    lib = gs.load_library()
    for rc in (lib.gs_sh_quantize(None, 1, None, None), lib.gs_sh_dequantize(None, 1, None, None),
               lib.gs_sh_color(None, 1, None, None, 3, 0, None, None, None),
               lib.gs_sh_color_backward(None, 1, None, None, 3, 0, None, None, None, 0, None, None),
               lib.gs_opacity_dropout(None, 1, None, 0, .1, 0, 0, None, None),
               lib.gs_opacity_dropout_backward(None, 1, None, 0, .1, 0, 0, None, None, 0, None)):
        assert rc < 0 and b"ctx is NULL" in lib.gs_last_error()
