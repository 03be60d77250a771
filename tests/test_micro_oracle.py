"""The ray-head operators without a GPU: the oracle against brute force and
differences, the header's declarations, and the refusals that need no device."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from tests import micro_oracle as O
from vorotracing_amd import _lib, micro

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "vt_micro_abi.h")


def test_nearest_takes_every_tie_to_the_even_code():
    for values in (O.E2M1, O.E4M3):
        a = np.concatenate([values, (values[1:] + values[:-1]) / 2, np.linspace(0, values[-1] * 1.2, 4001)])
        got = O.nearest(values, a)
        d = np.abs(values[None] - a[:, None])
        best = d.min(1)
        assert np.array_equal(d[np.arange(len(a)), got], best)
        tied = (d == best[:, None]).sum(1) > 1
        assert np.all(got[tied] % 2 == 0) and tied.sum() >= len(values) - 1


def test_e4m3_table_is_torchs():
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(O.f64(codes.view(torch.float8_e4m3fn).float()), O.E4M3)


def test_scales_and_formats():
    x = np.zeros((6, 40))
    x[0, :3] = [7.9, -6.0, 0.3]       # floor(log2) 2: scale 1, 7.9 held to 6
    x[1, 32] = 2.0 ** -140            # a subnormal's block: the smallest scale
    x[2, 0], x[2, 33] = np.nan, 1.0   # the first block is NaN, the second is not
    x[3, 35] = -np.inf
    x[4, :2] = [1.0, 2.0 ** -40]
    codes, scales, v = O.mx4(x)
    assert codes.shape == (6, 32) and scales.shape == (6, 2)
    assert scales[0].tolist() == [127, 0] and v[0, :3].tolist() == [6.0, -6.0, 0.5]
    assert scales[1, 1] == 0 and v[1, 32] == 0
    assert np.isnan(v[2, :32]).all() and v[2, 33] == 1.0 and scales[2].tolist() == [255, 125]
    assert np.isnan(v[3, 32:]).all() and (v[3, :32] == 0).all()
    codes, scales, v = O.ckpt8(x)
    assert codes.shape == (6, 40) and scales.shape == (6, 2)
    assert v[0, :3].tolist() == [8.0, -6.0, 0.3125] and scales[0, 0] == 122
    assert v[1, 32] == 2.0 ** -136    # zero only for zeros
    assert np.isnan(v[2, 0]) and v[2, 1] == 0 and codes[2, 0] == 127 and v[2, 33] == 1
    assert np.isnan(v[3, 35]) and codes[3, 35] == 127 and v[3, 36] == 0
    assert v[4, 1] == 2.0 ** -16


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
def test_slopes_against_differences(name):
    z = np.concatenate([np.linspace(-9, 9, 1801), [1e-3, -1e-3]])
    z = z[np.abs(z) > 1e-4]  # relu has no slope at 0
    h = 1e-5
    d = (O.act(z + h, name) - O.act(z - h, name)) / (2 * h)
    # the third derivative is below 2: h^2 / 3, and 1e-16 * 9 / h of rounding
    assert np.abs(d - O.slope(z, name)).max() < 1e-9


def _declarations():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"\b(?:int|size_t)\s+(vt_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}


def test_header_binding_and_library_agree():
    d = _declarations()
    assert len(d) == 11, sorted(d)
    lib = _lib.load()
    for name, n in d.items():
        assert getattr(lib, name, None) is not None, name
        assert len(_lib.SIGNATURES[name][0]) == n, name


def test_entries_reject_before_any_launch():
    lib = _lib.load()
    p = C.c_void_p(16)
    assert lib.vt_mx4_quantize(0, None, 4, 3, 4, p, p, None) == 1 and b"null pointer" in lib.vt_last_error()
    assert lib.vt_mx4_quantize(3, p, 4, 3, 4, p, p, None) == 1 and b"dtype 3" in lib.vt_last_error()
    assert lib.vt_mx4_quantize(0, None, 4, 0, 4, None, None, None) == 0  # no rows, no work
    assert lib.vt_mx4_dequantize(p, p, 3, 4, 5, p, None) == 1 and b"dtype 5" in lib.vt_last_error()
    assert lib.vt_mx4_linear(4, p, 4, p, 3, 4, p, p, 2, None, 0, 0, p, p, None) == 1
    assert b"x dtype 4" in lib.vt_last_error()
    assert lib.vt_mx4_linear(3, p, 4, None, 3, 4, p, p, 2, None, 0, 0, p, p, None) == 1
    assert b"scales" in lib.vt_last_error()
    assert lib.vt_mx4_linear(0, p, 4, None, 3, 4, p, p, 2, None, 0, 3, p, p, None) == 1
    assert b"dtype 3" in lib.vt_last_error()
    assert lib.vt_act_checkpoint(0, 4, p, 4, 3, 4, p, p, p, None) == 1 and b"activation 4" in lib.vt_last_error()
    assert lib.vt_act_checkpoint(0, 1, p, 4, 3, 4, None, p, p, None) == 1 and b"null" in lib.vt_last_error()
    assert lib.vt_act_input_grad(0, -1, p, p, p, 4, 3, 4, p, None) == 1 and b"activation -1" in lib.vt_last_error()
    assert lib.vt_act_weight_grad(7, 0, p, p, p, 4, 3, 4, 2, p, p, p, None) == 1 and b"dtype 7" in lib.vt_last_error()
    layers = (micro._LayerC * 2)()
    for e, (w, o) in zip(layers, ((8, 4), (5, 3))):
        e.codes = e.scales = 16
        e.width, e.out = w, o
    at = C.addressof(layers)
    assert lib.vt_mx4_mlp(0, p, 8, 3, at, 2, 0, p, p, None) == 1
    assert b"layer 1 takes 5 values, the one before gives 4" in lib.vt_last_error()
    assert lib.vt_mx4_mlp(0, p, 8, 3, at, 17, 0, p, p, None) == 1 and b"1 to 16 layers" in lib.vt_last_error()
    assert lib.vt_mx4_linear_workspace_size(3, 10 ** 6, 256, 256) == 0  # stored rows need none
    assert lib.vt_mx4_mlp_workspace_size(0, 3, None, 2) == 0


def test_python_refusals_without_a_gpu():
    x = torch.zeros(3, 4)
    for call in (lambda: micro.quantize_mx4(x), lambda: micro.checkpoint_activation(x, "relu")):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        micro.quantize_mx4(x.double())
    with pytest.raises(TypeError, match="expected a tensor"):
        micro.quantize_mx4([1.0])
    with pytest.raises(ValueError, match="uint8 tensor on the GPU"):
        micro.Mx4(torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.uint8), 5)
    with pytest.raises(ValueError, match="none of none, relu, silu, gelu"):
        micro.Checkpoint8(torch.zeros(2, 4, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), "tanh")
