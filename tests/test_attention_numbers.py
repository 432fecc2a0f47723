"""Scales and caps that the C entries refuse, because what they make of them is not finite."""

from __future__ import annotations

import ctypes

import pytest

from torchmatch_amd import _native


@pytest.mark.parametrize("changes,code", [
    ({"scale": float("inf")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"scale": -float("inf")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"scale": 3e38}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": float("inf")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": float("nan")}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": 3e38}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": 1e-39}, _native.TM_ERR_INVALID_ARGUMENT),
    ({"cap": 1e-39, "scale": 0.0}, _native.TM_OK),
    ({"cap": 1e-36}, _native.TM_OK),
    ({"scale": 1e37, "cap": 30.0}, _native.TM_OK),
    ({"scale": -1e37}, _native.TM_OK),
])
def test_refusals(changes, code):
    fields = {"B": 0, "Lq": 3, "Lk": 5, "H": 2, "Hkv": 2, "D": 64, "dtype": _native.TM_F32,
              "scale": 0.125, "q": 4096, "k": 4096, "v": 4096, **changes}
    a = _native.Attention(**fields)
    assert _native.lib().tm_attention_forward(ctypes.byref(a), 4096, None, None, None, 0,
                                              None) == code
