"""Numbers that do not fit an argument structure's field (no device needed)."""
import importlib

import pytest


@pytest.mark.parametrize("value", [2 ** 31, -2 ** 31 - 1, 2 ** 40, 1.5])
def test_integers_out_of_range(pkg, value):
    kv = importlib.import_module("gemma-webgpu-engine_b200.kv_cache")
    good = [0] * 13 + [1, 1, 1, 1, 0, 0, 0.5]
    assert len(pkg._lib.pack_args(kv._ATTENTION_ARGS, *good)) == kv._ATTENTION_ARGS.size
    for field in (15, 16, 17, 18):  # max_q, max_kv, window, sinks
        bad = list(good)
        bad[field] = value
        with pytest.raises(ValueError, match="range"):
            pkg._lib.pack_args(kv._ATTENTION_ARGS, *bad)


def test_floats_out_of_range(pkg):
    norm = importlib.import_module("gemma-webgpu-engine_b200.norm")
    good = [0] * 17 + [1e-6, 0.0, 0.0]
    assert len(pkg._lib.pack_args(norm._RMS_NORM_ARGS, *good)) == norm._RMS_NORM_ARGS.size
    for field in (17, 18, 19):
        bad = list(good)
        bad[field] = 1e300
        with pytest.raises(ValueError, match="range"):
            pkg._lib.pack_args(norm._RMS_NORM_ARGS, *bad)
