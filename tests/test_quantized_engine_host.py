"""``EngineConfig.kv_cache_dtype`` (no GPU)."""

import pytest

from microinfer_amd.engine.config import EngineConfig


def test_kv_cache_dtype_names():
    assert EngineConfig().kv_cache_dtype is None
    for kind in ("fp8", "int8"):
        assert EngineConfig(kv_cache_dtype=kind).kv_cache_dtype == kind
    for bad in ("e5m2", "", 8, True):
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            EngineConfig(kv_cache_dtype=bad)
