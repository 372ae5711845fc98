"""CPU tests of the layer configuration with 8 bits in every layer."""

import pytest

from turboquant.integration import paged_backend
from turboquant.integration.paged_backend import (TurboQuantPaged8State, TurboQuantPagedConfig, TurboQuantPagedImpl,
                                                  TurboQuantPagedState)
from turboquant.kernels.paged8 import Paged8Format


def test_every_layer_at_8_bits():
    """The states fit the cache shape that get_kv_cache_shape(k_bits=8) gives; protected layers keep their own format."""
    cfg = TurboQuantPagedConfig(128, num_layers=6, num_protected_layers=1, k_bits=8, block_size=32, encoding="int8", protected_bits=8)
    st = cfg.get_state(3)
    assert isinstance(st, TurboQuantPaged8State) and st.k_format == Paged8Format.for_keys("int8", 32) and cfg.get_state(3) is st
    assert st.kv_cache_shape(5, 2) == TurboQuantPagedImpl.get_kv_cache_shape(5, 32, 2, 128, k_bits=8)
    assert cfg.get_state(0).k_format == Paged8Format.for_keys("e4m3", 32)
    assert TurboQuantPagedConfig(128, num_layers=6, k_bits=8, v_bits=8).get_state(0) is None
    low = TurboQuantPagedConfig(128, num_layers=6, k_bits=8, protected_bits=4)
    assert isinstance(low.get_state(0), TurboQuantPagedState) and isinstance(low.get_state(3), TurboQuantPaged8State)
    for kw in (dict(v_bits=4), dict(k_qjl=True)):
        with pytest.raises(ValueError):
            TurboQuantPagedConfig(128, num_layers=6, k_bits=8, **kw)
    with pytest.raises(ValueError):
        TurboQuantPagedConfig(128, k_bits=8, encoding="int4").get_state(0)
    try:
        paged_backend.reset_tq_paged_config()
        assert paged_backend.get_tq_paged_config(num_layers=6, k_bits=8, encoding="int8").get_state(2).k_format.encoding == "int8"
    finally:
        paged_backend.reset_tq_paged_config()
