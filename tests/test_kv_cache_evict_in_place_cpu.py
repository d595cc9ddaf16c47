"""An eviction's new lengths and weights are other memory than the old ones, which its blocks still read."""
import pytest

from ring_swa import _lib
from test_kv_cache_cpu import params

# (all else is refused for its budget, behind these checks)
OTHERS = {"seqlens": 4096, "new_seqlens": 12288, "weights": 16384, "new_weights": 20480, "new_max_pages": 0}


@pytest.mark.parametrize("fill", [{"new_seqlens": 4096}, {"new_weights": 16384}])
def test_results_in_the_place_of_what_is_read(fill):
    L = _lib.lib()
    assert L.rswa_cache_evict(params({**OTHERS, **fill}), None) == -1
    assert "others than the old" in L.rswa_last_error().decode()


def test_results_of_their_own():
    L = _lib.lib()
    assert L.rswa_cache_evict(params(OTHERS), None) == -1 and "may stay" in L.rswa_last_error().decode()
    none = {"weights": 0, "new_weights": 0, "weights_len": 0}
    assert L.rswa_cache_evict(params({**OTHERS, **none}), None) == -1 and "may stay" in L.rswa_last_error().decode()
