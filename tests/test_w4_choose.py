"""ammon_w4_choose without a device."""
from ammon_amd import _abi
from ammon_amd._abi import lib


def test_no_runtime_is_refused():
    for tile, way in ((None, None), (b"long", b"flat")):
        assert lib.ammon_w4_choose(None, tile, way) == _abi.E_VALIDATION
        assert "runtime" in _abi.last_error()
