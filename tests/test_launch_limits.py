"""A launch of 2^32 threads and more, which HIP cuts short without an error, is refused by every entry
point that sizes could lead there, before the device is touched."""

from __future__ import annotations


def test_weights_that_no_grid_holds():
    from mambo_amd import _native
    lib = _native.lib()
    for rc in (lib.mambo_iq3s_prepare(16, 2**28, 1, 111, 111, 1, None, None, None, None, None, 16, None),
               lib.mambo_iq3s_prepare(16, 2**30, 1, 110, 110, 1, None, None, None, None, None, 16, None),
               lib.mambo_iq3s_pack(16, 16, 16, 16, 16, 2**30, 1, 16, None)):
        assert rc == _native.MAMBO_ERR_VALUE
        assert "too large for one launch" in lib.mambo_last_error().decode()


def test_a_refused_launch_does_not_stay_with_the_thread():
    """The next call is judged by itself."""
    from mambo_amd import _native
    lib = _native.lib()
    assert lib.mambo_iq3s_pack(16, 16, 16, 16, 16, 2**30, 1, 16, None) == _native.MAMBO_ERR_VALUE
    assert lib.mambo_fp8_block_matmul(None, 32, None, 1, 1, 0, None, None, 8, 32, None, 0, 8, None) == _native.MAMBO_OK
    assert lib.mambo_iq3s_pack(None, 16, 16, 16, 16, 2**30, 1, 16, None) == _native.MAMBO_ERR_VALUE
    assert "null pointer" in lib.mambo_last_error().decode()
