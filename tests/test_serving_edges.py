"""The ends of what the norms, the pages and the chunks over the cache take, without a GPU."""
import ctypes

import pytest

from larder_amd import _lib

P = ctypes.c_void_p(16)  # never dereferenced: every call below is refused while its arguments are checked


@pytest.mark.parametrize("T,heads", [(0x7ffff000, 2), (0x7ffff000 // 2, 3), (1 << 30, 2)])
def test_chunks_of_more_threads_than_a_launch_takes_are_refused(built_lib, T, heads):
    """Workgroups of 512 threads (width 128, many rows): 2^23 of them are 2^32 threads, which no grid holds."""
    assert T * heads // 256 * 512 >= 2 ** 32 > T * heads // 256 * 256
    rc = built_lib.lmoe_kv_chunk(P, 1, 128 * heads, 128, T, heads, heads, 128, P, P, 1, P, 2000, P, P, P, P, 1, 64, 100000, 0.1,
                                 None, 0, P, None)
    assert rc == _lib.ESHAPE and b"more than a launch" in built_lib.lmoe_error(), (rc, built_lib.lmoe_error())
