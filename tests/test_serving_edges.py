"""The ends of what the norms, the pages and the chunks over the cache take, without a GPU."""
import ctypes

import pytest
import torch

from larder_amd import _lib, attention, pages, trunk

P = ctypes.c_void_p(16)  # never dereferenced: every call below is refused while its arguments are checked


@pytest.mark.parametrize("T,heads", [(0x7ffff000, 2), (0x7ffff000 // 2, 3), (1 << 30, 2)])
def test_chunks_of_more_threads_than_a_launch_takes_are_refused(built_lib, T, heads):
    """Workgroups of 512 threads (width 128, many rows): 2^23 of them are 2^32 threads, which no grid holds."""
    assert T * heads // 256 * 512 >= 2 ** 32 > T * heads // 256 * 256
    rc = built_lib.lmoe_kv_chunk(P, 1, 128 * heads, 128, T, heads, heads, 128, P, P, 1, P, 2000, P, P, P, P, 1, 64, 100000, 0.1,
                                 None, 0, P, None)
    assert rc == _lib.ESHAPE and b"more than a launch" in built_lib.lmoe_error(), (rc, built_lib.lmoe_error())


def test_sizes_past_an_int_are_refused(monkeypatch):
    """What the library takes as an int would wrap: 2^32 + 64 channels would be 64 of them. (Tensors without memory.)"""
    def empty(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device="meta")

    launched = []
    monkeypatch.setattr(attention, "_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda *a: launched.append(a))
    monkeypatch.setattr(pages, "_device", lambda *a: 0)
    monkeypatch.setattr(pages, "_launch", lambda *a: launched.append(a))
    monkeypatch.setattr(trunk, "call", lambda *a: launched.append(a))
    far, bf = 2 ** 32 + 64, torch.bfloat16
    cache = attention.KVCache.empty(2, 1, 64, device="meta")
    q = empty(1, 1, 64, dtype=bf)
    for call in (lambda: trunk.norm_rows(empty(1, far, dtype=bf), empty(far, dtype=bf)),
                 lambda: trunk.norm_rows(empty(1, far, dtype=bf), empty(far, dtype=bf), group=32),
                 lambda: trunk.norm_rows(empty(1, far, 1, dtype=bf), empty(1, dtype=bf)),
                 lambda: trunk.read_codes(empty(1, far, dtype=torch.float8_e4m3fn), empty(1, 1, dtype=torch.float32)),
                 lambda: pages.take_pages(empty(far), empty(1, 1), empty(1)),
                 lambda: pages.take_pages(empty(4), empty(far, 1), empty(far)),
                 lambda: pages.free_pages(empty(4), empty(1, far), empty(1)),
                 lambda: pages.fork_pages(empty(4), empty(1, 1), empty(far)),
                 lambda: pages.compact_pages(empty(4), empty(1, 1), empty(far, 1)),
                 lambda: pages.copy_pages(cache, empty(far), empty(far)),
                 lambda: attention.chunk_rows(q, cache, empty(1, far), empty(1)),
                 lambda: attention.attend_rows(q, cache, empty(1, far), empty(1)),
                 lambda: attention.append_rows(cache, None, q, q, empty(1, far), empty(1)),
                 lambda: attention.read_rows(cache, empty(1, far), empty(2), 1)):
        with pytest.raises(ValueError, match="an int counts"):
            call()
    assert not launched
    trunk.norm_rows(empty(1, 64, dtype=bf), empty(64, dtype=bf))  # (these stand in for the kernels' launch)
    pages.take_pages(empty(4), empty(1, 1), empty(1))
    assert len(launched) == 2


def test_a_broadcast_total_is_refused(monkeypatch):
    """Rows that would all be written to one place; a dense axis of one may have any stride."""
    monkeypatch.setattr(attention, "_device", lambda *a: 0)
    monkeypatch.setattr(attention, "_launch", lambda *a: None)
    x, w = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    for total in (x[:1].expand(3, 2, 64), x[:, :1].expand(3, 2, 64)):
        with pytest.raises(ValueError, match="every element"):
            trunk.norm_rows(x, w, total=total)
        trunk.norm_rows(total, w, residual=x)  # (read, they are rows like any)
    trunk.norm_rows(x[:1], w, total=x[:1].as_strided((1, 2, 64), (0, 64, 1)))
    trunk.norm_rows(x[..., :1], w[:1], total=x[..., :1].as_strided((3, 2, 1), (128, 64, 0)))
