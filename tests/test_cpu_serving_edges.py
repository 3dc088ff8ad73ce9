"""What the serving operators refuse beyond shapes and types: memory that a call would write while it reads it, and sizes that 32 bits
do not hold.  The C entries check before any CUDA call; the Python entries are run up to their C call, which is replaced."""
import ctypes as C

import pytest
import torch

from hydra_b200 import _lib
from tests.test_cpu_serving_ops import _cache, _last

M = 1 << 32   # addresses far from one another that no call below gets far enough to use


# ------------------------------------------------------------------------------------------------------ memory: C entries
# two requests of 32 heads of 64 on a cache of 8 pages, 4 heads and 16 rows: q and out take 8192 bytes, a cache 65536
def _attention(out=6 * M, lse=7 * M, q=M, table=4 * M, lens=5 * M, cache=None):
    c = cache or _cache(k=2 * M, v=3 * M)
    return _lib.lib().hb200_paged_decode_attention(C.byref(c), q, 2048, 64, out, lse, table, 4, 4, lens, 2, 32, 0.125, 8 * M, 1 << 40, None)


@pytest.mark.parametrize("bad", [
    dict(out=M), dict(out=M - 8192 + 16), dict(out=M + 8192 - 16), dict(out=2 * M + 65536 - 16), dict(out=2 * M - 8192 + 16), dict(out=3 * M + 4096),
    dict(out=4 * M - 8176), dict(out=5 * M - 8176), dict(lse=M + 64), dict(lse=2 * M), dict(lse=3 * M + 65532), dict(lse=4 * M + 28), dict(lse=5 * M + 4),
    dict(out=7 * M - 8176), dict(lse=6 * M + 8188),
    dict(cache=_cache(k=2 * M, v=3 * M, k_stride_page=-4096), out=2 * M - 7 * 8192), dict(cache=_cache(k=2 * M, v=3 * M, v_stride_page=1 << 20), out=3 * M + (7 << 21)),
])
def test_attention_refuses_results_among_its_inputs(bad):
    assert _attention(**bad) == -1 and "overlap" in _last()


# -------------------------------------------------------------------------------------------------- memory: Python entries
def test_reach_of_strided_tensors():
    from hydra_b200.kernels import _overlap
    room = torch.zeros(4, 100)
    assert _overlap(room[0], room[0, 99:]) and not _overlap(room[0], room[1]) and not _overlap(room[:2], room[2:])
    assert _overlap(room[::2, 10:20], room[1])                            # between its rows
    assert not _overlap(room[0, :0], room) and not _overlap(room[:, :10].t()[9:], room[0, :9])
    assert _overlap(room[:1].expand(3, 100), room[0, 99:]) and not _overlap(room[:1].expand(3, 100), room[1])
