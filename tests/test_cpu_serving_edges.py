"""What the serving operators refuse beyond shapes and types: memory that a call would write while it reads it, and sizes that 32 bits
do not hold.  The C entries check before any CUDA call; the Python entries are run up to their C call, which is replaced."""
import ctypes as C

import pytest
import torch

from hydra_b200 import _lib
from tests.test_cpu_serving_ops import _cache as _cache_struct, _last

M = 1 << 32   # addresses far from one another that no call below gets far enough to use: its type is none that is built, which is
NONE = 7      # what a call that passes all checks is refused for, with or without a GPU


def _cache(**kw):
    return _cache_struct(**{"dtype": NONE, **kw})


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


# 4 tokens of 8 query and 4 key heads of 64 into the same cache
def _append(cache, **kw):
    s = {f"{t}_stride_{d}": n for t in ("q", "k", "v", "q_out", "k_out") for d, n in (("batch", 0), ("token", 512), ("head", 64))}
    d = dict(q=10 * M, k=11 * M, v=12 * M, q_out=13 * M, k_out=None, slots=14 * M, positions=15 * M, cos=16 * M, sin=17 * M, q_weight=18 * M,
             k_weight=19 * M, **s, table_rows=128, table_ld=32, B=1, S=4, Hq=8, Hkv=4, hd=64, rot=64, layout=1, norm=1,
             dtype=NONE, eps=1e-6, q_scale=1.0, k_scale=1.0)
    a = _lib.QkNormRopeArgs(**{**d, **kw})
    return _lib.lib().hb200_qk_norm_rope(C.byref(a), C.byref(cache), None)


K = dict(k=2 * M, v=3 * M)


@pytest.mark.parametrize("cache", [
    dict(K, k_stride_row=32), dict(K, v_stride_head=960), dict(K, k_stride_page=4032), dict(K, k_stride_row=64, k_stride_head=64),
    dict(K, v_stride_row=-63), dict(K, k_stride_page=64, k_stride_row=512 - 8),
    dict(k=2 * M, v=2 * M), dict(k=2 * M, v=2 * M + 64), dict(k=2 * M, v=2 * M + 8192 * 7), dict(k=2 * M, v=2 * M - 4096),
    dict(k=2 * M, v=2 * M + 128, v_stride_row=256, v_stride_head=64, v_stride_page=4096),
])
def test_append_refuses_caches_on_top_of_themselves_or_one_another(cache):
    assert _append(_cache(**cache)) == -1 and "on top" in _last()


@pytest.mark.parametrize("bad", [
    dict(q=2 * M + 65536 - 128), dict(q=2 * M - 4096 + 2), dict(k=3 * M), dict(v=2 * M + 640), dict(q_out=3 * M - 2048), dict(slots=2 * M - 24),
    dict(positions=3 * M + 65532), dict(cos=2 * M - 128 * 32 * 4 + 4), dict(sin=3 * M), dict(q_weight=2 * M + 256), dict(k_weight=3 * M - 252),
])
def test_append_refuses_inputs_in_the_cache(bad):
    assert _append(_cache(**K), **bad) == -1 and "overlap" in _last()


def test_append_takes_what_it_does_not_read_from_anywhere():
    for unread in (dict(rot=0, cos=2 * M, sin=3 * M), dict(positions=None, positions_stride=M // 2, B=2), dict(q_weight=None, k_weight=None),
                   dict(Hq=0, q=2 * M, q_out=3 * M)):
        assert _append(_cache(**K), **unread) == -4 and "dtype" in _last(), _last()


def _layouts():
    """Ways to keep keys and values side by side: [2, pages, ...], [pages, 2, ...], heads or values of a row in turn, token-major."""
    for shape, at in (((2, 8, 4, 16, 64), 0), ((8, 2, 4, 16, 64), 1), ((8, 4, 2, 16, 64), 2), ((8, 4, 16, 2, 64), 3)):
        yield torch.empty(shape, dtype=torch.bfloat16).unbind(at)
    yield torch.empty(8, 2, 16, 4, 64, dtype=torch.bfloat16).transpose(2, 3).unbind(1)
    pool = torch.empty(16, 4, 16, 64, dtype=torch.bfloat16)
    yield pool[:8], pool[8:]
    yield pool[::2], pool[1::2]
    yield pool[1::2], pool[::2]
    yield torch.empty(8, 3, 2, 4, 16, 64, dtype=torch.bfloat16)[:, 1].unbind(1)      # one of three layers


def test_caches_side_by_side_are_taken():
    """Layouts whose rows lie apart byte by byte pass all checks; the same tensor for both does not."""
    for k, v in _layouts():
        for a, b, good in ((k, v, True), (k, k, False)):
            strides = {f"{n}_stride_{d}": s for n, t in (("k", a), ("v", b)) for d, s in zip(("page", "head", "row"), t.stride())}
            at = min(a.data_ptr(), b.data_ptr())
            status = _append(_cache(k=2 * M + a.data_ptr() - at, v=2 * M + b.data_ptr() - at, **strides))
            assert (status, "dtype" in _last()) == (-4, True) if good else (status, "on top" in _last()) == (-1, True), (k.stride(), _last())


# two requests, tables of 4 in rows of 8, 8 free pages, 8 rows.
def _plan(**kw):
    a = dict(context=M, new=2 * M, table=3 * M, free=4 * M, start=5 * M, lens=6 * M, cu=7 * M, pos=8 * M, slots=9 * M, out=10 * M, status=11 * M)
    a.update(kw)
    return _lib.lib().hb200_paged_plan(a["context"], a["new"], 2, a["table"], 8, 4, 16, a["free"], 8, a["start"], a["lens"], a["cu"], a["pos"],
                                       a["slots"], 8, a["out"], a["status"], None)


@pytest.mark.parametrize("bad", [
    dict(context=3 * M + 44), dict(new=3 * M - 4), dict(free=3 * M + 16), dict(start=3 * M), dict(lens=M + 4), dict(cu=2 * M - 8), dict(pos=4 * M + 16),
    dict(slots=4 * M - 48), dict(out=5 * M), dict(status=M), dict(lens=3 * M + 40), dict(pos=9 * M + 48), dict(out=11 * M), dict(cu=6 * M + 4),
])
def test_plan_refuses_results_among_its_inputs(bad):
    assert _plan(**bad) == -1 and "overlap" in _last()


# -------------------------------------------------------------------------------------------------- memory: Python entries
def test_reach_of_strided_tensors():
    from hydra_b200.kernels import _overlap
    room = torch.zeros(4, 100)
    assert _overlap(room[0], room[0, 99:]) and not _overlap(room[0], room[1]) and not _overlap(room[:2], room[2:])
    assert _overlap(room[::2, 10:20], room[1])                            # between its rows
    assert not _overlap(room[0, :0], room) and not _overlap(room[:, :10].t()[9:], room[0, :9])
    assert _overlap(room[:1].expand(3, 100), room[0, 99:]) and not _overlap(room[:1].expand(3, 100), room[1])


# --------------------------------------------------------------------------------------------------------------- sizes
class Taken(Exception):
    pass


@pytest.fixture
def up_to_the_c_call(monkeypatch):
    """The Python entries on tensors without memory, up to their C call."""
    from contextlib import nullcontext
    from hydra_b200 import kernels

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                raise Taken(name)
            return call
    lib = Lib()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(kernels, "_require_cuda", lambda *t: torch.device("meta"))
    monkeypatch.setattr(kernels, "_on", lambda dev: nullcontext())
    monkeypatch.setattr(kernels, "_stream", lambda dev: 0)
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: M)
    monkeypatch.setattr(kernels, "_empty_strided", lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype, device="meta"))


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_sizes_past_32_bits_are_refused(up_to_the_c_call):
    """ctypes cuts an int to 32 bits: 2^32 + 16 rows of a page were 16."""
    from hydra_b200.kernels import fused_qk_norm_rope
    from hydra_b200.paged import paged_append, paged_decode_attention, paged_plan
    from hydra_b200.sampling import token_logprobs
    i32, i64, f32, big = dict(dtype=torch.int32), dict(dtype=torch.int64), dict(dtype=torch.float32), (1 << 32) + 4

    def plan(B=2, width=4, page=16, room=8):
        return paged_plan(_meta(B, **i32), _meta(B, **i32), _meta(B, width, **i32), _meta(9, **i32), page, room)

    def rope(T=4, hq=4, hkv=2, hd=64, table=8):
        return fused_qk_norm_rope(_meta(T, hq, hd), _meta(T, hkv, hd), _meta(table, 4, **f32), _meta(table, 4, **f32), _meta(T, **i32))

    def rope4(B=1, S=4):
        return fused_qk_norm_rope(_meta(B, 2, S, 8), _meta(B, 1, S, 8), _meta(S, 4, **f32), _meta(S, 4, **f32))

    def append(T=4, pages=8, page=16):
        x, c = _meta(T, 2, 16), _meta(pages, 2, page, 16)
        return paged_append(x, x, x, c, c, _meta(T, **i64), _meta(8, 8, **f32), _meta(8, 8, **f32), _meta(T, **i32))

    def attention(B=2, hq=4, pages=8, page=16, hd=16, width=4):
        c = _meta(pages, 2, page, hd)
        return paged_decode_attention(_meta(B, hq, hd), c, c, _meta(B, width, **i32), _meta(B, **i32))

    def logprobs(N=2, V=64, vocab=None):
        return token_logprobs(_meta(N, V), _meta(N, **i64), vocab=vocab)

    for call, sizes in ((plan, ("B", "width", "page", "room")), (rope, ("T", "hq", "hkv", "hd")), (rope4, ("B", "S")), (append, ("T", "pages", "page")),
                        (attention, ("B", "hq", "pages", "page", "hd", "width")), (logprobs, ("V",))):
        with pytest.raises(Taken):
            call()
        for size in sizes:
            with pytest.raises(ValueError):
                call(**{size: big})
    with pytest.raises(Taken):
        logprobs(V=big, vocab=64)
    with pytest.raises(Taken):
        rope(table=big)


def test_tables_of_several_sequences_are_refused(up_to_the_c_call):
    """cos and sin [1, 1, rows, rot / 2] are one table; of a table per sequence or head the first one served for all."""
    from hydra_b200.kernels import fused_qk_norm_rope
    q, k = _meta(2, 4, 8, 16), _meta(2, 2, 8, 16)
    t = lambda *s: _meta(*s, dtype=torch.float32)                         # noqa: E731
    for cos, sin in ((t(8, 8), t(8, 8)), (t(1, 1, 8, 8), t(1, 1, 8, 8))):
        with pytest.raises(Taken):
            fused_qk_norm_rope(q, k, cos, sin)
    for cos, sin in ((t(2, 1, 8, 8), t(2, 1, 8, 8)), (t(1, 4, 8, 8), t(1, 4, 8, 8)), (t(1, 1, 8, 8), t(2, 1, 8, 8)), (t(1, 1, 8, 8), t(8, 8)),
                     (t(8, 8), t(1, 1, 8, 8)), (t(0, 1, 8, 8), t(0, 1, 8, 8))):
        with pytest.raises(ValueError, match="rotated"):
            fused_qk_norm_rope(q, k, cos, sin)
