"""What the serving operators (paged cache, norm + rotation, token log probabilities) refuse, on a machine without a GPU: the
C entries check their arguments before any CUDA call, the Python entries refuse CPU tensors instead of falling back."""
import ctypes as C

import pytest
import torch

from hydra_b200 import _lib

P = 1 << 20   # a 16-byte aligned address that no call below gets far enough to use


def _last() -> str:
    return _lib.lib().hb200_last_error().decode()


def _plan(B=2, table=P, ld=4, width=4, page=16, n_free=8, room=8, context=P, new=P, free=P, lens=P, cu=P, pos=P, slots=P, out=P, status=P):
    return _lib.lib().hb200_paged_plan(context, new, B, table, ld, width, page, free, n_free, None, lens, cu, pos, slots, room, out,
                                       status, None)


@pytest.mark.parametrize("bad, status, text", [
    (dict(B=-1), -1, "bad shape"), (dict(page=0), -1, "bad shape"), (dict(width=5), -1, "bad shape"), (dict(room=-1), -1, "bad shape"),
    (dict(B=4097), -4, "4096"), (dict(n_free=1 << 31), -4, "free list"), (dict(context=None), -1, "null"), (dict(table=None), -1, "null"),
    (dict(slots=None), -1, "null"), (dict(status=None), -1, "null"), (dict(free=None), -1, "null"), (dict(pos=P + 4), -1, "aligned"),
])
def test_paged_plan_refuses(bad, status, text):
    assert _plan(**bad) == status and text in _last()


def _cache(**kw):
    d = dict(k=P, v=P, k_stride_page=4096, k_stride_head=1024, k_stride_row=64, v_stride_page=4096, v_stride_head=1024, v_stride_row=64,
             num_pages=8, page_size=16, n_kv_heads=4, head_dim=64, dtype=_lib.HB200_BF16)
    return _lib.PagedCache(**{**d, **kw})


def _attention(cache=None, q=P, sb=2048, sh=64, out=P, table=P, ld=4, width=4, lens=P, B=2, Hq=32, scale=0.125, ws=P, n=1 << 40):
    c = _cache() if cache is None else cache
    return _lib.lib().hb200_paged_decode_attention(C.byref(c), q, sb, sh, out, None, table, ld, width, lens, B, Hq, scale, ws, n, None)


@pytest.mark.parametrize("bad, status, text", [
    (dict(Hq=30), -1, "multiple"), (dict(Hq=2048), -4, "1024"), (dict(B=4097), -4, "4096"), (dict(B=-1), -1, "shape"),
    (dict(q=None), -1, "null"), (dict(ws=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(table=None), -1, "bad cache or table"),
    (dict(width=5), -1, "bad cache or table"), (dict(q=P + 2), -1, "aligned"), (dict(sh=60), -1, "multiples of 8"),
    (dict(cache=_cache(head_dim=60)), -4, "head_dim"), (dict(cache=_cache(head_dim=264)), -4, "head_dim"),
    (dict(cache=_cache(v_stride_row=4)), -1, "multiples of 8"), (dict(cache=_cache(page_size=0)), -1, "bad cache or table"),
    (dict(cache=_cache(k=None)), -1, "null"), (dict(scale=float("nan")), -1, "NaN"), (dict(scale=float("inf")), -1, "infinite"), (dict(ld=1 << 27, width=1 << 27), -4, "too far"),
    (dict(B=4096, ld=1 << 24, width=1 << 24), -4, "too far"),
])
def test_paged_attention_refuses(bad, status, text):
    assert _attention(**bad) == status and text in _last()


def test_paged_attention_without_requests_is_nothing():
    assert _attention(B=0) == 0


def _rope(cache=None, **kw):
    s = {f"{t}_stride_{d}": n for t in ("q", "k", "v", "q_out", "k_out") for d, n in (("batch", 0), ("token", 512), ("head", 64))}
    d = dict(q=P, k=P, v=P, q_out=P, k_out=P, slots=P, positions=P, cos=P, sin=P, **s, table_rows=128, table_ld=32, B=1, S=4, Hq=8, Hkv=4, hd=64, rot=64, norm=1, dtype=_lib.HB200_BF16, eps=1e-6,
             q_scale=1.0, k_scale=1.0)
    a = _lib.QkNormRopeArgs(**{**d, **kw})
    return _lib.lib().hb200_qk_norm_rope(C.byref(a), C.byref(cache) if cache is not None else None, None)


@pytest.mark.parametrize("bad, status, text", [
    (dict(S=-1), -1, "bad shape"), (dict(hd=0), -1, "bad shape"), (dict(hd=257, rot=64), -4, "256"), (dict(rot=66), -1, "rotated"),
    (dict(rot=33), -1, "rotated"), (dict(layout=2), -1, "layout"), (dict(norm=3), -1, "norm"), (dict(table_ld=31), -1, "table"), (dict(table_rows=0), -1, "table"),
    (dict(positions=None, S=129), -1, "129"), (dict(q=None), -1, "null"), (dict(k_out=None), -1, "null"), (dict(cos=None), -1, "null"),
    (dict(dtype=7), -4, "dtype"), (dict(cache=_cache(), slots=None), -1, "null"), (dict(cache=_cache(n_kv_heads=2)), -1, "cache"),
    (dict(cache=_cache(head_dim=32)), -1, "cache"), (dict(cache=_cache(dtype=_lib.HB200_F16)), -1, "cache"),
    (dict(cache=_cache(v=None)), -1, "null"), (dict(cache=_cache(k_stride_page=0)), -1, "on top"), (dict(cache=_cache(v_stride_row=0)), -1, "on top"),
])
def test_qk_norm_rope_refuses(bad, status, text):
    assert _rope(**bad) == status and text in _last()


def _logprobs(x=P, t=P, rows=2, cols=64, ld=64, temperature=1.0, top=4, lp=P, h=P, tl=P, ti=P, dtype=_lib.HB200_BF16):
    return _lib.lib().hb200_token_logprobs(x, t, rows, cols, ld, -100, temperature, top, lp, h, tl, ti, dtype, None)


@pytest.mark.parametrize("bad, status, text", [
    (dict(rows=-1), -1, "bad shape"), (dict(cols=0), -1, "bad shape"), (dict(ld=63), -1, "bad shape"), (dict(temperature=0.0), -1, "temperature"),
    (dict(temperature=float("nan")), -1, "temperature"), (dict(temperature=float("inf")), -1, "temperature"), (dict(top=33), -4, "32"),
    (dict(top=-1), -4, "alternatives"), (dict(cols=3, top=4), -1, "alternatives"), (dict(x=None), -1, "null"), (dict(ti=None), -1, "null"),
    (dict(x=P + 1), -1, "misaligned"), (dict(dtype=9), -4, "dtype"),
])
def test_token_logprobs_refuses(bad, status, text):
    assert _logprobs(**bad) == status and text in _last()


def test_python_entries_refuse_cpu_tensors():
    from hydra_b200 import kernels, paged, sampling
    i = torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(2, 4, 16, dtype=torch.bfloat16), torch.zeros(3, 4, 16, 16, dtype=torch.bfloat16)
    t = torch.zeros(8, 8)
    for call in (lambda: paged.paged_plan(i, i, torch.zeros(2, 4, dtype=torch.int32), i, 16, 8),
                 lambda: paged.paged_append(q, q, q, c, c, i.long(), t, t, i),
                 lambda: paged.paged_decode_attention(q, c, c, torch.zeros(2, 4, dtype=torch.int32), i),
                 lambda: kernels.fused_qk_norm_rope(q, q, t, t), lambda: sampling.token_logprobs(q[0], i.long())):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_struct_layouts_match_the_header():
    assert C.sizeof(_lib.PagedCache) == 8 * 8 + 5 * 4 + 4                        # trailing padding to 8
    assert C.sizeof(_lib.QkNormRopeArgs) == 11 * 8 + 15 * 8 + 3 * 8 + 10 * 4 + 3 * 4 + 4
