"""fused_qk_norm_rope and paged_append against a plain computation in 64 bits.

Tolerance, per value: half a step of the storage type (the one rounding) relative to the value, plus 2^-16 of the row's
largest value for the 32-bit arithmetic: the sum of up to 256 squares in lanes of 8 and five shuffles, rsqrt, three products
and the rotation's sum come to at most 20 roundings of 2^-24 relative to terms of at most twice that value, 2^-18.7."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def tables(rows, rot, base=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1))[None]
    return a.cos().float(), a.sin().float()


def exact(x, w, cos, sin, norm, eps, scale, layout):
    """x [T, H, hd]; cos, sin [T, rot / 2], all as 64 bits."""
    x = x.double()
    if norm:
        x = x / (x.square().sum(-1, keepdim=True) / (x.shape[-1] if norm == "rms" else 1) + eps).sqrt()
    if w is not None:
        x = x * w.double()
    x = x * scale
    c, s = cos.double()[:, None], sin.double()[:, None]
    r = c.shape[-1]
    y = x.clone()
    a, b = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def check(got, want, dtype, what=""):
    got = got.double().cpu()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -16 * want.abs().amax(-1, keepdim=True)
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp_min(1e-30)).max()):.2f} tolerances"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("T,hq,hkv,hd,rot,norm", [
    (1, 8, 2, 32, 32, "l2"), (7, 4, 4, 128, 128, "rms"), (33, 5, 1, 80, 40, "rms"), (3, 6, 2, 64, 16, None), (2, 3, 3, 256, 256, "rms"),
    (9, 1, 1, 8, 8, "rms"), (5, 2, 1, 6, 4, "rms"), (4, 3, 1, 17, 10, "l2"), (6, 4, 2, 96, 94, "rms"), (300, 32, 8, 64, 64, "rms"),
    (2, 2, 1, 100, 0, "rms"), (3, 2, 2, 2, 2, None),
    (5000, 5, 3, 64, 32, "rms"), (2501, 9, 1, 24, 24, "l2"), (1300, 3, 3, 256, 64, "rms"), (4097, 1, 1, 16, 8, None)])
def test_packed_tokens(dtype, layout, T, hq, hkv, hd, rot, norm):
    from hydra_b200.kernels import fused_qk_norm_rope
    g = torch.Generator().manual_seed(T * 1000 + hd)
    rows = torch.randn(T, hq + 2 * hkv, hd, generator=g).to(dtype)
    wq, wk = (1 + 0.2 * torch.randn(2, hd, generator=g)) if norm == "rms" else (None, None)
    cos, sin = tables(50, rot)
    pos = torch.randint(0, 50, (T,), generator=g)
    dev = rows.cuda()
    q, k = fused_qk_norm_rope(dev[:, :hq], dev[:, hq:hq + hkv], cos.cuda(), sin.cuda(), pos.int().cuda(), norm=norm, eps=1e-5,
                              q_weight=None if wq is None else wq.cuda(), k_weight=None if wk is None else wk.cuda(),
                              q_scale=0.25, k_scale=3.0, layout=layout)
    assert q.is_contiguous() and k.is_contiguous() and q.shape == (T, hq, hd) and k.shape == (T, hkv, hd)
    check(q, exact(rows[:, :hq], wq, cos[pos], sin[pos], norm, 1e-5, 0.25, layout), dtype, "q")
    check(k, exact(rows[:, hq:hq + hkv], wk, cos[pos], sin[pos], norm, 1e-5, 3.0, layout), dtype, "k")
    q2, _ = fused_qk_norm_rope(dev[:, :hq], dev[:, hq:hq + hkv], cos.cuda(), sin.cuda(), pos.cuda(), norm=norm, eps=1e-5,
                               q_weight=None if wq is None else wq.cuda(), q_scale=0.25, k_scale=3.0, layout=layout)
    assert torch.equal(q, q2)                                             # int64 positions


@pytest.mark.parametrize("view", ["bhsd", "bshd", "misaligned", "sliced"])
def test_heads_first_layouts_and_strides(view):
    from hydra_b200.kernels import fused_qk_norm_rope
    g = torch.Generator().manual_seed(3)
    B, hq, hkv, S, hd = 3, 4, 2, 21, 32
    if view == "bshd":
        q, k = (torch.randn(B, S, h, hd, generator=g).cuda().transpose(1, 2) for h in (hq, hkv))
    elif view == "misaligned":
        q, k = (torch.randn(B, h, S, hd + 1, generator=g).cuda()[..., 1:] for h in (hq, hkv))
    elif view == "sliced":
        q, k = (torch.randn(B, h, S, 2 * hd, generator=g).cuda()[..., ::2] for h in (hq, hkv))
    else:
        q, k = (torch.randn(B, h, S, hd, generator=g).cuda() for h in (hq, hkv))
    cos, sin = tables(64, hd)
    flat = lambda t: t.cpu().transpose(1, 2).reshape(B * S, -1, hd)      # noqa: E731
    pos = torch.randint(0, 64, (B, S), generator=g)
    for p in (pos, pos[0], None):
        qo, ko = fused_qk_norm_rope(q, k, cos[None, None].cuda(), sin[None, None].cuda(), None if p is None else p.cuda(), norm="rms")
        at = (torch.arange(S) if p is None else p).expand(B, S).reshape(-1)
        assert qo.is_contiguous() and qo.shape == (B, hq, S, hd)
        check(flat(qo), exact(flat(q), None, cos[at], sin[at], "rms", 1e-6, 1.0, "interleaved"), torch.float32, view)
        check(flat(ko), exact(flat(k), None, cos[at], sin[at], "rms", 1e-6, 1.0, "interleaved"), torch.float32, view)


def test_equals_the_two_ops_that_it_joins():
    """fused_qk_norm ("rsqrt" mode, eps 1e-8) and then fused_rope, without the rounding in between (fp32)."""
    from hydra_b200 import kernels as K
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(2, 8, 40, 32, generator=g).cuda(), torch.randn(2, 2, 40, 32, generator=g).cuda()
    cos, sin = (t.cuda() for t in tables(40, 32))
    a, b = K.fused_qk_norm(q, k, 5.0, 1.7)
    want_q, want_k = K.fused_rope(a, cos, sin), K.fused_rope(b, cos, sin)
    got_q, got_k = K.fused_qk_norm_rope(q, k, cos, sin, norm="l2", eps=1e-8, q_scale=5.0, k_scale=5.0 * 1.7)
    assert float((got_q - want_q).abs().max()) <= 1e-5 and float((got_k - want_k).abs().max()) <= 2e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout,order,hd,rot,page", [("half", "hnd", 128, 128, 16), ("interleaved", "nhd", 64, 32, 24), ("half", "nhd", 80, 40, 1),
                                                      ("half", "hnd", 20, 6, 5)])
def test_append_writes_its_slots_and_nothing_else(dtype, layout, order, hd, rot, page):
    from hydra_b200.paged import paged_append
    g = torch.Generator().manual_seed(hd + page)
    T, hq, hkv, pages = 37, 6, 3, 60 // page + 3
    rows = torch.randn(T, hq + 2 * hkv, hd, generator=g).to(dtype)
    wq, wk = 1 + 0.2 * torch.randn(2, hd, generator=g)
    shape = (pages, hkv, page, hd) if order == "hnd" else (pages, page, hkv, hd)
    kc0, vc0 = torch.randn(2, *shape, generator=g).to(dtype)
    kc, vc = kc0.cuda(), vc0.cuda()
    if order == "nhd":
        kc, vc, kc0, vc0 = (t.transpose(1, 2) for t in (kc, vc, kc0, vc0))
    cos, sin = tables(99, rot)
    pos, slots = torch.randint(0, 99, (T,), generator=g), torch.randperm(pages * page, generator=g)[:T]
    pos[30:], slots[33:] = -1, -1                                         # padding; three of them with a slot all the same
    slots[5] = -1                                                         # a token without a page: computed, not stored
    slots[6], pos[7] = pages * page, 99                                   # out of the cache; out of the tables
    dev = rows.cuda()
    q = paged_append(dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:], kc, vc, slots.cuda(), cos.cuda(), sin.cuda(), pos.int().cuda(),
                     q_weight=wq.cuda(), k_weight=wk.cuda(), layout=layout)
    good = [t for t in range(30) if t not in (6, 7)]
    at = pos.clamp(0, 98)
    want_q = exact(rows[:, :hq], wq, cos[at], sin[at], "rms", 1e-6, 1.0, layout)
    want_k = exact(rows[:, hq:hq + hkv], wk, cos[at], sin[at], "rms", 1e-6, 1.0, layout)
    check(q[good], want_q[good], dtype, "q")
    assert (q[30:] == 0).all() and q[6].isnan().all() and q[7].isnan().all()
    kc, vc = kc.cpu(), vc.cpu()
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for t in range(30):
        s = int(slots[t])
        if 0 <= s < pages * page:
            touched[s // page, s % page] = True
            if t == 7:
                assert kc[s // page, :, s % page].isnan().all()
            else:
                check(kc[s // page, :, s % page], want_k[t], dtype, f"k of token {t}")
            assert torch.equal(vc[s // page, :, s % page], rows[t, hq + hkv:])
    keep = ~touched[:, None, :, None].expand(kc.shape)
    assert torch.equal(kc[keep], kc0[keep]) and torch.equal(vc[keep], vc0[keep])


def test_special_values_stay_in_their_rows_and_unrotated_parts():
    from hydra_b200.kernels import fused_qk_norm_rope
    q = torch.zeros(4, 2, 16)
    q[1, 0, 12], q[1, 1, 3] = float("inf"), float("nan")
    q[2] = 3e19                                                           # the squares overflow
    q[3] = 1e-30
    cos, sin = (t.cuda() for t in tables(8, 8))
    a, _ = fused_qk_norm_rope(q.cuda(), q[:, :1].cuda(), cos, sin, norm=None)
    a = a.cpu()
    assert a[1, 0, 12] == float("inf") and a[1, 0].isfinite().sum() == 15     # the part behind `rot` is passed through
    assert a[1, 1].isnan().sum() == 2 and torch.equal(a[1, 1, 8:], q[1, 1, 8:])
    b, _ = fused_qk_norm_rope(q.cuda(), q[:, :1].cuda(), cos, sin, norm="rms")
    assert (b[0] == 0).all() and (b[2] == 0).all() and (b[3].abs() < 1e-25).all()   # rsqrt(inf) = 0; eps holds tiny rows down


def test_no_tokens_and_refusals():
    from hydra_b200.kernels import fused_qk_norm_rope
    from hydra_b200.paged import paged_append
    cos, sin = (t.cuda() for t in tables(8, 8))
    q, k = torch.zeros(0, 4, 8).cuda(), torch.zeros(0, 2, 8).cuda()
    a, b = fused_qk_norm_rope(q, k, cos, sin)
    assert a.shape == (0, 4, 8) and b.shape == (0, 2, 8)
    q, k = torch.zeros(3, 4, 8).cuda(), torch.zeros(3, 2, 8).cuda()
    c = torch.zeros(2, 2, 4, 8).cuda()
    s, p = torch.zeros(3, dtype=torch.int64).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="norm"):
        fused_qk_norm_rope(q, k, cos, sin, norm="layer")
    with pytest.raises(ValueError, match="layout"):
        fused_qk_norm_rope(q, k, cos, sin, layout="split")
    with pytest.raises(ValueError, match="rotated"):
        fused_qk_norm_rope(q[..., :6], k[..., :6], cos, sin)
    with pytest.raises(ValueError, match="cover"):
        fused_qk_norm_rope(torch.zeros(9, 4, 8).cuda(), torch.zeros(9, 2, 8).cuda(), cos, sin)
    with pytest.raises(TypeError, match="positions"):
        fused_qk_norm_rope(q, k, cos, sin, p.float())
    with pytest.raises(ValueError, match="positions"):
        fused_qk_norm_rope(q, k, cos, sin, p[:2])
    with pytest.raises(ValueError, match="q_weight"):
        fused_qk_norm_rope(q, k, cos, sin, q_weight=torch.ones(7).cuda())
    with pytest.raises(RuntimeError, match="inference only"):
        fused_qk_norm_rope(q.clone().requires_grad_(), k, cos, sin)
    with pytest.raises(ValueError, match="dtype"):
        paged_append(q, k, k, c.half(), c.half(), s, cos, sin, p)
    with pytest.raises(ValueError, match="fit"):
        paged_append(q, k, k, c[:, :1], c[:, :1], s, cos, sin, p)
    with pytest.raises(ValueError, match="slots"):
        paged_append(q, k, k, c, c, s.int(), cos, sin, p)
    with pytest.raises(ValueError, match="slots"):
        paged_append(q, k, k, c, c, s[:2], cos, sin, p)
    with pytest.raises(ValueError, match="contiguous"):
        paged_append(q, k, k, c.transpose(2, 3), c.transpose(2, 3), s, cos, sin, p)
    with pytest.raises(RuntimeError, match="inference only"):
        paged_append(q, k.clone().requires_grad_(), k, c, c, s, cos, sin, p)
