"""Serving operators at the ends of their ranges."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


# ------------------------------------------------------------------------------------------- token log probabilities
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,top", [(3, 4, 4), (2, 32, 32), (3, 700, 20), (400, 700, 3), (1000, 200, 2), (1, 200000, 32), (2, 200000, 1)])
def test_nan_in_the_first_column_is_the_first_alternative(dtype, N, V, top):
    """NaN is above +inf and the lowest index comes first: ids in order whatever column it lies in, the first slice's or a later
    slice's first among them (rows of 200000 columns are split over a cluster)."""
    from hydra_b200.sampling import token_logprobs
    x = torch.randn(N, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    x[:, 0] = NAN
    x[-1, V // 2], x[-1, V - 1] = NAN, INF
    r = token_logprobs(x.cuda(), torch.ones(N, dtype=torch.int64).cuda(), top=top)
    key = x.float().nan_to_num(nan=INF, posinf=3e38)
    assert torch.equal(r.top_ids.cpu(), torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top])
    assert r.logprobs.isnan().all() and r.entropy.isnan().all() and r.top_logprobs.isnan().all()


# ------------------------------------------------------------------------------------------------------------ attention
def pages_of(k, v, page, seed=0):
    """k, v [B, n, hkv, hd] -> caches [pages, hkv, page, hd] with the pages in any order, and the table"""
    B, n, hkv, hd = k.shape
    W = -(-n // page)
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(B * W, generator=g).view(B, W)
    kc, vc = (torch.zeros(B * W, hkv, page, hd, dtype=t.dtype) for t in (k, v))
    for c, t in ((kc, k), (vc, v)):
        full = torch.zeros(B, W * page, hkv, hd, dtype=t.dtype)
        full[:, :n] = t
        c[ids.flatten()] = full.view(B * W, page, hkv, hd).transpose(1, 2)
    return kc.cuda(), vc.cuda(), ids.int().cuda()


def attend(q, k, v, scale):
    """One kv head.  -> out, lse and sum of weights times |v|, in 64 bits"""
    s = torch.einsum("bhd,bnd->bhn", q.double(), k[:, :, 0].double()) * scale
    p = torch.softmax(s, 2)
    return torch.einsum("bhn,bnd->bhd", p, v[:, :, 0].double()), torch.logsumexp(s, 2), torch.einsum("bhn,bnd->bhd", p, v[:, :, 0].double().abs())


@pytest.mark.parametrize("dtype,top", [(torch.bfloat16, 2.0 ** 20), (torch.bfloat16, 2.0 ** 40), (torch.float16, 2.0 ** 15), (torch.float16, 2.0 ** 10)])
@pytest.mark.parametrize("heads,hd", [(1, 128), (8, 64), (20, 16), (3, 256)])
@pytest.mark.parametrize("n", [70, 5000])
def test_scores_of_any_size(dtype, top, heads, hd, n):
    """Scores of up to 2^80 * scale: their distances decide, whatever the size.  Two keys share the largest one, all others lie below
    by at least 2^-10 of it: the answer is the two values' mean (2^-22 of the weights' exponentials, one rounding)."""
    from hydra_b200.paged import paged_decode_attention
    scale = hd ** -0.5
    g = torch.Generator().manual_seed(n + heads)
    q, k = torch.zeros(2, heads, hd), torch.zeros(2, n, 1, hd)
    q[:, :, :4] = top
    k[..., :4] = (top * (0.25 + 0.5 * torch.rand(2, n, 1, 1, generator=g)))
    k[1] = -k[1]                                                          # and a request of scores far below zero
    k[0, 3, 0, :4] = k[0, n - 2, 0, :4] = top
    k[1, 3, 0, :4] = k[1, n - 2, 0, :4] = -top / 8
    v = torch.randn(2, n, 1, hd, generator=g)
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    kc, vc, table = pages_of(k, v, 16)
    out, l = (t.double().cpu() for t in paged_decode_attention(q.cuda(), kc, vc, table, torch.full((2,), n, dtype=torch.int32).cuda(), scale=scale,
                                                               return_lse=True))
    want, lse, mass = attend(q, k, v, scale)
    half = torch.finfo(dtype).eps / 2
    assert ((out - want).abs() <= half * want.abs() + 2.0 ** -16 * mass + 2.0 ** -25).all(), float((out - want).abs().max())
    assert float(((l - lse).abs() / (1 + lse.abs())).max()) <= 1e-5
    small = paged_decode_attention(q.cuda(), kc, vc, table, torch.full((2,), n, dtype=torch.int32).cuda(), scale=-scale).double().cpu()
    want = attend(q, k, v, -scale)[0]
    if n == 70:                                                           # (one share: the order turned round)
        assert small.isfinite().all() and float((small - want).abs().max()) <= 2 * half * 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 8, 20])
@pytest.mark.parametrize("B,n,at", [(64, 4096, 0), (64, 4096, 4095), (200, 1000, 500), (1, 4096, 0), (1, 60000, 7), (3, 20000, 19999)])
def test_a_token_that_takes_nearly_all_and_gives_nothing(dtype, heads, B, n, at):
    """One key 10 to 20 nats above thousands of equal others, its value row zero: the output is what the others leave.

    Per value: half a step of the type (2^-25 in f16 below its normal range) for the rounding; the weights as two summands: f16
    ones are held up to 2^15 in steps of 2^-24, so each is off by at most 2^-40 of the largest, or 2^-17 of itself (bf16; f16:
    2^-22); exponentials 2^-22 and 2^-24 times an exponent of at most 2^6 (log2(e) 20 + 15) twice: 2^-17; the sums of n / 16
    products 2^-24 each, at most twice (numerator and denominator): n 2^-27."""
    from hydra_b200.paged import paged_decode_attention
    hd, scale = 64, 0.125
    g = torch.Generator().manual_seed(n)
    q = torch.zeros(B, heads, hd)
    q[:, :, 0] = 10.0 + (torch.arange(heads) % 9) * 1.25                  # scores: 8 q scale = 10 .. 20
    k = torch.randn(B, n, 1, hd, generator=g)
    k[..., 0] = 0.0
    v = (0.5 + torch.rand(B, n, 1, hd, generator=g)) * 8
    k[:, at, :, 0], v[:, at] = 8.0, 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    want, lse, mass = attend(q, k, v, scale)
    kc, vc, table = pages_of(k, v, 16)
    out, l = paged_decode_attention(q.cuda(), kc, vc, table, torch.full((B,), n, dtype=torch.int32).cuda(), scale=scale, return_lse=True)
    half = torch.finfo(dtype).eps / 2
    off = (out.double().cpu() - want).abs()
    tol = half * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0) + n * 2.0 ** -40 * 12 + (2.0 ** -16 + n * 2.0 ** -27) * mass
    assert (off <= tol).all(), f"off by {float((off / tol).max()):.2f} tolerances, {float((off / want).max()):.2e} of the value"
    assert float(((l.double().cpu() - lse).abs() / (1 + lse.abs())).max()) <= 1e-5

@pytest.mark.parametrize("heads,hd", [(4, 64), (20, 16)])
@pytest.mark.parametrize("n", [1, 37, 3000])
@pytest.mark.parametrize("power,scale", [(60, 2.0 ** -119), (60, -2.0 ** -119), (60, 0.0), (0, 0.0), (30, -0.0), (-70, 2.0 ** 126), (-70, -2.0 ** 127.5), (63, 2.0 ** -140)])
def test_scales_of_any_size(heads, hd, n, power, scale):
    """Scores near 2^(2 power) times a scale near its inverse: weights, mean values and sums as at ordinary sizes (2^-16 of the
    weights' exponents, whose size is below 2^7; a scale of zero weighs all tokens alike)."""
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(n + hd)
    q, k, v = torch.zeros(2, heads, hd), torch.zeros(2, n, 1, hd), torch.randn(2, n, 1, hd, generator=g)
    q[..., 0] = 2.0 ** power
    k[..., 0] = (torch.randint(-64, 64, (2, n, 1), generator=g) / 32) * 2.0 ** power
    q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    kc, vc, table = pages_of(k, v, 16)
    out, l = (t.double().cpu() for t in paged_decode_attention(q.cuda(), kc, vc, table, torch.full((2,), n, dtype=torch.int32).cuda(), scale=scale,
                                                               return_lse=True))
    want, lse, mass = attend(q, k, v, torch.tensor(scale, dtype=torch.float32).item())
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -14 + n * 2.0 ** -27) * mass).all(), float((out - want).abs().max())
    assert float(((l - lse).abs() / (1 + lse.abs())).max()) <= 1e-5


def test_out_within_what_is_read_is_refused():
    from hydra_b200.paged import paged_decode_attention
    arena = torch.zeros(3, 4, 2, 16, 64, dtype=torch.float16, device="cuda")
    kc, vc, spare = arena.unbind(0)
    q = torch.randn(2, 8, 64, device="cuda").half()
    ints = torch.zeros(4096, dtype=torch.int32, device="cuda")
    table, n = ints[:4].view(2, 2), ints[4:6].fill_(20)
    as_out = lambda t: t.view(torch.float16).flatten()[:q.numel()].view(q.shape)   # noqa: E731
    for name, out in (("k_cache", as_out(kc)), ("v_cache", as_out(vc[2])), ("block_tables", as_out(ints)), ("kv_lens", as_out(ints[4:]))):
        with pytest.raises(ValueError, match=f"overlap {name}"):
            paged_decode_attention(q, kc, vc, table, n, out=out)
    assert (arena == 0).all() and (ints[:4] == 0).all()
    want = paged_decode_attention(q, kc, vc, table, n)
    assert torch.equal(paged_decode_attention(q, kc, vc, table, n, out=as_out(spare)), want)


@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_keys_and_values_in_one_tensor(at):
    """Caches that lie between one another are filled like any others; one tensor for both, or rows that overlap, are refused."""
    from hydra_b200.paged import paged_append
    sizes = [6, 2, 8, 16]
    room = torch.zeros(*sizes[:at], 2, *sizes[at:], device="cuda")
    kc, vc = room.unbind(at)
    apart = torch.zeros(6, 2, 8, 16, device="cuda"), torch.zeros(6, 2, 8, 16, device="cuda")
    cos, sin = torch.ones(32, 8, device="cuda"), torch.zeros(32, 8, device="cuda")
    x, y, z = torch.randn(3, 5, 2, 16, device="cuda")
    slots, pos = torch.tensor([3, 47, 0, 16, 9]).cuda(), torch.arange(5).cuda()
    q = paged_append(x, y, z, kc, vc, slots, cos, sin, pos)
    assert torch.equal(q, paged_append(x, y, z, *apart, slots, cos, sin, pos)) and torch.equal(kc, apart[0]) and torch.equal(vc, apart[1])
    before = room.clone()
    for k, v in ((kc, kc), (kc, kc.as_strided(kc.shape, kc.stride())), (kc[:1].expand(6, -1, -1, -1), vc),
                 (apart[0].as_strided((6, 2, 8, 16), (256, 128, 8, 1)), vc)):
        with pytest.raises(RuntimeError, match="on top"):
            paged_append(x, y, z, k, v, slots, cos, sin, pos)
    with pytest.raises(RuntimeError, match="overlap"):
        paged_append(kc[:5, :, 0], y, z, kc, vc, slots, cos, sin, pos)
    assert torch.equal(room, before)


def test_plan_with_a_free_list_in_its_tables_is_refused():
    from hydra_b200.paged import paged_plan
    room = torch.arange(40, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        paged_plan(n, n + 5, room[:8].view(2, 4), room[6:20], 16, 16)
    assert torch.equal(room, torch.arange(40, device="cuda").int())
    plan = paged_plan(n, n + 5, room[:8].view(2, 4), room[8:20], 16, 16)
    assert room[:8].tolist() == [8, 1, 2, 3, 9, 5, 6, 7] and int(plan.status) == 0


# ------------------------------------------------------------------------------------------------------------- autograd
def small_server():
    i32 = dict(dtype=torch.int32, device="cuda")
    kc, vc = torch.zeros(2, 6, 2, 8, 16, device="cuda").unbind(0)
    cos, sin = torch.ones(32, 8, device="cuda"), torch.zeros(32, 8, device="cuda")
    return i32, kc.clone(), vc.clone(), cos, sin


def test_writes_in_place_are_seen_by_autograd():
    """A tensor that a call writes counts as changed: a backward pass that needs its old contents says so."""
    from hydra_b200.paged import paged_append, paged_decode_attention, paged_plan
    i32, kc, vc, cos, sin = small_server()
    w = torch.ones_like(kc, requires_grad=True)
    table = torch.full((2, 3), -1, **i32)
    kept = (w * kc).sum(), (w * vc).sum()
    version = table._version
    plan = paged_plan(torch.zeros(2, **i32), torch.tensor([3, 1], **i32), table, torch.arange(6, **i32), 8, 4)
    assert table._version > version
    x = torch.randn(4, 2, 16, device="cuda")
    paged_append(x, x, x, kc, vc, plan.slots, cos, sin, plan.positions)
    for y in kept:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():                                          # (inference tensors keep no versions)
        a, b = torch.zeros_like(kc), torch.zeros_like(vc)
        paged_append(x, x, x, a, b, plan.slots, cos, sin, plan.positions)
        assert torch.equal(a, kc) and torch.equal(b, vc)
    h = torch.randn(2, 2, 16, device="cuda").half()
    out = torch.zeros_like(h)
    version = out._version
    paged_decode_attention(h, kc.half(), vc.half(), table, plan.kv_lens, out=out)
    assert out._version > version


def test_forward_mode_tangents_are_refused():
    """A derivative that would be dropped in silence is refused, in forward mode too, under no_grad too (which does not end it)."""
    import torch.autograd.forward_ad as fwd
    from hydra_b200.kernels import fused_qk_norm_rope
    from hydra_b200.paged import paged_append, paged_decode_attention
    from hydra_b200.sampling import token_logprobs
    i32, kc, vc, cos, sin = small_server()
    x = torch.randn(4, 2, 16, device="cuda")
    where = torch.arange(4, **i32)
    n = torch.tensor([1, 2, 3, 4], **i32)
    table = torch.zeros(4, 1, **i32)
    h, hk, hv = x.half(), kc.half(), vc.half()
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))                # noqa: E731
        for call in (lambda: fused_qk_norm_rope(d(x), x, cos, sin), lambda: fused_qk_norm_rope(x, x, d(cos), sin),
                     lambda: fused_qk_norm_rope(x, x, cos, sin, q_weight=d(torch.ones(16, device="cuda"))),
                     lambda: paged_append(x, x, d(x), kc, vc, where.long(), cos, sin, where),
                     lambda: paged_append(x, x, x, d(kc), vc, where.long(), cos, sin, where),
                     lambda: paged_decode_attention(d(h), hk, hv, table, n), lambda: paged_decode_attention(h, hk, d(hv), table, n),
                     lambda: token_logprobs(d(x[0]), torch.zeros(2, dtype=torch.int64, device="cuda"))):
            with pytest.raises(RuntimeError, match="inference only"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="inference only"):
                call()
        fused_qk_norm_rope(x, x, cos, sin)                                # without tangents: as ever


# ---------------------------------------------------------------------------------------------------------------- model
def test_model_scores_ids_of_any_integer_type():
    """HydraB200Model.token_logprobs takes what forward and eval_loss take."""
    from tests import golden_io as G
    from tests.test_gpu_model import build
    fx, cfg, w = G.model_fixture("model_hd32.npz")
    m = build(w, cfg)
    ids = torch.from_numpy(fx["ids"]).clamp(0, cfg.vocab_size - 1).cuda()
    want = m.token_logprobs(ids, top=2)
    for got in (m.token_logprobs(ids.int(), top=2), m.token_logprobs(ids[:, :-1].int(), ids[:, 1:].int(), top=2)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
