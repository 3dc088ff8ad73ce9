"""token_logprobs against a plain computation in 64 bits on the same logits.

Tolerance: 1e-5 + 1e-6 |x|.  A log probability is a difference of 32-bit values: (x - max) / T carries two roundings (2^-23
relative), ln Z the roundings of a sum of positive terms whose exponentials are right to 2^-22 relative plus 2^-23 times
their exponent's size (at most 150 before they vanish), so below 2^-15 of terms that matter least; what remains is under 1e-5."""
import pytest
import torch

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def exact(x, tokens, top, temperature):
    x = x.cpu()
    z = x.double() / temperature
    lp = torch.log_softmax(z, 1)                                          # (relative to the maximum: right at 1e38 too)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    ids = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    given = lp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    return given, h, lp.gather(1, ids), ids


def close(got, want, what):
    got = got.double().cpu()
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    d = (got - want).abs()[~inf]
    tol = (1e-5 + 1e-6 * want.abs())[~inf]
    assert (d <= tol).all(), f"{what}: off by {float(d.max()):.3e}"


def check(x, vocab=None, top=0, temperature=1.0, seed=0, tokens=None):
    from hydra_b200.sampling import token_logprobs
    V = vocab or x.shape[1]
    t = torch.randint(0, V, (x.shape[0],), generator=torch.Generator().manual_seed(seed)) if tokens is None else tokens
    r = token_logprobs(x, t.cuda(), top=top, temperature=temperature, vocab=vocab)
    lp, h, tl, ti = exact(x[:, :V], t, top, temperature)
    close(r.logprobs, lp, "logprobs")
    close(r.entropy, h, "entropy")
    close(r.top_logprobs, tl, "top_logprobs")
    assert torch.equal(r.top_ids.cpu(), ti), "top_ids"
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,V,ld,top", [(1, 1, 1, 1), (3, 2, 2, 2), (5, 37, 41, 32), (2, 33, 64, 32), (4, 1000, 1000, 5), (33, 777, 790, 20), (7, 4099, 4099, 32),
                                        (1, 50257, 50304, 20), (64, 50257, 50304, 5), (2, 152064, 152064, 8), (600, 1500, 1536, 1), (9, 20000, 20001, 0)])
def test_against_64_bits(dtype, N, V, ld, top):
    g = torch.Generator().manual_seed(N + V)
    x = (torch.randn(N, ld, generator=g) * 3).to(dtype)
    x[:, V:] = 90.0                                                       # padding columns must not count
    check(x.cuda(), vocab=V, top=top, temperature=0.7 if N % 2 else 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,V,top", [(900, 3001, 4), (1000, 5000, 5), (900, 5003, 0), (2000, 300, 32), (890, 70001, 20), (400, 9000, 3), (400, 9000, 30)])
def test_many_rows(dtype, N, V, top):
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(N, V + 5, generator=g, device="cuda") * 3).to(dtype)
    check(x[:, :V], top=top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 30.0, 1e6])
@pytest.mark.parametrize("N,V", [(3, 700), (2, 40000)])
def test_extreme_temperatures(dtype, temperature, N, V):
    """Differences of logits over a temperature near nothing are far beyond what e^x holds, or one token takes all."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(N, V, generator=g) * 4).to(dtype)
    x[0, 5:90] = -INF
    x[1] -= 20.0                                                          # a row of negative logits
    check(x.cuda(), top=8, temperature=temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nearly_certain_tokens(dtype):
    """ln p and the entropy of rows in which one token takes all but a small part e of the mass are of the size of e, and right to
    the roundings of the sum 1 + e.  Each of them is off by at most 2^-24 (half a step between one and two).  The sum that holds
    the one is added to by its thread's other columns, in pairs (at most 15 of 30000 in four slices over 512 threads: 8
    times), once by its second half, five times over the lanes, four over the warps and three over the slices: 21 roundings.
    The terms' own are 2^-22 of e each and the product and the sum of the result a few 2^-24 of it: 2^-20 relative."""
    g = torch.Generator().manual_seed(6)
    for V in (1000, 30000):
        x = torch.randn(40, V, generator=g)
        x[:, 7] = torch.linspace(9.0, 30.0, 40)
        x = x.to(dtype)
        from hydra_b200.sampling import token_logprobs
        t = torch.full((40,), 7)
        r = token_logprobs(x.cuda(), t.cuda(), top=1)
        lp, h, tl, ti = exact(x, t, 1, 1.0)
        for got, want in ((r.logprobs, lp), (r.top_logprobs[:, 0], tl[:, 0])):
            assert ((got.double().cpu() - want).abs() <= 21 * 2.0 ** -24 + 2.0 ** -20 * want.abs()).all()
        # (an entropy's terms are e times distances of up to 34: their sum is rounded where e times 34 is, at less than 2^-24 of
        # the entropy each; the one's roundings come in through ln Z and through the division)
        assert ((r.entropy.double().cpu() - h).abs() <= 2 * 21 * 2.0 ** -24 + 2.0 ** -19 * h.abs()).all()


@pytest.mark.parametrize("scale", [1e5, 1e8, 1e30, -1e30])
@pytest.mark.parametrize("N", [2, 300])
def test_huge_logits(scale, N):
    """The distances between logits stay small, or come out in whole steps of the type, whatever their size."""
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        x = (scale * (1 + 1e-6 * torch.randn(N, 9000, generator=g))).to(dtype)
        check(x.cuda(), top=6)
        x[:, ::2] = -INF
        check(x.cuda(), top=6, tokens=torch.ones(N, dtype=torch.int64))
    x = torch.full((N, 20000), -65504.0, dtype=torch.float16)             # half precision masked by its lowest value
    x[:, 3::7] = -INF
    check(x.cuda(), top=4, temperature=100.0, tokens=torch.zeros(N, dtype=torch.int64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [1, 3, 7])
def test_rows_off_16_byte_boundaries(dtype, shift):
    x = torch.randn(6, 9001, generator=torch.Generator().manual_seed(shift)).to(dtype).cuda()
    check(x[:, shift:], top=9)
    check(x[:, shift:shift + 5], top=5)                                   # shorter than the way to the boundary
    check(x[1:2, shift:].expand(3, -1), top=2)                            # overlapping rows


@pytest.mark.parametrize("V", [6, 500, 30000, 120000])
@pytest.mark.parametrize("N", [1, 40, 300])
def test_ties_and_masks(V, N):
    """All equal; a few allowed tokens, fewer than `top`; the lowest finite value as a mask; two levels; signed zeros."""
    top = min(V, 20)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(N, V, dtype=dtype)
        x[:, 1::2] = -0.0
        check(x.cuda(), top=top)
        x = torch.full((N, V), -INF, dtype=dtype)
        x[:, V // 2], x[:, V - 1] = 1.5, 2.0
        check(x.cuda(), top=top, tokens=torch.full((N,), V // 2))
        x = torch.full((N, V), torch.finfo(dtype).min, dtype=dtype)
        x[:, ::5] = -2.0
        check(x.cuda(), top=top, tokens=torch.zeros(N, dtype=torch.int64))
        x = torch.full((N, V), torch.finfo(dtype).min, dtype=dtype)       # nothing but the lowest value: uniform
        check(x.cuda(), top=top)
        x = torch.where(torch.arange(V) % 3 == 1, 4.0, -1.0).to(dtype).expand(N, V).contiguous()
        check(x.cuda(), top=top)


def test_sorted_rows_and_many_candidates():
    """Rows in which one thread's columns hold all of the largest logits, or each tile is above the one before."""
    for x in (torch.linspace(-9, 9, 40000)[None], torch.linspace(9, -9, 40000)[None].repeat(200, 1)):
        check(x.contiguous().cuda(), top=32)
    x = torch.full((3, 100000), -5.0)
    x[:, ::4096] = torch.arange(25.0)                                     # one thread's pieces, if 512 threads take 8 columns each
    check(x.to(torch.bfloat16).cuda(), top=32)
    x = torch.full((160, 60000), -5.0)
    x[:, (torch.arange(60000) // 8) % 512 < 30] = 1.0 + torch.rand(160, int(((torch.arange(60000) // 8) % 512 < 30).sum()),
                                                                    generator=torch.Generator().manual_seed(1))
    check(x.to(torch.bfloat16).float().cuda(), top=32)                    # more logits above the bound than the list holds
    check(x.to(torch.bfloat16).cuda(), top=32)


def test_rows_without_a_distribution():
    from hydra_b200.sampling import token_logprobs
    for V in (64, 30000):
        x = torch.randn(6, V, generator=torch.Generator().manual_seed(2))
        x[1] = -INF
        x[2, 7] = NAN
        x[3, 9] = INF
        x[4, 5], x[4, 11], x[4, 3] = NAN, INF, NAN
        r = token_logprobs(x.cuda(), torch.zeros(6, dtype=torch.int64).cuda(), top=4)
        for t in (r.logprobs, r.entropy, r.top_logprobs):
            assert t[1:5].isnan().all() and t[[0, 5]].isfinite().all()
        ids = r.top_ids.cpu()
        assert ids[1].tolist() == [0, 1, 2, 3] and ids[2, 0] == 7 and ids[3, 0] == 9 and ids[4, :3].tolist() == [3, 5, 11]
        check(x[[0, 5]].cuda(), top=4)


def test_tokens_that_are_not_scored():
    from hydra_b200.sampling import cross_entropy_rows, token_logprobs
    x = (torch.randn(6, 5000, generator=torch.Generator().manual_seed(3)) * 2).to(torch.bfloat16).cuda()
    t = torch.tensor([3, -100, 5000, -1, 4999, 0])
    r = token_logprobs(x, t.cuda(), top=2)
    assert r.logprobs[1] == 0 and r.logprobs[2].isnan() and r.logprobs[3].isnan() and r.entropy.isfinite().all()
    ok = [0, 1, 4, 5]
    nll = cross_entropy_rows(x[ok], t[ok].cuda())
    assert float((r.logprobs[ok] + nll).abs().max()) < 1e-4
    assert token_logprobs(x, t.cuda(), ignore_index=-1).logprobs[3] == 0


def test_sizes_streams_graphs_and_refusals():
    from hydra_b200.sampling import token_logprobs
    x = torch.randn(5, 30000, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    t = torch.arange(5).cuda()
    r = token_logprobs(x[:0], t[:0], top=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    want = token_logprobs(x, t, top=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, t, top=3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    y = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(y, t, top=3)
    for shift in (0, 1):
        y.copy_(x.roll(shift, 0))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(token_logprobs(y, t, top=3), got))
    for bad, text in ((dict(top=33), "top"), (dict(top=-1), "top"), (dict(temperature=0.0), "temperature"), (dict(vocab=30001), "vocab"), (dict(vocab=0), "vocab")):
        with pytest.raises(ValueError, match=text):
            token_logprobs(x, t, **bad)
    with pytest.raises(ValueError, match="token per row"):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="token per row"):
        token_logprobs(x, t[:4])
    with pytest.raises(ValueError, match="column stride"):
        token_logprobs(x.t(), t)
    with pytest.raises(TypeError, match="float32, bfloat16"):
        token_logprobs(x.double(), t)
    with pytest.raises(RuntimeError, match="inference only"):
        token_logprobs(x.float().requires_grad_(), t)


def test_model_and_session_entry_points():
    """HydraB200Model.token_logprobs beside eval_loss and the model's own logits, DecodeSession.token_logprobs beside the
    logits of the step."""
    from hydra_b200.sampling import token_logprobs
    from tests import golden_io as G
    from tests.test_gpu_model import build
    fx, cfg, w = G.model_fixture("model_hd32.npz")
    m = build(w, cfg)
    ids = torch.from_numpy(fx["ids"]).clamp(0, cfg.vocab_size - 1).cuda()
    r = m.token_logprobs(ids, top=3)
    B, S = ids.shape
    assert r.logprobs.shape == (B, S - 1) and r.top_ids.shape == (B, S - 1, 3)
    assert float((r.logprobs + m.eval_loss(ids, reduction="none")).abs().max()) < 1e-4
    lg = m(ids[:, :-1]).float()
    close(r.entropy, torch.distributions.Categorical(logits=lg.double()).entropy().cpu(), "entropy")
    assert torch.equal(r.top_ids[..., 0], lg.argmax(-1))
    with pytest.raises(ValueError):
        m.token_logprobs(ids[:, :1])
    s = m.new_decode_session(B, 16)
    with pytest.raises(RuntimeError):
        s.token_logprobs()
    s.prefill(ids[:, :8])
    for _ in range(2):
        got = s.token_logprobs(top=2)
        assert torch.equal(got.top_ids[:, 0], s.tokens) and torch.equal(got.logprobs, got.top_logprobs[:, 0])
        assert torch.equal(got.logprobs, token_logprobs(s.last_logits, s.tokens, vocab=cfg.vocab_size).logprobs)
        s.step()
