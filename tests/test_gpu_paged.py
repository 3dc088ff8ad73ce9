"""The paged cache: paged_plan against a request-by-request computation, paged_decode_attention against softmax in 64 bits,
and whole serving steps of plan, append, attention and log probabilities.

Tolerance of the attention, per value: half a step of the output's type relative to the value (the one rounding), plus 2^-14
of the largest |v| a request attends to: the weights enter the products as two summands (2^-17 left out of bf16 ones), their
exponentials are right to 2^-21 (2^-22 of the instruction, 2^-24 times an exponent below 8 in weights that matter), and the
32-bit sums of up to 4096 / 16 tile products add at most 2^-24 * 256 = 2^-16 each in two sums.  Over all values the error is
the rounding's: at most half a step in the 2-norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


# ---------------------------------------------------------------------------------------------------------------- plan
def plan_by_hand(context, new, table, free, page, room, start=0):
    """One request, one token, one page after another.  -> table, kv_lens, cu, positions, slots, next, status"""
    W = table.shape[1]
    table, status, taken = table.clone(), 0, start
    pos, slots, cu, lens = [], [], [0], []
    for b, (c, n) in enumerate(zip(context.tolist(), new.tolist())):
        if c < 0 or n < 0:
            status |= 8
            c, n = max(c, 0), max(n, 0)
        held, want = -(-c // page), -(-(c + n) // page)
        if want > W:
            status |= 2
        for j in range(min(held, W), min(want, W)):
            if taken < len(free):
                table[b, j] = free[taken]
            else:
                table[b, j] = -1
                status |= 1
            taken += 1
        for t in range(c, c + n):
            pos.append(t)
            p = int(table[b, t // page]) if t // page < W else -1
            slots.append(p * page + t % page if p >= 0 else -1)
        cu.append(cu[-1] + n)
        lens.append(c + n)
    if len(pos) > room:
        status |= 4
    pad = [-1] * max(0, room - len(pos))
    return table, lens, cu, (pos + pad)[:room], (slots + pad)[:room], min(taken, len(free)), status


def run_plan(context, new, table, free, page, room, start=None):
    from hydra_b200.paged import paged_plan
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32)   # noqa: E731
    context, new, free = i32(context), i32(new), i32(free)
    want = plan_by_hand(context, new, table, free, page, room, start or 0)
    dev = table.cuda()
    args = (context.cuda(), new.cuda(), dev, free.cuda(), page, room, None if start is None else i32([start]).cuda())
    for _ in range(2):                                                    # the same call again gives the same
        p = paged_plan(*args)
        got = (dev.cpu(), p.kv_lens.tolist(), p.cu_new.tolist(), p.positions.tolist(), p.slots.tolist(), int(p.free_start), int(p.status))
        assert torch.equal(got[0], want[0])
        assert got[1:] == want[1:], [(a, b) for a, b in zip(got[1:], want[1:]) if a != b]
    return p


def random_requests(g, B, W, page, most_new):
    pages = torch.randperm(4 * B * W + 8, generator=g).int()
    context = torch.randint(0, max(1, W * page - most_new), (B,), generator=g)
    table = pages[:B * W].view(B, W).clone()
    for b in range(B):
        table[b, -(-int(context[b]) // page):] = -7                       # what lies behind the pages held is not read
    new = torch.randint(0, most_new + 1, (B,), generator=g)
    return context, new, table, pages[B * W:]


@pytest.mark.parametrize("B,W,page,most_new", [(1, 1, 1, 1), (1, 8, 16, 100), (3, 5, 7, 20), (64, 40, 16, 1), (257, 9, 16, 64), (300, 3, 1, 2),
                                               (1500, 4, 24, 40), (4096, 2, 16, 3)])
def test_plan(B, W, page, most_new):
    g = torch.Generator().manual_seed(B + W)
    context, new, table, free = random_requests(g, B, W, page, min(most_new, W * page))
    total = int(new.sum())
    run_plan(context, new, table, free, page, total + 5)
    run_plan(context, new, table, free, page, total, start=3)
    if total > 1:
        run_plan(context, new, table, free, page, total // 2)             # more tokens than rows


def test_plan_edges():
    t = torch.full((3, 4), -1, dtype=torch.int32)
    run_plan([0, 0, 0], [0, 0, 0], t, [5, 6], 16, 0)
    run_plan([0, 0, 0], [0, 0, 0], t, [], 16, 9)
    run_plan([0, 0, 0], [16, 17, 1], t, [5, 6, 7, 8], 16, 40)            # whole pages, one over
    run_plan([0, 0, 0], [16, 17, 1], t, [5, 6], 16, 40)                  # the free list ends inside the second request
    run_plan([0, 0, 0], [16, 17, 1], t, [5, 6, 9, 4], 16, 40, start=2)
    run_plan([0, 0, 0], [2, 65, 1], t, list(range(9)), 16, 70)           # the second outgrows its row of four pages
    run_plan([0, -3, 2], [5, 2, -1], torch.zeros((3, 4), dtype=torch.int32), list(range(9)), 16, 20)
    run_plan([30, 0, 63], [40, 0, 1], torch.arange(12, dtype=torch.int32).view(3, 4), list(range(20, 40)), 16, 50)
    run_plan([], [], torch.empty((0, 4), dtype=torch.int32), [1], 16, 7)
    wide = torch.full((3, 9), -1, dtype=torch.int32).cuda()               # a table that is part of a wider one
    from hydra_b200.paged import paged_plan
    p = paged_plan(torch.zeros(3, dtype=torch.int32).cuda(), torch.full((3,), 20, dtype=torch.int32).cuda(), wide[:, 2:6],
                   torch.arange(10, dtype=torch.int32).cuda(), 16, 60)
    assert wide.tolist() == [[-1, -1, 2 * b, 2 * b + 1, -1, -1, -1, -1, -1] for b in range(3)] and int(p.free_start) == 6
    big = torch.full((1, 4), 1 << 27, dtype=torch.int32)                  # slots past 32 bits
    q = run_plan([17], [3], big, [3], 64, 4)
    assert q.slots.tolist()[0] == (1 << 33) + 17
    huge = paged_plan(torch.tensor([2 ** 31 - 5], dtype=torch.int32).cuda(), torch.tensor([90], dtype=torch.int32).cuda(), big.cuda(),
                      torch.arange(4, dtype=torch.int32).cuda(), 64, 8)
    assert int(huge.status) & 8 and int(huge.kv_lens) == 2 ** 31 - 1


def test_plan_refusals():
    from hydra_b200.paged import paged_plan
    i = torch.zeros(2, dtype=torch.int32).cuda()
    t = torch.zeros((2, 4), dtype=torch.int32).cuda()
    for args, text in (((i.long(), i, t, i, 16, 8), "context_lens"), ((i, i[:1], t, i, 16, 8), "new lengths"), ((i, i, t[:1], i, 16, 8), "block tables"),
                       ((i, i, t.long(), i, 16, 8), "block tables"), ((i, i, t, i, 0, 8), "page_size"), ((i, i, t, i, 16, -1), "max_new_tokens"),
                       ((i, i, t[:, ::2], i, 16, 8), "rows"), ((i, i, t[:1].expand(2, 4), i, 16, 8), "rows"), ((i, i, t, i, 16, 8, i), "free_start")):
        with pytest.raises(ValueError, match=text):
            paged_plan(*args)


# ----------------------------------------------------------------------------------------------------------- attention
def cache_of(g, lens, hkv, hd, page, dtype, order="hnd", junk=NAN, spare=2):
    """Random pages for requests of these lengths; what no request holds, and the rows behind each one's end, is `junk`."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    k, v = torch.randn(2, pages, hkv, page, hd, generator=g).to(dtype)
    W = max(need + [1])
    table = torch.full((len(lens), W), 10 ** 6, dtype=torch.int32)        # entries behind a request's end are not read
    ids = torch.randperm(pages, generator=g)
    at = 0
    free = torch.ones(pages, dtype=torch.bool)
    for b, n in enumerate(lens):
        mine = ids[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = mine.int()
        free[mine] = False
        if n % page:
            k[mine[-1], :, n % page:], v[mine[-1], :, n % page:] = junk, junk
    k[free], v[free] = junk, junk
    if order == "nhd":
        kd, vd = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v))
    else:
        kd, vd = k.cuda(), v.cuda()
    return k, v, kd, vd, table


def attend(q, k, v, table, lens, scale):
    """-> out, lse in 64 bits, and the largest |v| that each request attends to"""
    B, Hq, hd = q.shape
    page, group = k.shape[2], Hq // k.shape[1]
    out, lse, big = torch.zeros(B, Hq, hd, dtype=torch.float64), torch.full((B, Hq), -INF, dtype=torch.float64), torch.zeros(B)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = table[b, :-(-n // page)].long()
        kk = k[ids].transpose(1, 2).reshape(-1, k.shape[1], hd)[:n].double().repeat_interleave(group, 1)
        vv = v[ids].transpose(1, 2).reshape(-1, k.shape[1], hd)[:n].double().repeat_interleave(group, 1)
        s = torch.einsum("hd,nhd->hn", q[b].double(), kk) * scale
        lse[b] = torch.logsumexp(s, 1)
        out[b] = torch.einsum("hn,nhd->hd", torch.softmax(s, 1), vv)
        big[b] = vv.abs().max()
    return out, lse, big


def check(got, lse_got, want, lse, big, dtype):
    got, lse_got = got.double().cpu(), lse_got.double().cpu()
    half = torch.finfo(dtype).eps / 2
    tol = half * want.abs() + 2.0 ** -14 * big[:, None, None]
    worst = ((got - want).abs() / tol.clamp_min(1e-30)).max()
    assert not got.isnan().any() and worst <= 1, f"off by {float(worst):.2f} tolerances"
    rel = float((got - want).norm() / want.norm().clamp_min(1e-30))
    assert rel <= half, f"2-norm {rel:.3e}"
    fine = lse.isfinite()
    assert torch.equal(lse_got[~fine], lse[~fine])
    assert float(((lse_got - lse).abs() / (1 + lse.abs()))[fine].max() if fine.any() else 0) <= 1e-5


def run(lens, hq, hkv, hd, page, dtype=torch.bfloat16, order="hnd", scale=None, seed=0):
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(seed + hd + page + sum(lens))
    k, v, kd, vd, table = cache_of(g, lens, hkv, hd, page, dtype, order)
    q = (1.5 * torch.randn(len(lens), hq, hd, generator=g)).to(dtype)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = paged_decode_attention(q.cuda(), kd, vd, table.cuda(), n, scale=scale, return_lse=True)
    assert out.dtype == dtype and out.is_contiguous() and lse.dtype == torch.float32
    check(out, lse, *attend(q, k, v, table, lens, hd ** -0.5 if scale is None else scale), dtype)
    again = paged_decode_attention(q.cuda(), kd, vd, table.cuda(), n, scale=scale)
    assert torch.equal(out, again)                                        # equal bits, with or without lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 4, 128), (8, 2, 32), (32, 4, 16), (12, 3, 64), (2, 1, 256), (5, 1, 80), (16, 1, 8), (20, 1, 64), (40, 2, 128),
                                       (33, 1, 24), (6, 2, 200), (3, 3, 40), (20, 1, 256), (48, 2, 16), (9, 1, 32), (26, 1, 64), (51, 1, 128),
                                       (17, 1, 16), (64, 1, 32)])
def test_heads_and_sizes(dtype, order, hq, hkv, hd):
    run([1, 17, 64, 0, 333, 2], hq, hkv, hd, 16, dtype, order)


@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
@pytest.mark.parametrize("hd", [16, 64, 128])
def test_pages_that_end_inside_a_tile(page, hd):
    run([15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1], 8, 2, hd, page)


@pytest.mark.parametrize("lens", [[1], [4096], [3], [0, 0, 0], [0], [0, 5, 0, 0, 9, 0], [4000] + [1] * 63, [1] * 700, [50] * 300, [2500, 0, 7, 2500],
                                  list(range(90)), [3000, 1] * 40 + [0] * 7 + [17] * 200, [6000, 5000, 1, 0, 2]])
def test_lengths(lens):
    run(lens, 8, 2, 64, 16)
    if len(lens) < 100:
        run(lens, 4, 1, 128, 16)
        run(lens, 20, 2, 32, 64)


def test_large_batch_and_odd_scales():
    run([i % 7 for i in range(4096)], 2, 1, 32, 4)
    run([100, 700, 40], 8, 4, 64, 16, scale=-0.3)
    run([100, 700, 40], 8, 4, 64, 16, scale=0.0)
    run([100, 700, 40], 8, 4, 64, 16, scale=2.0)                          # nearly one token takes it all


def test_a_long_cache_whose_offsets_pass_32_bits():
    """Pages of one sequence at both ends of a cache of more than 2^31 elements (4.6 GB each for K and V)."""
    from hydra_b200.paged import paged_decode_attention
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    hkv, hd, page, pages = 2, 128, 64, 140000
    k, v = (torch.empty(pages, hkv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    g = torch.Generator().manual_seed(5)
    small_k, small_v = torch.randn(2, 4, hkv, page, hd, generator=g).to(torch.bfloat16)
    ids = torch.tensor([[pages - 1, 0, pages - 2, 70000]], dtype=torch.int32)
    k[ids[0].long().cuda()], v[ids[0].long().cuda()] = small_k.cuda(), small_v.cuda()
    q = torch.randn(1, 4, hd, generator=g).to(torch.bfloat16)
    out, lse = paged_decode_attention(q.cuda(), k, v, ids.cuda(), torch.tensor([250], dtype=torch.int32).cuda(), return_lse=True)
    check(out, lse, *attend(q, small_k, small_v, torch.tensor([[0, 1, 2, 3]]), [250], hd ** -0.5), torch.bfloat16)


def test_bad_tables_and_lengths_are_nan_and_stay_with_their_request():
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(6)
    lens = [40, 40, 40, 40, 2000, 40]
    k, v, kd, vd, table = cache_of(g, lens, 2, 64, 16, torch.bfloat16)
    q = torch.randn(6, 8, 64, generator=g).to(torch.bfloat16)
    want, lse, big = attend(q, k, v, table, lens, 0.125)
    n = torch.tensor(lens, dtype=torch.int32)
    table[1, 1], table[2, 0], table[4, 70] = -1, k.shape[0], 2 ** 31 - 1
    n[3], n[5] = table.shape[1] * 16 + 1, -4
    out, l = paged_decode_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), return_lse=True)
    assert out[[1, 2, 3, 4]].isnan().all() and l[[1, 2, 3, 4]].isnan().all()
    assert (out[5] == 0).all() and (l[5] == -INF).all()                   # a negative length is an empty request
    check(out[:1], l[:1], want[:1], lse[:1], big[:1], torch.bfloat16)
    none = paged_decode_attention(q.cuda(), kd, vd, table[:, :0].cuda(), n.cuda())
    assert none[:5].isnan().all() and (none[5] == 0).all()                # a length without any table


def test_infinite_scores_and_values():
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(7)
    lens = [100, 100, 100]
    k, v, _, _, table = cache_of(g, lens, 1, 64, 16, torch.bfloat16, junk=0.0)
    q = torch.ones(3, 2, 64).to(torch.bfloat16)
    page = lambda b, t: (int(table[b, t // 16]), 0, t % 16)               # noqa: E731
    for t in range(0, 60):
        k[page(0, t)][3] = -INF                                           # 60 tokens shut out, among them whole tiles
    k[page(1, 50)][3] = INF
    v[page(2, 99)][5] = INF
    out, lse = (t.cpu() for t in paged_decode_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                                        return_lse=True))
    want, wl, _ = attend(q, k, v, table, lens, 0.125)
    assert float((out[0] - want[0]).abs().max()) < 2e-2 and float((lse[0] - wl[0]).abs().max()) < 1e-4
    assert out[1].isnan().all()
    assert not out[2, :, 5].isfinite().any() and float((out[2, :, 6:] - want[2, :, 6:]).abs().max()) < 2e-2


def test_strided_queries_streams_out_and_refusals():
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(8)
    lens = [70, 300, 5]
    k, v, kd, vd, table = cache_of(g, lens, 2, 64, 16, torch.bfloat16)
    wide = torch.randn(3, 12, 64, generator=g).to(torch.bfloat16).cuda()
    tb, n = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    want = paged_decode_attention(wide[:, :8].contiguous(), kd, vd, tb, n)
    assert torch.equal(paged_decode_attention(wide[:, :8], kd, vd, tb, n), want)
    odd = torch.empty(3 * 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 8, 64).copy_(wide[:, :8])
    assert torch.equal(paged_decode_attention(odd, kd, vd, tb, n), want)
    assert torch.equal(paged_decode_attention(wide[:, :8].transpose(1, 2).contiguous().transpose(1, 2), kd, vd, tb, n), want)
    out = torch.empty_like(want)
    assert paged_decode_attention(wide[:, :8], kd, vd, tb, n, out=out) is out and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_decode_attention(wide[:, :8], kd, vd, tb, n)
    side.synchronize()
    assert torch.equal(got, want)
    assert paged_decode_attention(wide[:0, :8], kd, vd, tb[:0], n[:0]).shape == (0, 8, 64)
    q = wide[:, :8]
    for args, text in (((q.float(), kd, vd, tb, n), "dtype"), ((q, kd, vd[:, :1], tb, n), "one shape"), ((wide[:, :7], kd, vd, tb, n), "fit"),
                       ((q[..., :32], kd, vd, tb, n), "fit"), ((q, kd, vd, tb.long(), n), "block_tables"), ((q, kd, vd, tb, n.long()), "kv_lens"),
                       ((q, kd, vd, tb[:2], n), "table rows"), ((q, kd[:0], vd[:0], tb, n), "empty cache"),
                       ((q[..., :60], kd[..., :60], vd[..., :60], tb, n), "head_dim")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            paged_decode_attention(*args)
    with pytest.raises(ValueError, match="16-byte"):
        paged_decode_attention(q[..., :56], kd[..., 4:60], vd[..., 4:60], tb, n)
    with pytest.raises(ValueError, match="scale"):
        paged_decode_attention(q, kd, vd, tb, n, scale=INF)
    with pytest.raises(ValueError, match="out must"):
        paged_decode_attention(q, kd, vd, tb, n, out=out[:2])
    with pytest.raises(RuntimeError, match="inference only"):
        paged_decode_attention(q.clone().requires_grad_(), kd, vd, tb, n)


def test_shared_pages_and_two_streams_at_once():
    """Requests that hold the same pages (a common prompt), and two calls that overlap on two streams, many times over."""
    from hydra_b200.paged import paged_decode_attention
    g = torch.Generator().manual_seed(9)
    k, v, kd, vd, table = cache_of(g, [900], 2, 64, 16, torch.bfloat16)
    lens = [900, 896, 1, 450, 900]
    q = torch.randn(5, 8, 64, generator=g).to(torch.bfloat16)
    tb = table.expand(5, -1).contiguous()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = paged_decode_attention(q.cuda(), kd, vd, tb.cuda(), n, return_lse=True)
    check(out, lse, *attend(q, k, v, tb, lens, 0.125), torch.bfloat16)
    k2, v2, kd2, vd2, table2 = cache_of(g, [3000, 20, 777], 1, 128, 16, torch.float16)
    q2, n2 = torch.randn(3, 4, 128, generator=g).half().cuda(), torch.tensor([3000, 20, 777], dtype=torch.int32).cuda()
    want2 = paged_decode_attention(q2, kd2, vd2, table2.cuda(), n2)
    qd, td, td2 = q.cuda(), tb.cuda(), table2.cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(30):
        with torch.cuda.stream(streams[0]):
            a = paged_decode_attention(qd, kd, vd, td, n)
        with torch.cuda.stream(streams[1]):
            b = paged_decode_attention(q2, kd2, vd2, td2, n2)
        got.append((a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(a, out) and torch.equal(b, want2) for a, b in got)


# ------------------------------------------------------------------------------------------------------- whole steps
def product(a, b):
    """a @ b in an order that is the same eagerly and in a graph."""
    return (a[:, :, None] * b).sum(1)


class Server:
    """Two layers' worth of random projections over one plan per step; `step` is what a server captures into a graph."""

    def __init__(self, seed=0, B=5, rows=32, hq=8, hkv=2, hd=64, page=16, width=12, vocab=501, dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")        # noqa: E731
        self.hq, self.hkv, self.hd, self.page, self.rows, self.vocab = hq, hkv, hd, page, rows, vocab
        pages = B * width
        self.x = torch.zeros(rows, 96, device="cuda")
        self.w = [(0.1 * r(96, (hq + 2 * hkv) * hd)) for _ in range(2)]
        self.wo = [(0.05 * r(hq * hd, 96)) for _ in range(2)]
        self.head = 0.3 * r(96, vocab)
        self.norms = [(1 + 0.1 * r(hd), 1 + 0.1 * r(hd)) for _ in range(2)]
        self.kc = [torch.full((pages, hkv, page, hd), NAN, dtype=dtype, device="cuda") for _ in range(2)]
        self.vc = [torch.full((pages, hkv, page, hd), NAN, dtype=dtype, device="cuda") for _ in range(2)]
        i = torch.arange(width * page, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2) / hd)[None].double()
        self.cos, self.sin = i.cos().float().cuda(), i.sin().float().cuda()
        self.table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.start = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.context = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.tokens = torch.zeros(B, dtype=torch.int64, device="cuda")

    def step(self):
        """The decode half: one token for each request that has one (new = 1), through both layers to log probabilities."""
        from hydra_b200.paged import paged_append, paged_decode_attention, paged_plan
        from hydra_b200.sampling import token_logprobs
        B = self.context.shape[0]
        plan = paged_plan(self.context, self.new, self.table, self.free, self.page, self.rows, self.start)
        x, keep = self.x, []
        for l in range(2):
            qkv = product(x, self.w[l]).to(self.kc[l].dtype).view(self.rows, -1, self.hd)
            q = paged_append(qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.hkv], qkv[:, self.hq + self.hkv:], self.kc[l], self.vc[l], plan.slots,
                             self.cos, self.sin, plan.positions, q_weight=self.norms[l][0], k_weight=self.norms[l][1], layout="half")
            last = (plan.cu_new[1:].long() - 1).clamp(min=0)              # each request's newest row
            o = paged_decode_attention(q[last], self.kc[l], self.vc[l], self.table, plan.kv_lens)
            keep.append((qkv, q, o))
            x = x.clone()
            x.index_add_(0, last, product(o.float().view(B, -1), self.wo[l]) * (self.new > 0)[:, None])
        logits = product(x[last], self.head).to(torch.bfloat16)
        return plan, keep, logits, token_logprobs(logits, self.tokens, top=3)


def test_steps_of_a_server():
    """Prefill of two requests, then steps in which others join, pause and leave; every attention is checked against the keys
    and values that the projections gave, gathered by position on the host."""
    s = Server()
    B = 5
    past = [[([], []) for _ in range(B)] for _ in range(2)]               # per layer and request: keys, values (64 bits)
    g = torch.Generator(device="cuda").manual_seed(1)
    context = [0] * B
    for new in ([20, 0, 9, 0, 0], [1, 0, 1, 0, 0], [1, 14, 1, 0, 0], [0, 1, 1, 0, 3], [1, 1, 1, 0, 1], [16, 1, 0, 2, 1], [1, 1, 1, 1, 1]):
        s.new.copy_(torch.tensor(new, dtype=torch.int32))
        s.x.copy_(torch.randn(s.x.shape, generator=g, device="cuda"))
        s.tokens.copy_(torch.randint(0, s.vocab, (B,), generator=g, device="cuda"))
        plan, keep, logits, lp = s.step()
        assert int(plan.status) == 0
        context = [c + n for c, n in zip(context, new)]
        assert plan.kv_lens.tolist() == context
        cu = plan.cu_new.tolist()
        for l, (qkv, q, o) in enumerate(keep):
            rows, wq, wk = qkv.double().cpu(), *(w.double().cpu() for w in s.norms[l])
            half = s.hd // 2
            def turned(x, w, t):
                x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
                c, n = s.cos[t].double().cpu(), s.sin[t].double().cpu()
                return torch.cat([x[..., :half] * c - x[..., half:] * n, x[..., :half] * n + x[..., half:] * c], -1)
            for b in range(B):
                for i in range(new[b]):
                    t, row = context[b] - new[b] + i, rows[cu[b] + i]
                    past[l][b][0].append(turned(row[s.hq:s.hq + s.hkv], wk, t).to(torch.bfloat16))
                    past[l][b][1].append(row[s.hq + s.hkv:].to(torch.bfloat16))
                if new[b]:
                    qq = turned(rows[cu[b + 1] - 1, :s.hq], wq, context[b] - 1)
                    kk, vv = (torch.stack(p).double().repeat_interleave(s.hq // s.hkv, 1) for p in past[l][b])
                    w = torch.softmax(torch.einsum("hd,nhd->hn", qq, kk) * s.hd ** -0.5, 1)
                    want = torch.einsum("hn,nhd->hd", w, vv)
                    # the query is rounded to bf16 once (2^-9 of scores of at most 8 * sqrt(64) / 8): weights within 2^-6
                    assert float((o[b].double().cpu() - want).abs().max()) <= 2.0 ** -6 * float(vv.abs().max())
        ref = torch.log_softmax(logits.double(), -1).cpu()
        assert float((lp.logprobs.cpu() - ref.gather(1, s.tokens.cpu()[:, None])[:, 0]).abs().max()) <= 1e-4
        s.context.copy_(plan.kv_lens)
        s.start.copy_(plan.free_start)
    # request 2 leaves: its pages serve again
    held = -(-context[2] // s.page)
    free = torch.cat([s.free[int(s.start):], s.table[2, :held]])
    assert len(set(free.tolist())) == free.numel() and not set(free.tolist()) & set(s.table[0, :-(-context[0] // s.page)].tolist())


def test_a_captured_step_replays_with_new_lengths_beside_another_graph():
    """Two servers' steps captured into two graphs and replayed turn by turn, one of them also eagerly in between: the same bits
    as the eager steps, while lengths, tables and inputs change under the graphs."""
    a, b = (Server(seed=s) for s in (2, 2))
    other = Server(seed=3, hd=128, hq=4, hkv=1)
    g = torch.Generator(device="cuda").manual_seed(4)
    graphs = []
    for s in (a, other):
        s.new.fill_(1)
        with torch.cuda.stream(torch.cuda.Stream()):
            s.step()                                                      # set-up calls outside the capture
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, s.step()))
        graphs[-1] = (gr, graphs[-1][1])
    for turn, new in enumerate(([1, 1, 1, 1, 1], [1, 0, 1, 1, 0], [1, 1, 0, 0, 1], [5, 1, 1, 1, 1])):
        x = torch.randn(a.x.shape, generator=g, device="cuda")
        for s in (a, b, other):
            s.new.copy_(torch.tensor(new, dtype=torch.int32))
            s.x.copy_(x)
        graphs[0][0].replay()
        graphs[1][0].replay()
        want = b.step()
        got = graphs[0][1]
        for u, v in zip(got[0], want[0]):
            assert torch.equal(u, v)
        for (_, q1, o1), (_, q2, o2) in zip(got[1], want[1]):
            rows = int(want[0].cu_new[-1])
            assert torch.equal(q1[:rows], q2[:rows]) and torch.equal(o1, o2)
        assert all(torch.equal(u, v) for u, v in zip(got[3], want[3]))
        for s, p in ((a, got[0]), (b, want[0]), (other, graphs[1][1][0])):
            s.context.copy_(p.kv_lens)
            s.start.copy_(p.free_start)


def test_outputs_that_overlap_queries_or_record_gradients_are_refused():
    from hydra_b200.paged import paged_append, paged_decode_attention
    g = torch.Generator().manual_seed(21)
    lens = [40, 3]
    k, v, kd, vd, table = cache_of(g, lens, 2, 64, 16, torch.bfloat16)
    q = torch.randn(2, 8, 64, generator=g).to(torch.bfloat16).cuda()
    tb, n = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    room = torch.cat([q, q, q])            # q lies at the end, an output at the beginning touches it or just does not
    want = paged_decode_attention(q, kd, vd, tb, n)
    for q_at, out_at in ((2, 2), (2, 3), (3, 2)):
        with pytest.raises(ValueError, match="overlap"):
            paged_decode_attention(room[q_at:q_at + 2], kd, vd, tb, n, out=room[out_at:out_at + 2])
    assert torch.equal(room, torch.cat([q, q, q]))
    assert torch.equal(paged_decode_attention(room[2:4], kd, vd, tb, n, out=room[:2]), want) and torch.equal(room[2:], torch.cat([q, q]))
    assert torch.equal(paged_decode_attention(room[2:4], kd, vd, tb, n, out=room[4:]), want) and torch.equal(room[2:4], q)
    with pytest.raises(RuntimeError, match="inference only"):
        paged_decode_attention(q, kd, vd, tb, n, out=torch.empty_like(q).requires_grad_())
    cos = torch.ones(8, 32, device="cuda", requires_grad=True)
    where = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="inference only"):
        paged_append(q, q[:, :2], q[:, 2:4], kd, vd, where.long(), cos, cos, where)
