"""The latent cache: append (bit for bit against the symmetric format's rule) and absorbed
attention against 64 bits, over dims, heads, tokens, lengths, page sizes, holes, strides,
streams and captured graphs.

Tolerance of the attention, derived from the kernel's roundings.  With p the softmax and
A = sum_j p_j |scale_j c_j| of an output element: P rounds once to fp16 (half a step, 2^-11
of each p), a score is off by delta <= sm_scale * (max|q| / 32639 / 2) * max_j |c_j|_1 from
the 16-bit fixed point of q (each side of the quotient, so 2 delta of p) plus fp32 sums
(2^-24 * (dc + dr) of sum |q c| sm_scale, less than 2^-12 here for normal data), and the
output rounds once: |err| <= (2^-11 + 2 delta + 2^-12) A + half |out| + 2^-24."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def fs():
    import flashspec_b200

    return flashspec_b200


def make_cache(lens, dc, dr, page, dtype, seed, slack=2, extra_cols=0):
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    total = max(1, sum(need) + slack)
    perm = torch.randperm(total, generator=g)
    cols = max(1, max(need)) + extra_cols
    table = torch.full((len(lens), cols), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    values = torch.randint(-127, 128, (total, page, dc), generator=g).to(torch.int8)
    # scales over several orders, so that a token's weight and its size differ
    scale = torch.exp(torch.randn((total, page), generator=g) * 1.5 - 4).float()
    ropes = torch.randn((total, page, dr), generator=g).to(dtype)
    return fs().LatentKVCache(values.cuda(), scale.cuda(), ropes.cuda(), table.cuda(), torch.tensor(lens).cuda(),
                              max(max(lens), 1))


def queries(b, t, h, dc, dr, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((b, t, h, dc), generator=g).to(dtype).cuda(),
            torch.randn((b, t, h, dr), generator=g).to(dtype).cuda())


def expect(q, qr, cache, sm_scale):
    """(out, bound) in 64 bits."""
    b, t, h, dc = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    page = cache.block_size
    half = torch.finfo(q.dtype).eps / 2
    table, lens = cache.block_table.cpu(), cache.lengths.cpu().tolist()
    for i in range(b):
        n = min(lens[i], cache.max_seq_len, table.shape[1] * page)
        if n <= 0:
            continue
        pages = table[i, : (n + page - 1) // page]
        here = ((pages >= 0) & (pages < cache.values.shape[0])).repeat_interleave(page)[:n].cuda()
        at = torch.where((pages >= 0) & (pages < cache.values.shape[0]), pages, 0).cuda()
        c = (cache.values[at].double() * cache.scale[at].double()[..., None]).flatten(0, 1)[:n]
        r = cache.ropes[at].double().flatten(0, 1)[:n]
        for k in range(t):
            seen = here & (torch.arange(n, device="cuda") <= n - t + k)
            if not bool(seen.any()):
                continue
            cs, rs = c[seen], r[seen]
            qk, qrk = q[i, k].double(), qr[i, k].double()
            p = torch.softmax((qk @ cs.T + qrk @ rs.T) * sm_scale, -1)
            out[i, k] = p @ cs
            delta = sm_scale * qk.abs().amax(1) / 32639 / 2 * cs.abs().sum(1).max()
            bound[i, k] = (2 ** -11 + 2 * delta[:, None] + 2 ** -12) * (p @ cs.abs())
    return out, bound + half * out.abs() + 2 ** -24


def check(q, qr, cache, sm_scale=None, **kw):
    sm = (cache.latent_dim + cache.rope_dim) ** -0.5 if sm_scale is None else sm_scale
    want, bound = expect(q, qr, cache, sm)
    out = fs().latent_attention_cuda(q, qr, cache, sm_scale=sm_scale, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return out


F, B = torch.float16, torch.bfloat16
CASES = [
    # lens, T, H, dc, dr, page, dtype
    ([1], 1, 1, 512, 64, 64, F),
    ([777], 1, 16, 512, 64, 64, F),
    ([0, 1, 63, 64, 65, 300], 1, 16, 512, 64, 16, B),
    ([500, 129], 1, 32, 512, 64, 32, F),
    ([500, 129], 1, 17, 512, 32, 64, B),
    ([260, 1000], 1, 64, 512, 64, 64, B),
    ([260, 0, 90], 2, 64, 512, 64, 128, F),
    ([333, 10], 1, 128, 512, 64, 64, F),
    ([2, 40], 3, 5, 512, 64, 64, F),  # the first queries of the short request see nothing
    ([700, 64], 1, 16, 256, 32, 16, F),
    ([700, 64], 1, 30, 256, 64, 64, B),
    ([700, 64], 2, 40, 256, 32, 64, F),
    ([700, 64], 1, 9, 128, 64, 16, B),
    ([700, 64], 1, 32, 128, 32, 64, F),
    ([700, 64], 1, 100, 128, 64, 64, F),
]


@pytest.mark.parametrize("lens,t,h,dc,dr,page,dtype", CASES)
def test_absorbed_attention(lens, t, h, dc, dr, page, dtype):
    cache = make_cache(lens, dc, dr, page, dtype, seed=dc + h)
    q, qr = queries(len(lens), t, h, dc, dr, dtype, seed=h)
    check(q, qr, cache)


def test_many_requests_and_long_ones():
    lens = [50 * i for i in range(90)] + [30000]
    cache = make_cache(lens, 512, 64, 64, F, seed=3)
    q, qr = queries(len(lens), 1, 16, 512, 64, F, seed=4)
    check(q, qr, cache, sm_scale=0.07)


def test_one_long_request_over_all_shares():
    for h in (16, 128):
        cache = make_cache([40000], 512, 64, 64, B, seed=5)
        q, qr = queries(1, 1, h, 512, 64, B, seed=6)
        check(q, qr, cache)


def test_peaked_scores_and_small_scales():
    """One token far ahead of the rest, scales down to the format's floor."""
    cache = make_cache([400], 512, 64, 64, F, seed=7)
    cache.scale.mul_(1e-3)
    cache.scale[cache.block_table[0, 2], 5] = 1e-8
    q, qr = queries(1, 1, 16, 512, 64, F, seed=8)
    cache.ropes[cache.block_table[0, 2], 5] = qr[0, 0, 3] * 4
    check(q, qr, cache)


def test_holes_and_pages_outside_the_pool():
    cache = make_cache([300, 200], 512, 64, 16, F, seed=9)
    q, qr = queries(2, 1, 16, 512, 64, F, seed=10)
    outs = []
    for bad in (-1, 10 ** 13):
        table = cache.block_table.clone()
        table[0, 4] = bad
        table[1] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        c = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, table, cache.lengths, 300)
        outs.append(check(q, qr, c, device_status=status))
        assert int(status) == (0 if bad < 0 else 1)
    assert torch.equal(*outs)
    assert float(outs[0][1].abs().sum()) == 0.0  # no page at all: zeros


def test_nothing_behind_the_length_is_read():
    """Rows behind a request's length and unlisted pages may hold anything."""
    cache = make_cache([100, 37], 512, 64, 64, B, seed=11)
    q, qr = queries(2, 1, 16, 512, 64, B, seed=12)
    ref = fs().latent_attention_cuda(q, qr, cache)
    for i, n in enumerate((100, 37)):
        page = cache.block_table[i, n // 64]
        cache.ropes[page, n % 64:] = float("nan")
        cache.scale[page, n % 64:] = float("inf")
    assert torch.equal(fs().latent_attention_cuda(q, qr, cache), ref)


def test_nan_in_a_query_stays_in_its_row():
    cache = make_cache([100], 512, 64, 64, F, seed=13)
    q, qr = queries(1, 1, 16, 512, 64, F, seed=14)
    ref = fs().latent_attention_cuda(q, qr, cache)
    q[0, 0, 2, 7], qr[0, 0, 5, 1] = float("nan"), float("nan")
    out = fs().latent_attention_cuda(q, qr, cache)
    assert bool(out[0, 0, 2].isnan().all()) and bool(out[0, 0, 5].isnan().all())
    keep = [i for i in range(16) if i not in (2, 5)]
    assert torch.equal(out[0, 0, keep], ref[0, 0, keep])


def test_single_token_form_strides_stream_and_repeat():
    cache = make_cache([900, 5, 64], 512, 64, 64, F, seed=15)
    packed = torch.randn((3, 16, 576), generator=torch.Generator().manual_seed(1)).half().cuda()
    q, qr = packed[..., :512], packed[..., 512:]  # views of one projection
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        a = fs().latent_attention_cuda(q, qr, cache)
        b = fs().latent_attention_cuda(q.unsqueeze(1).contiguous(), qr.unsqueeze(1).contiguous(), cache)[:, 0]
        torch.cuda.synchronize()
    assert a.shape == (3, 16, 512) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("dc,dr,page", [(512, 64, 64), (256, 32, 16), (128, 64, 128)])
def test_append(dtype, dc, dr, page):
    g = torch.Generator().manual_seed(dc)
    cache = fs().LatentKVCache.empty(3, 200, dc, dr, page, dtype=dtype)
    cache.scale.fill_(9.0)
    held_len = torch.tensor([0, 17, 100])
    cache = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, cache.block_table, held_len.cuda(), 100)
    values, scale, ropes = cache.values.clone(), cache.scale.clone(), cache.ropes.clone()
    t = 50
    wide = torch.randn((3, t, dc + dr), generator=g).to(dtype).cuda()  # latent and rope of one projection
    wide[1, 3, :dc] = 0  # a zero vector takes the scale's floor
    counts = torch.tensor([50, 0, 31])
    out, held = cache.append(wide[..., :dc], wide[..., dc:], counts.cuda(), return_held=True)
    want_held = torch.zeros((3, t, dc), dtype=dtype, device="cuda")
    for b in range(3):
        for k in range(int(counts[b])):
            pos = int(held_len[b]) + k
            at = cache.block_table[b, pos // page], pos % page
            x = wide[b, k, :dc].float().cpu().numpy()
            sc = np.maximum(np.abs(x).max() / np.float32(127), np.float32(1e-8)).astype(np.float32)
            code = np.clip(np.rint(x / sc), -127, 127).astype(np.float32)
            values[at] = torch.from_numpy(code.astype(np.int8)).cuda()
            scale[at] = float(sc)
            ropes[at] = wide[b, k, dc:]
            want_held[b, k] = torch.from_numpy(code * sc).to(dtype).cuda()
    assert torch.equal(out.values, values) and torch.equal(out.scale, scale) and torch.equal(out.ropes, ropes)
    assert torch.equal(held, want_held)
    assert out.lengths.tolist() == [50, 17, 131] and cache.lengths.tolist() == [0, 17, 100]
    assert out.max_seq_len == 150 and out.values.data_ptr() == cache.values.data_ptr()


def test_append_codes_equal_the_symmetric_quantizer():
    x = torch.randn((1, 64, 512), generator=torch.Generator().manual_seed(5)).half().cuda() * 3
    cache = fs().LatentKVCache.empty(1, 64, dtype=F).append(x, x[..., :64].contiguous())
    sym = fs().quantize_int8_symmetric_per_token(x, 64)
    assert torch.equal(cache.values, sym.values) and torch.equal(cache.scale, sym.scale)


def test_append_drops_tokens_without_a_page():
    for bad in (-1, 99):
        cache = fs().LatentKVCache.empty(1, 128, dtype=B)
        table = cache.block_table.clone()
        table[0, 1] = bad
        c = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, table, cache.lengths, 0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        x = torch.ones((1, 200, 512), dtype=B, device="cuda")
        out, held = c.append(x, x[..., :64], return_held=True, device_status=status)
        assert int(status) == 1 and out.lengths.tolist() == [200] and out.max_seq_len == 128
        assert bool((out.values[0] != 0).all()) and not bool(out.values[1].any())
        assert bool((held == held[0, 0]).all())


def test_steps_of_append_and_attention_in_a_captured_graph():
    """A decode step recorded once: append one token, attend; replays see new inputs and keep
    counting through a length that is copied back.  Two graphs replay beside each other."""
    b, h = 3, 16
    g = torch.Generator().manual_seed(21)
    rand = lambda *s: torch.randn(s, generator=g).half().cuda()  # noqa: E731

    def build():
        cache = fs().LatentKVCache.empty(b, 256, dtype=F)
        cache = cache.append(rand(b, 90, 512), rand(b, 90, 64), torch.tensor([90, 3, 64]).cuda())
        cache = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, cache.block_table, cache.lengths, 256)
        return cache, rand(b, 1, 512), rand(b, 1, 64), rand(b, 1, h, 512), rand(b, 1, h, 64)

    def step(cache, c, r, q, qr):
        new = cache.append(c, r)
        out = fs().latent_attention_cuda(q, qr, new)
        cache.lengths.copy_(new.lengths)
        return out

    g.manual_seed(21)
    eager = build()
    twins = []
    for _ in range(2):
        g.manual_seed(21)
        st = build()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*st)
        twins.append((graph, st, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        fresh = [rand(*x.shape) for x in eager[1:]]
        for st in [eager] + [x[1] for x in twins]:
            for x, y in zip(st[1:], fresh):
                x.copy_(y)
        torch.cuda.synchronize()
        for (graph, _, _), s in zip(twins, streams):
            with torch.cuda.stream(s):
                graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        for _, st, out in twins:
            assert torch.equal(out, want) and torch.equal(st[0].values, eager[0].values)
    assert eager[0].lengths.tolist() == [94, 7, 68]
    check(eager[3], eager[4], eager[0])


def test_refusals():
    f = fs()
    cache = make_cache([64], 512, 64, 64, F, seed=30)
    q, qr = queries(1, 1, 4, 512, 64, F, seed=31)
    for bad in ((q[..., :256], qr), (q, qr[..., :32]), (q.bfloat16(), qr), (q, qr.bfloat16()), (q[:, 0], qr),
                (q.expand(2, 1, 4, 512), qr.expand(2, 1, 4, 64)), (q[:, :0], qr[:, :0])):
        with pytest.raises(ValueError):
            f.latent_attention_cuda(*bad, cache)
    with pytest.raises(RuntimeError):
        f.latent_attention_cuda(q.cpu(), qr.cpu(), cache)
    c = cache
    for broken in (f.LatentKVCache(c.values[..., :64], c.scale, c.ropes, c.block_table, c.lengths, 64),
                   f.LatentKVCache(c.values, c.scale.half(), c.ropes, c.block_table, c.lengths, 64),
                   f.LatentKVCache(c.values, c.scale, c.ropes[..., :16], c.block_table, c.lengths, 64),
                   f.LatentKVCache(c.values[:, :48], c.scale[:, :48], c.ropes[:, :48], c.block_table, c.lengths, 64),
                   f.LatentKVCache(c.values, c.scale, c.ropes, c.block_table, c.lengths[None], 64)):
        with pytest.raises(ValueError):
            f.latent_attention_cuda(q, qr, broken)
    x, r = q[:, :, 0], qr[:, :, 0]
    for bad in ((x[..., :500], r, None), (x, r[..., :10], None), (x.float(), r, None), (x[:, :0], r[:, :0], None),
                (x, r, torch.ones(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            cache.append(*bad)
    with pytest.raises(RuntimeError):
        cache.append(x, r, torch.ones(1, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        f.LatentKVCache.empty(1, 10, device="cpu")
    with pytest.raises(ValueError):
        f.LatentKVCache.empty(1, 10, latent_dim=100)
    with pytest.raises(ValueError):
        f.LatentKVCache.empty(0, 10)


def test_append_behind_the_largest_length_finds_no_page():
    cache = fs().LatentKVCache.empty(2, 128, dtype=B)
    lens = torch.tensor([2 ** 63 - 3, 2]).cuda()
    c = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, cache.block_table, lens, 128)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones((2, 9, 512), dtype=B, device="cuda")
    c.append(x, x[..., :64], device_status=status)
    assert int(status) == 1 and not bool(c.values[:2].any()) and bool((c.values[2, 2:11] == 127).all())
    assert int((c.values != 0).sum()) == 9 * 512


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("h,page,n", [(4, 64, 130), (16, 16, 64), (40, 64, 129)])
def test_a_bad_token_does_not_reach_queries_before_it(bad, h, page, n):
    """The last drafted tokens have an infinite or undefined scale: the queries that do not see
    them give what they gave before, the others NaN."""
    t = 3
    cache = make_cache([n, 200], 512, 64, page, F, seed=40 + h)
    q, qr = queries(2, t, h, 512, 64, F, seed=41)
    ref = fs().latent_attention_cuda(q, qr, cache)
    cache.scale[cache.block_table[0, (n - 1) // page], (n - 1) % page] = bad
    cache.scale[cache.block_table[0, (n - 2) // page], (n - 2) % page] = bad
    out = fs().latent_attention_cuda(q, qr, cache)
    assert torch.equal(out[0, 0], ref[0, 0]) and torch.equal(out[1], ref[1])
    assert bool(out[0, 1:].isnan().all())


def test_an_infinite_latent_of_a_draft_stays_behind_the_mask():
    g = torch.Generator().manual_seed(50)
    rand = lambda *s: torch.randn(s, generator=g).to(B).cuda()  # noqa: E731
    cache = fs().LatentKVCache.empty(1, 256, dtype=B).append(rand(1, 100, 512), rand(1, 100, 64))
    c, r, q, qr = rand(1, 2, 512), rand(1, 2, 64), rand(1, 2, 16, 512), rand(1, 2, 16, 64)
    ref = fs().latent_attention_cuda(q, qr, cache.append(c, r))
    c[0, 1, 77] = float("inf")
    out = fs().latent_attention_cuda(q, qr, cache.append(c, r))
    assert torch.equal(out[0, 0], ref[0, 0]) and bool(out[0, 1].isnan().all())


@pytest.mark.parametrize("h,near", [(16, 0), (16, 700), (64, 0)])
def test_many_far_tokens_beside_a_near_one(h, near):
    """One token takes nearly all of the weight and is zero in every dim but the first; the
    other dims are what 1000 tokens at e^-17 (2^-24.5) of it add up to.  Requests enough that a
    share holds the near token together with most of the others."""
    b, n = 320, 1000
    cache = make_cache([n] * b, 512, 64, 64, F, seed=60)
    g = torch.Generator(device="cuda").manual_seed(61)
    cache.values.copy_(torch.randint(40, 128, cache.values.shape, generator=g, device="cuda"))
    cache.values[..., 0] = 0
    cache.scale.fill_(1)
    cache.ropes.zero_()
    cache.ropes[..., 0] = -1
    page, row = cache.block_table[:, near // 64], near % 64
    cache.values[page, row] = 0
    cache.values[page, row, 0] = 127
    cache.ropes[page, row, 0] = 16
    q, qr = queries(b, 1, h, 512, 64, F, seed=62)
    q.zero_(), qr.zero_()
    qr[..., 0] = 1
    out = check(q, qr, cache, sm_scale=1.0)
    assert float(out[..., 1:].min()) > 2e-3


@pytest.mark.parametrize("longest", [2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 62])
def test_no_limit_on_the_length(longest):
    cache = make_cache([300, 77], 512, 64, 64, F, seed=70, extra_cols=1)
    q, qr = queries(2, 1, 16, 512, 64, F, seed=71)
    free = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, cache.block_table, cache.lengths, longest)
    assert torch.equal(check(q, qr, cache), fs().latent_attention_cuda(q, qr, free))
    assert free.append(q[:, :, 0], qr[:, :, 0]).max_seq_len == 6 * 64


def test_queries_of_a_request_that_has_outgrown_its_table():
    """append keeps counting where the table ends; a query's own position still is the one that
    its request's length gives it: of three at 62, 63 and 64, the first sees 63 tokens, the others
    all 64."""
    cache = make_cache([64, 64], 512, 64, 64, F, seed=80)
    q, qr = queries(2, 3, 16, 512, 64, F, seed=81)
    for whole, seen in ((64, (62, 63, 64)), (65, (63, 64, 64)), (66, (64, 64, 64)), (1000, (64, 64, 64))):
        c = fs().LatentKVCache(cache.values, cache.scale, cache.ropes, cache.block_table,
                               torch.tensor([whole, 64]).cuda(), 64)
        out = fs().latent_attention_cuda(q, qr, c)
        for k, n in enumerate(seen):
            one = fs().LatentKVCache(c.values, c.scale, c.ropes, c.block_table, torch.tensor([n, 62 + k]).cuda(), 64)
            want = fs().latent_attention_cuda(q[:, k: k + 1].contiguous(), qr[:, k: k + 1].contiguous(), one)
            assert torch.allclose(out[:, k: k + 1].float(), want.float(), rtol=2 ** -10, atol=2 ** -10)


def test_a_status_on_the_host_is_refused():
    """By every operator that reports bad pages; refused before any launch."""
    f, host = fs(), torch.zeros(1, dtype=torch.int32)
    cache = make_cache([64], 512, 64, 64, F, seed=90)
    q, qr = queries(1, 1, 4, 512, 64, F, seed=91)
    x = torch.zeros((2, 1, 96), dtype=F, device="cuda")
    o = torch.tensor([0, 2]).cuda()
    kq = f.quantize_int8_per_block(torch.zeros((4, 1, 16, 128), device="cuda"), 16)
    kv = f.PagedKVCache(kq, f.quantize_int8_per_block(torch.zeros((4, 1, 16, 128), device="cuda"), 16),
                        torch.zeros((1, 1), dtype=torch.int64, device="cuda"), torch.ones(1).long().cuda(), 16, 16)
    w, q1 = torch.zeros((4, 1, 16), device="cuda"), torch.zeros((1, 1, 128), dtype=F, device="cuda")
    for call in (lambda s: f.latent_attention_cuda(q, qr, cache, device_status=s),
                 lambda s: cache.append(q[:, :, 0], qr[:, :, 0], device_status=s),
                 lambda s: f.latent_prefill_attention_cuda(x, torch.zeros((2, 1, 128), dtype=F, device="cuda"),
                                                           x[:, 0, :32], o, o, device_status=s),
                 lambda s: f.evict_tokens_cuda(kv, w, 4, recent=1, device_status=s),
                 lambda s: f.paged_quant_attention_weights_cuda(q1, kv, w, device_status=s),
                 lambda s: f.paged_quant_attention_cuda(q1, kv, device_status=s)):
        with pytest.raises(RuntimeError):
            call(host)
        with pytest.raises(ValueError):
            call(torch.zeros(4, dtype=torch.uint8, device="cuda"))
        call(torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("large,share", [(100.0, 2e-3), (1000.0, 2e-2)])
def test_one_large_dim_in_q(large, share):
    """What the 16-bit fixed point of a row's queries costs when one dim is far above the others
    and its latents as far below: within the bound of every case, and within the stated share of
    the largest output."""
    cache = make_cache([500, 90], 512, 64, 64, F, seed=100)
    cache.scale.fill_(1 / 73)  # latents of size 1
    cache.values[..., 5] = (cache.values[..., 5].float() / large).round().to(torch.int8)
    q, qr = queries(2, 1, 16, 512, 64, F, seed=101)
    q[..., 5] *= large
    want, _ = expect(q, qr, cache, 576 ** -0.5)
    out = check(q, qr, cache)
    assert float((out.double() - want).abs().max() / want.abs().max()) < share
