"""Decode attention with accumulated weights against a 64-bit restatement: the output and
the weight every cached token receives, over formats, head groups, head dims, page sizes,
kernels (split, balanced, generic), empty and short requests, unallocated pages, shared
pages, other streams and captured graphs.

Tolerances.  A weight is 2^(x - LSE): x = q.k scaled is an fp32 sum of exact products
(24-bit fixed-point q in the tuned kernels, q itself in the generic one), so its error is at
most (D + 4) roundings of terms bounded by sum|q k| sm_scale log2e, and the exp2 turns it
into the same relative error; ex2.approx and the LSE add about 2^-21.  With normal data
sum|q k| sm_scale log2e <= 1.44 * D * 0.64 / sqrt(D) < 15 for D = 256, which gives
260 * 15 * 2^-24 * ln2 < 2e-4 as a worst case and its square root's order (2e-5) as what
happens; the tests allow 4e-5 of a weight, plus the same share of the largest."""

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


def make_cache(b, hkv, d, lens, page, fmt, seed, slack=3):
    """A cache of random codes on shuffled pages, with spare pages in the pool."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + slack
    perm = torch.randperm(total, generator=g)
    cols = max(1, max(need))
    table = torch.full((b, cols), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n

    def pool():
        x = torch.randn((total, hkv, page, d), generator=g).cuda()
        if fmt == "symmetric":
            return fs().quantize_int8_symmetric_per_token(x, page)
        return fs().quantize_int8_per_block(x, page)

    return fs().PagedKVCache(pool(), pool(), table.cuda(), torch.tensor(lens).cuda(), page, max(max(lens), 1))


def dense64(cache, i, n):
    """K and V of request i's first n tokens in 64 bits, [Hkv, n, D]; unallocated pages as None rows."""
    out = []
    pages = cache.block_table[i].cpu().tolist()
    for qt in (cache.k_quant, cache.v_quant):
        v = qt.values.double()
        if getattr(qt, "symmetric", False):
            x = v * qt.scale.double()[..., None]
        else:
            x = ((v + 128 - qt.zero_point.double()) * qt.scale.double()).flatten(2, 3)
        rows = [x[p] if p >= 0 else torch.full_like(x[0], float("nan")) for p in pages]
        out.append(torch.cat(rows, 1)[:, :n].cpu())
    return out


def expect(q, cache, weights):
    """(out, weights) in 64 bits."""
    b, hq, d = q.shape
    hkv, page = weights.shape[1:]
    w = weights.double().cpu().clone()
    out = torch.zeros((b, hq, d), dtype=torch.float64)
    table, lens = cache.block_table.cpu(), cache.lengths.cpu().tolist()
    for i in range(b):
        n = min(lens[i], cache.max_seq_len, table.shape[1] * page)
        if n == 0:
            continue
        k, v = dense64(cache, i, n)
        live = ~torch.isnan(k[0, :, 0])
        s = torch.einsum("hgd,hnd->hgn", q[i].double().cpu().view(hkv, -1, d), torch.nan_to_num(k)) / d ** 0.5
        s[..., ~live] = -float("inf")
        p = torch.nan_to_num(torch.softmax(s, -1))
        out[i] = torch.einsum("hgn,hnd->hgd", p, torch.nan_to_num(v)).reshape(hq, d)
        got = p.sum(1)
        for t in range(n):
            pg = int(table[i, t // page])
            if pg >= 0:
                w[pg, :, t % page] += got[:, t]
    return out, w


def check(q, cache, weights, **kw):
    before = weights.clone()
    ref_out, ref_w = expect(q, cache, weights)
    out = fs().paged_quant_attention_weights_cuda(q, cache, weights, **kw)
    torch.cuda.synchronize()
    err = (out.double().cpu() - ref_out).abs()
    half = torch.finfo(q.dtype).eps / 2
    # P and out each round once to 16 bits (half: fp16 P in the tuned kernels), |out| <= max|V| ~ 5
    assert bool((err <= 5 * half + 3 * half * ref_out.abs() + 1e-5).all()), err.max()
    werr = (weights.double().cpu() - ref_w).abs()
    assert bool((werr <= 4e-5 * (ref_w + ref_w.max())).all()), werr.max()
    untouched = ref_w == before.double().cpu()
    assert torch.equal(weights.cpu()[untouched], before.cpu()[untouched])
    return out


CASES = [
    # b, hq, hkv, d, page, lens, fmt, dtype
    (1, 1, 1, 128, 16, [1], "affine", torch.float16),
    (3, 8, 2, 128, 16, [0, 129, 16], "affine", torch.float16),
    (3, 8, 8, 128, 16, [5, 31, 400], "symmetric", torch.float16),
    (2, 24, 8, 128, 16, [1000, 1], "affine", torch.float16),
    (2, 16, 2, 128, 16, [3000, 2999], "symmetric", torch.float16),
    (2, 8, 2, 64, 16, [200, 37], "affine", torch.bfloat16),
    (2, 6, 2, 32, 16, [65, 0], "symmetric", torch.float16),
    (2, 4, 4, 256, 32, [100, 33], "affine", torch.bfloat16),
    (1, 5, 1, 64, 6, [77], "affine", torch.float16),
    (2, 4, 2, 128, 16, [2500, 90], "affine", torch.bfloat16),
]


@pytest.mark.parametrize("b,hq,hkv,d,page,lens,fmt,dtype", CASES)
def test_weights_and_output(b, hq, hkv, d, page, lens, fmt, dtype):
    cache = make_cache(b, hkv, d, lens, page, fmt, seed=b * 100 + d + page)
    q = torch.randn((b, hq, d), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    w = torch.rand((cache.k_quant.values.shape[0], hkv, page), generator=torch.Generator().manual_seed(2)).cuda()
    check(q, cache, w)
    check(q * 2, cache, w)  # a second step adds to the first


@pytest.mark.parametrize("kernel", ["split", "balanced"])
@pytest.mark.parametrize("splits", [None, 1, 5])
def test_both_tuned_kernels(monkeypatch, kernel, splits):
    if splits is None:
        monkeypatch.setenv("FLASHSPEC_DECODE_KERNEL", kernel)
    elif kernel == "balanced":
        pytest.skip("an explicit split count runs the split kernel")
    cache = make_cache(5, 4, 128, [700, 0, 333, 64, 1], 16, "affine", seed=9)
    q = torch.randn((5, 12, 128), generator=torch.Generator().manual_seed(3)).half().cuda()
    w = torch.zeros((cache.k_quant.values.shape[0], 4, 16), device="cuda")
    check(q, cache, w, num_splits=splits)


def test_many_pairs_run_the_balanced_kernel():
    lens = [100 + 13 * i for i in range(40)]
    cache = make_cache(40, 16, 128, lens, 16, "affine", seed=11)
    q = torch.randn((40, 16, 128), generator=torch.Generator().manual_seed(4)).half().cuda()
    check(q, cache, torch.zeros((cache.k_quant.values.shape[0], 16, 16), device="cuda"))


def test_weights_of_a_row_sum_to_one_per_query():
    cache = make_cache(2, 2, 128, [5000, 100], 16, "affine", seed=12)
    q = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(5)).half().cuda()
    w = torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda")
    fs().paged_quant_attention_weights_cuda(q, cache, w)
    for i in range(2):
        pages = cache.block_table[i]
        got = w[pages[pages >= 0]].double().sum((0, 2)).cpu()
        # n weights, each within 4e-5 of itself
        assert torch.allclose(got, torch.full((2,), 4.0, dtype=torch.float64), rtol=4e-5)


def test_unallocated_pages_and_capped_lengths():
    cache = make_cache(2, 2, 128, [200, 180], 16, "affine", seed=13)
    table = cache.block_table.clone()
    table[0, 3] = -1  # a hole inside the length
    q = torch.randn((2, 4, 128), generator=torch.Generator().manual_seed(6)).half().cuda()
    w = torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda")
    for lens, cap in ([200, 180], 200), ([10000, 180], 170):
        c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, torch.tensor(lens).cuda(), 16, cap)
        check(q, c, w)


def test_page_outside_the_pool_is_skipped_and_reported():
    cache = make_cache(1, 2, 128, [100], 16, "affine", seed=14)
    q = torch.randn((1, 4, 128), generator=torch.Generator().manual_seed(7)).half().cuda()
    hole, bad = cache.block_table.clone(), cache.block_table.clone()
    hole[0, 2], bad[0, 2] = -1, cache.k_quant.values.shape[0]
    outs = []
    for table in hole, bad:
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        w = torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda")
        c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, cache.lengths, 16, 100)
        o = fs().paged_quant_attention_weights_cuda(q, c, w, device_status=status)
        outs.append((o, w, int(status)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert outs[0][2] == 0 and outs[1][2] == 1


def test_shared_pages_add_up():
    cache = make_cache(1, 2, 128, [64], 16, "affine", seed=15)
    table = cache.block_table.repeat(3, 1)
    c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, torch.tensor([64, 64, 20]).cuda(), 16, 64)
    q = torch.randn((3, 4, 128), generator=torch.Generator().manual_seed(8)).half().cuda()
    check(q, c, torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda"))


def test_runs_repeat_bit_for_bit_and_match_the_plain_decode():
    cache = make_cache(3, 8, 128, [4000, 900, 17], 16, "affine", seed=16)
    q = torch.randn((3, 32, 128), generator=torch.Generator().manual_seed(9)).half().cuda()
    got = []
    for _ in range(2):
        w = torch.zeros((cache.k_quant.values.shape[0], 8, 16), device="cuda")
        got.append((fs().paged_quant_attention_weights_cuda(q, cache, w, num_splits=3), w))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    plain = fs().paged_quant_attention_cuda(q, cache, num_splits=3)
    # the plain decode's q has 16 bits: a score is off by at most 128 * 2^-16 * max|q k| sm_scale
    assert torch.allclose(plain.float(), got[0][0].float(), rtol=2e-3, atol=2e-3)


def test_other_stream_and_unaligned_weights():
    cache = make_cache(2, 2, 128, [300, 45], 16, "affine", seed=17)
    q = torch.randn((2, 4, 128), generator=torch.Generator().manual_seed(10)).half().cuda()
    pages = cache.k_quant.values.shape[0]
    w = torch.zeros(pages * 32 + 1, device="cuda")[1:].view(pages, 2, 16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check(q, cache, w)


def test_captured_graphs_share_nothing():
    cache = make_cache(4, 8, 128, [2000, 1500, 0, 77], 16, "affine", seed=18)
    pages = cache.k_quant.values.shape[0]
    q = torch.randn((4, 16, 128), generator=torch.Generator().manual_seed(11)).half().cuda()
    ref_w = torch.zeros((pages, 8, 16), device="cuda")
    ref = fs().paged_quant_attention_weights_cuda(q, cache, ref_w)
    graphs = []
    for _ in range(2):
        w = torch.zeros((pages, 8, 16), device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fs().paged_quant_attention_weights_cuda(q, cache, w)
        graphs.append((g, out, w))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for (g, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        # an eager call of another size beside the replays
        fs().paged_quant_attention_weights_cuda(q[:2], fs().PagedKVCache(
            cache.k_quant, cache.v_quant, cache.block_table[:2], cache.lengths[:2], 16, 2000),
            torch.zeros((pages, 8, 16), device="cuda"))
        torch.cuda.synchronize()
    for _, out, w in graphs:
        assert torch.equal(out, ref)
        assert torch.allclose(w, 3 * ref_w, rtol=1e-6)


@pytest.mark.parametrize("d,dtype", [(128, torch.float16), (64, torch.bfloat16)])
def test_nothing_behind_the_length_is_used(d, dtype):
    cache = make_cache(2, 2, d, [100, 39], 16, "symmetric", seed=20)
    q = torch.randn((2, 4, d), generator=torch.Generator().manual_seed(12)).to(dtype).cuda()
    w = torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda")
    ref = check(q, cache, w)
    for i, n in enumerate((100, 39)):
        page = cache.block_table[i, n // 16]
        cache.k_quant.scale[page, :, n % 16:] = float("nan")
        cache.v_quant.scale[page, :, n % 16:] = float("inf")
    w2 = torch.zeros_like(w)
    out = fs().paged_quant_attention_weights_cuda(q, cache, w2)
    assert torch.equal(out, ref) and torch.equal(w, w2)


def test_refusals():
    cache = make_cache(1, 2, 128, [40], 16, "affine", seed=19)
    pages = cache.k_quant.values.shape[0]
    q = torch.zeros((1, 4, 128), dtype=torch.float16, device="cuda")
    ok = torch.zeros((pages, 2, 16), device="cuda")
    f = fs().paged_quant_attention_weights_cuda
    for bad in (ok.half(), ok[:-1], ok.transpose(1, 2), ok.double()):
        with pytest.raises(ValueError):
            f(q, cache, bad)
    with pytest.raises(RuntimeError):
        f(q, cache, ok.cpu())
    with pytest.raises(RuntimeError):
        f(q.cpu(), cache, ok)
    with pytest.raises(ValueError):
        f(q.float(), cache, ok)
    with pytest.raises(ValueError):
        f(torch.zeros((1, 18, 128), dtype=torch.float16, device="cuda"), cache, ok)  # nine heads a kv head
    assert float(ok.abs().sum()) == 0.0


@pytest.mark.parametrize("longest", [2 ** 31, 2 ** 32, 2 ** 62])
@pytest.mark.parametrize("d", [128, 64])
def test_no_limit_on_the_length(longest, d):
    cache = make_cache(2, 2, d, [300, 45], 16, "affine", seed=21)
    c = fs().PagedKVCache(cache.k_quant, cache.v_quant, cache.block_table, cache.lengths, 16, longest)
    q = torch.randn((2, 4, d), generator=torch.Generator().manual_seed(13)).half().cuda()
    out = check(q, c, torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda"))
    assert torch.allclose(fs().paged_quant_attention_cuda(q, c).float(), out.float(), rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("size", [1.0, 6.0])
@pytest.mark.parametrize("b,hq,hkv,d,page,lens,fmt,dtype", [
    (2, 8, 2, 128, 16, [3000, 77], "affine", torch.float16),
    (2, 8, 2, 128, 16, [3000, 77], "symmetric", torch.float16),
    (40, 16, 16, 128, 16, [100 + 13 * i for i in range(40)], "affine", torch.float16),  # the balanced kernel
    (2, 8, 2, 64, 16, [900, 37], "affine", torch.bfloat16),
    (2, 4, 2, 256, 32, [700, 33], "symmetric", torch.bfloat16),
    (1, 5, 1, 64, 6, [77], "affine", torch.float16)])
def test_every_weight_is_precise_in_itself(b, hq, hkv, d, page, lens, fmt, dtype, size):
    """What a call adds to a token, light ones included, against 64 bits and relative to itself.

    With x a score in the log2 domain and u = 2^-24: x comes out of sums of terms that cancel, so its
    error is u times their size M = sm_scale log2(e) scale (sum |q c| + |offset| |sum q|) a few times
    over (8: conversions to fp32 and the join of the three byte sums), or D times in the generic
    kernel's chain of FMAs (without an offset); four roundings of x itself; and in the tuned kernels
    q's 24-bit fixed point, max|q| / 8355000 / 2 against sum |k|.  The LSE's error is at most that
    of the worst score, four roundings of itself and of the sum (n / 16 u); exp2 adds 2^-22 on either
    side.  ln 2 turns an error of the exponent into one of the weight; a weight below 2^-126 may be
    flushed."""
    u, ln2 = 2.0 ** -24, float(np.log(2))
    cache = make_cache(b, hkv, d, lens, page, fmt, seed=200 + d + page)
    q = (torch.randn((b, hq, d), generator=torch.Generator().manual_seed(14)) * size).to(dtype).cuda()
    pages = cache.k_quant.values.shape[0]
    w = torch.zeros((pages, hkv, page), device="cuda")
    fs().paged_quant_attention_weights_cuda(q, cache, w)
    tuned = d == 128 and page == 16 and dtype == torch.float16
    kq, table = cache.k_quant, cache.block_table
    worst = 0.0
    for i, n in enumerate(lens):
        at = table[i, : (n + page - 1) // page]
        if fmt == "symmetric":
            c, sc, off = kq.values[at].double(), kq.scale[at].double()[..., None], 0.0
        else:
            c = kq.values[at].double()[:, :, 0]
            sc = kq.scale[at].double()[:, :, 0]
            off = 128 - kq.zero_point[at].double()[:, :, 0]
        flat = lambda t: t.expand(len(at), hkv, page, t.shape[-1]).transpose(0, 1).flatten(1, 2)[:, :n]  # noqa: E731
        k = flat((c + off) * sc)
        qd = q[i].double().view(hkv, -1, d)
        x = torch.einsum("hgd,hnd->hgn", qd, k) * d ** -0.5 / ln2
        lse = torch.logsumexp(x * ln2, -1, keepdim=True) / ln2
        if tuned:
            m = torch.einsum("hgd,hnd->hgn", qd.abs(), flat(c.abs() * sc))
            if fmt == "affine":
                m = m + qd.sum(-1).abs()[..., None] * flat((off * sc).abs()).squeeze(-1)[:, None]
            e = 8 * u * m * d ** -0.5 / ln2
            e = e + qd.abs().amax(-1)[..., None] / 8355000 / 2 * k.abs().sum(-1)[:, None] * d ** -0.5 / ln2
        else:
            e = d * u * torch.einsum("hgd,hnd->hgn", qd.abs(), k.abs()) * d ** -0.5 / ln2
        e = e + 4 * u * x.abs()
        p = torch.exp2(x - lse)
        rel = ln2 * (e + e.amax(-1, keepdim=True) + 8 * u * lse.abs()) + 2.0 ** -21 + n / 16 * u
        got = w[at].double().transpose(0, 1).flatten(1)[:, :n]
        err, bound = (got - p.sum(1)).abs(), (p * rel).sum(1) + 2.0 ** -126
        worst = max(worst, float((err / bound).max()))
    assert worst <= 1, worst


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 0.0])
def test_weights_do_not_depend_on_v(fmt, bad):
    """A live token of V whose scale is infinite, undefined or zero: the output shows it, the weights
    are those of the scores.  Beside an infinite scale the reference lies 2^100 up, so tokens 2^-26
    below the heaviest no longer count towards the LSE (200 of them: 3e-6)."""
    cache = make_cache(2, 2, 128, [200, 39], 16, fmt, seed=22)
    q = torch.randn((2, 4, 128), generator=torch.Generator().manual_seed(15)).half().cuda()
    runs = []
    for scale in (None, bad):
        if scale is not None:
            s = cache.v_quant.scale.view(cache.v_quant.scale.shape[0], 2, -1)
            s[cache.block_table[0, 3], :, 0] = scale
        w = torch.zeros((cache.k_quant.values.shape[0], 2, 16), device="cuda")
        runs.append((fs().paged_quant_attention_weights_cuda(q, cache, w), w))
    assert torch.allclose(runs[1][1], runs[0][1], rtol=2e-5, atol=0)
    assert torch.equal(runs[1][0][1], runs[0][0][1])
    assert bool(runs[1][0][0].isfinite().all()) == (bad == 0.0)
