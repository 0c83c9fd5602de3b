"""Expanded latent attention for prompts against 64 bits: dims, types, ragged packed
requests, cached prefixes, queries that see nothing, padding rows, odd offsets, streams and
graphs; and a whole run, prompt and steps, where the expanded and the absorbed form of the
same model agree.

Tolerance: with A = sum_j p_j |v_j|, P rounds once to 16 bits (half a step h of each p), the
fp32 sums of a score add at most 2^-12 of p here (dn + dr products of normal values,
sm_scale 1 / sqrt(dn + dr)), and the output rounds once:
|err| <= (h + 2^-12) A + h |out| + 2^-24."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
F, B = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def fs():
    import flashspec_b200

    return flashspec_b200


def offsets(n):
    return torch.cumsum(torch.tensor([0] + list(n)), 0).cuda()


def make(nq, nk, h, dn, dr, dv, dtype, seed, spare=0):
    g = torch.Generator().manual_seed(seed)
    rows_q, rows_k = sum(nq) + spare, sum(nk) + spare
    q = torch.randn((rows_q, h, dn + dr), generator=g).to(dtype).cuda()
    kv = torch.randn((rows_k, h, dn + dv), generator=g).to(dtype).cuda()
    r = torch.randn((rows_k, dr), generator=g).to(dtype).cuda()
    return q, kv, r


def expect(q, kv, r, nq, nk, sm_scale):
    dr = r.shape[1]
    dn = q.shape[2] - dr
    h, dv = q.shape[1], kv.shape[2] - dn
    out = torch.zeros((q.shape[0], h, dv), dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    half = torch.finfo(q.dtype).eps / 2
    q0 = k0 = 0
    for a, b in zip(nq, nk):
        qd, kd, rd = q[q0:q0 + a].double(), kv[k0:k0 + b].double(), r[k0:k0 + b].double()
        s = torch.einsum("ihd,jhd->hij", qd[..., :dn], kd[..., :dn]) + torch.einsum("ihd,jd->hij", qd[..., dn:], rd)
        seen = torch.ones((a, b), dtype=torch.bool, device="cuda").tril(b - a)
        p = torch.nan_to_num(torch.softmax(s * sm_scale + torch.where(seen, 0.0, -float("inf")), -1))
        out[q0:q0 + a] = torch.einsum("hij,jhd->ihd", p, kd[..., dn:])
        bound[q0:q0 + a] = (half + 2 ** -12) * torch.einsum("hij,jhd->ihd", p, kd[..., dn:].abs())
        q0, k0 = q0 + a, k0 + b
    return out, bound + half * out.abs() + 2 ** -24


def check(nq, nk, h, dn, dr, dv, dtype, seed, sm_scale=None):
    q, kv, r = make(nq, nk, h, dn, dr, dv, dtype, seed)
    want, bound = expect(q, kv, r, nq, nk, (dn + dr) ** -0.5 if sm_scale is None else sm_scale)
    out = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk), sm_scale=sm_scale)
    assert out.dtype == dtype
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


CASES = [
    # nq, nk, H, dn, dr, dv, dtype
    ([1], [1], 1, 128, 64, 128, F),
    ([1], [700], 2, 128, 64, 128, B),
    ([127, 128, 129], [127, 128, 129], 2, 128, 64, 128, F),
    ([63, 64, 65, 1], [63, 64, 65, 1], 3, 128, 64, 128, B),
    ([300, 5], [1000, 64], 2, 128, 64, 128, F),
    ([0, 200, 0, 3], [40, 200, 0, 3], 2, 128, 64, 128, B),
    ([200, 9], [150, 2], 2, 128, 64, 128, F),  # more queries than keys: the first see nothing
    ([50], [0], 1, 128, 64, 128, F),
    ([400, 31], [450, 31], 2, 64, 32, 64, F),
    ([400, 31], [450, 31], 2, 64, 64, 128, B),
    ([400, 31], [450, 31], 2, 128, 32, 64, F),
    ([400, 31], [450, 31], 2, 64, 32, 128, B),
    ([400, 31], [450, 31], 1, 64, 64, 64, F),
    ([400, 31], [450, 31], 1, 128, 32, 128, B),
    ([400, 31], [450, 31], 1, 128, 64, 64, B),
    ([2000], [2000], 1, 128, 64, 128, B),
]


@pytest.mark.parametrize("nq,nk,h,dn,dr,dv,dtype", CASES)
def test_prefill(nq, nk, h, dn, dr, dv, dtype):
    check(nq, nk, h, dn, dr, dv, dtype, seed=sum(nq) + dn)


def test_many_requests():
    n = [(37 * i) % 150 for i in range(100)]
    check(n, [x + (i % 3) * 70 for i, x in enumerate(n)], 3, 64, 32, 64, F, seed=5, sm_scale=0.2)


def test_long_and_peaked():
    check([700], [9000], 2, 128, 64, 128, F, seed=6, sm_scale=1.0)


@pytest.mark.parametrize("sm_scale", [-0.1, 0.0])
def test_scales_of_any_sign(sm_scale):
    check([300, 77], [420, 77], 2, 128, 64, 128, B, seed=14, sm_scale=sm_scale)


def test_rows_of_no_request():
    """Padding rows behind the last request stay as they were, or are zeros."""
    nq = nk = [100, 30]
    q, kv, r = make(nq, nk, 2, 128, 64, 128, F, 7, spare=200)
    q[130:], kv[130:], r[130:] = float("nan"), float("nan"), float("inf")
    mine = torch.full((330, 2, 128), 5.0, dtype=F, device="cuda")
    a = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk), out=mine)
    b = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk))
    assert a.data_ptr() == mine.data_ptr() and bool((a[130:] == 5).all()) and not bool(b[130:].any())
    want, bound = expect(q[:130], kv[:130], r[:130], nq, nk, 192 ** -0.5)
    assert torch.equal(a[:130], b[:130]) and bool(((a[:130].double() - want).abs() <= bound).all())


def test_first_offset_and_offsets_outside_the_rows():
    nq = nk = [60, 40]
    q, kv, r = make(nq, nk, 1, 64, 32, 64, F, 8)
    late = torch.tensor([60, 100]).cuda()
    full = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk))
    part = fs().latent_prefill_attention_cuda(q, kv, r, late, late)
    assert torch.equal(part[60:], full[60:]) and not bool(part[:60].any())
    wild = torch.tensor([-50, 60, 10 ** 15]).cuda()
    assert torch.equal(fs().latent_prefill_attention_cuda(q, kv, r, wild, wild), full)
    falling = torch.tensor([60, 0, 30]).cuda()  # a request of no rows, then one of 30
    got = fs().latent_prefill_attention_cuda(q, kv, r, falling, falling)
    assert torch.equal(got[:30], full[:30]) and not bool(got[30:].any())


def test_infinite_values_stay_behind_the_mask():
    nq = nk = [150]
    q, kv, r = make(nq, nk, 1, 128, 64, 128, B, 9)
    ref = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk))
    kv[100:], r[100:] = float("inf"), float("nan")
    out = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk))
    assert torch.equal(out[:64], ref[:64])  # tiles without those keys
    assert bool(out[100:].isnan().all())


def test_strided_inputs_stream_and_graph():
    nq, nk = [70, 130], [90, 130]
    q, kv, r = make(nq, nk, 2, 128, 64, 128, F, 10)
    wide = torch.zeros((sum(nk), 2 * 256 + 64 + 3), dtype=F, device="cuda")
    wide[:, 3:67], wide[:, 67:] = r, kv.flatten(1)
    kv_v, r_v = wide[:, 67:].view(sum(nk), 2, 256), wide[:, 3:67]
    ref = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk))
    qo, ko = offsets(nq), offsets(nk)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert torch.equal(fs().latent_prefill_attention_cuda(q, kv_v, r_v, qo.int(), ko.int()), ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fs().latent_prefill_attention_cuda(q, kv, r, qo, ko)
    for _ in range(2):
        out.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_no_queries():
    q, kv, r = make([0], [5], 2, 64, 32, 64, F, 11)
    assert fs().latent_prefill_attention_cuda(q, kv, r, offsets([0]), offsets([5])).shape == (0, 2, 64)


def test_refusals():
    q, kv, r = make([10], [10], 2, 64, 32, 64, F, 12)
    f, o = fs().latent_prefill_attention_cuda, offsets([10])
    for bad in ((q[..., :80], kv, r), (q, kv[:, :1], r), (q, kv[:9], r), (q, kv, r[:, :16]), (q, kv.bfloat16(), r),
                (q.float(), kv.float(), r.float()), (q[0], kv, r)):
        with pytest.raises(ValueError):
            f(*bad, o, o)
    for bad in ((o[:1], o[:1]), (o, offsets([5, 5])), (o[None], o[None])):
        with pytest.raises(ValueError):
            f(q, kv, r, *bad)
    with pytest.raises(ValueError):
        f(q, kv, r, o, o, out=torch.zeros((10, 2, 64), device="cuda"))
    with pytest.raises(RuntimeError):
        f(q, kv, r, o.cpu(), o)
    with pytest.raises(RuntimeError):
        f(q.cpu(), kv.cpu(), r.cpu(), o.cpu(), o.cpu())


def test_prompt_then_steps_of_one_model():
    """A layer of a latent model: the prompt through the expanded form, the last tokens again
    through the absorbed form; both are the same attention.  The forms round in different
    places (the expanded one its keys and values, the absorbed one its queries), each 2^-11 of
    a product of normal values, so they agree to a few 2^-10 of the values' size."""
    g = torch.Generator().manual_seed(13)
    h, dn, dr, dv, dc, t = 4, 64, 32, 64, 256, 150
    rand = lambda *s: torch.randn(s, generator=g).half().cuda()  # noqa: E731
    w_uk, w_uv = rand(h, dn, dc) / 16, rand(h, dv, dc) / 16
    c, r = rand(2, t, dc), rand(2, t, dr)
    qn, qr = rand(2, t, h, dn), rand(2, t, h, dr)
    cache = fs().LatentKVCache.empty(2, 256, dc, dr, 64, dtype=F)
    counts = torch.tensor([150, 99]).cuda()
    cache, held = cache.append(c, r, counts, return_held=True)
    rows = torch.cat([torch.arange(150), 150 + torch.arange(99)]).cuda()
    flat = held.flatten(0, 1)[rows]
    kv = torch.cat([torch.einsum("nc,hdc->nhd", flat.float(), w.float()).half() for w in (w_uk, w_uv)], -1)
    q = torch.cat([qn, qr], -1).flatten(0, 1)[rows]
    o = offsets([150, 99])
    prompt = fs().latent_prefill_attention_cuda(q, kv, r.flatten(0, 1)[rows], o, o)
    last = torch.stack([torch.arange(147, 150), torch.arange(96, 99)]).cuda()
    pick = lambda x: torch.stack([x[b, last[b]] for b in range(2)])  # noqa: E731
    ql = torch.einsum("bthd,hdc->bthc", pick(qn).float(), w_uk.float()).half()
    lat = fs().latent_attention_cuda(ql, pick(qr).contiguous(), cache, sm_scale=(dn + dr) ** -0.5)
    step = torch.einsum("bthc,hdc->bthd", lat.float(), w_uv.float())
    want = torch.stack([prompt[147:150], prompt[246:249]]).float()
    assert torch.allclose(step, want, atol=6e-3, rtol=6e-3), (step - want).abs().max()


def test_out_over_an_input_is_refused():
    q, kv, r = make([10], [10], 2, 64, 64, 128, F, 14)
    f, o = fs().latent_prefill_attention_cuda, offsets([10])
    with pytest.raises(ValueError):
        f(q, kv, r, o, o, out=q)
    out = torch.empty_like(q)
    assert torch.equal(f(q, kv, r, o, o, out=out), f(q, kv, r, o, o)) and out.data_ptr() != q.data_ptr()


def expect_infinite(q, kv, r, nq, nk, sm_scale):
    """As expect, for values that may be infinite or NaN: (finite part and bound, where +inf, -inf, NaN)."""
    dn = q.shape[2] - r.shape[1]
    plain = kv.clone()
    plain[..., dn:] = torch.nan_to_num(plain[..., dn:], nan=0.0, posinf=0.0, neginf=0.0)
    out, bound = expect(q, plain, r, nq, nk, sm_scale)
    hits = [torch.zeros(out.shape, dtype=torch.bool, device="cuda") for _ in range(3)]
    q0 = k0 = 0
    for a, b in zip(nq, nk):
        v = kv[k0:k0 + b, :, dn:]
        seen = torch.ones((a, b), dtype=torch.double, device="cuda").tril(b - a)
        for hit, what in zip(hits, (v.isposinf(), v.isneginf(), v.isnan())):
            hit[q0:q0 + a] = torch.einsum("ij,jhd->ihd", seen, what.double()) > 0
        q0, k0 = q0 + a, k0 + b
    pos, neg, nan = hits
    nan = nan | (pos & neg)
    return out, bound, pos & ~nan, neg & ~nan, nan


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("nq,nk,sm_scale", [([300], [300], None), ([40, 500], [700, 520], None),
                                            ([40, 500], [700, 520], 1.0), ([200, 9], [150, 2], None)])
def test_infinite_values_by_the_definition(dtype, nq, nk, sm_scale):
    """Infinite and undefined values on the causal edge, far inside it, and under probabilities
    that 16 bits round to zero (sm_scale 1): a query that sees one gets infinity where all that
    it sees have one sign, else NaN; the other queries and dims what they had."""
    q, kv, r = make(nq, nk, 2, 128, 64, 128, dtype, 15)
    g = torch.Generator().manual_seed(16)
    for k in range(24):
        key = int(torch.randint(0, sum(nk), (1,), generator=g))
        kv[key, k % 2, 128 + 5 * k] = (float("inf"), -float("inf"), float("nan"), float("inf"))[k % 4]
    kv[3, 0, 200], kv[sum(nk) - 4, 0, 200] = float("inf"), -float("inf")  # of one dim
    out, bound, pos, neg, nan = expect_infinite(q, kv, r, nq, nk, 192 ** -0.5 if sm_scale is None else sm_scale)
    got = fs().latent_prefill_attention_cuda(q, kv, r, offsets(nq), offsets(nk), sm_scale=sm_scale).double()
    assert torch.equal(got.isposinf(), pos) and torch.equal(got.isneginf(), neg) and torch.equal(got.isnan(), nan)
    fine = ~(pos | neg | nan)
    assert bool(pos.any()) and bool(neg.any()) and bool(nan.any())
    assert bool(((got - out).abs() <= bound)[fine].all())


def test_every_value_infinite():
    """All of V: the largest number of elements to look over again."""
    q, kv, r = make([600], [2000], 2, 64, 32, 64, B, 17)
    kv[..., 64:] = float("inf")
    kv[1800:, 1, 64:] = -float("inf")
    out = fs().latent_prefill_attention_cuda(q, kv, r, offsets([600]), offsets([2000]))
    assert bool(out[:, 0].isposinf().all())
    assert bool(out[:400, 1].isposinf().all()) and bool(out[400:, 1].isnan().all())


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("near", [0, 100, 29000])
def test_many_far_keys_beside_a_near_one_without_value(dtype, near):
    """One key takes nearly all of the weight and has value zero (a sink); the output is what
    30000 keys at e^-17 of it add up to.  P keeps its relative precision down to 2^-25 (e^-17 is
    2^-24.5), so the bound of the other cases holds here too; without that fp16 gave zero."""
    n, nq = 30000, 300
    q = torch.zeros((nq, 1, 96), dtype=dtype, device="cuda")
    q[..., 0] = 1
    kv = torch.zeros((n, 1, 128), dtype=dtype, device="cuda")
    kv[..., 0], kv[near, 0, 0] = -1.0, 16.0
    kv[..., 64:] = (torch.rand((n, 1, 64), generator=torch.Generator().manual_seed(1)) + 0.5).to(dtype).cuda()
    kv[near, 0, 64:] = 0
    r = torch.zeros((n, 32), dtype=dtype, device="cuda")
    want, bound = expect(q, kv, r, [nq], [n], 1.0)
    out = fs().latent_prefill_attention_cuda(q, kv, r, offsets([nq]), offsets([n]), sm_scale=1.0)
    err = (out.double() - want).abs()
    assert float(want.min()) > 1e-3 and bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("b", [33, 100, 1025, 5000])
@pytest.mark.parametrize("longest", [3, 700])
def test_large_batches(b, longest):
    """Requests are searched for: none to several 256-query tiles each, empty ones in runs, prefixes,
    and rows before the first and behind the last."""
    g = torch.Generator().manual_seed(b)
    total = 12000
    n = torch.randint(0, longest + 1, (b,), generator=g)
    n[torch.rand(b, generator=g) < 0.4] = 0
    n = torch.where(torch.cumsum(n, 0) <= total, n, torch.zeros_like(n)).tolist()
    nk = [x + (i % 4 if x else 0) for i, x in enumerate(n)]
    front = 300
    q, kv, r = make([sum(n)], [sum(nk)], 2, 64, 32, 64, F, 18, spare=front)
    q[:front] = float("nan")
    # expect() walks from row 0: give it the part that the requests cover
    want, bound = expect(q[front:], kv, r, n, nk, 96 ** -0.5)
    qo, ko = offsets(n) + front, offsets(nk)
    got = fs().latent_prefill_attention_cuda(q, kv, r, qo, ko)
    assert bool(((got[front:].double() - want).abs() <= bound).all()) and not bool(got[:front].any())
    if b <= 4096:  # the same batch, padded with zeros behind its last request
        pad = torch.zeros(b // 3 if b < 2000 else 500, dtype=torch.int64, device="cuda")
        again = fs().latent_prefill_attention_cuda(q, kv, r, torch.cat([qo, pad]), torch.cat([ko, pad]))
        assert torch.equal(again, got)


def test_the_time_of_a_large_batch_is_linear():
    """16384 requests of one token: dealt, they would take some seconds."""
    n = [1] * 16384
    q, kv, r = make(n, n, 16, 64, 32, 64, F, 19)
    o = offsets(n)
    fs().latent_prefill_attention_cuda(q[:40], kv[:40], r[:40], o[:41], o[:41])
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    out = fs().latent_prefill_attention_cuda(q, kv, r, o, o)
    b.record()
    torch.cuda.synchronize()
    assert torch.equal(out, kv[..., 64:]) and a.elapsed_time(b) < 100
