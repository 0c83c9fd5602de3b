"""GPU parity of the symmetric per-token INT8 format (FS_KV_SYMMETRIC): the quantizer
bit-exact against the oracle's restatement of the format, and paged / contiguous decode
against the oracle's attention over the dequantized cache at
|got - ref| <= 2e-3 + 1e-2 |ref|."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import flashspec_oracle as O

pytestmark = pytest.mark.gpu

ATOL, RTOL = 2e-3, 1e-2


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def fs():
    import flashspec_b200

    return flashspec_b200


def close(got, ref):
    ref_t = torch.as_tensor(np.asarray(ref, dtype=np.float32))
    err = (got.detach().float().cpu() - ref_t).abs()
    bad = err > ATOL + RTOL * ref_t.abs()
    assert not bool(bad.any()), f"{int(bad.sum())} out of tolerance, max abs err {err.max().item():.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_symmetric_quantizer_bit_exact(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(3, 4, 37, 128, generator=g, device="cuda") * 3).to(dtype)
    x[0, 0, 5] = 0  # an all-zero token: scale floor 1e-8, values 0
    qt = fs().quantize_int8_symmetric_per_token(x, 16)
    vals, sc = O.quantize_symmetric(x.float().cpu().numpy())
    assert tuple(qt.values.shape) == (3, 4, 48, 128)
    np.testing.assert_array_equal(qt.values[..., :37, :].cpu().numpy(), vals)
    np.testing.assert_array_equal(qt.scale[..., :37].cpu().numpy().view(np.uint32), sc.view(np.uint32))
    assert bool((qt.values[..., 37:, :] == 0).all())


@pytest.mark.parametrize("hq,hkv,d,page", [(32, 32, 128, 16), (8, 2, 128, 32), (4, 4, 64, 16)])
def test_symmetric_paged_decode_vs_oracle(hq, hkv, d, page):
    g = torch.Generator(device="cuda").manual_seed(hq + d + page)
    b, s = 4, 700
    k = torch.randn(b, hkv, s, d, generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn(b, hkv, s, d, generator=g, device="cuda", dtype=torch.float16)
    q = torch.randn(b, hq, d, generator=g, device="cuda", dtype=torch.float16)
    bps = (s + page - 1) // page
    perm = torch.randperm(b * bps, generator=torch.Generator().manual_seed(3))
    lengths = torch.tensor([700, 1, 333, 16], dtype=torch.int64, device="cuda")
    cache = fs().paged_cache_symmetric(k, v, page, lengths=lengths, perm=perm)
    out, stats = fs().paged_quant_attention_cuda(q, cache, return_stats=True)
    kq, vq = cache.k_quant, cache.v_quant
    ref = O.symmetric_paged_attention(q.cpu().numpy(), kq.values.cpu().numpy(), kq.scale.cpu().numpy(),
                                      vq.values.cpu().numpy(), vq.scale.cpu().numpy(), cache.block_table.cpu().numpy(),
                                      lengths.cpu().numpy(), s)
    close(out, ref)
    assert stats["quant_kv_bytes"] > 0


def test_symmetric_fused_decode_vs_oracle():
    g = torch.Generator(device="cuda").manual_seed(9)
    b, h, s, d = 3, 8, 300, 128
    k = torch.randn(b, h, s, d, generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn(b, h, s, d, generator=g, device="cuda", dtype=torch.float16)
    q = torch.randn(b, h, d, generator=g, device="cuda", dtype=torch.float16)
    kq = fs().quantize_int8_symmetric_per_token(k, 16)
    vq = fs().quantize_int8_symmetric_per_token(v, 16)
    lengths = torch.tensor([300, 299, 17], dtype=torch.int64, device="cuda")
    out = fs().fused_dequant_attention_cuda(q, kq, vq, lengths)
    kd = fs().dequantize_int8_symmetric(kq).cpu().numpy()
    vd = fs().dequantize_int8_symmetric(vq).cpu().numpy()
    close(out, O.reference_attention(q.cpu().numpy(), kd, vd, lengths.cpu().numpy()))


@pytest.mark.parametrize("kernel", ["split", "balanced"])
def test_scales_of_one_page_do_not_reach_another(monkeypatch, kernel):
    """Scales that differ by 64 from page to page, over many times the ring's stages: a warp that
    read the scales of the page that comes next in its stage would be far off.

    Bound per output element, with A = sum_j p_j |v_j| and delta the score error of 16-bit
    fixed-point q (max|q| / 32639 / 2 * max_j |k_j|_1 / sqrt(D)): P rounds once to fp16 (2^-11),
    a score enters on both sides of the quotient (2 delta), V's offset of at most 1152 leaves n / 16
    MMA additions of 2^-23 each, fp32 sums and exp2 2^-12, and the output rounds once (2^-11)."""
    monkeypatch.setenv("FLASHSPEC_DECODE_KERNEL", kernel)
    g = torch.Generator().manual_seed(23)
    b, hkv, grp, d, page, pages = 3, 2, 4, 128, 16, 150
    n = page * pages
    perm = torch.randperm(b * pages, generator=g).view(b, pages)
    codes = [torch.randint(-127, 128, (b * pages, hkv, page, d), generator=g).to(torch.int8) for _ in "kv"]
    step = torch.tensor([1.0, 64.0, 8.0])[torch.arange(pages) % 3]
    scale = []
    for top in (0.02, 1.0):
        s = torch.rand((b * pages, hkv, page), generator=g) * 0.5 + 0.5
        s[perm.reshape(-1)] *= (top / step).repeat(b)[:, None, None]
        scale.append(s)
    q = torch.randn((b, hkv * grp, d), generator=g).half()
    pool = [fs().SymQuantizedTensor(c.cuda(), s.cuda(), page, (b * pages, hkv, page, d)) for c, s in zip(codes, scale)]
    cache = fs().PagedKVCache(*pool, perm.cuda(), torch.full((b,), n).cuda(), page, n)
    k, v = ((c.double() * s.double()[..., None])[perm].transpose(1, 2).reshape(b, hkv, n, d)
            for c, s in zip(codes, scale))
    qd = q.double().view(b, hkv, grp, d)
    p = torch.softmax(torch.einsum("bhgd,bhnd->bhgn", qd, k) / d ** 0.5, -1)
    want = torch.einsum("bhgn,bhnd->bhgd", p, v)
    delta = qd.abs().amax(-1) / 32639 / 2 * k.abs().sum(-1).amax(-1)[..., None] / d ** 0.5
    a = torch.einsum("bhgn,bhnd->bhgd", p, v.abs())
    bound = (2 ** -11 + 2 * delta[..., None] + 2 ** -12) * a + 2 ** -11 * want.abs() + n / 16 * 2 ** -23 * 1152 + 2 ** -24
    weights = torch.zeros((b * pages, hkv, page), device="cuda")
    for out in (fs().paged_quant_attention_cuda(q.cuda(), cache),
                fs().paged_quant_attention_weights_cuda(q.cuda(), cache, weights)):
        err = (out.double().cpu().view(want.shape) - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())
    got = weights.cpu()[perm].transpose(1, 2).reshape(b, hkv, n).double()
    assert torch.allclose(got, p.sum(2), rtol=1e-4, atol=1e-9)
