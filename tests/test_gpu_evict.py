"""Eviction by accumulated weight against a plain restatement: which tokens stay (ties, equal
weights, zeros, infinities, NaN), where they land (codes, scales, zero points bit for bit),
the weights that move with them, rows left alone, the allocator's bookkeeping, and a
serving run that cuts its requests.  Everything compared here is exact: positions are whole
numbers, moved codes are copies or follow from the format's own rounding, and moved weights
are copies."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import flashspec_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")


def fs():
    import flashspec_b200

    return flashspec_b200


def make_cache(hkv, d, lens, page, fmt, seed, slack=2, extra_cols=0):
    rng = np.random.default_rng(seed)
    need = [(n + page - 1) // page for n in lens]
    total = max(1, sum(need) + slack)
    perm = rng.permutation(total)
    cols = max(1, max(need)) + extra_cols
    table = np.full((len(lens), cols), -1, np.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    x = [torch.from_numpy(rng.standard_normal((total, hkv, page, d)).astype(np.float32)).cuda() for _ in "kv"]
    f = fs().quantize_int8_symmetric_per_token if fmt == "symmetric" else fs().quantize_int8_per_block
    cache = fs().PagedKVCache(f(x[0], page), f(x[1], page), torch.from_numpy(table).cuda(),
                              torch.tensor(lens, dtype=torch.int64).cuda(), page, max(max(lens), 1))
    w = np.exp(rng.standard_normal((total, hkv, page)) * 2).astype(np.float32)
    return cache, w


def expect_kept(w, n, budget, recent, sinks):
    """Positions kept of one head's n weights: NaN above all, then by value, ties to the lower position."""
    if n <= budget:
        return list(range(n))
    mid = range(sinks, n - recent)
    order = sorted(mid, key=lambda i: (0, 0.0, i) if np.isnan(w[i]) else (1, -float(w[i]), i))
    return list(range(sinks)) + sorted(order[: budget - recent - sinks]) + list(range(n - recent, n))


def expect(cache, w, budget, recent, sinks):
    """numpy copies of (kept, lengths, weights, [values, scale, zero] of K and V) after the cut."""
    table = cache.block_table.cpu().numpy()
    lens = cache.lengths.cpu().numpy()
    page, hkv = cache.block_size, w.shape[1]
    b = table.shape[0]
    kept = np.full((b, hkv, budget), -1, np.int32)
    new_lens = np.zeros(b, np.int64)
    w_out = w.copy()
    pools = []
    for qt in (cache.k_quant, cache.v_quant):
        v = qt.values.cpu().numpy().copy()
        sym = getattr(qt, "symmetric", False)
        v = v if sym else v[:, :, 0]
        sc = qt.scale.cpu().numpy().copy()
        z = None if sym else qt.zero_point.cpu().numpy().copy()
        pools.append([v, sc, z])
    old = [[None if x is None else x.copy() for x in p] for p in pools]
    for i in range(b):
        n = int(max(0, min(lens[i], cache.max_seq_len, table.shape[1] * page)))
        new_lens[i] = min(n, budget)
        for h in range(hkv):
            row = np.array([w[table[i, t // page], h, t % page] if table[i, t // page] >= 0 else -np.inf
                            for t in range(n)], np.float32)
            keep = expect_kept(row, n, budget, recent, sinks)
            kept[i, h, : len(keep)] = keep
            for t in range(table.shape[1] * page):
                pg = table[i, t // page]
                if pg >= 0:
                    src = keep[t] if t < len(keep) else -1
                    w_out[pg, h, t % page] = 0.0 if src < 0 or table[i, src // page] < 0 else row[src]
            if n <= budget:
                continue
            for lp in range((budget + page - 1) // page):
                at = keep[lp * page:(lp + 1) * page]
                dst = table[i, lp]
                if at == list(range(lp * page, lp * page + len(at))) or dst < 0:
                    continue
                for (v, sc, z), (ov, osc, oz) in zip(pools, old):
                    if z is None:
                        v[dst, h] = 0
                        sc[dst, h] = np.float32(1e-8)
                        for r, t in enumerate(at):
                            if table[i, t // page] >= 0:
                                v[dst, h, r] = ov[table[i, t // page], h, t % page]
                                sc[dst, h, r] = osc[table[i, t // page], h, t % page]
                        continue
                    x = np.zeros((page, v.shape[-1]), np.float32)
                    for r, t in enumerate(at):
                        p = table[i, t // page]
                        if p >= 0:
                            u = ov[p, h, t % page].astype(np.float32) + np.float32(128)
                            x[r] = (u - np.float32(oz[p, h, 0, 0, 0])) * osc[p, h, 0, 0, 0]
                    oq = O.quantize_int8_per_block(x, page)
                    v[dst, h] = oq.values.reshape(page, -1)
                    sc[dst, h] = oq.scale.reshape(())
                    z[dst, h] = oq.zero_point.reshape(())
    return kept, new_lens, w_out, pools


def check(cache, w, budget, recent, sinks, out=None, **kw):
    want = expect(cache, w, budget, recent, sinks)
    wd = torch.from_numpy(w).cuda()
    cut, kept = fs().evict_tokens_cuda(cache, wd, budget, recent=recent, sinks=sinks, weights_out=out, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(kept.cpu().numpy(), want[0])
    assert np.array_equal(cut.lengths.cpu().numpy(), want[1])
    got_w = (wd if out is None else out).cpu().numpy()
    if out is None:
        assert np.array_equal(got_w, want[2], equal_nan=True)
    else:  # pages outside the table keep what weights_out held
        pages = cache.block_table[cache.block_table >= 0].cpu().numpy()
        assert np.array_equal(got_w[pages], want[2][pages], equal_nan=True)
        assert np.array_equal(wd.cpu().numpy(), w, equal_nan=True)
    for qt, (v, sc, z) in zip((cut.k_quant, cut.v_quant), want[3]):
        assert np.array_equal(qt.values.cpu().numpy().reshape(v.shape), v)
        assert np.array_equal(qt.scale.cpu().numpy().reshape(sc.shape), sc)
        if z is not None:
            assert np.array_equal(qt.zero_point.cpu().numpy().reshape(z.shape), z)
    assert cut.max_seq_len == min(cache.max_seq_len, budget)
    return cut, kept


CASES = [
    # hkv, d, lens, page, budget, recent, sinks
    (1, 128, [17], 16, 16, 0, 0),
    (2, 128, [0, 1, 16, 33, 200], 16, 32, 8, 4),
    (3, 128, [500, 499, 64], 16, 100, 20, 3),
    (2, 64, [300, 20], 16, 150, 0, 16),
    (1, 64, [333], 32, 70, 70, 0),  # recent alone
    (2, 32, [100, 90], 16, 50, 25, 25),  # nothing left to choose
    (1, 256, [130, 65], 32, 64, 1, 0),
    (2, 64, [77, 50], 6, 31, 5, 2),
    (1, 128, [200], 64, 65, 10, 1),
    (1, 256, [120], 45, 80, 7, 1),
    (1, 128, [40], 16, 1, 0, 0),
    (1, 128, [40], 16, 1, 1, 0),
]


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
@pytest.mark.parametrize("hkv,d,lens,page,budget,recent,sinks", CASES)
def test_cut(fmt, hkv, d, lens, page, budget, recent, sinks):
    cache, w = make_cache(hkv, d, lens, page, fmt, seed=d + page + budget, extra_cols=1)
    check(cache, w, budget, recent, sinks)


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
def test_two_cuts_and_weights_out(fmt):
    cache, w = make_cache(2, 128, [600, 450, 10], 16, fmt, seed=5)
    out = torch.full(w.shape, 7.0, device="cuda")
    cut, _ = check(cache, w, 300, 50, 8, out=out)
    check(cut, out.cpu().numpy(), 77, 10, 2)


def test_long_rows_take_a_cluster():
    """Rows long enough for clusters of several CTAs in both kernels."""
    cache, w = make_cache(1, 32, [20000, 9000], 16, "symmetric", seed=6)
    check(cache, w, 5000, 300, 4)


@pytest.mark.parametrize("n", [390016, 400000])
def test_rows_at_and_past_what_shared_memory_holds(n):
    """390016 tokens fill the clusters' shared memory; with 400000 the keys are in the workspace."""
    page = 64
    pages = n // page
    g = torch.Generator(device="cuda").manual_seed(1)
    v = torch.randint(-127, 128, (pages, 1, page, 16), generator=g, device="cuda", dtype=torch.int8)
    sc = torch.rand((pages, 1, page), generator=g, device="cuda") + 0.1
    pool = lambda: fs().SymQuantizedTensor(v.clone(), sc.clone(), page, (pages, 1, page, 16))  # noqa: E731
    table = torch.randperm(pages, generator=g, device="cuda")[None]
    cache = fs().PagedKVCache(pool(), pool(), table, torch.tensor([n], device="cuda"), page, n)
    w = torch.randint(0, 1000, (pages, 1, page), generator=g, device="cuda").float()  # many ties
    flat = w[table[0], 0].reshape(-1)
    mid = flat[16: n - 100]
    order = torch.sort(mid, descending=True, stable=True).indices[: 50000 - 116]
    want = torch.cat([torch.arange(16, device="cuda"), torch.sort(order).values + 16,
                      torch.arange(n - 100, n, device="cuda")])
    tok = v[table[0], 0].reshape(n, 16)[want]
    cut, kept = fs().evict_tokens_cuda(cache, w, 50000, recent=100, sinks=16)
    assert torch.equal(kept[0, 0].long(), want)
    assert torch.equal(cut.k_quant.values[table[0], 0].reshape(n, 16)[:50000], tok)
    assert torch.equal(w[table[0], 0].reshape(-1)[:50000], flat[want])
    assert float(w[table[0], 0].reshape(-1)[50000:].abs().sum()) == 0.0


@pytest.mark.parametrize("what", ["equal", "zeros", "extremes"])
def test_ties_and_odd_weights(what):
    cache, w = make_cache(2, 64, [700, 70], 16, "symmetric", seed=7)
    if what == "equal":
        w[:] = 3.0
    elif what == "zeros":
        w[:] = np.where(np.random.default_rng(0).random(w.shape) < 0.5, 0.0, -0.0)
    else:
        pick = np.random.default_rng(1).choice([np.inf, np.nan, 0.0, 1e-45, 3e38, -1.0, -np.inf, 1e-20], w.shape)
        w[:] = pick.astype(np.float32)
    check(cache, w, 64, 5, 3)


def test_unallocated_pages_come_last():
    cache, w = make_cache(1, 64, [200], 16, "affine", seed=8)
    table = cache.block_table.clone()
    table[0, 5] = -1
    c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, cache.lengths, 16, 200)
    check(c, w, 120, 10, 2)


def test_page_outside_the_pool_counts_as_unallocated():
    got = []
    for bad in (-1, 10 ** 12):
        cache, w = make_cache(1, 64, [200], 16, "affine", seed=9)
        table = cache.block_table.clone()
        table[0, 7] = bad
        c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, cache.lengths, 16, 200)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        cut, kept = fs().evict_tokens_cuda(c, torch.from_numpy(w).cuda(), 130, recent=90, device_status=status)
        got.append((kept, cut.k_quant.values, int(status)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert got[0][2] == 0 and got[1][2] == 1


def test_capture_and_other_stream():
    cache, w = make_cache(2, 128, [400, 300], 16, "affine", seed=10)
    want = expect(cache, w, 100, 10, 4)
    wd = torch.from_numpy(w).cuda()
    out = torch.zeros_like(wd)
    pristine = [t.clone() for q in (cache.k_quant, cache.v_quant) for t in (q.values, q.scale, q.zero_point)]
    live = [t for q in (cache.k_quant, cache.v_quant) for t in (q.values, q.scale, q.zero_point)]
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        cut, kept = fs().evict_tokens_cuda(cache, wd, 100, recent=10, sinks=4, weights_out=out)
    for _ in range(2):
        for a, b in zip(live, pristine):
            a.copy_(b)
        kept.fill_(5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(kept.cpu().numpy(), want[0])
        assert np.array_equal(cut.lengths.cpu().numpy(), want[1])
        assert np.array_equal(cut.k_quant.values.cpu().numpy()[:, :, 0], want[3][0][0])


def test_refusals():
    cache, w = make_cache(1, 64, [60], 16, "affine", seed=11)
    wd = torch.from_numpy(w).cuda()
    f = fs().evict_tokens_cuda
    for kw in (dict(budget=0, recent=0), dict(budget=4, recent=5), dict(budget=4, recent=2, sinks=3),
               dict(budget=4, recent=-1), dict(budget=4, recent=1, sinks=-1)):
        with pytest.raises(ValueError):
            f(cache, wd, **kw)
    with pytest.raises(ValueError):
        f(cache, wd.half(), 8, recent=1)
    with pytest.raises(ValueError):
        f(cache, wd[1:], 8, recent=1)
    base = torch.zeros(2 * wd.numel(), device="cuda")
    with pytest.raises(ValueError):
        f(cache, base[: wd.numel()].view_as(wd), 8, recent=1, weights_out=base[4: wd.numel() + 4].view_as(wd))
    with pytest.raises(RuntimeError):
        f(cache, wd.cpu(), 8, recent=1)
    x = torch.randn((4, 1, 32, 64), device="cuda")
    two = fs().PagedKVCache(fs().quantize_int8_per_block(x, 16), fs().quantize_int8_per_block(x, 16),
                            torch.zeros((1, 1), dtype=torch.int64, device="cuda"), cache.lengths, 32, 32)
    with pytest.raises(ValueError):
        f(two, torch.zeros((4, 1, 32), device="cuda"), 8, recent=1)  # pages of two quantization blocks
    with pytest.raises(ValueError):
        f(fs().PagedKVCache(cache.k_quant, cache.k_quant, cache.block_table, cache.lengths, 16, 60), wd, 8, recent=1)
    with pytest.raises(ValueError):
        f(cache, wd, 1 << 30, recent=1)
    kq = cache.k_quant
    turned = fs().QuantizedTensor(kq.values.transpose(3, 4).contiguous().transpose(3, 4), kq.scale, kq.zero_point, 16,
                                  kq.original_shape)
    with pytest.raises(ValueError):
        f(fs().PagedKVCache(turned, cache.v_quant, cache.block_table, cache.lengths, 16, 60), wd, 8, recent=1)


def test_allocator_steps_of_attention_append_and_eviction():
    """A run as a server makes it; after every cut the cache equals one that the host cut."""
    f, rng = fs(), torch.Generator(device="cuda").manual_seed(3)
    hkv, hq, d = 2, 4, 128
    alloc = f.PagedKVAllocator(capacity_blocks=64, heads=hkv, head_dim=d, track_weights=True)
    rand = lambda *s: torch.randn(s, generator=rng, device="cuda", dtype=torch.float16)  # noqa: E731
    for rid, n in ((7, 90), (3, 200), (9, 31)):
        alloc.add_request(rid, rand(1, hkv, n, d), rand(1, hkv, n, d))
    ids = [3, 9, 7]
    for step in range(40):
        alloc.append_batch(ids, rand(len(ids), hkv, 1, d), rand(len(ids), hkv, 1, d))
        f.paged_quant_attention_weights_cuda(rand(len(ids), hq, d), alloc.to_cache(ids), alloc.weights)
        over = [i for i in ids if alloc._requests[i].length > 80]
        if over:
            before = alloc.to_cache(over)
            want = expect(before, alloc.weights.cpu().numpy(), 64, 16, 2)
            kept = alloc.evict_batch(over, 64, recent=16, sinks=2)
            assert np.array_equal(kept.cpu().numpy(), want[0])
            assert np.array_equal(alloc.weights.cpu().numpy(), want[2])
            assert np.array_equal(alloc.k_quant.values.cpu().numpy()[:, :, 0], want[3][0][0])
            after = alloc.to_cache(over)
            assert after.lengths.tolist() == [64] * len(over) and after.block_table.shape[1] == 4
            assert bool((after.block_table >= 0).all())
        if step == 20:
            alloc.release_request(9)
            ids.remove(9)
        free = torch.tensor(alloc.free_blocks, device="cuda")
        assert float(alloc.weights[free].abs().sum()) == 0.0
        used = alloc.to_cache(ids).block_table
        used = used[used >= 0].tolist()
        assert len(used) == len(set(used)) and not set(used) & set(alloc.free_blocks)
        assert len(used) + len(alloc.free_blocks) == 64
    with pytest.raises(ValueError):
        alloc.evict_batch([3, 3], 10, recent=1)
    with pytest.raises(KeyError):
        alloc.evict_batch([12345], 10, recent=1)
    with pytest.raises(RuntimeError):
        f.PagedKVAllocator(capacity_blocks=2, heads=1, head_dim=64).evict_batch([], 10, recent=1)


def test_serving_run_with_a_budget():
    from flashspec_b200.serving import ServingConfig, run

    cfg = ServingConfig(steps=60, arrival_rate=1.0, max_live=8, prompt_min=20, prompt_max=300, out_min=20, out_max=60,
                        heads=4, kv_budget=100, kv_slack=16, kv_recent=20)
    log = []
    res = run(cfg, recorder=log)
    assert res["cuts"] > 0 and any(op[0] == "evict" for op in log)
    alloc = log[-1][1]
    assert all(alloc._requests[i].length <= 116 for i in alloc.live_request_ids)
    attn = [op for op in log if op[0] == "attn"]
    assert all(np.isfinite(op[3].astype(np.float32)).all() for op in attn)


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
def test_pool_whose_parts_differ_in_size_is_refused(fmt):
    cache, w = make_cache(2, 64, [60], 16, fmt, seed=12)
    kq, wd = cache.k_quant, torch.from_numpy(w).cuda()
    short = fs().QuantizedTensor(kq.values, kq.scale[1:].contiguous(), kq.zero_point, 16, kq.original_shape) \
        if fmt == "affine" else type(kq)(kq.values, kq.scale[1:].contiguous(), kq.block_size, kq.original_shape)
    with pytest.raises(ValueError):
        fs().evict_tokens_cuda(fs().PagedKVCache(short, cache.v_quant, cache.block_table, cache.lengths, 16, 60), wd,
                               8, recent=1)


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
@pytest.mark.parametrize("bad", [-2, -2 ** 31, 3 - 2 ** 32, 3 - 2 ** 40, -2 ** 63])
def test_every_negative_table_entry_counts_as_unallocated(fmt, bad):
    """Entries whose low 32 bits name a page of the pool among them; none is reported as bad."""
    got = []
    for entry in (-1, bad):
        cache, w = make_cache(2, 64, [200], 16, fmt, seed=13)
        table = cache.block_table.clone()
        table[0, 1], table[0, 9] = entry, entry
        c = fs().PagedKVCache(cache.k_quant, cache.v_quant, table, cache.lengths, 16, 200)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        wd = torch.from_numpy(w).cuda()
        cut, kept = fs().evict_tokens_cuda(c, wd, 150, recent=100, sinks=40, device_status=status)
        got.append((kept, wd, cut.k_quant.values, cut.k_quant.scale, cut.v_quant.values))
        assert int(status) == 0
    assert all(torch.equal(x, y) for x, y in zip(*got))


def evict_args(cache, w, budget, recent, new_lengths, kept):
    from flashspec_b200 import _lib

    a, kq, vq = _lib.FsEvictArgs(), cache.k_quant, cache.v_quant
    a.kv_format = _lib.FS_KV_SYMMETRIC
    a.batch, a.kv_heads, a.head_dim, a.page_size = 1, w.shape[1], kq.values.shape[-1], cache.block_size
    a.table_cols, a.max_seq_len = cache.block_table.shape[1], cache.max_seq_len
    a.budget, a.recent, a.num_pages = budget, recent, w.shape[0]
    a.block_table, a.lengths = cache.block_table.data_ptr(), cache.lengths.data_ptr()
    a.k_values, a.k_scale = kq.values.data_ptr(), kq.scale.data_ptr()
    a.v_values, a.v_scale = vq.values.data_ptr(), vq.scale.data_ptr()
    a.weights = a.weights_out = w.data_ptr()
    a.kept, a.new_lengths = kept.data_ptr(), new_lengths.data_ptr()
    return a


def test_calls_on_several_host_threads():
    """Cuts that need much and little shared memory, entered from several threads at once
    (ctypes lets go of the interpreter during a call)."""
    import ctypes as C
    import threading

    from flashspec_b200 import _lib

    lib, states = _lib.load(), []
    for n in (300000, 40, 40, 40):
        cache, w = make_cache(1, 32, [n], 16, "symmetric", seed=n)
        wd = torch.from_numpy(w).cuda()
        new, kept = torch.empty(1, dtype=torch.int64, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        stream = torch.cuda.Stream()
        states.append((evict_args(cache, wd, n, 0, new, kept), stream, (cache, wd, new, kept), []))
    torch.cuda.synchronize()

    def work(a, stream, keep, codes):
        for i in range(1500):
            codes.append(lib.fs_evict_tokens(C.byref(a), stream.cuda_stream))
            if i % 50 == 0:
                stream.synchronize()

    threads = [threading.Thread(target=work, args=s) for s in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, _, (cache, wd, new, kept), codes in states:
        assert set(codes) == {0}, codes
        assert int(new) == a.budget and torch.equal(kept.cpu(), torch.arange(a.budget, dtype=torch.int32))


@pytest.mark.parametrize("longest", [2 ** 31, 2 ** 32, 2 ** 62])
def test_no_limit_on_the_length(longest):
    cache, w = make_cache(2, 64, [300, 20], 16, "affine", seed=14, extra_cols=1)
    c = fs().PagedKVCache(cache.k_quant, cache.v_quant, cache.block_table, cache.lengths, 16, longest)
    check(c, w, 100, 10, 2)


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (128, 64)])
def test_many_rows_move_in_rounds(fmt, d, page):
    """Rows enough that one CTA of four warps takes each, over several rounds of its pages."""
    lens = [150 + 7 * (i % 30) for i in range(75)]
    cache, w = make_cache(4, d, lens, page, fmt, seed=15)
    check(cache, w, 210, 20, 4)


@pytest.mark.parametrize("fmt", ["affine", "symmetric"])
@pytest.mark.parametrize("d,page", [(128, 16), (256, 32)])
def test_a_long_row_moves_in_rounds_of_a_cluster(fmt, d, page):
    cache, w = make_cache(1, d, [9000], page, fmt, seed=16)
    check(cache, w, 6000, 500, 16)
