"""CPU checks of the cache operators' C boundary: struct layouts, and refusals that the
entry points make before any CUDA call."""

from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parents[1] / "include" / "flashspec_b200.h"


def layouts():
    from flashspec_b200 import _lib

    return {"FsEvictArgs": _lib.FsEvictArgs, "FsLatentAppendArgs": _lib.FsLatentAppendArgs,
            "FsLatentArgs": _lib.FsLatentArgs, "FsLatentPrefillArgs": _lib.FsLatentPrefillArgs}


def test_struct_layouts_match_c(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for name, cls in layouts().items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True)
               .stdout.splitlines())
    for name, cls in layouts().items():
        assert int(got[name]) == C.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"


def decode_args():
    from flashspec_b200 import _lib

    a = _lib.FsDecodeArgs()
    a.layout = _lib.FS_LAYOUT_PAGED
    a.q = a.k_values = a.v_values = a.k_scale = a.v_scale = a.k_zero = a.v_zero = 4096
    a.block_table = a.lengths = a.out = 4096
    a.batch, a.q_heads, a.kv_heads, a.head_dim, a.block_size = 2, 8, 8, 128, 16
    a.num_blocks, a.table_cols, a.max_seq_len = 64, 4, 64
    a.sm_scale = 128 ** -0.5
    return a


@pytest.mark.parametrize("change,status", [
    (dict(layout=0), 1), (dict(q_heads=7), 1), (dict(out=None), 1), (dict(lengths=None), 1), (dict(q_heads=72), 2),
    (dict(head_dim=96), 2), (dict(k_values=4100), 5), (dict(q_dtype=2), 2)])
def test_weighted_decode_refuses(change, status):
    from flashspec_b200 import _lib

    a = decode_args()
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().fs_paged_decode_weights(C.byref(a), 4096, None) == status


def test_weighted_decode_refuses_missing_or_unaligned_weights():
    from flashspec_b200 import _lib

    lib = _lib.load()
    assert lib.fs_paged_decode_weights(C.byref(decode_args()), None, None) == 1
    assert lib.fs_paged_decode_weights(None, 4096, None) == 1
    assert lib.fs_paged_decode_weights(C.byref(decode_args()), 4097, None) == 5
    assert lib.fs_paged_decode_weights_workspace_size(C.byref(decode_args()), None, None) == 1


def evict_args():
    from flashspec_b200 import _lib

    a = _lib.FsEvictArgs()
    a.batch, a.kv_heads, a.head_dim, a.page_size, a.table_cols, a.max_seq_len = 2, 4, 128, 16, 8, 128
    a.budget, a.recent, a.sinks, a.num_pages = 32, 8, 4, 20
    a.block_table = a.lengths = a.k_values = a.k_scale = a.k_zero = a.v_zero = 4096
    a.v_values = a.v_scale = 16384
    a.weights = a.weights_out = a.kept = 4096
    a.new_lengths = 8192
    return a


@pytest.mark.parametrize("change,status", [
    (dict(budget=0), 1), (dict(recent=30), 1), (dict(sinks=-1), 1), (dict(kv_format=2), 1), (dict(k_zero=None), 1),
    (dict(kept=None), 1), (dict(new_lengths=4096), 1), (dict(page_size=65), 2), (dict(head_dim=72), 2),
    (dict(page_size=64, head_dim=256), 2), (dict(k_values=4104), 5), (dict(weights=4098), 5),
    (dict(table_cols=1 << 28), 2), (dict(num_pages=0), 1), (dict(table_cols=1 << 26), 2), (dict(budget=1 << 30), 2),
    (dict(v_values=4096), 1), (dict(v_scale=4096), 1), (dict(num_pages=1 << 31), 2)])
def test_evict_refuses(change, status):
    from flashspec_b200 import _lib

    a, n = evict_args(), C.c_size_t(0)
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().fs_evict_tokens(C.byref(a), None) == status
    assert _lib.load().fs_evict_workspace_size(C.byref(a), C.byref(n)) == status


def test_evict_workspace():
    from flashspec_b200 import _lib

    lib, a, n = _lib.load(), evict_args(), C.c_size_t(0)
    assert lib.fs_evict_workspace_size(C.byref(a), C.byref(n)) == 0 and n.value == 0
    a.table_cols, a.max_seq_len = 393216 // 16, 393216
    assert lib.fs_evict_workspace_size(C.byref(a), C.byref(n)) == 0 and n.value == 0
    a.table_cols, a.max_seq_len = 393216 // 16 + 16, 393216 + 256
    assert lib.fs_evict_workspace_size(C.byref(a), C.byref(n)) == 0 and n.value == 2 * 4 * (393216 + 256) * 4
    assert lib.fs_evict_tokens(C.byref(a), None) == 4  # FS_ERR_WORKSPACE


def latent_args():
    from flashspec_b200 import _lib

    a = _lib.FsLatentArgs()
    a.q = a.q_rope = a.out = a.values = a.scale = a.ropes = a.block_table = a.lengths = 4096
    a.batch, a.tokens, a.heads, a.latent_dim, a.rope_dim, a.page_size = 2, 1, 16, 512, 64, 64
    a.table_cols, a.max_seq_len, a.num_pages, a.sm_scale = 4, 256, 10, 0.1
    return a


@pytest.mark.parametrize("change,status", [
    (dict(q=None), 1), (dict(lengths=None), 1), (dict(tokens=0), 1), (dict(heads=0), 1), (dict(num_pages=0), 1),
    (dict(dtype=2), 2), (dict(latent_dim=192), 2), (dict(rope_dim=16), 2), (dict(page_size=48), 2),
    (dict(batch=4097), 2), (dict(tokens=1 << 17), 2), (dict(table_cols=1 << 24), 2), (dict(values=4104), 5),
    (dict(num_pages=1 << 25), 2),
    (dict(q=4098), 5), (dict(scale=4097), 5)])
def test_latent_attention_refuses(change, status):
    from flashspec_b200 import _lib

    a, n = latent_args(), C.c_size_t(0)
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().fs_latent_attention(C.byref(a), None) == status
    assert _lib.load().fs_latent_workspace_size(C.byref(a), C.byref(n)) == status


@pytest.mark.parametrize("change,status", [
    (dict(latent=None), 1), (dict(new_lengths=None), 1), (dict(new_lengths=4096), 1), (dict(tokens=0), 1),
    (dict(dtype=2), 2), (dict(latent_dim=64), 2), (dict(held=4097), 5)])
def test_latent_append_refuses(change, status):
    from flashspec_b200 import _lib

    a = _lib.FsLatentAppendArgs()
    a.latent = a.rope = a.values = a.scale = a.ropes = a.block_table = a.lengths = 4096
    a.new_lengths = 8192
    a.batch, a.tokens, a.latent_dim, a.rope_dim, a.page_size, a.table_cols, a.num_pages = 1, 1, 512, 64, 64, 1, 1
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().fs_latent_append(C.byref(a), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(q=None), 1), (dict(kv=None), 1), (dict(q_offsets=None), 1), (dict(batch=0), 1), (dict(heads=0), 1),
    (dict(q_rows=-1), 1), (dict(dtype=2), 2), (dict(nope_dim=96), 2), (dict(rope_dim=128), 2), (dict(value_dim=32), 2),
    (dict(k_rope=4098), 5), (dict(out=4104), 5), (dict(k_rows=1 << 30), 2), (dict(q_rows=0), 0)])
def test_latent_prefill_refuses(change, status):
    from flashspec_b200 import _lib

    a = _lib.FsLatentPrefillArgs()
    a.q = a.kv = a.k_rope = a.out = a.q_offsets = a.k_offsets = 4096
    a.q_rows = a.k_rows = 10
    a.batch, a.heads, a.nope_dim, a.rope_dim, a.value_dim = 1, 2, 128, 64, 128
    for k, v in change.items():
        setattr(a, k, v)
    assert _lib.load().fs_latent_prefill(C.byref(a), None) == status


def test_pool_whose_parts_differ_in_size_is_refused():
    import torch
    from flashspec_b200.evict import _check_pool

    pages, hkv, page, d = 5, 2, 16, 8
    for sym in (False, True):
        n = pages * hkv * (page if sym else 1)
        parts = [torch.zeros(pages * hkv * page * d, dtype=torch.int8)] * 2 + [torch.zeros(n)] * 2
        parts += [] if sym else [torch.zeros(n, dtype=torch.int16)] * 2
        _check_pool(parts, pages, hkv, page, d, sym)
        for i in range(len(parts)):
            short = list(parts)
            short[i] = parts[i][:-1]
            with pytest.raises(ValueError):
                _check_pool(short, pages, hkv, page, d, sym)


def test_overlap():
    import torch
    from flashspec_b200.latent import _overlap

    x = torch.zeros(4, 6)
    assert _overlap(x, x) and _overlap(x, x[3:]) and _overlap(x[:, 5:], x[1:2]) and _overlap(x[:2], x[1:])
    assert not _overlap(x[:2], x[2:]) and not _overlap(x, torch.zeros(4, 6)) and not _overlap(x[:0], x)
    assert not _overlap(x[:2, :3], x[2:]) and not _overlap(x[2:], x[:2, 3:])


def test_a_decode_stage_is_released_behind_its_last_read():
    """The decode's consumer hands a ring stage back to the copies; whatever it reads of the stage
    (K, V, the token scales) has to be read before that, or the next page's bytes may be there."""
    src = (HEADER.parents[1] / "flashspec_b200" / "csrc" / "decode.cu").read_text()
    body = src[src.index("void consume_page("):]
    body = body[:body.index("\n}\n")]
    release = body.index("mbar_arrive(empty_bar)")
    reads = [body.rindex(x) for x in ("sbase + off.k", "sbase + off.v", "si.tok +")]
    assert body.count("mbar_arrive(") == 1 and max(reads) < release


@pytest.mark.parametrize("offset,status", [(4, 5), (8, 5), (16, 5), (128, 5)])
def test_evict_refuses_an_unaligned_workspace(offset, status):
    """The keys of a long row are read and written 16 bytes at a time."""
    from flashspec_b200 import _lib

    lib, a, n = _lib.load(), evict_args(), C.c_size_t(0)
    a.table_cols, a.max_seq_len = 400000 // 16, 400000
    assert lib.fs_evict_workspace_size(C.byref(a), C.byref(n)) == 0 and n.value > 0
    a.workspace, a.workspace_bytes = 1 << 20 | offset, n.value
    assert lib.fs_evict_tokens(C.byref(a), None) == status


def test_longest_length_beyond_32_bits():
    """max_seq_len may say "no limit"; the C field has 32 bits and ctypes would drop the others."""
    from flashspec_b200.attention import _seq_cap

    assert [_seq_cap(n, 16, 10) for n in (0, 1000, 2 ** 31 - 1)] == [0, 1000, 2 ** 31 - 1]
    assert [_seq_cap(n, 16, 10) for n in (2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 62)] == [160] * 4
    assert _seq_cap(2 ** 40, 128, 2 ** 30) == 2 ** 31 - 1


def test_status_word():
    """The kernels write to it, so a host address or a short element must not get there."""
    import torch
    from flashspec_b200.quant import status_word

    cpu, gpu = torch.device("cpu"), torch.device("cuda", 0)
    assert status_word(None, gpu) is None
    for dtype in (torch.int32, torch.int64, torch.uint32):
        t = torch.zeros(2, dtype=dtype)
        assert status_word(t, cpu) == t.data_ptr()
        with pytest.raises(RuntimeError):
            status_word(t, gpu)
    for bad in (torch.zeros(4, dtype=torch.int8), torch.zeros(1), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError):
            status_word(bad, cpu)
    with pytest.raises(RuntimeError):
        status_word(0, cpu)


class Ring:
    """mbarriers of a ring of stages, as the hardware counts them: one completion a tile, in any
    order over the stages; wait(parity) passes when the phase of that parity has completed."""

    def __init__(self, stages):
        self.stages, self.done = stages, [0] * stages

    def complete(self, tile):
        assert self.done[tile % self.stages] == tile // self.stages  # in turn on one stage
        self.done[tile % self.stages] += 1

    def passes(self, tile):
        return (self.done[tile % self.stages] & 1) != ((tile // self.stages) & 1)


@pytest.mark.parametrize("stages", [2, 3])
def test_giving_up_waits_for_the_copies_in_flight(stages):
    """The latent attention gives up at tile `used` with tiles [used, issued) on their way (fewer
    than the stages): its last waits pass for each of them when it has come, and not before."""
    for used in range(4 * stages):
        for ahead in range(1, stages):
            for missing in range(used, used + ahead):
                ring = Ring(stages)
                for tile in range(used + ahead):
                    if tile != missing:
                        ring.complete(tile)
                for tile in range(used, used + ahead):
                    assert ring.passes(tile) == (tile != missing)
                ring.complete(missing)
                assert all(ring.passes(tile) for tile in range(used, used + ahead))
    src = (HEADER.parents[1] / "flashspec_b200" / "csrc" / "latent.cu").read_text()
    end = src[src.index("if (__syncthreads_or(here ? 0 : 1))"):]
    end = end[:end.index("return;")]
    assert "i = used; i != issued" in end and end.count("mbar_wait_bounded") == 1


def test_giving_up_in_a_prompt_waits_for_the_copies_in_flight():
    """The expanded attention keeps two K and two V tiles in flight at most: a tile is sent when the
    one two before it was consumed, so the last two sent are all that may be on their way."""
    for sent in range(1, 12):
        for arrived in range(max(0, sent - 2), sent + 1):
            ring = Ring(2)
            for tile in range(arrived):
                ring.complete(tile)
            waits = range(max(0, sent - 2), sent)
            assert [ring.passes(t) for t in waits] == [t < arrived for t in waits]
            for tile in range(arrived, sent):
                ring.complete(tile)
            assert all(ring.passes(t) for t in waits)
    src = (HEADER.parents[1] / "flashspec_b200" / "csrc" / "latent_prefill.cu").read_text()
    end = src[src.index("if (s_abort != 0) {"):src.index("tmem_dealloc(tmem")]
    assert all(x in end for x in ("bars.q_full", "bars.k_full", "bars.v_full", "mma_commit(smem_u32(&bars.drained))"))


def test_every_arrival_of_a_prompt_is_waited_for():
    """The commits that free the stages of the expanded attention, against the waits for them: K of
    tile i is free behind the scores of tile i, V behind its P V, and both are waited for by the
    copies of tile i + 2 alone.  An arrival that nobody waits for could reach a CTA that has ended."""
    src = (HEADER.parents[1] / "flashspec_b200" / "csrc" / "latent_prefill.cu").read_text()
    for line in ("if (tiles > 2) mma_commit(smem_u32(&bars.k_empty[0]))",
                 "if (j + 2 < tiles) mma_commit(smem_u32(&bars.v_empty[st]))",
                 "if (j + 3 < tiles) mma_commit(smem_u32(&bars.k_empty[st ^ 1]))",
                 "if (j >= 2 && !pre_wait(&bars.k_empty[st]", "if (j >= 2 && !pre_wait(&bars.v_empty[st]"):
        assert src.count(line) == 1, line
    assert src.count("mma_commit(smem_u32(&bars.k_empty") == 2 and src.count("mma_commit(smem_u32(&bars.v_empty") == 1
    for tiles in range(1, 12):
        k_free = ([0] if tiles > 2 else []) + [j + 1 for j in range(tiles) if j + 3 < tiles]
        v_free = [j for j in range(tiles) if j + 2 < tiles]
        assert k_free == v_free == [j - 2 for j in range(2, tiles)]
