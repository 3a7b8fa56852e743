"""The paged cache's host side (no GPU): sizes and refused shapes, and the
plain form that the GPU tests compare with, checked against torch."""
import ctypes

import numpy as np
import pytest
import torch

import ditch_amd
import pages_ref as ref
from ditch_amd import abi
from ditch_amd.hip import Device


def _pages(**over):
    a = dict(codes=1 << 20, codes_bytes=1 << 60, scales=1 << 20, scales_bytes=1 << 60, kind="int8", layers=2,
             n_pages=10, page_tokens=64, kv_heads=4, head_dim=128, v_head_dim=128)
    a.update(over)
    kind = a.pop("kind")
    p = Device.kv_pages(a["codes"], a["codes_bytes"], a["scales"], a["scales_bytes"], "int8", a["layers"],
                        a["n_pages"], a["page_tokens"], a["kv_heads"], a["head_dim"], a["v_head_dim"])
    p.kind = abi.KV_KIND.get(kind, kind)
    return p


def _bytes(p):
    lib = ditch_amd.load_library()
    return lib.ditch_hip_kv_pages_codes_bytes(ctypes.byref(p)), lib.ditch_hip_kv_pages_scales_bytes(ctypes.byref(p))


@pytest.mark.parametrize("hd,vd,width", [(128, 128, 256), (64, 64, 128), (80, 80, 256), (1, 1, 128), (192, 128, 320),
                                         (256, 256, 512)])
def test_pool_sizes(hd, vd, width):
    p = _pages(head_dim=hd, v_head_dim=vd)
    assert _bytes(p) == (2 * 10 * 4 * 64 * width, 2 * 10 * 4 * 8)


def test_pool_sizes_past_32_bits():
    assert _bytes(_pages(layers=60, n_pages=100000, kv_heads=8)) == (60 * 100000 * 8 * 64 * 256, 60 * 100000 * 8 * 8)


@pytest.mark.parametrize("over", [dict(kind=7), dict(layers=0), dict(n_pages=0), dict(page_tokens=16),
                                  dict(page_tokens=48), dict(kv_heads=0), dict(head_dim=0), dict(v_head_dim=0),
                                  dict(head_dim=257), dict(n_pages=1 << 31)])
def test_refused_shapes_have_no_size(over):
    assert _bytes(_pages(**over)) == (0, 0)
    lib = ditch_amd.load_library()
    assert lib.ditch_hip_kv_pages_codes_bytes(None) == 0
    batch = Device.kv_batch(1, 4, 1, 1, 1, 1, 1, 64)
    assert lib.ditch_hip_kv_pages_attention_workspace(ctypes.byref(_pages(**over)), ctypes.byref(batch), 8, abi.F32, 0,
                                                      0) == 0


def test_null_contexts_fail():
    lib = ditch_amd.load_library()
    assert lib.ditch_hip_kv_pages_append_device(None, None, 0, None, 0, None, None, None, None, None, 0,
                                                None) == abi.INVALID_ARGUMENT
    assert lib.ditch_hip_kv_pages_read_device(None, None, 0, None, 0, None, None, None) == abi.INVALID_ARGUMENT
    assert lib.ditch_hip_kv_pages_attention_device(None, None, 0, None, 0, None, None, 0, 1.0, 0, 0, None, 0,
                                                   None) == abi.INVALID_ARGUMENT
    assert lib.ditch_hip_kv_pages_fork_device(None, None, None, None, None, 0, None, None, None, 0, 0,
                                              None) == abi.INVALID_ARGUMENT
    assert lib.ditch_hip_beam_select_device(None, None, None, None, None, None, 0, 0, 0, 0, None, 0,
                                            None) == abi.INVALID_ARGUMENT


@pytest.mark.parametrize("prompts,beams,vocab,k", [(1, 0, 10, 1), (1, 65, 10, 1), (1, 2, 0, 1), (1, 2, 10, 0),
                                                   (1, 2, 300, 129), (1, 2, 10, 21), (1 << 17, 1, 10, 1)])
def test_refused_beam_shapes_have_no_workspace(prompts, beams, vocab, k):
    lib = ditch_amd.load_library()
    assert lib.ditch_hip_beam_select_workspace(prompts, beams, vocab, k) == 0
    assert lib.ditch_hip_beam_select_workspace(2, 4, 1000, 8) > 0


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ditch_hip.h"\nint main(void) { printf('
                   '"%zu %zu %zu %zu %zu %zu %zu", sizeof(ditch_kv_pages), offsetof(ditch_kv_pages, v_head_dim), '
                   'sizeof(ditch_kv_batch), offsetof(ditch_kv_batch, max_len), sizeof(ditch_kv_rows), '
                   'sizeof(ditch_kv_rope), offsetof(ditch_kv_rope, style)); return 0; }')
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-I", os.path.dirname(ditch_amd.HEADER_PATH), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(abi.KvPages), abi.KvPages.v_head_dim.offset, ctypes.sizeof(abi.KvBatch),
                   abi.KvBatch.max_len.offset, ctypes.sizeof(abi.KvRows), ctypes.sizeof(abi.KvRope),
                   abi.KvRope.style.offset]


# the plain form itself

def test_e4m3_codes_are_torchs():
    want = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    got = ref.decode_table("e4m3")
    np.testing.assert_array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    x = np.concatenate([np.random.default_rng(1).standard_normal(20000) * s for s in (0.003, 0.05, 1, 100)])
    x = np.concatenate([x, got[~np.isnan(got)], [0.0, 2.0 ** -10, 3 * 2.0 ** -11, 17.0, 19.0, 447.9, 1e4]])
    x = x.astype(np.float32)
    want = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(ref.decode_table("e4m3")[ref.encode(x.astype(np.float64), "e4m3")],
                                  ref.decode_table("e4m3")[want])


@pytest.mark.parametrize("page,hd,vd", [(32, 64, 64), (64, 128, 128), (128, 192, 128), (256, 256, 256), (64, 80, 80)])
def test_every_byte_of_a_page_has_one_place(page, hd, vd):
    k, v = ref.offsets(page, hd, vd)
    every = np.concatenate([k.ravel(), v.ravel()])
    assert np.array_equal(np.sort(every), np.arange(page * (ref.padded(hd) + ref.padded(vd))))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_appending_in_pieces_stays_within_half_a_step_a_rounding(kind):
    """Each value is off by at most half a step of the scale it was rounded at, once and once more for every
    larger scale after it."""
    rng = np.random.default_rng(3)
    pool = ref.Pool(kind, 1, 3, 32, 1, 64)
    table = np.array([[2, 0]])
    x = rng.standard_normal((40, 1, 64)).astype(np.float32) * np.linspace(0.5, 4, 40, dtype=np.float32)[:, None, None]
    for lo, hi in ((0, 3), (3, 30), (30, 40)):
        ref.append(pool, 0, table, np.array([0, hi - lo]), np.array([lo]), x[lo:hi], x[lo:hi])
    k, v = ref.sequence(pool, 0, table[0], 40)
    step = 1 / 127 if kind == "int8" else 2.0 ** -3
    bound = (np.abs(x[:, 0]).max() * step if kind == "int8" else np.abs(x[:, 0]) * step + 4 * 2.0 ** -9 / 448) * 1.01
    assert (np.abs(k[0] - x[:, 0]) <= bound).all() and np.array_equal(k, v)


def test_fork_keeps_every_page():
    rng = np.random.default_rng(5)
    for _ in range(200):
        beams, groups, page = int(rng.integers(1, 9)), int(rng.integers(1, 4)), 32
        cols, n = 5, groups * beams
        ids = rng.permutation(n * cols + n)
        table, spare = ids[:n * cols].reshape(n, cols).astype(np.int32), ids[n * cols:].astype(np.int32)
        lens = rng.integers(0, cols * page + 1, groups)
        parents = rng.integers(-1, beams + 1, n)
        t, s, copies = ref.fork(table, parents, spare, lens, page, beams)
        for g in range(groups):
            full = int(lens[g]) // page
            if int(lens[g]) % page and full < cols:
                was = list(table[g * beams:(g + 1) * beams, full]) + list(spare[g * beams:(g + 1) * beams])
                now = list(t[g * beams:(g + 1) * beams, full]) + list(s[g * beams:(g + 1) * beams])
                assert sorted(was) == sorted(now)
