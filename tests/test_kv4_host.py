"""Host side of the operators over a 4-bit cache and of the grouped int4 product: layouts, sizes, refusals.  No GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def refused(pkg, code, call, *args, **kw):
    with pytest.raises(pkg.StatusError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value
    return e.value.message


@pytest.mark.parametrize("n,k,group,offset", [(1, 2, 32, False), (16, 128, 128, True), (17, 130, 64, False), (33, 388, 32, True), (5, 254, 128, False)])
def test_grouped_image_element_by_element(pkg, n, k, group, offset):
    rng = np.random.Generator(np.random.PCG64(n * 1000 + k))
    q = rng.integers(0, 16, (n, k)).astype(np.uint8)
    groups = -(-k // group)
    scale, off = (rng.integers(0, 65536, (n, groups)).astype(np.uint16) for _ in range(2))
    img = pkg.ops.repack_w4_grouped(q[:, 0::2] | q[:, 1::2] << 4, scale, off if offset else None, group)
    per, blocks = 128 // group, -(-k // 128)
    size = 1024 + 32 * per * (2 if offset else 1)
    img = img.reshape(-(-n // 16), blocks, size)
    seen = np.zeros_like(img)
    for r in range(n):
        for j in range(k):
            c = j % 64
            at = j % 128 // 64 * 512 + (4 * (r % 8) + c % 16 // 4) * 16 + 4 * (2 * (c // 32) + c % 32 // 16) + c % 4
            byte = img[r // 16, j // 128, at]
            assert (byte >> 4 if r % 16 >= 8 else byte & 15) == q[r, j]
            seen[r // 16, j // 128, at] |= 0xF0 if r % 16 >= 8 else 0x0F
        for j in range(groups):
            at = 1024 + ((r % 8 * per + j % per) * 2 + r % 16 // 8) * 2
            for a, x in ((at, scale), (at + 32 * per, off if offset else None)):
                if x is not None:
                    assert img[r // 16, j // per, a:a + 2].view(np.uint16)[0] == x[r, j]
                    seen[r // 16, j // per, a:a + 2] = 255
    assert not (img & ~seen).any()                         # rows and k past the end are zero


def test_page_bytes(pkg):
    assert pkg.Kv4Cache.page_bytes(4, 256, 64) == 512 * 4 * (128 + 16)
    assert pkg.Kv4Cache.page_bytes(1, 64, 64) == 512 * (32 + 4)
    assert pkg.Kv4Cache.page_bytes(16, 128, 128) == 512 * 16 * (64 + 4)
    for hkv, hd, group, code in [(0, 128, 64, 3), (1, 96, 32, 12), (1, 64, 128, 12), (1, 128, 32, 12), (2000, 64, 64, 3)]:
        refused(pkg, code, pkg.Kv4Cache.page_bytes, hkv, hd, group)


def test_cache_layout_gives_every_element_a_nibble_of_its_own(tmp_path):
    exe = str(tmp_path / "kv4_layout")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "litert-lm_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "kv4_layout_test.cc"), "-o", exe], check=True)
    subprocess.run([exe], check=True)


P = 1 << 20      # an aligned address that is never looked at: the arguments are refused before


def test_gemv_refusals(pkg):
    ok = dict(w_dev=P, x_dev=P, y_dev=P, n=64, k=256, group=64)
    g = pkg.ops.gemv_w4_grouped
    for bad, code in [(dict(w_dev=0), 3), (dict(x_dev=0), 3), (dict(y_dev=0), 3), (dict(n=0), 3), (dict(k=0), 3), (dict(k=255), 3), (dict(k=-2), 3), (dict(group=16), 12), (dict(group=0), 12),
                      (dict(ncols=0), 3), (dict(ncols=9), 3), (dict(ncols=2, ldx=255), 3), (dict(ncols=2, ldy=63), 3), (dict(scale_type=0), 3), (dict(x_type=3), 3), (dict(y_type=-1), 3),
                      (dict(w_dev=P + 8), 3), (dict(x_dev=P + 2), 3), (dict(y_dev=P + 1, y_type=1), 3), (dict(n=1 << 31), 3)]:
        refused(pkg, code, g, **{**ok, **bad})
    with pytest.raises(pkg.StatusError):
        pkg.ops.repack_w4_grouped(np.zeros((4, 32), np.uint8), np.zeros((4, 2), np.float16), None, 64)     # one group of 64, two given
    with pytest.raises(pkg.StatusError):
        pkg.ops.repack_w4_grouped(np.zeros((4, 32), np.uint8), np.zeros((4, 4), np.float16), None, 16)


def test_rows_refusals(pkg):
    ok = dict(qkv_dev=P, type=1, qkv_stride=768, tokens=3, hq=4, hkv=1, hd=128, rot=128, q_gain_dev=P, k_gain_dev=P, eps=1e-6, cos_dev=P, sin_dev=P, rope_rows=10, pos_dev=P, q_out_dev=P, q_stride=512)
    f = lambda **kw: pkg.ops.qk_norm_rope(**{**ok, "k_out_dev": P, "k_stride": 128, **kw})          # noqa: E731
    for bad, code in [(dict(qkv_dev=0), 3), (dict(type=4), 3), (dict(qkv_stride=767), 3), (dict(tokens=-1), 3), (dict(hq=0), 3), (dict(hkv=0), 3), (dict(hd=96), 12), (dict(rot=144), 3), (dict(rot=24), 3),
                      (dict(rot=-8), 3), (dict(eps=-1.0), 3), (dict(eps=float("nan")), 3), (dict(cos_dev=0), 3), (dict(sin_dev=0), 3), (dict(rope_rows=0), 3), (dict(pos_dev=0), 3), (dict(q_out_dev=0), 3),
                      (dict(q_stride=511), 3), (dict(k_out_dev=0), 3), (dict(k_stride=127), 3), (dict(qkv_dev=P + 1), 3), (dict(q_gain_dev=P + 2), 3), (dict(status_dev=P + 2), 3)]:
        refused(pkg, code, f, **bad)
    cache = pkg.Kv4Cache(P, 8, P, 4, 2, 1, 128, 64)
    f = lambda **kw: pkg.ops.qk_norm_rope_append_kv4(**{**ok, "cache": cache, "seq_dev": P, **kw})   # noqa: E731
    for bad, code in [(dict(hd=64, qkv_stride=4096), 3), (dict(hkv=2, qkv_stride=4096), 3), (dict(seq_dev=0), 3), (dict(seq_dev=P + 1), 3), (dict(cos_dev=0), 3)]:
        refused(pkg, code, f, **bad)


def caches(pkg):
    good = dict(pages_dev=P, num_pages=8, page_table_dev=P, table_stride=4, batch=2, hkv=1, hd=128, group=64)
    for bad, code in [(dict(pages_dev=0), 3), (dict(pages_dev=P + 8), 3), (dict(num_pages=0), 3), (dict(num_pages=1 << 31), 3), (dict(page_table_dev=0), 3), (dict(page_table_dev=P + 2), 3),
                      (dict(table_stride=0), 3), (dict(table_stride=1 << 23), 3), (dict(batch=0), 3), (dict(batch=65536), 3), (dict(hkv=0), 3), (dict(hd=32), 12), (dict(group=32), 12), (dict(hd=64, group=128), 12)]:
        yield pkg.Kv4Cache(**{**good, **bad}), code


def test_cache_and_attention_refusals(pkg):
    att = dict(q_dev=P, q_type=0, q_stride=512, kv_len_dev=P, q_start_dev=P, tokens=2, max_q=1, max_kv=1024, hq=4, out_dev=P, out_stride=512, workspace_dev=P, workspace_bytes=1 << 30)
    for cache, code in caches(pkg):
        refused(pkg, code, pkg.ops.attention_kv4, cache, **att)
        refused(pkg, code, pkg.ops.kv4_read, cache, P, P, 1, 0, P, P)
    cache = pkg.Kv4Cache(P, 8, P, 4, 2, 1, 128, 64)
    for bad in [dict(q_dev=0), dict(q_type=3), dict(q_stride=511), dict(out_stride=511), dict(kv_len_dev=0), dict(tokens=-1), dict(max_q=0), dict(max_kv=-1), dict(max_kv=1025), dict(hq=0), dict(out_dev=0),
                dict(q_dev=P + 2), dict(out_dev=P + 2), dict(workspace_dev=P + 8), dict(q_start_dev=0, tokens=3), dict(q_start_dev=0, max_q=2), dict(q_start_dev=P + 2), dict(status_dev=P + 1)]:
        refused(pkg, 3, pkg.ops.attention_kv4, cache, **{**att, **bad})
    refused(pkg, 3, pkg.ops.attention_kv4, pkg.Kv4Cache(P, 8, P, 4, 2, 3, 128, 64), **att)                # four query heads on three
    cache.desc.struct_size = 8
    refused(pkg, 3, pkg.ops.attention_kv4, cache, **att)
    cache = pkg.Kv4Cache(P, 8, P, 4, 2, 1, 128, 64)
    for bad in [(P, 0, 1, 0, P, P), (P, P, -1, 0, P, P), (P, P, 1, 9, P, P), (P, P, 1, 0, 0, 0), (P, P, 1, 0, P + 2, P), (0, P, 3, 0, P, P), (P, P + 1, 1, 0, P, P)]:
        refused(pkg, 3, pkg.ops.kv4_read, cache, *bad)
    refused(pkg, 3, pkg.ops.device_status, 0)
    for bad in [(0, 1, 128, 4, 1, 100), (1, 3, 128, 4, 1, 100), (1, 1, 128, 4, 0, 100), (1, 1, 128, 4, 1, -1), (1, 1, 128, 4, 1 << 29, 100)]:
        refused(pkg, 3, pkg.ops.attention_kv4_workspace, *bad)
    refused(pkg, 12, pkg.ops.attention_kv4_workspace, 1, 1, 80, 4, 1, 100)


def test_error_strings_may_be_declined(pkg):
    lib = pkg.load_library()
    assert lib.B200LmOps_DeviceStatus(0, None, None, None, None) == 3
    n = C.c_int64(7)
    assert lib.B200LmOps_Kv4PageBytes(1, 96, 64, C.byref(n), None) == 12 and n.value == 7


def test_arguments_of_the_extension_module(pkg):
    """What is not a whole number, or does not fit its type, is refused before the library sees it."""
    ok = dict(w_dev=P, x_dev=P, y_dev=P, n=64, k=256, group=64)
    with pytest.raises(TypeError):
        pkg.ops.gemv_w4_grouped(**{**ok, "w_dev": 1.5})
    with pytest.raises(TypeError):
        pkg.ops.gemv_w4_grouped(**{**ok, "x_dev": None})
    with pytest.raises(OverflowError):
        pkg.ops.gemv_w4_grouped(**{**ok, "group": 1 << 40})
    with pytest.raises(OverflowError):
        pkg.ops.gemv_w4_grouped(**{**ok, "n": 1 << 70})
    assert "null" in refused(pkg, 3, pkg.ops.gemv_w4_grouped, **{**ok, "w_dev": np.int64(0)})
