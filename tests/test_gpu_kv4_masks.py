"""Masks at the ends of their range, and rows that see nothing."""
import pytest
import torch

from test_gpu_kv4 import TYPES, Attention, stream

pytestmark = pytest.mark.gpu

HEADS = [(4, 1, 256, 64), (8, 4, 256, 128), (8, 4, 128, 64), (5, 1, 64, 64)]


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens,counts", [([3, 70, 257], [7, 2, 260]), ([700, 300, 900], [720, 310, 5])])
def test_windows_as_large_as_their_type(pkg, hq, hkv, hd, group, typ, lens, counts):
    """Sequences with more query tokens than positions, under windows that hide nothing."""
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd + hq)
    for window in (2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, max(lens), max(lens) - 1):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        a.check(window)


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens,counts", [([3, 70, 0], [7, 72, 3]), ([700, 300, 900], [720, 310, 5])])
def test_rows_that_see_nothing_are_zero_whatever_they_hold(pkg, hq, hkv, hd, group, typ, lens, counts):
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd + hq)
    for b, (n, count) in enumerate(zip(lens, counts)):
        rows = a.q[int(a.start[b]):int(a.start[b]) + max(0, count - n)]
        rows[0::2, 5], rows[1::2, hd - 1] = float("nan"), float("inf")
    for window in (0, 40):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        for b, (n, count) in enumerate(zip(lens, counts)):
            rows = a.out[int(a.start[b]):int(a.start[b]) + count, :hq * hd]
            assert (rows[:max(0, count - n)] == 0).all(), (b, window)
            assert torch.isfinite(rows).all() and (rows[max(0, count - n):] != 0).any(-1).all()


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
def test_scales_as_small_as_their_type(pkg, hq, hkv, hd, group, typ):
    """All weights of a row are the same, those of masked keys zero; rows of zeros among the queries."""
    a = Attention(pkg, [700, 300, 900], [700, 300, 5], hq, hkv, hd, group, typ, seed=hd + hq)
    a.q[10:400:3] = 0
    for scale in (1e-12, 1e-25, 1e-40):
        for window in (0, 40):
            a.out.fill_(7.0)
            a(window=window, scale=scale)
            assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
            a.check(window, scale)


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,counts", [([1500, 600, 900], [1, 1, 1]), ([1500, 600, 900], [600, 200, 700])])
def test_a_bad_page_leaves_its_whole_sequence(pkg, hq, hkv, hd, group, typ, lens, counts):
    """Rows that do not reach the page themselves too, however rows share CTAs; pages ahead of every row's window are nobody's."""
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd)
    table = a.cache.table.clone()
    for page in (0, 3, 5):
        a.cache.table[0, page] = -1 if page else a.cache.n
        a.out.fill_(7.0)
        a()
        with pytest.raises(pkg.StatusError) as e:
            pkg.ops.device_status(a.status.data_ptr(), stream())
        assert e.value.code == pkg.INVALID_ARGUMENT
        assert (a.out[:counts[0]] == 7.0).all()
        a.check(skip=(0,))
        a.cache.table.copy_(table)
    a.cache.table[0, 0], a.cache.table[0, 1] = -1, 2 ** 31 - 1      # positions below 512; the first row's window begins behind 600
    a.out.fill_(7.0)
    a(window=200)
    assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
    a.check(200)
