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
