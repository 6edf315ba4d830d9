"""How exactly the attention over the 4-bit cache works ahead of storing a row in 16 bits.

A stored element is the 64-bit one rounded, unless that lies nearer to the border between two numbers of the type than the kernel is off.
Scores from exact integer sums are off by a few 2^-24 of themselves, ex2 by 2^-22, weights and their scales held in two fp16 terms by
2^-22: about 3e-7 a key, independent, so that a result is 3e-7 to 1e-6 of itself off.  Numbers of a type lie eps / 2 to eps of themselves
apart, so one element in 2 * 1e-6 / (eps / 2) comes out on the other side: bf16 5e-4, fp16 4e-3.  The tests allow four times that.  Weights
rounded to 11 bits (2^-11 / sqrt(3) each, three times) would bring 4e-2 in bf16.
"""
import math

import pytest
import torch

from test_gpu_kv4 import Attention

pytestmark = pytest.mark.gpu


def exact(a, b):
    """Rows of sequence b in 64 bits, [count, hq * hd]."""
    hq, hkv, hd = a.dims
    n, count = a.lens[b], a.counts[b]
    at = slice(int(a.start[b]), int(a.start[b]) + count)
    q = a.q[at, :hq * hd].double().view(count, hkv, hq // hkv, hd)
    x = torch.einsum("thgd,shd->hgts", q, a.k[b].double()) * hd ** -0.5
    x = x.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(n - count, n, device="cuda")[:, None], -math.inf)
    return at, torch.einsum("hgts,shd->thgd", torch.softmax(x, -1), a.v[b].double()).reshape(count, hq * hd)


@pytest.mark.parametrize("hq,hkv,hd,group", [(4, 1, 256, 64), (8, 4, 256, 128), (32, 16, 128, 128), (8, 4, 128, 64), (12, 4, 64, 64)])
@pytest.mark.parametrize("typ,share", [(torch.bfloat16, 2e-3), (torch.float16, 1.6e-2)])
def test_16_bit_rows_are_rounded_once(pkg, hq, hkv, hd, group, typ, share):
    for lens, counts in (([777, 300, 1300, 2500, 64], [1] * 5), ([900, 5000, 333], [3, 2, 3])):
        a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hq + hd)
        a()
        other = total = 0
        for b in range(len(lens)):
            at, want = exact(a, b)
            other += (a.out[at, :want.shape[1]] != want.to(typ)).sum().item()
            total += want.numel()
        assert other <= share * total, (other, total)
