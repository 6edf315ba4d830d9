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

from test_gpu_kv4 import TYPES, U, Attention, gen, put, rounded

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


@pytest.mark.parametrize("hq,hkv,hd,group", [(8, 4, 256, 64), (8, 4, 256, 128), (8, 4, 128, 64), (16, 2, 128, 128)])
@pytest.mark.parametrize("how", ["one dim", "offsets"])
def test_large_scores_of_chunks(pkg, hq, hkv, hd, group, how):
    """Chunks of bf16 rows where one dim carries a score of 50, or where all keys lie far from zero: a score that is off by a share of
    itself is off by percents of its key's weight.  Per row, as in test_gpu_kv4_chunks.py: storing costs 2^-8 |o|; ahead of that P is
    rounded once (2^-11 / sqrt(3) of itself), V once, and a score is off by 2^-20 sum |q k| scale (its sums and its exponent's)."""
    lens, counts = [900, 600, 2500], [600, 599, 200]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, torch.bfloat16, seed=hd + group)
    q = a.q[:, :hq * hd].view(-1, hq, hd)
    if how == "one dim":
        q[..., 0] = 6 * hd ** 0.5
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).cuda()
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    k, v = (torch.randn(len(seq), hkv, hd, device="cuda", generator=gen(s)) for s in (1, 2))
    if how == "one dim":
        k[..., 0] = 8 + 0.5 * k[..., 0]
    else:
        k += 40
    a.k, a.v = (x.split(lens) for x in put(pkg, a.cache, seq, pos, k, v))
    a()
    assert pkg.ops.device_status(a.status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    for b, (n, count) in enumerate(zip(lens, counts)):
        at = slice(int(a.start[b]), int(a.start[b]) + count)
        got = a.out[at, :hq * hd].double().view(count, hq, hd)
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - count, n, device="cuda")[:, None]
        for h in range(hq):
            qh, kh, vh = q[at, h].double(), a.k[b][:, h // (hq // hkv)].double(), a.v[b][:, h // (hq // hkv)].double()
            p = torch.softmax((qh @ kh.T * hd ** -0.5).masked_fill(~seen, -math.inf), -1)
            o, p2 = p @ vh, p * p
            tau = 2.0 ** -11 * vh.abs().amax() / 3 ** 0.5
            sigma = torch.sqrt((2.0 ** -20 * (qh.abs() @ kh.abs().T).amax(-1) * hd ** -0.5) ** 2 + (2.0 ** -11) ** 2 / 3)
            gap = p2 @ vh.square().sum(-1) - 2 * ((p2 @ vh) * o).sum(-1) + p2.sum(-1) * o.square().sum(-1)
            inner = 6 * torch.sqrt(sigma ** 2 * gap.clamp(min=0) + hd * tau ** 2 * p2.sum(-1)) + 64 * U * vh.abs().amax() * hd ** 0.5
            err = (got[:, h] - o).norm(dim=-1)
            assert (err <= 2.0 ** -8 * (o.norm(dim=-1) + inner) + inner).all(), (b, h, (err / o.norm(dim=-1)).max().item())


@pytest.mark.parametrize("hq,hkv,hd,group", [(4, 1, 256, 64), (8, 4, 256, 128), (4, 2, 128, 64)])
@pytest.mark.parametrize("typ", [torch.float32, torch.float16])
@pytest.mark.parametrize("count", [1, 4])
def test_small_groups_beside_large_ones(pkg, hq, hkv, hd, group, typ, count):
    """Groups of V three million times smaller than their neighbours, some of which grow on the way: each is as exact as it would be alone.
    2^-22 for the terms of a weight, 2 * 2^-20 for the weights (scores of up to 16), 64 u for the sums, of the group's largest value."""
    lens = [700, 1500, 90]
    a = Attention(pkg, lens, [count] * 3, hq, hkv, hd, group, typ, seed=hd, tail=0)
    size = torch.full((max(lens), hd // group), 1e-3, device="cuda")
    size[:, 0] = 3000.0
    size[:, -1] = torch.where(torch.arange(max(lens), device="cuda") > 300, 10.0, 1e-4)
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).cuda()
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    k, v = (torch.randn(len(seq), hkv, hd, device="cuda", generator=gen(s)) for s in (1, 2))
    a.k, a.v = (x.split(lens) for x in put(pkg, a.cache, seq, pos, k, v * size[pos.long()].repeat_interleave(group, 1)[:, None]))
    a()
    for b in range(3):
        at, want = exact(a, b)
        err = (a.out[at, :hq * hd].double() - want).abs().view(count, hkv, -1, hd // group, group)
        want = want.view_as(err)
        top = a.v[b].double().view(lens[b], hkv, 1, hd // group, group).abs().amax((0, 4), keepdim=True)
        bound = (2.0 ** -22 + 2.0 ** -19 + 64 * U) * top
        assert (err <= rounded(bound, want, typ)).all(), ((err - rounded(bound * 0, want, typ)) / top).amax((0, 1, 2, 4)).tolist()


@pytest.mark.parametrize("hq,hkv,hd,group", [(8, 4, 256, 64), (16, 2, 128, 128)])
@pytest.mark.parametrize("gap", [12.0, 18.0, 20.0])
@pytest.mark.parametrize("typ", TYPES)
def test_many_small_weights_beside_a_large_one(pkg, hq, hkv, hd, group, gap, typ):
    """One key `gap` above all others, whose value is zero, and thousands of e^-gap with values of one: what is left is their sum, to 2^-9
    ahead of storing it (weights to 2^-11, one exponent) and 2^-36 a key: fp16 numbers are 2^-24 apart below 2^-14, so a weight that is held
    times 2^11 is off by at most 2^-25-11 of the largest."""
    lens, counts = [9000, 3000], [200, 150]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=1, tail=0)
    a.q[:] = 0
    a.q[:, :hq * hd].view(-1, hq, hd)[..., 0] = 1.0
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).cuda()
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    k, v = torch.zeros(len(seq), hkv, hd, device="cuda"), torch.ones(len(seq), hkv, hd, device="cuda")
    first = pos == 3
    k[first, :, 0], v[first] = gap * hd ** 0.5, 0.0
    k, v = put(pkg, a.cache, seq, pos, k, v)
    assert (v[~first] == 1).all() and (v[first] == 0).all() and (k[~first] == 0).all()
    a()
    for b, (n, count) in enumerate(zip(lens, counts)):
        rows = a.out[int(a.start[b]):int(a.start[b]) + count, :hq * hd].double()
        rest = torch.arange(n - count, n, device="cuda", dtype=torch.float64) * torch.exp(-k[first][b, 0, 0].double() * hd ** -0.5)
        want = (rest / (1 + rest))[:, None]
        assert ((rows - want).abs() <= rounded(want * 2.0 ** -9 + n * 2.0 ** -36, want, typ)).all(), (rows / want).aminmax()


@pytest.mark.parametrize("hq,hkv,hd,group", [(4, 2, 256, 64), (8, 4, 128, 128), (5, 1, 64, 64)])
@pytest.mark.parametrize("count", [1, 3])
def test_small_weights_in_fp32(pkg, hq, hkv, hd, group, count):
    """As above with random values under the large key, each of weight e^-10.5 (2.8e-5): fp32 rows to 2e-6 in the 2-norm.  ex2 and the two terms
    of a weight are off by 2^-22 and 2^-22, those below the terms' range by 2^-36 of the largest (5e-7 of these), of which a
    third of the square is expected in the sum of independent ones: 4e-7, five times allowed."""
    lens = [9000, 5000]
    a = Attention(pkg, lens, [count] * 2, hq, hkv, hd, group, torch.float32, seed=1, tail=0)
    a.q[:] = 0
    a.q[:, :hq * hd].view(-1, hq, hd)[..., 0] = 1.0
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).cuda()
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    k, v = torch.zeros(len(seq), hkv, hd, device="cuda"), torch.randn(len(seq), hkv, hd, device="cuda", generator=gen(5))
    first = pos % 100 == 3                                 # each warp meets one
    k[first, :, 0], v[first] = 10.5 * hd ** 0.5, 0.0
    a.k, a.v = (x.split(lens) for x in put(pkg, a.cache, seq, pos, k, v))
    a()
    for b in range(2):
        at, want = exact(a, b)
        err = (a.out[at, :hq * hd].double() - want).view(count, hq, hd).norm(dim=-1)
        assert (err <= 2e-6 * want.view(count, hq, hd).norm(dim=-1)).all(), (err / want.view(count, hq, hd).norm(dim=-1)).max().item()
