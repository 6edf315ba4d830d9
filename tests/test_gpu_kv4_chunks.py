"""Chunks of bf16 rows over the 4-bit cache, where they take the tensor-core kernel: each row's error in the 2-norm, against what one tile
of keys left out would do; results that repeat bit for bit while other work delays the loads; last tiles that carry the result.

Tolerance of a row o = sum_k p_k v_k (d elements, 2-norms).  Storing it as bf16 costs at most 2^-8 |o|.  Ahead of that, to first order,
  e = sum_k p_k eps_k (v_k - o) + sum_k p_k eta_k,
eps_k the error of the key's score with that of its weight, eta_k that of the value.  K and V may enter as fp16 numbers with two roundings
of at most 2^-11 of the largest each, P with one of 2^-11 of itself.  These are independent, of variance a third of their bound's square:
  E |e|^2 <= sum_k p_k^2 (sigma^2 |v_k - o|^2 + d tau^2),   tau^2 = 2/3 (2^-11 max |v|)^2,
  sigma^2 = 2/3 (2^-11 max |k| |q| scale)^2 + 1/3 (2^-11)^2.
Six times the root of that is passed with a probability of 2e-9 a row if one key has all of it, less if many share it.  fp32 sums add
64 u max |v| sqrt(d), far less.
"""
import math

import pytest
import torch

from test_gpu_kv4 import U, Attention, gen

pytestmark = pytest.mark.gpu

HEADS = [(8, 4, 256, 64), (8, 4, 256, 128), (8, 4, 128, 64), (16, 2, 128, 128)]


def rows_of(a, b, window=0, drop=0):
    """(result, expected result, bound of the 2-norm of their difference) of sequence b's rows [heads, rows]; `drop` leaves that many keys
    at the end of each row out of the expected result."""
    hq, hkv, hd = a.dims
    n, count = a.lens[b], a.counts[b]
    at = slice(int(a.start[b]), int(a.start[b]) + count)
    q = a.q[at, :hq * hd].double().view(count, hkv, hq // hkv, hd).permute(1, 2, 0, 3)
    got = a.out[at, :hq * hd].double().view(count, hkv, hq // hkv, hd).permute(1, 2, 0, 3)
    k, v = a.k[b].double().transpose(0, 1), a.v[b].double().transpose(0, 1)
    pos = torch.arange(n - count, n, device="cuda")[:, None]
    key = torch.arange(n, device="cuda")[None]
    seen = (key <= pos) & ((key > pos - window) if window > 0 else (key >= 0))
    want, bound = torch.empty_like(got), torch.empty_like(got[..., 0])
    used = hd ** -0.5
    for h in range(hkv):
        x = (q[h] @ k[h].T * used).masked_fill(~(seen & (key <= pos - drop)), -math.inf)
        p = torch.nan_to_num(torch.softmax(x, -1))
        o = p @ v[h]
        want[h] = o
        tau = math.sqrt(2 / 3) * 2.0 ** -11 * v[h].abs().amax()
        sigma = torch.sqrt(2 / 3 * (2.0 ** -11 * k[h].abs().amax() * q[h].norm(dim=-1) * used) ** 2 + (2.0 ** -11) ** 2 / 3)
        p2 = p * p
        gap = p2 @ v[h].square().sum(-1) - 2 * ((p2 @ v[h]) * o).sum(-1) + p2.sum(-1) * o.square().sum(-1)      # sum p^2 |v - o|^2
        inner = 6 * torch.sqrt(sigma ** 2 * gap.clamp(min=0) + hd * tau ** 2 * p2.sum(-1)) + 64 * U * v[h].abs().amax() * math.sqrt(hd)
        bound[h] = 2.0 ** -8 * (o.norm(dim=-1) + inner) + inner
    return got, want, bound


def check_rows(a, window=0):
    for b, (n, count) in enumerate(zip(a.lens, a.counts)):
        if count == 0 or n == 0:
            continue
        got, want, bound = rows_of(a, b, window)
        err = (got - want).norm(dim=-1)
        assert (err <= bound).all(), (b, n, count, window, (err / bound).max().item())


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("lens,counts", [([700, 130, 5, 1025, 0, 64, 300], [700, 129, 5, 300, 9, 100, 1]), ([5000] * 3 + [100] * 9, [20] * 12), ([30000, 12], [100, 12])])
def test_each_row_in_the_2_norm(pkg, hq, hkv, hd, group, lens, counts):
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, torch.bfloat16, seed=hd * 7 + hq)
    for window in (0, 130, 1000):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        check_rows(a, window)


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
def test_a_tile_left_out_would_not_pass(pkg, hq, hkv, hd, group):
    """The bound above tells a row whose last 64 or 32 keys are missing from a right one, in every row that has a few times as many."""
    lens, counts = [700, 5000], [700, 20]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, torch.bfloat16, seed=hd * 7 + hq)
    for b in range(2):
        for drop in (64, 32):
            _, whole, bound = rows_of(a, b)
            _, less, _ = rows_of(a, b, drop=drop)
            full = torch.arange(lens[b] - counts[b], lens[b], device="cuda") >= 2 * drop
            assert ((less - whole).norm(dim=-1) > bound)[..., full].all()


# (lengths, query tokens of each): tiles of 64 keys that a CTA walks: 1, 2, 3, and many with one share or several
SHAPES = [([64] * 64, 64), ([128] * 64, 128), ([192, 130, 129, 64] * 16, 64), ([1500, 1470] * 8, 300), ([6000], 128), ([9000, 3000], 200)]


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("lens,count", SHAPES)
def test_chunks_repeat_bit_for_bit_beside_other_work(pkg, hq, hkv, hd, group, lens, count):
    counts = [min(n, count) for n in lens]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, torch.bfloat16, seed=len(lens) + hd)
    a()
    torch.cuda.synchronize()
    first = a.out.clone()
    side = torch.cuda.Stream()
    noise = torch.empty(2, 64 << 20, device="cuda", dtype=torch.uint8)
    for i in range(12):
        a.out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):                      # takes the bandwidth away for a while, from another moment each time
            for _ in range(i % 4):
                noise[i % 2].copy_(noise[1 - i % 2])
        a()
        torch.cuda.synchronize()
        assert torch.equal(a.out, first)
    for b in {lens.index(n) for n in lens}:
        got, want, bound = rows_of(a, b)
        assert ((got - want).norm(dim=-1) <= bound).all()


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
def test_last_tiles_that_carry_the_result(pkg, hq, hkv, hd, group):
    """Values a hundred times as large in the last 128 positions, so that a product that comes too late is most of the result."""
    lens, count = [1500, 1470, 1409] * 5, 300
    a = Attention(pkg, lens, [count] * len(lens), hq, hkv, hd, group, torch.bfloat16, seed=3)
    from test_gpu_kv4 import put
    g = gen(8)
    for b, n in enumerate(lens):
        k, v = (torch.randn(128, hkv, hd, device="cuda", generator=g) for _ in range(2))
        seq = torch.full((128,), b, dtype=torch.int32, device="cuda")
        k, v = put(pkg, a.cache, seq, torch.arange(n - 128, n, dtype=torch.int32, device="cuda"), k, 100 * v)
        a.k = a.k[:b] + (torch.cat([a.k[b][:n - 128], k]),) + a.k[b + 1:]
        a.v = a.v[:b] + (torch.cat([a.v[b][:n - 128], v]),) + a.v[b + 1:]
    for _ in range(3):
        a.out.fill_(7.0)
        a()
        check_rows(a)


def test_one_workspace_serves_calls_in_turn(pkg):
    """Chunks, drafted and single tokens of different sizes, one behind the other over one workspace, called and from one graph: each as alone,
    and the tickets at zero behind every call, bad pages and lengths among them."""
    makes = [([6000, 40], [128, 40], 8, 4, 256, 64), ([9000], [1], 4, 1, 256, 64), ([9000, 3000], [200, 150], 16, 2, 128, 128), ([700] * 6, [5] * 6, 8, 4, 128, 64), ([20000, 3], [1, 1], 12, 4, 64, 64)]
    calls = [Attention(pkg, lens, counts, hq, hkv, hd, group, torch.bfloat16, seed=i) for i, (lens, counts, hq, hkv, hd, group) in enumerate(makes)]
    room = torch.zeros(max(a.need for a in calls), device="cuda", dtype=torch.uint8)
    alone = []
    for a in calls:
        a()
        alone.append(a.out.clone())
        a.room, a.need = room, room.numel()
    for a, want in zip(calls, alone):
        a.out.fill_(7.0)
        a()
        assert torch.equal(a.out, want) and not room[:16384].any()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        for a in calls:
            a()
    for _ in range(5):
        for a in calls:
            a.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.out, want) for a, want in zip(calls, alone)) and not room[:16384].any()
    calls[0].cache.table[0, 20], calls[2].kv_len[1], calls[4].cache.table[0, 70] = -1, 9001, 2 ** 30
    graph.replay()
    torch.cuda.synchronize()
    assert not room[:16384].any()
    for i in (0, 2, 4):
        with pytest.raises(pkg.StatusError):
            pkg.ops.device_status(calls[i].status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert torch.equal(calls[i].out, alone[i])         # the last replay's results stay where they were not written
    for i in (1, 3):
        assert torch.equal(calls[i].out, alone[i])
