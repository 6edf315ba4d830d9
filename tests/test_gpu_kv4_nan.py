"""A group of the cache that stands for NaN: in V it makes its own dims NaN, in the rows that see the key; in K all of those rows.  The same
wherever the key lies in its tile or among the rows' masks, and on either kernel of the attention."""
import math

import pytest
import torch

from test_gpu_kv4 import U, Attention, put, rounded, stream

pytestmark = pytest.mark.gpu

HEADS = [(8, 4, 256, 64), (8, 4, 256, 128), (8, 4, 128, 64), (4, 4, 128, 128), (6, 2, 64, 64)]


def one(x):
    return torch.tensor([x], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,count", [([777, 300, 5000], 1), ([600, 300, 64], 4), ([900, 700, 1500], 300)])
def test_a_group_of_nan_spoils_its_own_dims(pkg, hq, hkv, hd, group, typ, lens, count):
    counts = [min(n, count) for n in lens]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd + count)
    hurt = torch.zeros(len(lens), max(lens), hkv, hd, dtype=torch.bool, device="cuda")
    k_hurt = torch.zeros(len(lens), max(lens), hkv, dtype=torch.bool, device="cuda")
    # (sequence, position from the end, kv head, dim) of a NaN in V: first and inner tiles, the last key, keys that some rows see
    places = [(0, lens[0], 0, 3), (0, 1, hkv - 1, hd - 1), (0, 200, 0, hd // 2), (1, counts[1] // 2 + 1, 0, 0), (1, 150, hkv - 1, 70 % hd), (2, 2, 0, hd - 1), (2, 40, hkv - 1, 1)]
    v_new, k_new = {}, {}
    for b, back, head, dim in places:
        at = lens[b] - back
        v = v_new.setdefault((b, at), torch.nan_to_num(a.v[b][at]).clone())
        v[head, dim] = float("nan")
        hurt[b, at, head, dim // group * group:(dim // group + 1) * group] = True
    k = k_new.setdefault((1, lens[1] - 100), a.k[1][lens[1] - 100].clone())
    k[0, hd // 3] = float("inf")
    k_hurt[1, lens[1] - 100, 0] = True
    for b, at in set(v_new) | set(k_new):
        got_k, got_v = put(pkg, a.cache, one(b), one(at), k_new.get((b, at), a.k[b][at])[None].contiguous(), v_new.get((b, at), a.v[b][at])[None].contiguous())
        assert torch.equal(torch.isnan(got_v[0]), hurt[b, at]) and torch.equal(torch.isnan(got_k[0]).any(-1), k_hurt[b, at])
        a.k[b][at], a.v[b][at] = got_k[0], got_v[0]
    for window in (0, 1, 130):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        for b, (n, c) in enumerate(zip(lens, counts)):
            rows = slice(int(a.start[b]), int(a.start[b]) + c)
            got = a.out[rows, :hq * hd].double().view(c, hkv, hq // hkv, hd)
            pos, key = torch.arange(n - c, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            seen = (key <= pos) & ((key > pos - window) if window > 0 else (key >= 0))
            bad = torch.einsum("ts,shd->thd", seen.double(), hurt[b, :n].double()) > 0
            bad |= (torch.einsum("ts,sh->th", seen.double(), k_hurt[b, :n].double()) > 0)[..., None]
            assert (torch.isnan(got) == bad[:, :, None]).all(), (b, window)
            # and what stays is right
            k, v, q = torch.nan_to_num(a.k[b]).double(), torch.nan_to_num(a.v[b]).double(), a.q[rows, :hq * hd].double().view(c, hkv, hq // hkv, hd)
            p = torch.softmax((torch.einsum("thgd,shd->hgts", q, k) * hd ** -0.5).masked_fill(~seen, -math.inf), -1)
            want = torch.einsum("hgts,shd->thgd", p, v)
            # weights to 2^-16 (scores of up to 16, their exponents), on the tensor-core kernel P and V to 2^-11: of the largest value
            bound = (2.0 ** -15 + (2.0 ** -10 if typ == torch.bfloat16 and count > 4 else 64 * U)) * v.abs().amax()
            fine = ~bad[:, :, None].expand_as(got)
            assert ((got - want).abs() <= rounded(bound, want, typ))[fine].all()
