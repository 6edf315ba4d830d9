"""QK norm over the whole range of its types: rows far from one, infinities, eps of zero.  Tolerances as in test_gpu_kv4.py."""
import pytest
import torch

from test_gpu_kv4 import TYPES, Cache, Rows, close, held, stream

pytestmark = pytest.mark.gpu

SIZES = [1e-44, 1e-38, 1e-30, 1e-25, 1e-19, 1.0, 1e15, 1e18, 3e19, 1e25, 1e30, 1e37]


def norm_rope(x, gain, cos, sin, rot, eps):
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    h = rot // 2
    a, b, c, s = y[..., :h], y[..., h:rot], cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, a * s + b * c, y[..., rot:]], -1)


def scaled(hq, hkv, hd, rot, typ, eps):
    """Rows whose heads are of the sizes above, neighbours of different ones."""
    t = len(SIZES) + 1
    r = Rows(t, hq, hkv, hd, rot, typ, seed=hd + rot)
    for i in range(t):
        for h in range(hq + 2 * hkv):
            size = SIZES[(i + h) % len(SIZES)] if h < hq + hkv else 1.0
            if typ == torch.float16:
                size = min(max(size, 1e-4), 1e4)
            r.rows[i, h * hd:(h + 1) * hd] = (r.rows[i, h * hd:(h + 1) * hd].double() * size).to(typ)
    return r, {**r.args(), "eps": eps}


@pytest.mark.parametrize("hq,hkv,hd,rot", [(4, 1, 256, 256), (8, 4, 128, 128), (5, 3, 64, 32)])
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-6])
def test_rows_of_every_size(pkg, hq, hkv, hd, rot, typ, eps):
    r, args = scaled(hq, hkv, hd, rot, typ, eps)
    eps = float(torch.tensor(eps))
    t = r.q.shape[0]
    k_out = torch.full((t, hkv * hd), 7.0, device="cuda", dtype=typ)
    pkg.ops.qk_norm_rope(k_out_dev=k_out.data_ptr(), k_stride=hkv * hd, **args)
    q, k, v = r.heads()
    at = r.pos.long()
    for got, x, gain in ((r.q, q, r.q_gain), (k_out, k, r.k_gain)):
        want = norm_rope(x, gain, r.cos[at], r.sin[at], rot, eps)
        ok = torch.isfinite(want)                          # rows of zeros without eps: 0 / 0
        assert ok.flatten(2).any(-1).float().mean() > 0.8
        size = torch.cat([(want[..., :rot // 2].abs() + want[..., rot // 2:rot].abs()).repeat(1, 1, 2), want[..., rot:].abs()], -1) * 1.5
        got = got.view_as(want)
        assert (torch.isfinite(got) == ok).all()
        close(got[ok], want[ok], typ, size[ok])
    cache = Cache(pkg, 1, 3, hkv, hd, 64)
    seq = torch.zeros(t, dtype=torch.int32, device="cuda")
    r.q.fill_(7.0)
    pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, seq_dev=seq.data_ptr(), **args)
    assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
    kw = norm_rope(k, r.k_gain, r.cos[at], r.sin[at], rot, eps)
    kg, vg = cache.read(pkg, seq, r.pos)
    ok = torch.isfinite(kw)
    assert (torch.isfinite(kg) == ok).all()
    assert torch.equal(kg.double()[ok], held(kw.float(), 64)[ok]) and torch.equal(vg.double(), held(v.float(), 64))


@pytest.mark.parametrize("hq,hkv,hd,rot", [(4, 1, 256, 256), (8, 4, 128, 64), (5, 3, 64, 64)])
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("t,pad", [(600, 0), (600, 8), (40, 3)])
def test_many_rows_of_every_size_in_their_own_places(pkg, hq, hkv, hd, rot, typ, t, pad):
    """Several passes a warp, ordinary heads beside far ones, results over the rows themselves."""
    r = Rows(t, hq, hkv, hd, rot, typ, pad, seed=hd + rot)
    sizes = torch.tensor(SIZES, device="cuda", dtype=torch.float64)
    pick = (torch.arange(t, device="cuda")[:, None] * 5 + torch.arange(hq + 2 * hkv, device="cuda")) % len(SIZES)
    if typ == torch.float16:
        sizes = sizes.clamp(1e-4, 1e4)
    r.rows.copy_((r.rows.double().unflatten(1, (-1, hd)) * sizes[pick][..., None]).flatten(1).to(typ))
    q, k, v = (x.clone() for x in r.heads())
    at, args, stride = r.pos.long(), r.args(), r.buf.numel() // t
    args.update(q_out_dev=r.buf.data_ptr(), q_stride=stride)
    pkg.ops.qk_norm_rope(k_out_dev=r.buf.data_ptr() + hq * hd * r.buf.element_size(), k_stride=stride, **args)
    assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
    got_q, got_k, got_v = r.heads()
    assert torch.equal(got_v, v)
    for got, x, gain in ((got_q, q, r.q_gain), (got_k, k, r.k_gain)):
        want = norm_rope(x, gain, r.cos[at], r.sin[at], rot, 1e-6)
        size = torch.cat([(want[..., :rot // 2].abs() + want[..., rot // 2:rot].abs()).repeat(1, 1, 2), want[..., rot:].abs()], -1) * 1.5
        close(got, want, typ, size)


@pytest.mark.parametrize("rot", [0, 128])
def test_an_infinity_in_a_key_spoils_its_groups(pkg, rot):
    """The other elements of the head are x / inf = 0; with rotation the element's partner is spoilt too."""
    r = Rows(3, 2, 1, 128, rot, torch.float32, seed=2)
    r.rows[1, 256 + 5] = float("inf")
    r.rows[2, 256 + 70] = float("nan")
    cache = Cache(pkg, 1, 3, 1, 128, 64)
    seq = torch.zeros(3, dtype=torch.int32, device="cuda")
    pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, seq_dev=seq.data_ptr(), **r.args())
    k, _ = cache.read(pkg, seq, r.pos)
    assert torch.isnan(k[1, 0, :64]).all()
    assert torch.isnan(k[1, 0, 64:]).all() if rot else (k[1, 0, 64:] == 0).all()
    assert torch.isnan(k[2]).all() and torch.isfinite(k[0]).all() and torch.isfinite(r.q).all()
