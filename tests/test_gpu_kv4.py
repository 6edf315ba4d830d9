"""Grouped int4 products, QK norm with rotation, the cache in 4 bits and the attention over it, against the same mathematics in
64 bits, at the sizes and masks where they can go wrong.

Tolerances.  u = 2^-24.  A stored value is off by half a step: eps / 2 of it, and of the smallest normal number below that.
  product    x enters in digits of seven bits, the largest |x| of a block of 128 at least 2^5 of the first one's unit: four digits are
             off by half of 2^-21 units, 2^-27 of that |x|, three (more than four columns of a 16-bit type) by 2^-20; a column is added up in fp32 along one chain of at most
             ceil(k / 32) + 2 adds a lane, joined by at most 12 more, each term behind two roundings: (ceil(k / 32) + 18) u sum |w x|
  norm       sum of hd / 32 + 5 adds, a root, a quotient: at most 16 u on the factor, four roundings behind it: 24 u (|a| + |b|)
  cache      codes are decided in 64 bits from values rounded once to 32: equal
  attention  a score is off by dS = 8 u sum |q k| scale + 2^-20 (the exponent's own error, 2^-22, and its argument's rounding among it),
             a weight by 2 dS and what it is held in, two fp16 terms (2^-22), or for bf16 rows one,
             where P, P s and m + 8 s are rounded to fp16 (three times half a step, 2^-11); with the
             sums' own error of 64 u that times the largest |v| bounds the result's.
             Chunks of bf16 rows (head sizes 128 and 256, 16 rows of a kv head and more) may meet K and V as fp16 numbers
             s (c - 8) + (m + 8 s), two roundings of at most 2^-11 of the largest |k| or |v| each.  The roundings of a key's elements
             are independent: by Hoeffding's bound the score is off by more than 6 * 2^-10 max |k| |q| scale (|q| the 2-norm) with
             probability 2 exp(-18) = 3e-8; that is added to dS, and 2^-10 to what multiplies the largest |v|
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def code_of(t):
    return TYPES.index(t)


def rounded(bound, want, t):
    """What storing in t adds: half a step, and below t's smallest normal number the step is that of the smallest."""
    return bound + torch.finfo(t).eps / 2 * (want.abs() + bound).clamp(min=torch.finfo(t).smallest_normal)


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------- products

def product(pkg, n, k, group, cols, x_type, y_type, s_type, offset, seed, ldx=0, ldy=0, shift=0, spread=False):
    g = gen(seed)
    q = torch.randint(-8, 8, (n, k), device="cuda", generator=g)
    groups = -(-k // group)
    scale = (0.02 * torch.rand(n, groups, device="cuda", generator=g) + 1e-3).to(s_type)
    off = (0.05 * torch.randn(n, groups, device="cuda", generator=g)).to(s_type) if offset else None
    nib = (q & 15).to(torch.uint8).cpu().numpy()
    raw = lambda t: None if t is None else t.view(torch.int16).cpu().numpy()          # noqa: E731
    img = torch.from_numpy(pkg.ops.repack_w4_grouped(nib[:, 0::2] | nib[:, 1::2] << 4, raw(scale), raw(off), group)).cuda()
    ldx, ldy = ldx or k, ldy or n
    x = torch.randn(cols * ldx + shift, device="cuda", generator=g)
    if spread:                                                                      # twenty powers of two between neighbours
        x = x * torch.exp2(torch.randint(-10, 11, x.shape, device="cuda", generator=g).float())
    x = x.to(x_type)[shift:]
    y = torch.full((cols * ldy,), 7.0, device="cuda", dtype=y_type)
    pkg.ops.gemv_w4_grouped(img.data_ptr(), x.data_ptr(), y.data_ptr(), n, k, group, ncols=cols, x_type=code_of(x_type), y_type=code_of(y_type), scale_type=code_of(s_type), has_offset=offset,
                            ldx=ldx, ldy=ldy, stream=stream())
    rows = torch.stack([x[c * ldx:c * ldx + k] for c in range(cols)]).double()
    w = q.double() * scale.double().repeat_interleave(group, 1)[:, :k]
    size = w.abs()
    if offset:
        o = off.double().repeat_interleave(group, 1)[:, :k]
        w, size = w + o, size + o.abs()
    blocks = torch.nn.functional.pad(rows.abs(), (0, -k % 128)).view(cols, -1, 128).amax(-1).repeat_interleave(128, 1)[:, :k]
    want = rows @ w.T
    bound = (-(-k // 32) + 18) * U * (rows.abs() @ size.T) + (2.0 ** -20 if cols > 4 and x_type != torch.float32 else 2.0 ** -27) * (blocks @ size.T)
    got = y.view(cols, ldy)
    assert (got[:, n:] == 7.0).all()
    err = (got[:, :n].double() - want).abs()
    assert (err <= rounded(bound, want, y_type)).all(), (err / want.abs().max()).max().item()


@pytest.mark.parametrize("n,k", [(1, 2), (1, 128), (15, 30), (16, 130), (17, 1152), (40, 4098), (1536, 1152), (320, 9000), (5000, 256)])
@pytest.mark.parametrize("group,offset", [(32, True), (32, False), (64, False), (64, True), (128, True), (128, False)])
def test_product_sizes(pkg, n, k, group, offset):
    for cols in (1, 2, 3, 8):
        product(pkg, n, k, group, cols, torch.float32, torch.float32, torch.float16, offset, n + k + cols)


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("y_type", TYPES)
@pytest.mark.parametrize("s_type", [torch.bfloat16, torch.float16])
def test_product_types_strides_alignment(pkg, x_type, y_type, s_type):
    for i, (cols, ldx, ldy, shift) in enumerate([(1, 0, 0, 0), (5, 0, 0, 1), (4, 521, 67, 0), (7, 516, 64, 3)]):
        product(pkg, 60, 514, 64, cols, x_type, y_type, s_type, i % 2 == 1, 100 + i, ldx, ldy, shift)


def test_product_of_values_far_apart(pkg):
    for cols in (1, 6):
        product(pkg, 96, 2048, 32, cols, torch.float32, torch.float32, torch.bfloat16, True, 9, spread=True)


def test_product_of_extreme_columns(pkg):
    """Zeros, the smallest and largest numbers, an infinity and a NaN: only the last two spoil their columns."""
    n, k = 48, 640
    q = torch.ones(n, k, dtype=torch.uint8)
    nib = q.numpy()
    one = np.full((n, k // 64), np.float16(1.0).view(np.uint16))
    img = torch.from_numpy(pkg.ops.repack_w4_grouped(nib[:, 0::2] | nib[:, 1::2] << 4, one, None, 64)).cuda()
    x = torch.zeros(8, k, device="cuda")
    x[1] = 1e-45
    x[2], x[2, 5] = 1.0, 1e30
    x[3, 100] = 3e38
    x[4], x[5] = 1.0, 2.0
    x[4, 77], x[5, 639] = float("inf"), float("nan")
    x[6], x[7] = -1.0, 1e-30
    y = torch.zeros(8, n, device="cuda")
    pkg.ops.gemv_w4_grouped(img.data_ptr(), x.data_ptr(), y.data_ptr(), n, k, 64, ncols=8, stream=stream())
    assert (y[0] == 0).all() and (y[1].abs() <= 1e-40).all() and torch.isnan(y[4]).all() and torch.isnan(y[5]).all()
    assert torch.allclose(y[2], torch.tensor(1e30, device="cuda")) and torch.allclose(y[3], torch.tensor(3e38, device="cuda"))
    assert (y[6] == -k).all() and torch.allclose(y[7], torch.tensor(k * 1e-30, device="cuda"), atol=0)


# ------------------------------------------------------------------------------------------------- rows and cache

def norm_rope(x, gain, cos, sin, rot):
    y = x if gain is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain.double()
    h = rot // 2
    a, b = y[..., :h], y[..., h:rot]
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    return torch.cat([a * c - b * s, a * s + b * c, y[..., rot:]], -1)


def held(x, group):
    """What the cache stands for, of x in fp32."""
    g = x.double().unflatten(-1, (-1, group))
    low, high = g.amin(-1), g.amax(-1)
    m, s = low.float().half().double(), ((high - low) / 15).float().half().double()
    c = torch.where(s[..., None] > 0, ((g - m[..., None]) / s[..., None]).round().clamp(0, 15), 0.0)
    return (s[..., None] * c + m[..., None]).flatten(-2)


class Rows:
    def __init__(self, t, hq, hkv, hd, rot, typ, pad=0, shift=0, seed=0, far=700, norm=True):
        g = gen(seed)
        self.dims, self.typ, self.far = (t, hq, hkv, hd, rot), typ, far
        width = (hq + 2 * hkv) * hd
        self.buf = torch.randn(t * (width + pad) + shift, device="cuda", generator=g).to(typ)[shift:]
        self.rows = self.buf.view(t, width + pad)[:, :width]
        self.q_gain, self.k_gain = (1 + 0.2 * torch.randn(2, hd, device="cuda", generator=g)).unbind(0) if norm else (None, None)
        angle = torch.rand(far, rot // 2, device="cuda", generator=g) * 6.3
        self.cos, self.sin = torch.cos(angle), torch.sin(angle)
        self.pos = torch.randperm(far, device="cuda", generator=g)[:t].to(torch.int32)
        self.q = torch.full((t, hq * hd + pad), 7.0, device="cuda", dtype=typ)
        self.status = torch.zeros(1, device="cuda", dtype=torch.int32)

    def args(self):
        t, hq, hkv, hd, rot = self.dims
        ptr = lambda x: 0 if x is None or x.numel() == 0 else x.data_ptr()          # noqa: E731
        return dict(qkv_dev=self.buf.data_ptr(), type=code_of(self.typ), qkv_stride=self.buf.numel() // t, tokens=t, hq=hq, hkv=hkv, hd=hd, rot=rot, q_gain_dev=ptr(self.q_gain), k_gain_dev=ptr(self.k_gain),
                    eps=1e-6, cos_dev=ptr(self.cos), sin_dev=ptr(self.sin), rope_rows=self.far, pos_dev=self.pos.data_ptr(), q_out_dev=self.q.data_ptr(), q_stride=self.q.shape[1],
                    status_dev=self.status.data_ptr(), stream=stream())

    def heads(self):
        t, hq, hkv, hd, _ = self.dims
        x = self.rows.double().unflatten(1, (-1, hd))
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    def want(self):
        at, rot = self.pos.long().clamp(min=0, max=self.far - 1), self.dims[4]
        q, k, v = self.heads()
        return norm_rope(q, self.q_gain, self.cos[at], self.sin[at], rot), norm_rope(k, self.k_gain, self.cos[at], self.sin[at], rot), v


def close(got, want, typ, size):
    """`size`: sum of the magnitudes that went into an element."""
    bound = 24 * U * size
    assert ((got.double() - want).abs() <= rounded(bound, want, typ)).all(), ((got.double() - want).abs() / want.abs().max()).max().item()


@pytest.mark.parametrize("hq,hkv,hd,rot", [(4, 1, 256, 256), (8, 4, 128, 128), (3, 3, 64, 64), (4, 2, 256, 64), (4, 2, 128, 80), (6, 2, 64, 16), (2, 1, 128, 0)])
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("t,pad,shift", [(1, 0, 0), (37, 5, 1), (600, 8, 0)])
def test_norm_and_rotation(pkg, hq, hkv, hd, rot, typ, t, pad, shift):
    for norm in (True, False):
        r = Rows(t, hq, hkv, hd, rot, typ, pad, shift, seed=t + hd + rot, norm=norm)
        k = torch.full((t, hkv * hd + 3), 7.0, device="cuda", dtype=typ)
        pkg.ops.qk_norm_rope(k_out_dev=k.data_ptr(), k_stride=hkv * hd + 3, **r.args())
        assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
        qw, kw, _ = r.want()
        for got, want, n in ((r.q, qw, hq * hd), (k, kw, hkv * hd)):
            size = torch.cat([(want[..., :rot // 2].abs() + want[..., rot // 2:rot].abs()).repeat(1, 1, 2) if rot else want[..., :0], want[..., rot:].abs()], -1) * 1.5
            close(got[:, :n], want.flatten(1), typ, size.flatten(1))
            assert (got[:, n:] == 7.0).all()


def test_norm_and_rotation_in_place_padding_and_bad_positions(pkg):
    r = Rows(40, 4, 2, 128, 128, torch.float32, seed=5)
    r.pos[3], r.pos[17], r.pos[39] = -1, r.far, 2 ** 31 - 1
    qw, kw, _ = r.want()
    before, a = r.rows.clone(), r.args()
    a.update(q_out_dev=r.buf.data_ptr(), q_stride=r.buf.numel() // 40)
    pkg.ops.qk_norm_rope(k_out_dev=r.buf.data_ptr() + 4 * 512, k_stride=r.buf.numel() // 40, **a)
    with pytest.raises(pkg.StatusError) as e:
        pkg.ops.device_status(r.status.data_ptr(), stream())
    assert e.value.code == pkg.INVALID_ARGUMENT and pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 17, 39]] = True
    assert torch.equal(r.rows[bad], before[bad]) and torch.equal(r.rows[:, 768:], before[:, 768:])
    close(r.rows[~bad][:, :512], qw[~bad].flatten(1), torch.float32, 3 * qw[~bad].flatten(1).abs() + 8)
    close(r.rows[~bad][:, 512:768], kw[~bad].flatten(1), torch.float32, 3 * kw[~bad].flatten(1).abs() + 8)


class Cache:
    def __init__(self, pkg, batch, per, hkv, hd, group, seed=0, spare=2, fill=None):
        g = gen(seed + 77)
        self.hkv, self.hd, self.group, self.n = hkv, hd, group, batch * per + spare
        self.bytes = pkg.Kv4Cache.page_bytes(hkv, hd, group)
        # codes at random, every scale NaN: what was never appended must not be looked at
        self.pages = torch.full((self.n, self.bytes), 0xFF if fill is None else fill, device="cuda", dtype=torch.uint8)
        self.table = torch.randperm(self.n, device="cuda", generator=g)[:batch * per].to(torch.int32).view(batch, per)
        self.c = pkg.Kv4Cache(self.pages.data_ptr(), self.n, self.table.data_ptr(), per, batch, hkv, hd, group)

    def read(self, pkg, seq, pos, typ=torch.float32):
        t = seq.numel()
        k, v = (torch.full((t, self.hkv, self.hd), 7.0, device="cuda", dtype=typ) for _ in range(2))
        pkg.ops.kv4_read(self.c, seq.data_ptr(), pos.data_ptr(), t, code_of(typ), k.data_ptr(), v.data_ptr(), stream=stream())
        return k, v


@pytest.mark.parametrize("hq,hkv,hd,rot,group", [(4, 1, 256, 256, 64), (4, 2, 256, 128, 128), (8, 4, 128, 128, 64), (4, 4, 128, 64, 128), (6, 2, 64, 64, 64)])
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("t,pad,shift", [(1, 0, 0), (300, 3, 1)])
def test_append_and_read(pkg, hq, hkv, hd, rot, group, typ, t, pad, shift):
    r = Rows(t, hq, hkv, hd, rot, typ, pad, shift, seed=t + hd + group)
    cache = Cache(pkg, 3, 3, hkv, hd, group, seed=t)
    seq = (torch.arange(t, device="cuda", dtype=torch.int32) * 7) % 3
    pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, seq_dev=seq.data_ptr(), **r.args())
    assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
    qw, kw, vw = r.want()
    close(r.q[:, :hq * hd], qw.flatten(1), typ, 3 * qw.flatten(1).abs() + 8)
    k, v = cache.read(pkg, seq, r.pos)
    assert torch.equal(k.double(), held(kw.float(), group)) and torch.equal(v.double(), held(vw.float(), group))
    for low in TYPES[1:]:
        k16, v16 = cache.read(pkg, seq, r.pos, low)
        assert torch.equal(k16, k.to(low)) and torch.equal(v16, v.to(low))
    # nothing but the tokens' own rows was written
    page = cache.table[seq.long(), r.pos.long() // 256].long()
    own = torch.zeros(cache.n, 256, dtype=torch.bool, device="cuda")
    own[page, r.pos.long() % 256] = True
    heads = cache.pages.view(cache.n, hkv, -1)
    at = 0
    for _ in range(2):
        for width in [min(hd, 128) // 2] * (hd // min(hd, 128)) + [4 * hd // group]:
            part = heads[:, :, at:at + 256 * width].view(cache.n, hkv, 256, width)
            assert (part.transpose(1, 2)[~own] == 0xFF).all()
            at += 256 * width
    assert at == heads.shape[2]


def test_append_of_special_groups(pkg):
    """Constant groups, groups with an infinity or NaN, groups beyond fp16's range, and tiny ones."""
    r = Rows(6, 1, 1, 128, 0, torch.float32, seed=3, norm=False)
    r.rows[0, 128:] = 2.5
    r.rows[1, 130], r.rows[1, 300] = float("inf"), float("nan")
    r.rows[2, 128:] = 1e6 * r.rows[2, 128:]
    r.rows[3, 128:] = 1e-9 * r.rows[3, 128:]
    r.rows[4, 128:256] = torch.arange(128, device="cuda") % 16 + 0.5
    cache = Cache(pkg, 1, 3, 1, 128, 64)
    seq = torch.zeros(6, dtype=torch.int32, device="cuda")
    pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, seq_dev=seq.data_ptr(), **r.args())
    k, v = cache.read(pkg, seq, r.pos)
    k, v = k[:, 0], v[:, 0]
    assert (k[0] == 2.5).all() and (v[0] == 2.5).all()
    assert torch.isnan(k[1, :64]).all() and torch.isfinite(k[1, 64:]).all() and torch.isnan(v[1, :64]).all() and torch.isfinite(v[1, 64:]).all()
    assert torch.isfinite(k[2]).all() and (k[2] >= -65504).all() and (k[2] <= 65504 * 16).all()
    assert ((k[3] - r.rows[3, 128:256]).abs() <= 2.0 ** -24).all()
    assert torch.equal(k[4], held(r.rows[4, 128:256], 64).float())
    assert torch.equal(v[5], held(r.rows[5, 256:], 64).float())


def test_append_and_read_padding_and_bad_places(pkg):
    r = Rows(50, 2, 1, 128, 128, torch.bfloat16, seed=8, far=2000)
    cache = Cache(pkg, 2, 3, 1, 128, 64)
    seq = torch.arange(50, device="cuda", dtype=torch.int32) % 2
    r.pos.copy_(torch.randperm(768, device="cuda", generator=gen(1))[:50])
    bad = [4, 9, 20, 31, 44]
    r.pos[4], r.pos[9], seq[20], seq[31], r.pos[44] = -5, 768, 2, -1, 1999
    cache.table[1, 2] = cache.n
    wrong = (seq == 1) & (r.pos >= 512) & (r.pos < 768)
    wrong[bad] = True
    pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, seq_dev=seq.data_ptr(), **r.args())
    with pytest.raises(pkg.StatusError):
        pkg.ops.device_status(r.status.data_ptr(), stream())
    assert (r.q[wrong] == 7.0).all() and not (r.q[~wrong] == 7.0).all(1).any()
    k, v = cache.read(pkg, seq, r.pos)
    _, kw, vw = r.want()
    assert (k[wrong] == 7.0).all() and (v[wrong] == 7.0).all()
    assert torch.equal(k[~wrong].double(), held(kw.float(), 64)[~wrong]) and torch.equal(v[~wrong].double(), held(vw.float(), 64)[~wrong])


# ------------------------------------------------------------------------------------------------- attention

def put(pkg, cache, seq, pos, k, v):
    """Appends rows k, v [t, hkv, hd] as they are; returns what the cache stands for."""
    t, hkv, hd = k.shape
    rows = torch.cat([torch.zeros(t, hd, device="cuda"), k.flatten(1), v.flatten(1)], 1).contiguous()
    q = torch.empty(t, hd, device="cuda")
    pkg.ops.qk_norm_rope_append_kv4(rows.data_ptr(), 0, rows.shape[1], t, 1, hkv, hd, 0, 0, 0, 0.0, 0, 0, 0, pos.data_ptr(), q.data_ptr(), hd, cache.c, seq.data_ptr(), stream=stream())
    return cache.read(pkg, seq, pos)


class Attention:
    def __init__(self, pkg, lens, counts, hq, hkv, hd, group, typ, seed=0, k_size=1.0, tail=3):
        g = gen(seed)
        self.pkg, self.lens, self.counts, self.dims, self.typ = pkg, lens, counts, (hq, hkv, hd), typ
        per = max(1, -(-max(lens) // 256))
        self.cache = Cache(pkg, len(lens), per, hkv, hd, group, seed)
        seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).cuda()
        pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
        k, v = (torch.randn(max(1, len(seq)), hkv, hd, device="cuda", generator=g) for _ in range(2))
        self.k, self.v = (x.split(lens) for x in put(pkg, self.cache, seq, pos, k_size * k[:len(seq)], v[:len(seq)])) if len(seq) else ([k[:0]] * len(lens), [v[:0]] * len(lens))
        self.tokens = sum(counts)
        self.q = torch.randn(self.tokens + tail, hq * hd + 5, device="cuda", generator=g).to(typ)
        self.out = torch.full((self.tokens + tail, hq * hd + 2), 7.0, device="cuda", dtype=typ)
        self.kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.start = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, device="cuda", dtype=torch.int32)
        self.max_q, self.max_kv = max(1, max(counts)), max(lens)
        need = pkg.ops.attention_kv4_workspace(len(lens), hkv, hd, hq, self.max_q, self.max_kv)
        self.room = torch.zeros(max(16, need), device="cuda", dtype=torch.uint8)
        self.need = need

    def __call__(self, window=0, scale=0.0, plain_start=False):
        hq, hkv, hd = self.dims
        self.pkg.ops.attention_kv4(self.cache.c, self.q.data_ptr(), code_of(self.typ), self.q.shape[1], self.kv_len.data_ptr(), 0 if plain_start else self.start.data_ptr(),
                                   self.tokens if plain_start else self.q.shape[0], self.max_q, self.max_kv, hq, self.out.data_ptr(), self.out.shape[1], self.room.data_ptr() if self.need else 0, self.need,
                                   window=window, scale=scale, status_dev=self.status.data_ptr(), stream=stream())

    def check(self, window=0, scale=0.0, skip=()):
        hq, hkv, hd = self.dims
        used = scale if scale > 0 else hd ** -0.5
        for b, (n, count) in enumerate(zip(self.lens, self.counts)):
            if b in skip or count == 0:
                continue
            rows = slice(int(self.start[b]), int(self.start[b]) + count)
            q = self.q[rows, :hq * hd].double().view(count, hkv, hq // hkv, hd)
            k, v = self.k[b].double(), self.v[b].double()
            x = torch.einsum("thgd,shd->hgts", q, k) * used
            size = torch.einsum("thgd,shd->hgts", q.abs(), k.abs()) * used
            at = torch.arange(n - count, n, device="cuda")[:, None]
            key = torch.arange(n, device="cuda")[None]
            seen = (key <= at) & ((key > at - window) if window > 0 else (key >= 0))
            p = torch.where(seen, torch.softmax(x.masked_fill(~seen, -math.inf), -1), 0.0) if n else x
            want = torch.einsum("hgts,shd->thgd", p, v)
            d = 8 * U * (size.amax() if n else 0) + 2.0 ** -20
            held_in = 3 * 2.0 ** -11 if self.typ == torch.bfloat16 else 2.0 ** -22
            if self.typ == torch.bfloat16 and hd >= 128 and self.max_q * (hq // hkv) >= 16 and n:
                d = d + 6 * 2.0 ** -10 * k.abs().amax() * q.norm(dim=-1).amax() * used
                held_in += 2.0 ** -10
            bound = (2 * d + held_in + 64 * U) * (v.abs().amax() if n else 0)
            got = self.out[rows, :hq * hd].double().view_as(want)
            err = (got - want).abs()
            assert (err <= rounded(bound, want, self.typ)).all(), (b, n, count, err.max().item(), float(bound))
            empty = ~seen.any(-1)
            assert (got[empty] == 0).all()
        assert (self.out[self.tokens:] == 7.0).all() and (self.out[:, hq * hd:] == 7.0).all()


HEADS = [(4, 1, 256, 64), (8, 4, 256, 128), (8, 4, 128, 64), (4, 4, 128, 128), (6, 2, 64, 64), (16, 2, 128, 64), (10, 1, 128, 128), (5, 1, 64, 64)]


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
def test_attention_of_single_tokens(pkg, hq, hkv, hd, group, typ):
    lens = [1, 0, 15, 16, 17, 31, 33, 64, 255, 256, 257, 511, 777, 1300]
    a = Attention(pkg, lens, [1] * len(lens), hq, hkv, hd, group, typ, seed=hd + hq, tail=0)
    for window in (0, 1, 100, 5000):
        a(window=window, plain_start=True)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        a.check(window)
    a(window=-3, scale=0.31)
    a.check(0, 0.31)


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
def test_attention_of_several_tokens(pkg, hq, hkv, hd, group, typ):
    # none, more tokens than positions (the first ones see nothing), all of a sequence, its end
    lens, counts = [5, 300, 3, 0, 70, 600, 257], [5, 0, 7, 2, 1, 33, 4]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd * 3 + hq)
    for window in (0, 1, 7, 300):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        a.check(window)


@pytest.mark.parametrize("hq,hkv,hd,group", HEADS)
@pytest.mark.parametrize("typ", TYPES)
def test_attention_of_chunks(pkg, hq, hkv, hd, group, typ):
    lens, counts = [700, 130, 5, 1025, 0, 64, 300], [700, 129, 5, 300, 9, 100, 1]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=hd * 5 + hq)
    for window in (0, 1, 130):
        a.out.fill_(7.0)
        a(window=window)
        assert pkg.ops.device_status(a.status.data_ptr(), stream()) == 0
        a.check(window)


@pytest.mark.parametrize("hq,hkv,hd,group,lens", [(4, 1, 256, 64, [20001]), (32, 16, 128, 128, [9000, 12, 30000]), (8, 4, 256, 64, [5000] * 3 + [100] * 9), (12, 4, 64, 64, [40000, 1])])
@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
def test_attention_of_long_caches(pkg, hq, hkv, hd, group, lens, typ):
    a = Attention(pkg, lens, [1] * len(lens), hq, hkv, hd, group, typ, seed=len(lens))
    for window in (0, 4096):
        for _ in range(2):                                 # the second call finds the workspace as the first left it
            a.out.fill_(7.0)
            a(window=window)
            a.check(window)
    # long chunks over long caches, and more splits than keys allow for the short ones
    counts = [min(n, 20) for n in lens]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=len(lens) + 1)
    a()
    a.check()


def test_attention_of_peaked_and_flat_scores(pkg):
    for size in (0.0, 12.0):
        a = Attention(pkg, [900, 40], [3, 1], 8, 4, 128, 64, torch.float32, seed=4, k_size=size)
        a()
        a.check()


def test_attention_shows_what_is_not_a_number(pkg):
    """A NaN in a seen row spoils the rows that see it and no others; masked and stale ones do nothing."""
    a = Attention(pkg, [300, 300], [4, 4], 4, 2, 128, 64, torch.float32, seed=6)
    k = torch.randn(1, 2, 128, device="cuda")
    k[0, 0, 3] = float("nan")
    put(pkg, a.cache, torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([298], dtype=torch.int32, device="cuda"), k, k)
    a()
    a.check(skip=(1,))
    got = a.out[4:8, :512].view(4, 4, 128)
    assert torch.isfinite(got[:2]).all() and torch.isfinite(got[:, 2:]).all() and torch.isnan(got[2:, :2]).any()
    a(window=1)                                            # the last token's window no longer holds position 298
    assert torch.isfinite(a.out[7, :512]).all()


@pytest.mark.parametrize("typ", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,hd,group", [(8, 4, 256, 64), (8, 2, 128, 128)])
def test_chunks_show_what_is_not_a_number_and_bad_pages(pkg, typ, hq, hkv, hd, group):
    """As below, at sizes that take the tensor-core kernel: sequence 1 has a NaN in one key, sequence 2 in one value, sequence 3 a
    page outside the pool."""
    lens, counts = [900, 700, 900, 800], [600, 500, 800, 300]
    a = Attention(pkg, lens, counts, hq, hkv, hd, group, typ, seed=12)
    one = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")               # noqa: E731
    k, v = torch.randn(1, hkv, hd, device="cuda"), torch.randn(1, hkv, hd, device="cuda")
    k[0, 0, 3] = float("nan")
    put(pkg, a.cache, one(1), one(650), k, v)
    k[0, 0, 3], v[0, 1, hd - 1] = 0.0, float("inf")
    put(pkg, a.cache, one(2), one(500), k, v)
    a.cache.table[3, 2] = -7
    a()
    with pytest.raises(pkg.StatusError) as e:
        pkg.ops.device_status(a.status.data_ptr(), stream())
    assert e.value.code == pkg.INVALID_ARGUMENT
    a.check(skip=(1, 2, 3))
    g = hq // hkv
    rows = lambda b: a.out[int(a.start[b]):int(a.start[b]) + counts[b], :hq * hd].view(counts[b], hq, hd)      # noqa: E731
    for b, pos, head in ((1, 650, 0), (2, 500, 1)):
        sees = torch.arange(lens[b] - counts[b], lens[b], device="cuda") >= pos
        bad = torch.isnan(rows(b)[:, head * g:(head + 1) * g]).any(-1)
        assert bad[sees].all() and not bad[~sees].any()
        others = [h for h in range(hq) if h // g != head]
        assert torch.isfinite(rows(b)[:, others]).all()
    # tiles of rows that do not reach the bad page may be served; those that do are left alone
    last = rows(3)[-60:]
    assert (last == 7.0).all()


def test_attention_reports_bad_lengths_and_pages(pkg):
    a = Attention(pkg, [300, 400, 500, 200, 600], [1, 2, 3, 1, 1], 4, 2, 128, 64, torch.bfloat16, seed=9)
    a.kv_len[1], a.kv_len[3] = 601, -1
    a.cache.table[4, 1] = a.cache.n
    a()
    with pytest.raises(pkg.StatusError) as e:
        pkg.ops.device_status(a.status.data_ptr(), stream())
    assert e.value.code == pkg.INVALID_ARGUMENT
    a.check(skip=(1, 3, 4))
    assert (a.out[1:3] == 7.0).all() and (a.out[6] == 7.0).all()
    a.kv_len.copy_(torch.tensor(a.lens))
    a.cache.table[4, 1] = a.cache.table[4, 0]
    b = a.start.clone()
    a.start[2], a.start[5] = 0, 100                        # rows that run backwards and past the end
    a.out.fill_(7.0)
    a()
    with pytest.raises(pkg.StatusError):
        pkg.ops.device_status(a.status.data_ptr(), stream())
    a.start.copy_(b)
    assert (a.out[a.tokens:] == 7.0).all()


def test_calls_on_another_stream_and_in_a_graph(pkg):
    """Append and attention captured once, replayed with other rows, lengths and pages in the same places, while another workspace
    serves calls on another stream."""
    hq, hkv, hd = 8, 4, 128
    a = Attention(pkg, [3000, 700], [1, 1], hq, hkv, hd, 64, torch.bfloat16, seed=2, tail=0)
    b = Attention(pkg, [9000], [1], hq, hkv, hd, 64, torch.bfloat16, seed=3, tail=0)
    a()
    a.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a()
    g = gen(5)
    for i in range(3):
        a.q.copy_(torch.randn(a.q.shape, device="cuda", generator=g))
        lens = [3000 - 700 * i, 300 * i + 1]
        a.kv_len.copy_(torch.tensor(lens))
        a.out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b()
        graph.replay()
        torch.cuda.synchronize()
        full_k, full_v, full = a.k, a.v, a.lens
        a.k, a.v, a.lens = [x[:n] for x, n in zip(a.k, lens)], [x[:n] for x, n in zip(a.v, lens)], lens
        a.check()
        a.k, a.v, a.lens = full_k, full_v, full
        b.check()


def test_workspace_is_asked_for_and_checked(pkg):
    a = Attention(pkg, [30000], [1], 4, 1, 256, 64, torch.float32, seed=1)
    assert a.need == pkg.ops.attention_kv4_workspace(1, 1, 256, 4, 1, 30000)
    for smaller in [(1, 1, 256, 4, 1, 5000), (1, 1, 256, 4, 1, 0)]:
        assert pkg.ops.attention_kv4_workspace(*smaller) <= a.need
    sizes = [pkg.ops.attention_kv4_workspace(b, 4, 128, 8, q, 9000) for b in (1, 7, 64, 300, 3000) for q in (1, 40)]
    assert sizes[0::2] == sorted(sizes[0::2]) and sizes[1::2] == sorted(sizes[1::2])      # a larger one serves smaller calls
    if a.need:
        for ptr, size in ((0, a.need), (a.room.data_ptr(), a.need - 1)):
            with pytest.raises(pkg.StatusError) as e:
                pkg.ops.attention_kv4(a.cache.c, a.q.data_ptr(), 0, a.q.shape[1], a.kv_len.data_ptr(), 0, 1, 1, 30000, 4, a.out.data_ptr(), a.out.shape[1], ptr, size)
            assert e.value.code == pkg.INVALID_ARGUMENT


# ------------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("hidden,hq,hkv,hd", [(1152, 4, 1, 256), (520, 8, 4, 128)])
def test_the_attention_half_of_a_layer(pkg, hidden, hq, hkv, hd):
    """QKV product -> norm, rotation and append -> attention -> output product, six steps of three sessions, against 64 bits that
    use the cache's own values."""
    g, cols, steps, group = gen(hidden), 3, 6, 64
    width = (hq + 2 * hkv) * hd

    def weights(n, k):
        q = torch.randint(-8, 8, (n, k), device="cuda", generator=g)
        s = (0.01 * torch.rand(n, -(-k // group), device="cuda", generator=g) + 1e-3).bfloat16()
        nib = (q & 15).to(torch.uint8).cpu().numpy()
        img = torch.from_numpy(pkg.ops.repack_w4_grouped(nib[:, 0::2] | nib[:, 1::2] << 4, s.view(torch.int16).cpu().numpy(), None, group)).cuda()
        return img, q.double() * s.double().repeat_interleave(group, 1)[:, :k]

    w_in, d_in = weights(width, hidden)
    w_out, d_out = weights(hidden, hq * hd)
    r = Rows(cols, hq, hkv, hd, hd, torch.float32, seed=1, far=300)
    cache = Cache(pkg, cols, 2, hkv, hd, group)
    out, y = torch.empty(cols, hq * hd, device="cuda"), torch.empty(cols, hidden, device="cuda")
    need = pkg.ops.attention_kv4_workspace(cols, hkv, hd, hq, 1, 300)
    room = torch.zeros(max(16, need), device="cuda", dtype=torch.uint8)
    first = torch.tensor([0, 250, 100], dtype=torch.int32, device="cuda")
    fill = torch.randn(350, 2, hkv, hd, device="cuda", generator=g)
    seq = torch.tensor([1] * 250 + [2] * 100, dtype=torch.int32, device="cuda")
    put(pkg, cache, seq, torch.cat([torch.arange(250), torch.arange(100)]).to(torch.int32).cuda(), fill[:, 0].contiguous(), fill[:, 1].contiguous())
    for step in range(steps):
        x = torch.randn(cols, hidden, device="cuda", generator=g)
        r.pos.copy_(first + step)
        kv_len = r.pos + 1
        pkg.ops.gemv_w4_grouped(w_in.data_ptr(), x.data_ptr(), r.buf.data_ptr(), width, hidden, group, ncols=cols, scale_type=1, stream=stream())
        pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, **r.args())
        pkg.ops.attention_kv4(cache.c, r.q.data_ptr(), 0, hq * hd, kv_len.data_ptr(), 0, cols, 1, 300, hq, out.data_ptr(), hq * hd, room.data_ptr(), need, status_dev=r.status.data_ptr(), stream=stream())
        pkg.ops.gemv_w4_grouped(w_out.data_ptr(), out.data_ptr(), y.data_ptr(), hidden, hq * hd, group, ncols=cols, scale_type=1, stream=stream())
        assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
        rows = x.double() @ d_in.T
        assert ((r.rows.double() - rows).norm() <= 1e-6 * rows.norm()).item()
        at = r.pos.long()
        qw = norm_rope(rows.view(cols, -1, hd)[:, :hq], r.q_gain, r.cos[at], r.sin[at], hd)
        for b in range(cols):
            n = int(kv_len[b])
            k, v = cache.read(pkg, torch.full((n,), b, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda"))
            p = torch.softmax(torch.einsum("hgd,shd->hgs", qw[b].view(hkv, -1, hd), k.double()) / hd ** 0.5, -1)
            want = torch.einsum("hgs,shd->hgd", p, v.double()).flatten()
            assert ((out[b].double() - want).norm() <= 2e-5 * want.norm()).item()
            want = want @ d_out.T
            assert ((y[b].double() - want).norm() <= 4e-5 * want.norm()).item()


def test_the_chain_in_a_graph_repeats_bit_for_bit(pkg):
    """Product -> append -> attention -> product captured once: replays give the bits of the plain calls, step after step, with the
    tokens' positions, page table and inputs changed in place.  Sums have a fixed order, the joins of shares too."""
    g, cols, hidden, hq, hkv, hd, group, high = gen(77), 5, 1152, 8, 4, 128, 64, 5000
    width = (hq + 2 * hkv) * hd
    images = []
    for n, k in ((width, hidden), (hidden, hq * hd)):
        nib = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8).cpu().numpy()
        scale = (0.01 * torch.rand(n, -(-k // group), device="cuda", generator=g) + 1e-3).half()
        images.append(torch.from_numpy(pkg.ops.repack_w4_grouped(nib, scale.view(torch.int16).cpu().numpy(), None, group)).cuda())
    cache = Cache(pkg, cols, 20, hkv, hd, group, fill=0x11)
    r = Rows(cols, hq, hkv, hd, hd, torch.bfloat16, seed=3, far=high)
    x = torch.empty(cols, hidden, device="cuda", dtype=torch.bfloat16)
    out, y = torch.empty(cols, hq * hd, device="cuda", dtype=torch.bfloat16), torch.empty(cols, hidden, device="cuda")
    kv_len = torch.empty(cols, device="cuda", dtype=torch.int32)
    need = pkg.ops.attention_kv4_workspace(cols, hkv, hd, hq, 1, high)
    room = torch.zeros(need, device="cuda", dtype=torch.uint8)

    def chain():
        pkg.ops.gemv_w4_grouped(images[0].data_ptr(), x.data_ptr(), r.buf.data_ptr(), width, hidden, group, ncols=cols, x_type=1, y_type=1, stream=stream())
        pkg.ops.qk_norm_rope_append_kv4(cache=cache.c, **{**r.args(), "stream": stream()})
        pkg.ops.attention_kv4(cache.c, r.q.data_ptr(), 1, hq * hd, kv_len.data_ptr(), 0, cols, 1, high, hq, out.data_ptr(), hq * hd, room.data_ptr(), need, status_dev=r.status.data_ptr(), stream=stream())
        pkg.ops.gemv_w4_grouped(images[1].data_ptr(), out.data_ptr(), y.data_ptr(), hidden, hq * hd, group, ncols=cols, x_type=1, stream=stream())

    def step(i):
        torch.manual_seed(i)
        x.copy_(torch.randn(cols, hidden))
        r.pos.copy_(torch.tensor([7 + i, 300 + i, 1279 + i, 2600 + i, 4900 + i]))
        kv_len.copy_(r.pos + 1)
        torch.cuda.synchronize()

    step(0)
    chain()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        chain()
    for i in range(4):
        step(i)
        got = []
        for run in (chain, graph.replay, chain, graph.replay):
            y.fill_(7.0)
            run()
            torch.cuda.synchronize()
            got.append((y.clone(), out.clone(), cache.pages.clone()))
        assert torch.isfinite(got[0][0]).all() and (got[0][0] != 7.0).any()
        for other in got[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    assert pkg.ops.device_status(r.status.data_ptr(), stream()) == 0
