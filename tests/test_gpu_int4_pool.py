"""The 4-bit paged pool: per-head norm + rotation + quantised write, read-back, decode / verify attention and
prompt chunks, against their formulas in 64 bits.

Tolerances (a rounding is off by at most half a step, eps / 2 of its type: bf16 2^-8, fp16 2^-11, f32 2^-24):
  codes, scales, read-back   equal (codes are those of exact arithmetic, the scale is one rounding)
  q_rot                      2^-8 |exact| for the store, and 12 f32 roundings (square sum, root, weight, rotation) of the
                             pair's larger value: 12 * 2^-24 * 2 max(|a|, |b|)
  attention                  2^-8 |exact| for the store; P is fp16: 2^-11 sum p |v|; q is a 16-bit integer round(q 32639 /
                             max |q|), off by at most max |q| / 65278 < 1.01 2^-17 2 max |q|, times |c| <= 7, and a logit is
                             three f32 roundings of an exact integer: p is off by twice dl, 2 dl sum p |v|, dl = scale
                             max(s_k) (7 d 1.01 2^-16 max |q| + 4 * 2^-24 * 7 sum |q|), and by 2^-20 for exp2; the sums over
                             u = c + 8 instead of c add at most 16 sum p s_v (steps + 16) 2^-23, steps = 16-position steps of
                             a warp; and what lies below the range of fp16: p s_v is kept times mult >= 2^8 / max(s_v) in
                             steps of 2^-24, so each of the n positions is off by at most 2^-25 / mult <= 2^-33 max(s_v),
                             times |c| <= 7, over a sum of p of at least 1: 7 n 2^-33 max(s_v)
  prefill through the 8-bit kernels (32 rows and more): that form's own bar, 0.01 + 2^-8 |exact|, tests/test_gpu_attn_prefill_tc.py
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TOP = {4: 7, 8: 127}
EPS = float(np.float32(1e-6))


@pytest.fixture(scope="module")
def K():
    import granite4_b200  # noqa: F401
    from granite4_b200 import capi, kernels
    capi.lib()
    yield kernels
    assert capi.lib().device_status() == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def tables(max_pos, d):
    freq = 1e7 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    a = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * freq
    return a.cos().float(), a.sin().float()


def pack(c):
    u = (c + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def unpack(u):
    return torch.stack((u & 15, u >> 4), -1).flatten(-2).to(torch.int8) - 8


def quantise64(x, bits):
    """(codes int8, scale f32) of float64 rows."""
    s = (x.abs().amax(-1) / TOP[bits]).float()
    t = torch.where(s[..., None] > 0, x.abs() / s.double()[..., None], 0.0)
    return (torch.floor(t + 0.5).clamp(max=TOP[bits]) * torch.sign(x)).to(torch.int8), s


def write64(qkv, wq, wk, cos, sin, pos, Hq, Hk, d, bits):
    rows = qkv.shape[0]
    q, k, v = qkv.double().view(rows, Hq + 2 * Hk, d).split((Hq, Hk, Hk), 1)
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]

    def turned(x, w):
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)
    q = turned(q, wq)
    return q, *quantise64(turned(k, wk), bits), *quantise64(v, bits)


class Pool:
    def __init__(self, stride, Hk, d, bits, fill=0x5A):
        width = d // 2 if bits == 4 else d
        kind = torch.uint8 if bits == 4 else torch.int8
        self.ck, self.cv = (torch.full((Hk, stride, width), fill, dtype=kind, device=DEV) for _ in range(2))
        self.ks, self.vs = (torch.full((Hk, stride), float("nan"), device=DEV) for _ in range(2))
        self.all = (self.ck, self.cv, self.ks, self.vs)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("norm", ["both", "q", "k", "none"])
@pytest.mark.parametrize("rows,Hq,Hk,d", [(1, 32, 8, 128), (3, 4, 4, 64), (16, 32, 8, 128), (17, 5, 1, 128), (37, 16, 2, 64),
                                          (500, 32, 8, 128), (2500, 24, 8, 64), (1003, 40, 16, 128)])
def test_write_equals_the_formula(K, rows, Hq, Hk, d, norm, bits):
    g = gen(rows * 7 + d + bits)
    stride, max_pos = rows + 29, rows + 1000
    qkv = torch.randn(rows, (Hq + 2 * Hk) * d, generator=g, device=DEV).to(torch.bfloat16)
    qkv.view(rows, -1, d)[:, ::3] *= 37.0
    qkv.view(rows, -1, d)[rows // 2, -1] = 0  # a value head of zeros
    qkv.view(rows, -1, d)[rows // 3, Hq] = 0  # a key head of zeros
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2))
    wq, wk = (wq if norm in ("both", "q") else None), (wk if norm in ("both", "k") else None)
    cos, sin = tables(max_pos, d)
    pos = torch.randint(0, max_pos, (rows,), generator=g, device=DEV, dtype=torch.int32)
    kvr = torch.randperm(stride, generator=g, device=DEV)[:rows].to(torch.int32)
    p = Pool(stride, Hk, d, bits)
    before = [t.clone() for t in p.all]
    q_rot = torch.full((rows + 1, Hq * d), 3.0, dtype=torch.bfloat16, device=DEV)
    assert K.qk_norm_rope_kv_paged(qkv, wq, wk, EPS, cos, sin, pos, kvr, Hq, Hk, d, stride, max_pos, bits, q_rot[:rows],
                                   *p.all) == 0
    q, ck, sk, cv, sv = write64(qkv, wq, wk, cos, sin, pos, Hq, Hk, d, bits)
    got = q_rot[:rows].double().view(rows, Hq, d)
    pair = torch.maximum(q[..., : d // 2].abs(), q[..., d // 2:].abs()).repeat(1, 1, 2)
    assert ((got - q).abs() <= 2.0**-8 * q.abs() + 24 * 2.0**-24 * pair).all()
    assert (q_rot[rows] == 3.0).all()
    at = kvr.long()
    for cache, scale, codes, s in ((p.ck, p.ks, ck, sk), (p.cv, p.vs, cv, sv)):
        assert torch.equal(scale[:, at], s.t())
        have = cache[:, at].transpose(0, 1)
        assert torch.equal(unpack(have) if bits == 4 else have, codes)
    rest = torch.ones(stride, dtype=torch.bool, device=DEV)
    rest[at] = False
    for t, b in zip(p.all, before):
        assert torch.equal(t[:, rest].nan_to_num(-1.0) if t.is_floating_point() else t[:, rest],
                           b[:, rest].nan_to_num(-1.0) if b.is_floating_point() else b[:, rest])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_codes_between_two_steps(K, d, bits):
    """Values that lie exactly on the border of two codes, or a rounding of the scale away from it: every bf16 mantissa
    of amax, values amax (2 k + 1) / (2 top) rounded both ways; subnormal and huge rows."""
    rows, Hk = 128 * 5, 1
    m = torch.arange(128, device=DEV)
    amax = torch.cat([((e << 7) | m).to(torch.int16) for e in (1, 60, 127, 128, 250)]).view(torch.bfloat16)
    k2 = 2 * torch.arange(TOP[bits], device=DEV) + 1
    steps = (amax.double()[:, None] * k2 / (2 * TOP[bits])).repeat(1, -(-d // k2.numel()))[:, : d - 1]
    v = torch.cat((amax[:, None], steps.to(torch.bfloat16)), 1)
    v[:, 1::2] *= -1
    v[:, 2::3] = torch.nextafter(v[:, 2::3], torch.zeros_like(v[:, 2::3]))
    qkv = torch.zeros(rows, 3, d, dtype=torch.bfloat16, device=DEV)
    qkv[:, 2] = v
    qkv[:, 1] = v  # not normed, at position 0: the rotation leaves K as it is
    cos, sin = tables(8, d)
    zero = torch.zeros(rows, dtype=torch.int32, device=DEV)
    p = Pool(rows, Hk, d, bits)
    q_rot = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    at = torch.arange(rows, dtype=torch.int32, device=DEV)
    assert K.qk_norm_rope_kv_paged(qkv.view(rows, -1), None, None, EPS, cos, sin, zero, at, 1, Hk, d, rows, 8, bits, q_rot,
                                   *p.all) == 0
    codes, s = quantise64(v.double(), bits)
    for cache, scale in ((p.ck, p.ks), (p.cv, p.vs)):
        assert torch.equal(scale[0], s)
        assert torch.equal(unpack(cache[0]) if bits == 4 else cache[0], codes)


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_out_of_range_are_skipped_and_read_as_zeros(K, bits):
    Hq, Hk, d, stride, max_pos, rows = 8, 2, 128, 40, 16, 6
    g = gen(bits)
    qkv = torch.randn(rows, (Hq + 2 * Hk) * d, generator=g, device=DEV).to(torch.bfloat16)
    cos, sin = tables(max_pos, d)
    pos = torch.tensor([0, -1, 16, 15, 3, 4], dtype=torch.int32, device=DEV)
    kvr = torch.tensor([5, 6, 7, 40, -3, 39], dtype=torch.int32, device=DEV)
    p = Pool(stride, Hk, d, bits)
    q_rot = torch.full((rows, Hq * d), 3.0, dtype=torch.bfloat16, device=DEV)
    assert K.qk_norm_rope_kv_paged(qkv, None, None, EPS, cos, sin, pos, kvr, Hq, Hk, d, stride, max_pos, bits, q_rot,
                                   *p.all) == 0
    assert [(q_rot[r] == 3.0).all().item() for r in range(rows)] == [False, True, True, True, True, False]
    written = [r for r in range(stride) if not p.ks[0, r].isnan()]
    assert written == [5, 39]
    ko, vo = (torch.full((4, Hk, d), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    want = torch.tensor([39, -1, 40, 5], dtype=torch.int32, device=DEV)
    assert K.kv_read_paged(*p.all, want, bits, Hk, d, stride, ko, vo) == 0
    assert (ko[1:3] == 0).all() and (vo[1:3] == 0).all() and ko[0].any() and vo[3].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,Hk,d", [(1, 8, 128), (1, 1, 64), (33, 3, 64), (777, 8, 128), (5000, 5, 128)])
def test_read_back(K, rows, Hk, d, bits):
    g = gen(rows + bits)
    stride = rows // 2 + 7  # rows repeat
    p = Pool(stride, Hk, d, bits)
    low, high = (-7, 8) if bits == 4 else (-127, 128)
    codes = [torch.randint(low, high, (Hk, stride, d), generator=g, device=DEV).to(torch.int8) for _ in range(2)]
    for c, x in zip((p.ck, p.cv), codes):
        c.copy_(pack(x) if bits == 4 else x)
    for s in (p.ks, p.vs):
        s.copy_(torch.rand(Hk, stride, generator=g, device=DEV) * 10.0 ** torch.randint(-6, 6, (Hk, stride), generator=g, device=DEV))
    at = torch.randint(0, stride, (rows,), generator=g, device=DEV, dtype=torch.int32)
    outs = [torch.full((rows + 1, Hk, d), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    assert K.kv_read_paged(*p.all, at, bits, Hk, d, stride, outs[0][:rows], outs[1][:rows]) == 0
    for o, c, s in zip(outs, codes, (p.ks, p.vs)):
        want = (c[:, at.long()].float() * s[:, at.long()][..., None]).transpose(0, 1)
        assert torch.equal(o[:rows], want.to(torch.bfloat16))
        assert (o[rows] == 9.0).all()


# ---- attention ------------------------------------------------------------------------------------------------
def random_pool(stride, Hk, d, g, spread=0.0):
    p = Pool(stride, Hk, d, 4)
    codes = [torch.randint(-7, 8, (Hk, stride, d), generator=g, device=DEV).to(torch.int8) for _ in range(2)]
    for c, x in zip((p.ck, p.cv), codes):
        c.copy_(pack(x))
    for s in (p.ks, p.vs):
        s.copy_((torch.rand(Hk, stride, generator=g, device=DEV) + 0.5) * 0.2 *
                torch.exp2(spread * torch.randn(Hk, stride, generator=g, device=DEV)))
    return p, codes


def attention64(q, p, codes, tables_, row_pos, per, Hq, Hk, d, scale, window, steps):
    """(exact, tolerance) [rows, Hq, d]; tables_[s]: pool rows of sequence s."""
    rows, G = q.shape[0], Hq // Hk
    out, tol = (torch.zeros(rows, Hq, d, dtype=torch.float64, device=DEV) for _ in range(2))
    qd = q.double().view(rows, Hq, d)
    for r in range(rows):
        pos = int(row_pos[r])
        if pos < 0:
            continue
        lo = max(0, pos + 1 - window) if window else 0
        at = tables_[r // per][lo:pos + 1].long()
        for h in range(Hk):
            k = codes[0][h, at].double() * p.ks[h, at].double()[:, None]
            v = codes[1][h, at].double() * p.vs[h, at].double()[:, None]
            x = qd[r, h * G:(h + 1) * G]
            w = torch.softmax(scale * x @ k.t(), -1)
            dl = abs(scale) * p.ks[h, at].max().double() * (7 * d * 1.01 * 2.0**-16 * x.abs().amax(-1) +
                                                            28 * 2.0**-24 * x.abs().sum(-1))
            e = w @ v
            off = 2.0**-8 * e.abs() + (2.0**-11 + 2.0**-20 + 2 * dl)[:, None] * (w @ v.abs())
            off += 16 * (steps + 16) * 2.0**-23 * (w @ p.vs[h, at].double())[:, None]
            off += 7 * len(at) * 2.0**-33 * p.vs[h, at].max().double()
            out[r, h * G:(h + 1) * G], tol[r, h * G:(h + 1) * G] = e, off
    return out, tol


def addresses(tabs, per, rows):
    base = torch.tensor([t.data_ptr() for t in tabs], dtype=torch.int64, device=DEV)
    return base[torch.arange(rows, device=DEV) // per].contiguous()


def run_attention(K, seqs, per, ctxs, Hq, Hk, d, window=0, empty=(), seed=0, scale=None, spread=0.0, max_len=None,
                  scratch="none", sigma=2.0):
    """Sequences of ctxs[s] positions, their last `per` rows as queries; pages anywhere in the pool, everything that is
    not a position of theirs poisoned (NaN scales)."""
    g = gen(seed * 1000003 + sum(ctxs) + d)
    scale = scale or 1.0 / 64
    rows, G = seqs * per, Hq // Hk
    max_len = max_len or max(max(ctxs), 1)
    stride = sum(-(-c // 16) * 16 for c in ctxs) + 48
    p, codes = random_pool(stride, Hk, d, g, spread)
    order = torch.randperm(stride, generator=g, device=DEV).to(torch.int32)
    tabs, used = [], 0
    for c in ctxs:
        t = torch.full((max_len,), 0x7FFFFFF0, dtype=torch.int32, device=DEV)  # entries past the end mean nothing
        t[:c] = order[used:used + c]
        used += c
        tabs.append(t)
    p.ks[:, order[used:].long()] = float("nan")
    p.vs[:, order[used:].long()] = float("nan")
    pos = torch.cat([torch.arange(c - per, c, device=DEV) for c in ctxs]).to(torch.int32)
    for s in empty:
        pos[s * per:(s + 1) * per] = -1 - s
    q = (sigma * torch.randn(rows, Hq * d, generator=g, device=DEV)).to(torch.bfloat16)
    out = torch.full((rows + 1, Hq * d), 3.0, dtype=torch.bfloat16, device=DEV)
    need = K.attn_decode_int4_scratch_bytes(rows, per, Hq, Hk, d, max_len)
    assert need >= 0
    buf = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device=DEV) if scratch == "poisoned" else None
    assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, stride, max_len, scale, out[:rows], rows_per_group=per,
                                    row_pt=addresses(tabs, per, rows), window=window, scratch=buf) == 0
    steps = 2 * -(-max(ctxs) // 32)
    want, tol = attention64(q, p, codes, tabs, pos, per, Hq, Hk, d, scale, window, steps)
    got = out[:rows].double().view(rows, Hq, d)
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, worst
    for s in empty:
        assert (out[s * per:(s + 1) * per] == 0).all()
    assert (out[rows] == 3.0).all()
    return got


HEADS = [(32, 8, 128), (16, 2, 64), (8, 8, 128), (24, 8, 64), (16, 1, 128), (3, 1, 64), (64, 2, 128), (40, 8, 128)]


@pytest.mark.parametrize("Hq,Hk,d", HEADS)
@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 1000, 4099])
def test_decode_one_sequence(K, Hq, Hk, d, ctx):
    run_attention(K, 1, 1, [ctx], Hq, Hk, d, scratch="poisoned", seed=Hq)


@pytest.mark.parametrize("Hq,Hk,d", HEADS)
def test_decode_ragged_batch_with_idle_slots(K, Hq, Hk, d):
    run_attention(K, 7, 1, [1, 4000, 33, 64, 2049, 700, 16], Hq, Hk, d, empty=(0, 4), scratch="poisoned")
    run_attention(K, 3, 1, [5, 9, 40], Hq, Hk, d, empty=(0, 1, 2), max_len=5000)  # nothing to attend to at all


@pytest.mark.parametrize("per", [2, 3, 4, 5])
@pytest.mark.parametrize("Hq,Hk,d", [(32, 8, 128), (8, 8, 64), (24, 8, 64), (16, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("window", [0, 1, 2, 40, 700])
def test_verify_groups_and_windows(K, Hq, Hk, d, per, window):
    if per * Hq // Hk > 64:
        pytest.skip("more columns than a group has")
    run_attention(K, 4, per, [per, 700, 33 + per, 2500], Hq, Hk, d, window=window, empty=(1,), seed=per, scratch="poisoned")


@pytest.mark.parametrize("seqs,ctx", [(300, 200), (1100, 130), (64, 40), (130, 4000)])
def test_many_sequences(K, seqs, ctx):
    """More segments than CTAs, more groups than a launch scans, caches of one tile a warp."""
    ctxs = [max(1, (ctx * (i % 7 + 1)) // 7) for i in range(seqs)]
    run_attention(K, seqs, 1, ctxs, 8, 2, 64, empty=(3,), max_len=ctx)


@pytest.mark.parametrize("Hq,Hk,d", HEADS)
def test_forms_agree(K, monkeypatch, Hq, Hk, d):
    """A segment by one cluster, or with clusters off by shares of the line or one CTA: each within the bound."""
    for seqs, per, ctxs in ((2, 1, [3000, 1]), (5, 1, [700, 33, 1500, 900, 64]), (1, 1, [260])):
        for off in ("0", "1"):
            monkeypatch.setenv("G4_CLUSTER", off)
            run_attention(K, seqs, per, ctxs, Hq, Hk, d, empty=(1,) if seqs > 1 else (), scratch="poisoned", seed=3)
            run_attention(K, seqs, per, ctxs, Hq, Hk, d, max_len=20000, scratch="poisoned", seed=4)


def test_long_cache_of_one_kv_head(K):
    run_attention(K, 1, 1, [120000], 16, 1, 128, scratch="poisoned", sigma=0.5)
    run_attention(K, 2, 2, [60001, 3], 8, 4, 64, scratch="poisoned", sigma=0.5)


@pytest.mark.parametrize("spread", [4.0, 12.0])
def test_scales_over_many_magnitudes(K, spread):
    """Row scales from 2^-3 spread to 2^+3 spread: the largest comes late or early, a tile or the cache apart."""
    for seed in range(4):
        run_attention(K, 2, 1, [3000, 900], 32, 8, 128, seed=seed, spread=spread, scale=2.0**-spread / 256)


def test_zero_scales_and_peaked_softmax(K):
    Hq, Hk, d, n = 32, 8, 128, 600
    g = gen(1)
    p, codes = random_pool(n, Hk, d, g)
    p.vs[:, :400] = 0.0
    p.ks[:, 100:200] = 0.0
    q = (60 * torch.randn(1, Hq * d, generator=g, device=DEV)).to(torch.bfloat16)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    tab = torch.arange(n, dtype=torch.int32, device=DEV)
    for scale in (1.0, -1.0, 1e-30, 1.0 / 64):
        out = torch.empty(1, Hq * d, dtype=torch.bfloat16, device=DEV)
        assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, scale, out) == 0
        want, tol = attention64(q, p, codes, [tab], pos, 1, Hq, Hk, d, scale, 0, 40)
        assert ((out.double().view(1, Hq, d) - want).abs() <= tol).all(), scale


def test_a_table_for_all_rows_identity_and_positions_past_max_len(K):
    Hq, Hk, d, n = 8, 2, 128, 500
    g = gen(5)
    p, codes = random_pool(n, Hk, d, g)
    q = torch.randn(3, Hq * d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([499, 3, 1200], dtype=torch.int32, device=DEV)  # the last counts as max_len - 1
    perm = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    for tab in (None, perm):
        out = torch.empty(3, Hq * d, dtype=torch.bfloat16, device=DEV)
        assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, 0.05, out, pt=tab) == 0
        t = torch.arange(n, device=DEV) if tab is None else tab
        want, tol = attention64(q, p, codes, [t] * 3, pos.clamp(max=n - 1), 1, Hq, Hk, d, 0.05, 0, 40)
        assert ((out.double().view(3, Hq, d) - want).abs() <= tol).all()


@pytest.mark.parametrize("n", [60, 900, 30000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_head_that_is_not_a_number_stays_one(K, n, bad):
    Hq, Hk, d = 32, 8, 128
    g = gen(n)
    p, _ = random_pool(n, Hk, d, g)
    q = torch.randn(2, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([n - 1, n - 2], dtype=torch.int32, device=DEV)
    outs = []
    for spoilt in (False, True):
        if spoilt:
            q[1, 5, 17] = bad
        out = torch.empty_like(q)
        assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, 0.05, out, rows_per_group=2) == 0
        outs.append(out)
    assert outs[1][1, 5].isnan().all()
    outs[1][1, 5] = outs[0][1, 5]
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("which,bad", [("k", float("nan")), ("v", float("nan")), ("v", float("inf"))])
@pytest.mark.parametrize("n,per,window", [(60, 3, 0), (900, 4, 0), (30000, 3, 0), (5000, 2, 40), (129, 16, 3)])
def test_a_scale_that_is_not_a_number_stays_with_the_rows_that_see_it(K, n, per, window, which, bad):
    Hq, Hk, d, scale = 8, 4, 128, 1.0 / 64
    g = gen(n + per)
    p, codes = random_pool(n, Hk, d, g)
    q = torch.randn(per, Hq * d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.arange(n - per, n, device=DEV, dtype=torch.int32)
    tab = torch.arange(n, dtype=torch.int32, device=DEV)
    want, tol = attention64(q, p, codes, [tab] * per, pos, per, Hq, Hk, d, scale, window, 2 * n // 32 + 2)
    for at in (n - 1, max(0, n - per + 1 - window) if window else n - per + 1):
        t = p.ks if which == "k" else p.vs
        old = t[2, at].item()
        t[2, at] = bad
        out = torch.empty(per, Hq * d, dtype=torch.bfloat16, device=DEV)
        assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, scale, out, rows_per_group=per, window=window) == 0
        t[2, at] = old
        got = out.double().view(per, Hq, d)
        sees = (pos >= at) & (pos - window < at if window else pos >= at)
        hit = sees[:, None] & (torch.arange(Hq, device=DEV) // (Hq // Hk) == 2)[None]
        assert hit.any() and not hit.all()
        assert got[hit].isnan().all()
        assert ((got - want).abs() <= tol)[~hit].all()


def test_output_between_two_words_and_other_streams(K):
    Hq, Hk, d, n = 32, 8, 128, 2000
    g = gen(6)
    p, codes = random_pool(n, Hk, d, g)
    q = torch.randn(1, Hq * d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    want = torch.empty(1, Hq * d, dtype=torch.bfloat16, device=DEV)
    assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, 0.05, want) == 0
    buf = torch.zeros(Hq * d + 1, dtype=torch.bfloat16, device=DEV)
    odd = buf[1:].view(1, -1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, 0.05, odd) == 0
    side.synchronize()
    assert torch.equal(odd, want)


@pytest.mark.parametrize("rows,base", [(1, 0), (1, 77), (5, 1000), (31, 3), (32, 0), (33, 100), (63, 129), (63, 130), (64, 704), (64, 705),
                                       (77, 1203), (130, 5), (192, 3), (193, 3), (600, 2000)])
@pytest.mark.parametrize("Hq,Hk,d", [(32, 8, 128), (16, 2, 64), (6, 6, 128)])
def test_prefill_chunks(K, rows, base, Hq, Hk, d):
    g = gen(rows + base)
    n = base + rows
    stride = n + 60
    p, codes = random_pool(stride, Hk, d, g)
    tab = torch.randperm(stride, generator=g, device=DEV)[:n].to(torch.int32).contiguous()
    spare = torch.ones(stride, dtype=torch.bool, device=DEV)
    spare[tab.long()] = False
    p.ks[:, spare] = float("nan")
    p.vs[:, spare] = float("nan")
    q = torch.randn(rows, Hq * d, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.full((rows + 1, Hq * d), 3.0, dtype=torch.bfloat16, device=DEV)
    scale = 1.0 / 64
    assert K.prefill_attention_int4(q, scale, Hq, Hk, d, base, stride, out[:rows], *p.all, pt=tab) == 0
    pos = torch.arange(base, n, device=DEV)
    pick = torch.unique(torch.cat((torch.arange(min(rows, 20)), torch.arange(max(0, rows - 20), rows))))
    want, tol = attention64(q[pick.to(DEV)], p, codes, [tab] * len(pick), pos[pick.to(DEV)], 1, Hq, Hk, d, scale, 0, 2 * n // 32 + 2)
    if rows >= 32 and Hq == 4 * Hk and d == 128:
        tol = 0.01 + 2.0**-8 * want.abs()
    assert ((out[pick.to(DEV)].double().view(-1, Hq, d) - want).abs() <= tol).all()
    assert (out[rows] == 3.0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("Hq,Hk,d,per", [(32, 8, 128, 4), (16, 2, 64, 3), (8, 8, 64, 7), (32, 8, 128, 16)])
@pytest.mark.parametrize("window", [0, 90])
def test_rows_of_a_group_at_any_positions(K, Hq, Hk, d, per, window):
    """Rows of one sequence in no order, the same position twice, idle rows among them, a last group that is not full."""
    g = gen(per + window)
    n, rows = 900, 2 * per + 1
    p, codes = random_pool(n, Hk, d, g)
    tab = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    pos = torch.randint(0, n, (rows,), generator=g, device=DEV, dtype=torch.int32)
    pos[1], pos[2], pos[per] = -1, pos[0], -7
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    out = torch.full((rows, Hq, d), 3.0, dtype=torch.bfloat16, device=DEV)
    assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, n, 0.03, out, rows_per_group=per, pt=tab, window=window) == 0
    want, tol = attention64(q.view(rows, -1), p, codes, [tab] * 3, pos, per, Hq, Hk, d, 0.03, window, 64)
    assert ((out.double() - want).abs() <= tol).all()
    assert (out[1] == 0).all() and (out[per] == 0).all()


def test_offsets_past_32_bits(K):
    """A pool whose codes, and whose byte offsets within a head's rows, pass 2^31: rows at its ends written, read, attended to."""
    Hq, Hk, d, rows, max_pos = 8, 2, 128, 40, 64
    stride = (1 << 31) // (d // 2) + 1000  # a head's codes alone are over 2 GiB
    g = gen(9)
    p = Pool(stride, Hk, d, 4, fill=0x88)
    qkv = torch.randn(rows, (Hq + 2 * Hk) * d, generator=g, device=DEV).to(torch.bfloat16)
    cos, sin = tables(max_pos, d)
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    kvr = torch.cat((torch.arange(rows // 2, device=DEV), stride - 1 - torch.arange(rows - rows // 2, device=DEV))).to(torch.int32)
    q_rot = torch.empty(rows, Hq * d, dtype=torch.bfloat16, device=DEV)
    assert K.qk_norm_rope_kv_paged(qkv, None, None, EPS, cos, sin, pos, kvr, Hq, Hk, d, stride, max_pos, 4, q_rot, *p.all) == 0
    _, ck, sk, cv, sv = write64(qkv, None, None, cos, sin, pos, Hq, Hk, d, 4)
    ko, vo = (torch.empty(rows, Hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert K.kv_read_paged(*p.all, kvr, 4, Hk, d, stride, ko, vo) == 0
    assert torch.equal(ko, (ck.float() * sk[..., None]).to(torch.bfloat16))
    assert torch.equal(vo, (cv.float() * sv[..., None]).to(torch.bfloat16))
    last = torch.tensor([rows - 1], dtype=torch.int32, device=DEV)
    small = Pool(rows, Hk, d, 4)
    at = torch.arange(rows, dtype=torch.int32, device=DEV)
    for t, s in zip(small.all, p.all):
        t.copy_(s[:, kvr.long()])
    out, want = (torch.empty(1, Hq * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert K.attn_decode_int4_paged(q_rot[-1:], *p.all, last, Hq, Hk, d, stride, rows, 0.05, out, pt=kvr) == 0
    assert K.attn_decode_int4_paged(q_rot[-1:], *small.all, last, Hq, Hk, d, rows, rows, 0.05, want, pt=at) == 0
    assert torch.equal(out, want)
    chunk = torch.empty(rows, Hq * d, dtype=torch.bfloat16, device=DEV)
    assert K.prefill_attention_int4(q_rot, 0.05, Hq, Hk, d, 0, stride, chunk, *p.all, pt=kvr) == 0
    ref = torch.empty_like(chunk)
    assert K.prefill_attention_int4(q_rot, 0.05, Hq, Hk, d, 0, rows, ref, *small.all, pt=at) == 0
    assert torch.equal(chunk, ref)


def test_tensors_too_small_or_of_other_kinds_are_refused(K):
    Hq, Hk, d, n = 8, 2, 128, 64
    p, _ = random_pool(n, Hk, d, gen(1))
    q = torch.zeros(2, Hq * d, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    def call(**kw):
        a = dict(q=q, ck=p.ck, cv=p.cv, ks=p.ks, vs=p.vs, pos=pos, out=torch.empty_like(q))
        a.update(kw)
        return K.attn_decode_int4_paged(a["q"], a["ck"], a["cv"], a["ks"], a["vs"], a["pos"], Hq, Hk, d, n, n, 0.1, a["out"])
    assert call() == 0
    for bad in ({"ck": p.ck[:1]}, {"ks": p.ks[:, :-1].contiguous()}, {"pos": pos[:1]}, {"out": q[:1].clone()}, {"q": q[:, ::2]},
                {"vs": p.vs.cpu()}, {"cv": p.cv[:, :, ::2]}):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in ({"ck": p.ck.view(torch.int8)}, {"pos": pos.long()}, {"q": q.float()}, {"ks": p.ks.double()}):
        with pytest.raises(TypeError):
            call(**bad)
    cos, sin = tables(16, d)
    qkv = torch.zeros(2, (Hq + 2 * Hk) * d, dtype=torch.bfloat16, device=DEV)
    def write(**kw):
        a = dict(qkv=qkv, w=None, cos=cos, kvr=pos, q=torch.empty_like(q), ck=p.ck)
        a.update(kw)
        return K.qk_norm_rope_kv_paged(a["qkv"], a["w"], None, EPS, a["cos"], sin, pos, a["kvr"], Hq, Hk, d, n, 16, 4, a["q"],
                                       a["ck"], p.cv, p.ks, p.vs)
    for bad in ({"qkv": qkv[:, :-8].contiguous()}, {"w": qkv[0, : d - 1].clone()}, {"cos": cos[:8]}, {"kvr": pos[:1]},
                {"q": q[:1].clone()}, {"ck": p.ck[:, :-1].contiguous()}):
        with pytest.raises(ValueError):
            write(**bad)
    with pytest.raises(TypeError):
        write(ck=p.ck.view(torch.int8))
    ko = torch.empty(2, Hk, d, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        K.kv_read_paged(*p.all, pos, 4, Hk, d, n, ko, ko[:1])
    with pytest.raises(ValueError):
        K.prefill_attention_int4(q, 0.1, Hq, Hk, d, 5, n, torch.empty_like(q), *p.all, pt=pos)


def test_repeats_to_the_bit(K):
    a = run_attention(K, 5, 3, [4100, 3000, 2500, 4000, 3300], 32, 8, 128, scratch="poisoned")
    for _ in range(5):
        assert torch.equal(a, run_attention(K, 5, 3, [4100, 3000, 2500, 4000, 3300], 32, 8, 128))


def test_a_decode_loop_captured_into_a_graph(K):
    """Write, attend and read back as a loop of one layer would, with two sessions that grow: eager and replayed steps
    agree to the bit, and the pool's rows are those of the formula."""
    Hq, Hk, d, stride, max_pos, rows, steps = 32, 8, 128, 512, 512, 2, 6
    g = gen(11)
    cos, sin = tables(max_pos, d)
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2))
    inputs = torch.randn(steps, rows, (Hq + 2 * Hk) * d, generator=g, device=DEV).to(torch.bfloat16)
    start, tab = random_pool(stride, Hk, d, g)[0], torch.randperm(stride, generator=g, device=DEV).to(torch.int32).view(2, -1)
    pt = addresses([tab[0], tab[1]], 1, rows)
    first = torch.tensor([100, 7], dtype=torch.int32, device=DEV)
    scratch = torch.empty(K.attn_decode_int4_scratch_bytes(rows, 1, Hq, Hk, d, 256), dtype=torch.uint8, device=DEV)
    results = []
    for graphed in (False, True):
        p = Pool(stride, Hk, d, 4)
        for t, s in zip(p.all, start.all):
            t.copy_(s)
        qkv, pos = inputs[0].clone(), first.clone()
        kvr = torch.empty(rows, dtype=torch.int32, device=DEV)
        q_rot, out = (torch.empty(rows, Hq * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ko, vo = (torch.empty(rows, Hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))

        def step():
            kvr.copy_(tab.gather(1, pos.long()[:, None])[:, 0])
            assert K.qk_norm_rope_kv_paged(qkv, wq, wk, EPS, cos, sin, pos, kvr, Hq, Hk, d, stride, max_pos, 4, q_rot, *p.all) == 0
            assert K.attn_decode_int4_paged(q_rot, *p.all, pos, Hq, Hk, d, stride, 256, 1.0 / 64, out, row_pt=pt,
                                            scratch=scratch) == 0
            assert K.kv_read_paged(*p.all, kvr, 4, Hk, d, stride, ko, vo) == 0
            pos.add_(1)
        if graphed:
            keep = [t.clone() for t in p.all]
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                step()  # warm-up
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            for t, s in zip(p.all, keep):
                t.copy_(s)
            pos.copy_(first)
        seen = []
        for i in range(steps):
            qkv.copy_(inputs[i])
            graph.replay() if graphed else step()
            seen.append([t.clone() for t in (q_rot, out, ko, vo)])
        torch.cuda.synchronize()
        results.append((seen, [t.clone() for t in p.all]))
    for a, b in zip(results[0][0], results[1][0]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(results[0][1], results[1][1]))
    last = steps - 1
    _, ck, sk, cv, sv = write64(inputs[last], wq, wk, cos, sin, first + last, Hq, Hk, d, 4)
    ko, vo = results[0][0][last][2:]
    assert torch.equal(ko, (ck.float() * sk[..., None]).to(torch.bfloat16))
    assert torch.equal(vo, (cv.float() * sv[..., None]).to(torch.bfloat16))


def test_two_captured_calls_at_once(K):
    """Two graphs, of a cut call and of one by clusters, replayed side by side on two streams, each with a scratch of its own."""
    Hq, Hk, d, n = 32, 8, 128, 40000
    g = gen(21)
    p, _ = random_pool(n, Hk, d, g)
    jobs = []
    for rows, per, length in ((1, 1, n), (6, 3, 3000)):
        q = torch.randn(rows, Hq * d, generator=g, device=DEV).to(torch.bfloat16)
        pos = torch.full((rows,), length - 1, dtype=torch.int32, device=DEV) - torch.arange(rows, device=DEV, dtype=torch.int32) % per
        scratch = torch.empty(max(16, K.attn_decode_int4_scratch_bytes(rows, per, Hq, Hk, d, length)), dtype=torch.uint8, device=DEV)
        out = torch.empty_like(q)

        def call(q=q, pos=pos, length=length, per=per, out=out, scratch=scratch):
            assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, Hk, d, n, length, 0.02, out, rows_per_group=per, scratch=scratch) == 0
        call()
        torch.cuda.synchronize()
        want = out.clone()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(20):
                call()
        jobs.append((graph, stream, out, want, call))  # (call keeps what the graph reads)
    for _ in range(5):
        for _, _, out, _, _ in jobs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream, _, _, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, _, out, want, _ in jobs)


def test_kv_move_of_a_4_bit_pool(K):
    Hk, d, stride = 4, 128, 64
    p, _ = random_pool(stride, Hk, d, gen(3))
    before = [t.clone() for t in p.all]
    ck, cv = (t.view(torch.int8).view(1, Hk, stride, d // 2) for t in (p.ck, p.cv))
    assert K.kv_move([5, 9], [2, 3], 8, ck, cv, p.ks.view(1, Hk, stride), p.vs.view(1, Hk, stride), 1, Hk, stride, d // 2) == 0
    for t, b in zip(p.all, before):
        assert torch.equal(t[:, 2], b[:, 5]) and torch.equal(t[:, 3], b[:, 9])
        b[:, 2], b[:, 3] = b[:, 5], b[:, 9]
        assert torch.equal(t, b)


@pytest.mark.parametrize("rows,base", [(20, 5), (40, 0), (130, 2000), (300, 0), (64, 16000)])
@pytest.mark.parametrize("which,bad", [("k", float("nan")), ("v", float("nan")), ("v", float("inf"))])
def test_a_chunk_with_a_scale_that_is_not_a_number(K, rows, base, which, bad):
    """The rows before the position are as without it, to the bit; those that see it NaN."""
    Hq, Hk, d = 32, 8, 128
    g = gen(rows + base)
    n = base + rows
    p, _ = random_pool(n, Hk, d, g)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    outs = []
    first = rows // 2 + 1
    for spoilt in (False, True):
        if spoilt:
            (p.ks if which == "k" else p.vs)[3, base + first] = bad
        out = torch.empty_like(q)
        assert K.prefill_attention_int4(q, 1.0 / 64, Hq, Hk, d, base, n, out, *p.all) == 0
        outs.append(out)
    assert torch.isfinite(outs[0]).all()
    assert outs[1][first:, 12:16].isnan().all()
    assert torch.equal(outs[0][:first], outs[1][:first])
    assert torch.equal(outs[0][:, :12], outs[1][:, :12]) and torch.equal(outs[0][:, 16:], outs[1][:, 16:])


@pytest.mark.parametrize("rows,base", [(40, 0), (130, 2000)])
def test_a_chunk_with_values_past_fp16(K, rows, base):
    """A widened chunk holds V in fp16: a position past its range gives NaN where it is seen and nothing elsewhere."""
    Hq, Hk, d = 32, 8, 128
    g = gen(rows)
    n = base + rows
    p, _ = random_pool(n, Hk, d, g)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    first = rows - 3
    outs = []
    for vs in (1.0, 9300.0, 9400.0):  # times 7: 65100, 65800
        p.vs[3, base + first] = vs
        out = torch.empty_like(q)
        assert K.prefill_attention_int4(q, 1.0 / 64, Hq, Hk, d, base, n, out, *p.all) == 0
        outs.append(out)
    assert torch.isfinite(outs[1]).all()
    assert outs[2][first:, 12:16].isnan().all()
    outs[2][first:, 12:16] = outs[1][first:, 12:16]
    assert torch.equal(outs[1], outs[2]) and torch.equal(outs[0][:first], outs[1][:first])
