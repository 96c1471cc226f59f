"""Attention over the 4-bit pool where row scales and logits are anything but alike: value scales that some rows of a group do
not see, or give no weight to, many magnitudes above the rest; scales over many magnitudes; peaked softmaxes.

The reference, in 64 bits, takes q as the kernel holds it, the 16-bit integer round(q 32639 / max |q|) of its head times max |q|
/ 32639, so that what is left to bound are roundings (a rounding is off by at most half a step: bf16 2^-8, fp16 2^-11, f32
2^-24 of the value):
  store                  2^-8 |exact|
  p v_scale as fp16      2^-11 sum p |v|; its floor: the largest p s is held at 2^10 or more and steps under fp16's normal range
                         are 2^-24, so each of the n positions is off by at most 2^-35 max(p s), times |c| <= 7 (and 1 % for the
                         logarithm that decides on it); a scale counts as 2^-80 at least: 7 n (1.01 2^-35 max(p s) + 2^-115)
  logits                 an exact integer, to f32 (1), times k_scale (scale log2(e) max |q| / 32639) (5, the constant's among
                         them), less a logit in an fma and less a number under 64 (what is left is under 64 for every position
                         whose weight counts): in powers of two under 8 * 2^-24 |l| + 64 * 2^-24; exp2 itself 2^-22; numerator
                         and sum both: twice
  sums                   16 sum p s (steps + 16) 2^-23 over u = c + 8, steps = 16-position steps of a warp
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def K():
    import granite4_b200  # noqa: F401
    from granite4_b200 import capi, kernels
    capi.lib()
    yield kernels
    assert capi.lib().device_status() == 0


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Pool:
    """A 4-bit pool of random codes; k_scale 0.1 to 0.3, v_scale as given or the same."""

    def __init__(self, g, stride, Hk, d, vs=None):
        self.Hk, self.d, self.stride = Hk, d, stride
        self.codes = [torch.randint(-7, 8, (Hk, stride, d), generator=g, device=DEV).to(torch.int8) for _ in range(2)]
        self.ck, self.cv = (((c[..., 0::2] + 8) | ((c[..., 1::2] + 8) << 4)).to(torch.uint8).contiguous() for c in self.codes)
        self.ks = (torch.rand(Hk, stride, generator=g, device=DEV) + 0.5) * 0.2
        self.vs = (torch.rand(Hk, stride, generator=g, device=DEV) + 0.5) * 0.2 if vs is None else vs
        self.all = (self.ck, self.cv, self.ks, self.vs)


def held_q(q):
    """q as the kernel holds it, [rows, Hq, d] float64."""
    top = q.float().abs().amax(-1, keepdim=True).clamp(min=1e-30)
    return torch.round(q.float() * (32639.0 / top)).double() * top.double() / 32639.0


def reference(p, q, pos, scale, window=0, table=None):
    """(exact, bar, sum p |v|), [rows, Hq, d]; q [rows, Hq, d], pos one position per row."""
    rows, Hq, d = q.shape
    G, hq = Hq // p.Hk, held_q(q)
    exact, bar = torch.zeros(rows, Hq, d, dtype=torch.float64, device=DEV), torch.zeros(rows, Hq, d, dtype=torch.float64, device=DEV)
    for r in range(rows):
        last = int(pos[r])
        if last < 0:
            continue
        first = max(0, last + 1 - window) if window else 0
        at = torch.arange(first, last + 1, device=DEV)
        if table is not None:
            at = table[at].long()
        n = len(at)
        k = p.codes[0][:, at].double() * p.ks[:, at].double()[..., None]
        v = p.codes[1][:, at].double() * p.vs[:, at].double()[..., None]
        logits = scale * torch.einsum("hgd,htd->hgt", hq[r].view(p.Hk, G, d), k)
        w = torch.softmax(logits, -1)
        e = torch.einsum("hgt,htd->hgd", w, v)
        mass = torch.einsum("hgt,htd->hgd", w, v.abs())
        ws = w * p.vs[:, at].double()[:, None]
        size = logits.abs().amax(-1) / math.log(2.0)
        rel = 2.0**-11 + 2 * (2.0**-22 + math.log(2.0) * 2.0**-24 * (8 * size + 64))
        steps = 2 * -(-n // 32)
        off = 2.0**-8 * e.abs() + rel[..., None] * mass + (7 * n * (1.01 * 2.0**-35 * ws.amax(-1) + 2.0**-115) + 16 * (steps + 16) * 2.0**-23 * ws.sum(-1))[..., None]
        exact[r], bar[r] = e.view(Hq, d), off.view(Hq, d)
    return exact, bar


def decode(K, p, q, pos, scale, per=1, window=0, max_len=None):
    rows, Hq, d = q.shape
    out = torch.empty_like(q)
    assert K.attn_decode_int4_paged(q, *p.all, pos, Hq, p.Hk, d, p.stride, max_len or p.stride, scale, out, rows_per_group=per,
                                    window=window) == 0
    return out.double()


def check(got, want, bar, sharp):
    """Within the bar, and the bar says something: half of the values are more than `sharp` times as large."""
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / bar.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, worst
    assert (want.abs() / bar.clamp(min=1e-300)).median().item() >= sharp


@pytest.mark.parametrize("loud", [1e6, 1e12, 1e18, 1e28])
@pytest.mark.parametrize("Hq,Hk,d", [(8, 4, 128), (16, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("n,per,window", [(4, 4, 0), (60, 3, 0), (900, 4, 0), (30000, 3, 0), (5000, 2, 40), (129, 4, 3)])
def test_a_large_value_scale_stays_with_the_rows_that_see_it(K, n, per, window, Hq, Hk, d, loud):
    """At the last row's own position, and where a window has left later rows behind."""
    g = gen(n + per + d)
    p = Pool(g, n, Hk, d)
    q = torch.randn(per, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.arange(n - per, n, device=DEV, dtype=torch.int32)
    for at in (n - 1, max(0, n - per + 1 - window) if window else n - per + 1):
        old = p.vs[:, at].clone()
        p.vs[:, at] = loud
        want, bar = reference(p, q, pos, 1.0 / 64, window)
        check(decode(K, p, q, pos, 1.0 / 64, per, window), want, bar, 0.0)
        p.vs[:, at] = old


@pytest.mark.parametrize("n,per", [(33, 1), (700, 2), (30000, 1)])
def test_a_large_value_scale_without_weight(K, n, per):
    """A position whose value is 2^20 - 2^50 times the others' and whose weight is as far below: what is left of it counts,
    and takes nothing from the others, wherever in the cache it lies."""
    Hq, Hk, d = 32, 8, 128
    g = gen(n)
    p = Pool(g, n, Hk, d)
    q = (0.2 * torch.randn(per, Hk, 1, d, generator=g, device=DEV)).expand(per, Hk, Hq // Hk, d).to(torch.bfloat16).contiguous()
    pos = torch.arange(n - per, n, device=DEV, dtype=torch.int32)
    for at in (0, n // 2, n - per):
        for bits in (20, 35, 50):
            # codes of the key against q's signs: a logit far under the others'
            side = -torch.sign(q.float().mean(0)[:, 0]).to(torch.int8) * 7
            keep = [t[:, at].clone() for t in (p.codes[0], p.ck, p.ks, p.vs)]
            p.codes[0][:, at] = side
            p.ck[:, at] = ((side[:, 0::2] + 8) | ((side[:, 1::2] + 8) << 4)).to(torch.uint8)
            size = 7 * q.float().abs().sum(-1).amin() * 0.5
            p.ks[:, at] = bits * math.log(2.0) / (size * 0.25)
            p.vs[:, at] = 0.2 * 2.0**bits
            want, bar = reference(p, q.view(per, Hq, d), pos, 0.25)
            check(decode(K, p, q.view(per, Hq, d), pos, 0.25, per), want, bar, 1.0)
            for t, k in zip((p.codes[0], p.ck, p.ks, p.vs), keep):
                t[:, at] = k


@pytest.mark.parametrize("spread", [2.0, 6.0, 10.0])
@pytest.mark.parametrize("n", [40, 3000, 40000])
@pytest.mark.parametrize("Hq,Hk,d", [(32, 8, 128), (16, 2, 64)])
def test_value_scales_over_many_magnitudes(K, n, spread, Hq, Hk, d):
    """Row scales from 2^-3 spread to 2^+3 spread, the largest anywhere; logits of ordinary size."""
    for seed in range(3):
        g = gen(seed + n)
        vs = 0.2 * torch.exp2((spread * torch.randn(Hk, n, generator=g, device=DEV)).clamp(-35, 50))
        p = Pool(g, n, Hk, d, vs)
        q = torch.randn(2, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
        pos = torch.tensor([n - 1, n // 2], dtype=torch.int32, device=DEV)
        want, bar = reference(p, q, pos, 1.0 / 16)
        check(decode(K, p, q, pos, 1.0 / 16), want, bar, 10.0 if n < 10000 else 2.0)  # (the bound of the sums grows with n)


@pytest.mark.parametrize("small", [1e-3, 1e-6, 1e-9, 1e-11, 1e-16, 1e-22])
def test_small_values_keep_their_bits(K, small):
    Hq, Hk, d = 32, 8, 128
    for n in (50, 2000):
        g = gen(n)
        p = Pool(g, n, Hk, d)
        p.vs *= small
        q = torch.randn(1, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
        pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
        want, bar = reference(p, q, pos, 1.0 / 16)
        check(decode(K, p, q, pos, 1.0 / 16), want, bar, 10.0)


@pytest.mark.parametrize("scale", [0.25, -0.5, 1.0, 4.0])
@pytest.mark.parametrize("n,per,window", [(37, 1, 0), (700, 4, 0), (4099, 3, 500), (40000, 1, 0)])
@pytest.mark.parametrize("Hq,Hk,d", [(32, 8, 128), (16, 2, 64), (16, 1, 128)])
def test_peaked_softmax(K, n, per, window, scale, Hq, Hk, d):
    """Logits spread by 10 to 200 powers of two: few positions count, and the running base moves many times."""
    g = gen(n)
    p = Pool(g, n, Hk, d)
    q = (2.0 * torch.randn(per, Hq, d, generator=g, device=DEV)).to(torch.bfloat16)
    pos = torch.arange(n - per, n, device=DEV, dtype=torch.int32)
    want, bar = reference(p, q, pos, scale, window)
    check(decode(K, p, q, pos, scale, per, window), want, bar, 10.0)


def test_weight_on_values_of_zero(K):
    """The largest weight lies on a position whose value scale is zero; the others' share is 2^-20 and counts in full."""
    Hq, Hk, d, n = 32, 8, 128, 1000
    g = gen(2)
    p = Pool(g, n, Hk, d)
    q = torch.rand(1, Hq, d, generator=g, device=DEV).to(torch.bfloat16) + 0.5
    p.codes[0][:, 7], p.ck[:, 7] = 7, 0xFF
    p.vs[:, 7] = 0.0
    p.ks[:, 7] = 20 * math.log(2.0) / (7 * q.float().sum(-1).mean().item() / 64)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    want, bar = reference(p, q, pos, 1.0 / 64)
    check(decode(K, p, q, pos, 1.0 / 64), want, bar, 10.0)
    p.vs[:] = 0.0
    assert (decode(K, p, q, pos, 1.0 / 64) == 0).all()


@pytest.mark.parametrize("n", [40, 2000, 40000])
def test_zeros_then_a_large_value(K, n):
    """Value scales of zero or 1e-20, then 1e12 - 1e28 at one position: what the others weigh is not lost on the way."""
    Hq, Hk, d = 32, 8, 128
    g = gen(n)
    p = Pool(g, n, Hk, d)
    q = torch.randn(1, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    for low in (0.0, 1e-20):
        for loud in (1e12, 1e20, 1e28):
            for at in (n - 2, 3, n // 2):
                p.vs[:] = low
                p.vs[:, at] = loud
                want, bar = reference(p, q, pos, 1.0 / 16)
                check(decode(K, p, q, pos, 1.0 / 16), want, bar, 10.0 if n < 10000 else 2.0)


@pytest.mark.parametrize("scale", [1e5, -1e6, 1e8, 1e12])
@pytest.mark.parametrize("n", [37, 3000, 40000])
def test_logits_of_any_size(K, n, scale):
    """Logits of 1e6 to 1e14, a few hundred thousand steps of f32 apart: the output is the value of the largest one's position, whatever
    the others' scales are."""
    Hq, Hk, d = 32, 8, 128
    g = gen(n)
    p = Pool(g, n, Hk, d)
    q = torch.randn(1, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    k = p.codes[0].double() * p.ks.double()[..., None]
    logits = scale * torch.einsum("hgd,htd->hgt", held_q(q)[0].view(Hk, Hq // Hk, d), k)
    top2 = logits.topk(2, -1)
    clear = (top2.values[..., 0] - top2.values[..., 1] > 200 + 20 * 2.0**-24 * logits.abs().amax(-1)).view(Hq)
    assert clear.float().mean() > 0.8
    at = top2.indices[..., 0].view(Hq)
    kv = torch.arange(Hq, device=DEV) // (Hq // Hk)
    for loud in (0.0, 1e12):
        vs = p.vs.clone()
        if loud:
            best = torch.zeros(Hk, n, dtype=torch.bool, device=DEV)
            best[kv, at] = True
            p.vs[~best & (torch.rand(Hk, n, generator=g, device=DEV) < 0.1)] = loud
        got = decode(K, p, q, pos, scale)[0]
        want = p.codes[1][kv, at].double() * p.vs[kv, at].double()[:, None]
        # the store, the fp16 product, the sums over u, of a position of weight 1
        bar = (2.0**-8 + 2.0**-11) * want.abs() + 16 * p.vs[kv, at].double()[:, None] * (2 * -(-n // 32) + 16) * 2.0**-23
        check(got[clear], want[clear], bar[clear], 10.0 if n < 10000 else 2.0)
        p.vs.copy_(vs)


def test_columns_do_not_depend_on_their_neighbours(K):
    """The bits of a query head are the same whatever the other heads and rows of its group hold."""
    Hq, Hk, d = 32, 8, 128
    for n in (300, 30000):
        g = gen(n)
        p = Pool(g, n, Hk, d)
        q = (2.0 * torch.randn(3, Hq, d, generator=g, device=DEV)).to(torch.bfloat16)
        pos = torch.tensor([n - 1, n - 2, n - 1], dtype=torch.int32, device=DEV)
        first = decode(K, p, q, pos, 1.0, 3)
        other = q.clone()
        other[1] = (5.0 * torch.randn(Hq, d, generator=g, device=DEV)).to(torch.bfloat16)
        other[2, ::2] = float("nan")
        second = decode(K, p, other, pos, 1.0, 3)
        assert torch.equal(first[0], second[0]) and torch.equal(first[2, 1::2], second[2, 1::2])
