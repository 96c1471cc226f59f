"""Attention over the 4-bit pool where row scales and logits are anything but alike: value scales that some rows of a group do
not see, or give no weight to, many magnitudes above the rest; scales over many magnitudes; peaked softmaxes.

The reference, in 64 bits, takes q as the kernel holds it, the 16-bit integer round(q 32639 / max |q|) of its head times max |q|
/ 32639, so that what is left to bound are roundings (a rounding is off by at most half a step: bf16 2^-8, fp16 2^-11, f32
2^-24 of the value):
  store                  2^-8 |exact|
  p v_scale as fp16      2^-11 sum p |v|; its floor: the largest p s is held at 2^10 or more and steps under fp16's normal range
                         are 2^-24, so each of the n positions is off by at most 2^-35 max(p s), times |c| <= 7 (and 1 % for the
                         logarithm that decides on it); a scale counts as 2^-40 at least: 7 n (1.01 2^-35 max(p s) + 2^-75)
  logits                 an exact integer, to f32 (1), times k_scale (scale log2(e) max |q| / 32639) (4), less the base (1 of its
                         own size): in powers of two 6 * 2^-24 |l| + 2^-24 (|l| + |base|), |base| <= max |l| + 40 + 24;
                         exp2 itself 2^-22; numerator and sum both: twice
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
        off = 2.0**-8 * e.abs() + rel[..., None] * mass + (7 * n * (1.01 * 2.0**-35 * ws.amax(-1) + 2.0**-75) + 16 * (steps + 16) * 2.0**-23 * ws.sum(-1))[..., None]
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
