"""The quantised write at the ends of the types: codes and scales equal those of the formula in 64 bits (f32 of the scale its one
rounding) wherever that is finite, and a head that holds what is not a number keeps saying so."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TOP = {4: 7, 8: 127}


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


def unpack(u):
    return torch.stack((u & 15, u >> 4), -1).flatten(-2).to(torch.int8) - 8


class Case:
    """rows of Hq + 2 Hk heads written into a fresh pool at positions 0, 1, ... (identity rows)."""

    def __init__(self, K, qkv, wk, eps, Hq, Hk, d, bits):
        rows = self.rows = qkv.shape[0]
        kind, width = (torch.uint8, d // 2) if bits == 4 else (torch.int8, d)
        self.ck, self.cv = (torch.full((Hk, rows, width), 0x5A, dtype=kind, device=DEV) for _ in range(2))
        self.ks, self.vs = (torch.full((Hk, rows), -1.0, device=DEV) for _ in range(2))
        self.q = torch.empty(rows, Hq * d, dtype=torch.bfloat16, device=DEV)
        self.cos, self.sin = tables(rows, d)
        at = torch.arange(rows, dtype=torch.int32, device=DEV)
        assert K.qk_norm_rope_kv_paged(qkv.reshape(rows, -1), None, wk, eps, self.cos, self.sin, at, at, Hq, Hk, d, rows, rows, bits,
                                       self.q, self.ck, self.cv, self.ks, self.vs) == 0
        self.codes = [(unpack(c) if bits == 4 else c).transpose(0, 1) for c in (self.ck, self.cv)]  # [rows, Hk, d]
        self.scales = [s.t() for s in (self.ks, self.vs)]


def formula(x, w, eps, cos, sin, bits):
    """(codes, scales) of key rows [rows, Hk, d] float64; w None, cos None: of value rows."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is not None:
        a, b = x.chunk(2, -1)
        c, s = cos.double()[:, None], sin.double()[:, None]
        x = torch.cat((a * c - b * s, b * c + a * s), -1)
    scale = (x.abs().amax(-1) / TOP[bits]).float()
    t = torch.where(scale[..., None] > 0, x.abs() / scale.double()[..., None], 0.0)
    return (torch.floor(t + 0.5).clamp(max=TOP[bits]) * torch.sign(x)).to(torch.int8), scale


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("x,w", [
    (3.3e38, None),     # a rotated pair passes f32's end, its scale does not
    (1e38, None), (1e-38, None), (1e-40, None),
    (1e30, 1e12), (3e38, 3e38), (1e36, 0.5),   # x w passes it
    (1e-25, 1e-18), (1e-20, 1e-25), (1e-30, 1e30), (1e-38, 3.0)])  # x w falls under it, or its smaller elements do
@pytest.mark.parametrize("eps", [1e-6, 1e-37])
def test_keys_and_values_near_the_ends_of_f32(K, x, w, eps, d, bits):
    rows, Hq, Hk = 70, 2, 3
    g = gen(d + bits)
    head = torch.rand(rows, Hq + 2 * Hk, d, generator=g, device=DEV, dtype=torch.float64) * 2 - 1
    head[..., 0] = 1.0  # the largest of a head is x itself
    head[:, Hq + 1] *= 0.01
    head[:, Hq + 1, 1::2] *= 1e-3  # a head of few large elements
    qkv = (head * x).to(torch.bfloat16)
    qkv[:, :Hq] = 1.0
    eps = float(torch.tensor(eps))
    wk = None if w is None else ((0.5 + torch.rand(d, generator=g, device=DEV, dtype=torch.float64) / 2) * w).to(torch.bfloat16)
    assert torch.isfinite(qkv).all() and (wk is None or torch.isfinite(wk).all())
    c = Case(K, qkv, wk, eps, Hq, Hk, d, bits)
    codes, scales = formula(qkv[:, Hq:Hq + Hk].double(), wk, eps, c.cos, c.sin, bits)
    assert torch.equal(c.scales[0], scales)
    assert torch.equal(c.codes[0], codes)
    codes, scales = formula(qkv[:, Hq + Hk:].double(), None, eps, None, None, bits)
    assert torch.equal(c.scales[1], scales)
    assert torch.equal(c.codes[1], codes)
