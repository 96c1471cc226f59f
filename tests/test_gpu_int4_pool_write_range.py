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


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("bits,d", [(4, 128), (4, 64), (8, 128), (8, 64)])
def test_a_head_that_is_not_a_number_stays_one(K, bits, d, side, norm, bad):
    """Codes 0 and a scale that is not finite; the row reads back as NaN; every other head as without it."""
    rows, Hq, Hk = 40, 4, 2
    g = gen(d + bits)
    qkv = torch.randn(rows, Hq + 2 * Hk, d, generator=g, device=DEV).to(torch.bfloat16)
    wk = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16) if norm else None
    clean = Case(K, qkv, wk, 1e-6, Hq, Hk, d, bits)
    spoilt = qkv.clone()
    hit = torch.zeros(rows, Hk, dtype=torch.bool, device=DEV)
    for row, dim in ((0, 0), (0, d - 1), (3, 5), (17, d // 2 + 1), (39, d // 2 - 1)):  # row 0 is not turned
        head = (row + dim) % Hk
        spoilt[row, Hq + (Hk if side == "v" else 0) + head, dim] = bad
        hit[row, head] = True
    c = Case(K, spoilt, wk, 1e-6, Hq, Hk, d, bits)
    mine, other = (0, 1) if side == "k" else (1, 0)
    assert not torch.isfinite(c.scales[mine][hit]).any() and (c.codes[mine][hit] == 0).all()
    assert torch.equal(c.scales[mine][~hit], clean.scales[mine][~hit]) and torch.equal(c.codes[mine][~hit], clean.codes[mine][~hit])
    assert torch.equal(c.scales[other], clean.scales[other]) and torch.equal(c.codes[other], clean.codes[other])
    assert torch.equal(c.q, clean.q)
    outs = [torch.empty(rows, Hk, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    at = torch.arange(rows, dtype=torch.int32, device=DEV)
    assert K.kv_read_paged(c.ck, c.cv, c.ks, c.vs, at, bits, Hk, d, rows, *outs) == 0
    assert outs[mine][hit].isnan().all() and torch.isfinite(outs[mine][~hit]).all() and torch.isfinite(outs[other]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("rows", [40, 100, 260])
def test_what_is_not_a_number_reaches_who_sees_it(K, rows, side, bad):
    """Written, then attended to by rows one by one, in groups and as a chunk: the rows before it are as without it."""
    Hq, Hk, d = 8, 2, 128
    g = gen(rows)
    qkv = torch.randn(rows, Hq + 2 * Hk, d, generator=g, device=DEV).to(torch.bfloat16)
    first = rows // 2 + 3
    spoilt = qkv.clone()
    spoilt[first, Hq + (Hk if side == "v" else 0) + 1, 9] = bad
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    seen = []
    for x in (qkv, spoilt):
        c = Case(K, x, None, 1e-6, Hq, Hk, d, 4)
        outs = [torch.empty(rows, Hq, d, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
        pool = (c.ck, c.cv, c.ks, c.vs)
        assert K.attn_decode_int4_paged(c.q, *pool, pos, Hq, Hk, d, rows, rows, 1.0 / 64, outs[0]) == 0
        assert K.attn_decode_int4_paged(c.q, *pool, pos, Hq, Hk, d, rows, rows, 1.0 / 64, outs[1], rows_per_group=4) == 0
        assert K.prefill_attention_int4(c.q, 1.0 / 64, Hq, Hk, d, 0, rows, outs[2], *pool) == 0
        seen.append(outs)
    for a, b in zip(*seen):
        assert torch.isfinite(a).all()
        assert b[first:, 4:].isnan().all()
        assert torch.equal(a[:first], b[:first]) and torch.equal(a[:, :4], b[:, :4])
