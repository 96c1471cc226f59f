"""Attention over the 8-bit pool scales queries by a power of two into fp16: the bits of the output do not depend on how large they
are, to the end of bf16."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("power", [-40, 20, 100, 112, 122])
@pytest.mark.parametrize("rows", [1, 4, 20, 70])
def test_queries_of_any_power_of_two(rows, power):
    import granite4_b200  # noqa: F401
    from granite4_b200 import kernels as K
    Hq, Hk, d, base = 32, 8, 128, 300
    g = torch.Generator(device=DEV).manual_seed(rows)
    n = base + rows
    ck, cv = (torch.randint(-127, 128, (Hk, n, d), generator=g, device=DEV).to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand(Hk, n, generator=g, device=DEV) * 0.02 for _ in range(2))
    q = (4 * torch.randn(rows, Hq * d, generator=g, device=DEV)).to(torch.bfloat16)
    pos = torch.arange(base, n, dtype=torch.int32, device=DEV)
    outs = []
    for p in (0, power):
        x, scale = (q.float() * 2.0**p).to(torch.bfloat16), 2.0 ** (-3 - p)
        assert torch.isfinite(x).all()
        pair = [torch.empty_like(q) for _ in range(2)]
        assert K.prefill_attention_int8(x, scale, Hq, Hk, d, base, n, pair[0], ck, cv, ks, vs) == 0
        assert K.attn_decode_int8_paged(x, ck, cv, ks, vs, pos, Hq, Hk, d, n, n, scale, pair[1]) == 0
        outs.append(pair)
    for a, b in zip(*outs):
        assert torch.isfinite(a).all() and torch.equal(a, b)
