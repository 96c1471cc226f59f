"""What the entry points around the 4-bit pool refuse before any launch, and what the Python side refuses; no GPU."""
import pytest


@pytest.fixture(scope="module")
def lib():
    import granite4_b200
    from granite4_b200 import _build, capi
    if _build.is_stale():
        _build.build()
    assert granite4_b200
    return capi.lib()


def write(lib, **kw):
    a = dict(qkv=16, wq=16, wk=16, eps=1e-6, cos=16, sin=16, pos=16, kvr=16, rows=4, Hq=32, Hk=8, d=128, stride=64, max_pos=64,
             bits=4, q=16, ck=16, cv=16, ks=16, vs=16)
    a.update(kw)
    return lib.granite4_kernel_qk_norm_rope_kv_paged(*a.values())


@pytest.mark.parametrize("bad", [
    {"qkv": None}, {"cos": None}, {"sin": None}, {"pos": None}, {"kvr": None}, {"q": None}, {"ck": None}, {"cv": None},
    {"ks": None}, {"vs": None}, {"rows": 0}, {"rows": -1}, {"Hq": 0}, {"Hk": 0}, {"stride": 0}, {"max_pos": 0},
    {"eps": 0.0}, {"eps": float("nan")}, {"eps": float("inf")}, {"d": 96}, {"d": 256}, {"bits": 5}, {"bits": 16},
    {"qkv": 24}, {"wq": 8}, {"wk": 24}, {"cos": 20}, {"sin": 20}, {"q": 18}, {"ck": 24}, {"cv": 17}])
def test_write_refusals(lib, bad, capfd):
    assert write(lib, **bad) == -1
    assert capfd.readouterr().err.startswith("granite4: granite4_kernel_qk_norm_rope_kv_paged: ")


def read(lib, **kw):
    a = dict(ck=16, cv=16, ks=16, vs=16, kvr=16, rows=4, bits=4, Hk=8, d=128, stride=64, ko=16, vo=16)
    a.update(kw)
    return lib.granite4_kernel_kv_read_paged(*a.values())


@pytest.mark.parametrize("bad", [{"ck": None}, {"cv": None}, {"ks": None}, {"vs": None}, {"kvr": None}, {"ko": None},
                                 {"vo": None}, {"rows": 0}, {"bits": 3}, {"Hk": 0}, {"d": 32}, {"stride": 0}, {"ck": 24},
                                 {"ko": 18}, {"vo": 24}, {"cv": 8}])
def test_read_refusals(lib, bad, capfd):
    assert read(lib, **bad) == -1
    assert capfd.readouterr().err.startswith("granite4: granite4_kernel_kv_read_paged: ")


def decode(lib, **kw):
    a = dict(q=16, ck=16, cv=16, ks=16, vs=16, pos=16, row_pt=None, pt=None, rows=2, per=1, Hq=32, Hk=8, d=128, stride=131072,
             max_len=131072, window=0, scale=0.1, scratch=None, bytes=0, out=16)
    a.update(kw)
    return lib.granite4_kernel_attn_decode_int4_paged(*a.values())


@pytest.mark.parametrize("bad", [
    {"q": None}, {"ck": None}, {"cv": None}, {"ks": None}, {"vs": None}, {"pos": None}, {"out": None}, {"rows": 0},
    {"per": 0}, {"per": 17}, {"Hq": 33}, {"Hk": 0}, {"Hq": 0}, {"Hq": 1040}, {"d": 96}, {"stride": 0}, {"max_len": 0},
    {"max_len": 131073}, {"window": -1}, {"scale": float("nan")}, {"q": 18}, {"ck": 24}, {"cv": 8},
    {},  # a scratch is wanted at this length
    {"scratch": 24, "bytes": 1 << 30}, {"scratch": 16, "bytes": 64}])
def test_decode_refusals(lib, bad, capfd):
    assert decode(lib, **bad) == -1
    assert capfd.readouterr().err.startswith("granite4: granite4_kernel_attn_decode_int4_paged: ")


def test_scratch_sizes(lib):
    size = lib.granite4_attn_decode_int4_scratch_bytes
    assert size(1, 1, 32, 8, 128, 131072) > 0
    assert size(1, 1, 32, 8, 128, 128) == 0  # one tile a warp: nothing is split
    assert size(1, 1, 32, 8, 128, 4096) == 0  # a cluster per kv head
    assert size(1, 1, 33, 8, 128, 4096) == -1 and size(0, 1, 32, 8, 128, 4096) == -1
    assert size(1, 1, 32, 8, 96, 4096) == -1 and size(1, 1, 32, 8, 128, 0) == -1 and size(4, 17, 32, 8, 128, 64) == -1
    assert size(1 << 30, 4, 32, 8, 128, 1 << 30) >= 0
    pre = lib.granite4_prefill_attention_int4_scratch_bytes
    assert pre(32, 100, 32, 8, 128) >= 132 * 8 * 2 * 132
    assert pre(0, 0, 32, 8, 128) == -1 and pre(1, -1, 32, 8, 128) == -1 and pre(2, (1 << 31) - 1, 32, 8, 128) == -1


def prefill(lib, **kw):
    a = dict(q=16, scale=0.1, Hq=32, Hk=8, d=128, base=10, rows=40, stride=64, out=16, ck=16, cv=16, ks=16, vs=16, pt=None,
             scratch=None, bytes=0)
    a.update(kw)
    return lib.granite4_prefill_attention_int4(*a.values())


@pytest.mark.parametrize("bad", [
    {"q": None}, {"ck": None}, {"cv": None}, {"ks": None}, {"vs": None}, {"out": None}, {"rows": 0}, {"base": -1},
    {"base": (1 << 31) - 5}, {"stride": 49}, {"stride": 0}, {"scale": float("inf")}, {"d": 96}, {"Hq": 31}, {"Hk": 0},
    {"q": 24}, {"ck": 24}, {"cv": 20},
    {}, {"scratch": 16, "bytes": 100}, {"scratch": 24, "bytes": 1 << 30}])
def test_prefill_refusals(lib, bad, capfd):
    assert prefill(lib, **bad) == -1
    assert capfd.readouterr().err.startswith("granite4: granite4_prefill_attention_int4: ")


def test_cpu_tensors_are_refused(lib):
    import torch
    from granite4_b200 import kernels as k
    z = torch.zeros(2, 48 * 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(8, 16, 64, dtype=torch.uint8)
    s = torch.zeros(8, 16)
    with pytest.raises(ValueError):
        k.qk_norm_rope_kv_paged(z, None, None, 1e-6, s, s, i, i, 32, 8, 128, 16, 16, 4, z, c, c, s, s)
    with pytest.raises(ValueError):
        k.kv_read_paged(c, c, s, s, i, 4, 8, 128, 16, z, z)
    with pytest.raises(ValueError):
        k.attn_decode_int4_paged(z, c, c, s, s, i, 32, 8, 128, 16, 16, 0.1, z, scratch=torch.zeros(16, dtype=torch.uint8))
    with pytest.raises(ValueError):
        k.prefill_attention_int4(z, 0.1, 32, 8, 128, 0, 16, z, c, c, s, s, scratch=torch.zeros(16, dtype=torch.uint8))
