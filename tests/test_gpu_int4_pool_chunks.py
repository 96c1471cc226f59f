"""Prompt chunks over the 4-bit pool against their formula in 64 bits, with values that tell positions apart, peaked softmaxes, and
values of any magnitude.

Bounds (a rounding is off by at most half a step: bf16 2^-8, fp16 2^-11, f32 2^-24 of the value):
  store              2^-8 |exact|
  P and V            fp16: P 2^-11, V as fp16(code * fp16(v_scale)) 2 * 2^-11, of sum p |v|; the largest P is 1 or more, and a P
                     under 2^-14 is off by at most 2^-25: 2^-25 max(p) |v| for each position with p under 2^-14 max(p)
  logits             q in fp16 (exact where it is normal: off by at most 2^-25 max(1, max |q|)), codes exact, 128 products in 8
                     steps of 16, each lined up and cut 17 times at 2^-23: dl = |scale| max(k_scale) 7 (d 2^-25 max(1, max |q|) +
                     136 * 2^-23 sum |q|) and 4 * 2^-24 |l| for the factors; exp2 2^-22; numerator and sum both: twice
  sums               (n / 16 + 16) steps, cut 17 times at 2^-23 of at most sum p |v|
Chunks that the decode form takes are closer than that, but for q: the reference takes it as that form holds it, the integer
round(q 32639 / max |q|) of its head times max |q| / 32639.
"""
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


def widened(rows, base, Hq, Hk, d):
    """The chunks that run on the kernels for an 8-bit pool."""
    if rows < 32 or d != 128 or Hq != 4 * Hk:
        return False
    if rows < 64:
        return base <= 192 - rows
    places = 3 * torch.cuda.get_device_properties(0).multi_processor_count
    return -(-rows // 4) * Hk > places or (2 * base + rows) * rows * Hk >= 2800000


class Pool:
    def __init__(self, g, stride, Hk, d):
        self.Hk, self.d, self.stride = Hk, d, stride
        self.codes = [torch.randint(-7, 8, (Hk, stride, d), generator=g, device=DEV).to(torch.int8) for _ in range(2)]
        self.ck, self.cv = (((c[..., 0::2] + 8) | ((c[..., 1::2] + 8) << 4)).to(torch.uint8).contiguous() for c in self.codes)
        self.ks, self.vs = ((torch.rand(Hk, stride, generator=g, device=DEV) + 0.5) * 0.2 for _ in range(2))
        self.all = (self.ck, self.cv, self.ks, self.vs)


def chunk(K, p, q, base, scale, out=None, pt=None):
    rows, Hq, d = q.shape
    out = torch.empty(rows, Hq, d, dtype=torch.bfloat16, device=DEV) if out is None else out
    assert K.prefill_attention_int4(q, scale, Hq, p.Hk, d, base, p.stride, out, *p.all, pt=pt) == 0
    return out


def reference(p, q, base, scale, pick, pt=None):
    """(exact, bound) [len(pick), Hq, d] of the rows `pick`."""
    rows, Hq, d = q.shape
    G, out = Hq // p.Hk, []
    x_all = q.double()
    if not widened(rows, base, Hq, p.Hk, d):
        top = q.float().abs().amax(-1, keepdim=True).clamp(min=1e-30)
        x_all = torch.round(q.float() * (32639.0 / top)).double() * top.double() / 32639.0
    qmax = max(1.0, q.float().abs().max().item())
    for r in pick:
        n = base + r + 1
        at = torch.arange(n, device=DEV) if pt is None else pt[:n].long()
        k, v = (p.codes[i][:, at].double() * s[:, at].double()[..., None] for i, s in ((0, p.ks), (1, p.vs)))
        x = x_all[r].view(p.Hk, G, d)
        logits = scale * torch.einsum("hgd,htd->hgt", x, k)
        w = torch.softmax(logits, -1)
        e, mass = torch.einsum("hgt,htd->hgd", w, v), torch.einsum("hgt,htd->hgd", w, v.abs())
        dl = abs(scale) * 7 * p.ks[:, at].double().amax(-1)[:, None] * (
            d * 2.0**-25 * qmax + 136 * 2.0**-23 * x.abs().sum(-1)) + 4 * 2.0**-24 * logits.abs().amax(-1)
        rel = 3 * 2.0**-11 + 2 * (2.0**-22 + dl) + (n / 16 + 16) * 17 * 2.0**-23
        bound = 2.0**-8 * e.abs() + rel[..., None] * mass 
        bound += 2.0**-25 * w.amax(-1)[..., None] * torch.einsum("hgt,htd->hgd", (w < 2.0**-14 * w.amax(-1, keepdim=True)).double(), v.abs())
        out.append((e.view(Hq, d), bound.view(Hq, d)))
    return tuple(torch.stack(t) for t in zip(*out))


def check(got, want, bound):
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() / bound.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, worst


CHUNKS = [(32, 0), (33, 100), (63, 129), (63, 130), (64, 703), (64, 705), (77, 1203), (130, 700), (192, 3), (193, 3), (300, 0), (600, 2000),
          (64, 3000), (77, 2500), (130, 1400), (225, 3), (256, 0)]


@pytest.mark.parametrize("rows,base", CHUNKS)
@pytest.mark.parametrize("Hq,Hk,d", [(32, 8, 128), (8, 2, 128), (16, 2, 64)])
def test_every_row_sees_up_to_its_own_position(K, rows, base, Hq, Hk, d):
    """A value scale 400 times the others' in each kv head, at positions around the edges of tiles and blocks: a row that misses its own
    position, or sees the next, is off by many times the bound."""
    g = gen(rows + base + d)
    n, G = base + rows, Hq // Hk
    p = Pool(g, n + 30, Hk, d)
    pt = torch.randperm(n + 30, generator=g, device=DEV)[:n].to(torch.int32)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    marks = sorted({m for m in (1, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, rows - 2, rows - 1) if 0 < m < rows})
    plain = p.vs.clone()
    for i in range(0, len(marks), Hk):
        chosen = marks[i:i + Hk]
        p.vs.copy_(plain)
        for head, m in enumerate(chosen):
            p.vs[head, pt[base + m].long()] *= 400.0
        pick = sorted({r for m in chosen for r in (m - 1, m)} | {0, rows - 1})
        want, bound = reference(p, q, base, 1.0 / 64, pick, pt)
        check(chunk(K, p, q, base, 1.0 / 64, pt=pt)[pick], want, bound)
        for head, m in enumerate(chosen):  # what the mark adds to its row, for a code of 1 and an even softmax
            own = p.vs[head, pt[base + m].long()].item() / (base + m + 1)
            for r in (m - 1, m):
                assert own > 3 * bound[pick.index(r), head * G:(head + 1) * G].median().item()


@pytest.mark.parametrize("scale", [0.25, -1.0, 4.0])
@pytest.mark.parametrize("rows,base", [(40, 60), (64, 800), (300, 5), (100, 5000), (64, 3000)])
def test_peaked_softmax(K, rows, base, scale):
    Hq, Hk, d = 32, 8, 128
    g = gen(rows)
    p = Pool(g, base + rows, Hk, d)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    pick = sorted({0, 1, rows // 3, rows // 2, rows - 2, rows - 1})
    want, bound = reference(p, q, base, scale, pick)
    check(chunk(K, p, q, base, scale)[pick], want, bound)
    assert (want.abs() / bound.clamp(min=1e-300)).median().item() > 10.0


@pytest.mark.parametrize("small", [1e-2, 1e-4, 1e-6, 1e-9, 1e-20])
@pytest.mark.parametrize("rows,base", [(40, 60), (64, 800), (300, 5), (77, 1203), (64, 3000), (77, 2500)])
def test_small_values_keep_their_bits(K, rows, base, small):
    """Scaled by a power of two, to the bit the scaled output (of the widened form: the other's probabilities are taken against a rounded
    logarithm of the scales); by another number, within the bound. Other heads as they are."""
    Hq, Hk, d = 32, 8, 128
    g = gen(rows)
    p = Pool(g, base + rows, Hk, d)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    plain, first = p.vs.clone(), chunk(K, p, q, base, 1.0 / 16)
    p.vs[1::2] = plain[1::2] * small
    pick = [0, rows // 2, rows - 1]
    want, bound = reference(p, q, base, 1.0 / 16, pick)
    got = chunk(K, p, q, base, 1.0 / 16)
    small_heads = (torch.arange(Hq, device=DEV) // 4) % 2 == 1
    check(got[pick], want, bound)
    assert torch.equal(got[:, ~small_heads], first[:, ~small_heads])
    if not widened(rows, base, Hq, Hk, d):
        return
    power = 2.0 ** round(torch.log2(torch.tensor(small)).item())
    p.vs[1::2] = plain[1::2] * power
    got = chunk(K, p, q, base, 1.0 / 16)
    assert torch.equal(got[:, small_heads].float(), first[:, small_heads].float() * power)


@pytest.mark.parametrize("rows,base", [(40, 60), (300, 5), (77, 2500)])
def test_a_value_past_fp16_leaves_small_ones_alone(K, rows, base):
    """7 v_scale over 65504: NaN to the rows that see it, and nothing to the others, whose values are of 1e-6."""
    Hq, Hk, d = 32, 8, 128
    assert widened(rows, base, Hq, Hk, d)
    g = gen(rows)
    p = Pool(g, base + rows, Hk, d)
    p.vs *= 1e-6
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    first = chunk(K, p, q, base, 1.0 / 16)
    at = rows - 7
    p.vs[1, base + at] = 1e5
    got = chunk(K, p, q, base, 1.0 / 16)
    assert got[at:, 4:8].isnan().all()
    got[at:, 4:8] = first[at:, 4:8]
    assert torch.equal(got, first)


@pytest.mark.parametrize("rows,base", [(40, 60), (64, 800), (300, 5), (64, 3000)])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_an_output_on_any_boundary(K, rows, base, shift):
    Hq, Hk, d = 32, 8, 128
    g = gen(rows)
    p = Pool(g, base + rows, Hk, d)
    q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
    buf = torch.full((rows * Hq * d + 8,), 3.0, dtype=torch.bfloat16, device=DEV)
    out = buf[shift:shift + rows * Hq * d].view(rows, Hq, d)
    chunk(K, p, q, base, 1.0 / 16, out=out)
    pick = [0, rows // 2, rows - 1]
    want, bound = reference(p, q, base, 1.0 / 16, pick)
    # (which form an unaligned output takes is not said here: the bound of both)
    check(out[pick], want, bound + 2 * 7 * 128 * 2.0**-16 * 0.3 / 16 * 5.0 * want.abs().amax())
    assert (buf[:shift] == 3.0).all() and (buf[shift + rows * Hq * d:] == 3.0).all()


@pytest.mark.parametrize("rows,base", [(20, 7), (40, 60), (63, 129), (64, 800), (300, 5), (64, 3000)])
@pytest.mark.parametrize("size", [3e38, 1e9, 7e4, 1e-6, 1e-12])
def test_queries_of_any_size(K, rows, base, size):
    """Queries that fp16 does not hold, with a softmax scale that leaves their logits as they are: to the bit those of the queries
    scaled by a power of two, within the bound else."""
    Hq, Hk, d = 32, 8, 128
    g = gen(rows)
    p = Pool(g, base + rows, Hk, d)
    unit = torch.rand(rows, Hq, d, generator=g, device=DEV, dtype=torch.float64) * 2 - 1
    q = (unit * size).to(torch.bfloat16)
    assert torch.isfinite(q).all()
    pick = [0, rows // 2, rows - 1]
    unit = (q.double() / size).float()  # (what q stands for, in a type that holds it)
    want, bound = reference(p, unit, base, 1.0 / 16, pick)
    check(chunk(K, p, q, base, 1.0 / 16 / size)[pick], want, bound)
    power = 2.0 ** round(torch.log2(torch.tensor(size)).item() - 2)
    one = (unit * 4).to(torch.bfloat16)
    if size > 1e38:  # scale * log2(e) = 1.44 * 2^-132 is a multiple of 2^-149 in f32: a factor of the logits off by up to 2^-18
        return
    assert torch.equal(chunk(K, p, (one.float() * power).to(torch.bfloat16), base, 1.0 / 64 / power), chunk(K, p, one, base, 1.0 / 64))


@pytest.mark.parametrize("rows,base", [(20, 300), (40, 60), (64, 3000), (300, 5)])
def test_chunks_captured_and_replayed(K, rows, base):
    """Two graphs of a chunk each, with a scratch of its own, replayed side by side with inputs that change in between: to the bit what
    the calls give."""
    from granite4_b200 import capi
    Hq, Hk, d, scale = 32, 8, 128, 1.0 / 16
    g = gen(rows)
    need = max(16, capi.lib().granite4_prefill_attention_int4_scratch_bytes(rows, base, Hq, Hk, d))
    jobs = []
    for _ in range(2):
        p = Pool(g, base + rows, Hk, d)
        q = torch.randn(rows, Hq, d, generator=g, device=DEV).to(torch.bfloat16)
        out, scratch = torch.empty_like(q), torch.full((need,), 0xFF, dtype=torch.uint8, device=DEV)

        def call(p=p, q=q, out=out, scratch=scratch):
            assert K.prefill_attention_int4(q, scale, Hq, Hk, d, base, p.stride, out, *p.all, scratch=scratch) == 0
        call()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):
                call()
        jobs.append((p, q, out, call, graph, stream))
    for size in (1.0, 1e-3, 30.0):
        want = []
        for p, q, out, call, _, _ in jobs:
            q.copy_(torch.randn(rows, Hq, d, generator=g, device=DEV))
            p.vs.copy_((torch.rand(Hk, base + rows, generator=g, device=DEV) + 0.5) * size)
            call()
            want.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
        for _, _, _, _, graph, stream in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out, _, _, _), w in zip(jobs, want):
            assert torch.equal(out, w)
