"""Performance cases of the operators around the quantised KV pool, each in its plain form (elementary
torch operations) and as the framework's calls.

Four kinds:

  write    one layer's new token rows: per-head RMSNorm of q and k, rotation, K and V quantised into the
           4- or 8-bit paged pool, and the written rows read back as bf16 values (what a program does that
           hands the rows on, e.g. to a draft model or to a check)
  read     rows of a pool read back as bf16 values: a prefix exported or moved to another pool
  decode   attention of the newest token(s) of each sequence over its 4-bit pool rows; `per` rows of one
           sequence are a verify group, `window` > 0 is sliding-window attention, `empty` makes the last
           sequence an idle slot (position -1, zeros out)
  prefill  causal attention of a prompt chunk over the 4-bit pool

The pool: codes uint8 [Hk][stride][d / 2] (two codes c + 8 a byte, the even dim in the low half) or int8
[Hk][stride][d], scales float32 [Hk][stride], value = code * scale.
"""
import math

import torch

own = False

PAGE = 16
EPS = float(torch.tensor(1e-6, dtype=torch.float32))  # the value a float32 argument holds
THETA = 1e7
LEVELS = {4: 7, 8: 127}


def listed():
    return [
        # a single session's decode step, 4-bit pool: pure latency
        {"name": "write_1_row_b4", "kind": "write", "rows": 1, "Hq": 32, "Hk": 8, "d": 128, "bits": 4, "norm": True},
        # a short chunk with narrow heads into an 8-bit pool, an odd row count
        {"name": "write_37_d64_b8", "kind": "write", "rows": 37, "Hq": 16, "Hk": 2, "d": 64, "bits": 8, "norm": True},
        # a large prompt batch
        {"name": "write_16384_b4", "kind": "write", "rows": 16384, "Hq": 32, "Hk": 8, "d": 128, "bits": 4, "norm": True},
        # a short prefix, and a long one, moved out of the pool
        {"name": "read_777_b4", "kind": "read", "rows": 777, "Hk": 8, "d": 128, "bits": 4},
        {"name": "read_65536_b4", "kind": "read", "rows": 65536, "Hk": 8, "d": 128, "bits": 4},
        # the first tokens of one chat; one session at the model's longest context
        {"name": "decode_1_ctx_37", "kind": "decode", "seqs": 1, "per": 1, "ctx": 37, "Hq": 32, "Hk": 8, "d": 128,
         "window": 0, "empty": False},
        {"name": "decode_1_ctx_131072", "kind": "decode", "seqs": 1, "per": 1, "ctx": 131072, "Hq": 32, "Hk": 8,
         "d": 128, "window": 0, "empty": False},
        # a full batch of long sessions of different lengths, one slot idle
        {"name": "decode_16_ctx_24000", "kind": "decode", "seqs": 16, "per": 1, "ctx": 24000, "Hq": 32, "Hk": 8,
         "d": 128, "window": 0, "empty": True},
        # verify step: five sessions, three rows each
        {"name": "verify_5x3_ctx_4100", "kind": "decode", "seqs": 5, "per": 3, "ctx": 4100, "Hq": 32, "Hk": 8, "d": 128,
         "window": 0, "empty": False},
        # a busy server of a model with narrow heads, eight query heads a KV head, sliding window
        {"name": "decode_40_d64_window", "kind": "decode", "seqs": 40, "per": 1, "ctx": 6001, "Hq": 16, "Hk": 2, "d": 64,
         "window": 4096, "empty": False},
        # prompt chunks: a follow-up question in a chat, a long document
        {"name": "prefill_77_at_1203", "kind": "prefill", "rows": 77, "base": 1203, "Hq": 32, "Hk": 8, "d": 128},
        {"name": "prefill_2048_at_6000", "kind": "prefill", "rows": 2048, "base": 6000, "Hq": 32, "Hk": 8, "d": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "write", "read", "decode", "decode", "decode", "prefill"))
    Hq, Hk, d = rng.choice(((32, 8, 128), (32, 8, 128), (16, 2, 64), (8, 8, 128), (24, 8, 64), (16, 1, 128)))
    if kind == "write":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "Hq": Hq, "Hk": Hk, "d": d, "bits": rng.choice((4, 4, 8)),
                "norm": rng.random() < 0.7}
    if kind == "read":
        return {"kind": kind, "rows": _log(rng, 1, 65536), "Hk": Hk, "d": d, "bits": rng.choice((4, 4, 8))}
    if kind == "prefill":
        return {"kind": kind, "rows": _log(rng, 1, 2048), "base": rng.choice((0, _log(rng, 1, 6000))), "Hq": 32, "Hk": 8,
                "d": 128}
    per = rng.choice((1, 1, 1, 2, 3, 4)) if Hq <= 4 * Hk else 1
    seqs = _log(rng, 1, 64)
    ctx = max(per, _log(rng, 1, min(131072, 16 * 24000 // seqs)))
    return {"kind": kind, "seqs": seqs, "per": per, "ctx": ctx, "Hq": Hq, "Hk": Hk, "d": d,
            "window": rng.choice((0, 0, _log(rng, 1, ctx))), "empty": seqs > 1 and rng.random() < 0.3}


# ---- inputs ---------------------------------------------------------------------------------------------
def _tables(max_pos, d, device):
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cos(angle).float(), torch.sin(angle).float()


def _paged(n, pages, gen):
    """Pool rows of n positions whose pages lie in any order, for each of len(pages) // need sequences."""
    need = -(-n // PAGE)
    order = torch.randperm(pages, generator=gen, device=gen.device)[: pages // need * need].reshape(-1, need)
    rows = (order[:, :, None] * PAGE + torch.arange(PAGE, device=gen.device)).reshape(order.shape[0], -1)[:, :n]
    return rows.to(torch.int32).contiguous()


def _random_pool(stride, Hk, d, bits, gen):
    """A pool as written from N(0, 1) rows: keys with a few strong dims, values without."""
    dev = gen.device
    loud = 1.0 + 3.0 * (torch.rand(Hk, 1, d, generator=gen, device=dev) < 0.04)
    pool = []
    for gain in (loud, 1.0):
        x = torch.randn(Hk, stride, d, generator=gen, device=dev) * gain
        s = (x.abs().amax(-1) / LEVELS[bits]).float()
        c = torch.round(x / s[..., None]).clamp_(-LEVELS[bits], LEVELS[bits]).to(torch.int8)
        pool += [_pack(c) if bits == 4 else c, s]
    return pool


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, Hk, d = case["kind"], case["Hk"], case["d"]
    st = {"case": case}
    if kind == "write":
        rows, Hq, bits = case["rows"], case["Hq"], case["bits"]
        pages = -(-rows // PAGE) + 3
        st["stride"], st["max_pos"] = pages * PAGE, 2 * rows + 64
        st["cos"], st["sin"] = _tables(st["max_pos"], d, dev)
        st["qkv"] = torch.randn(rows, (Hq + 2 * Hk) * d, generator=gen, device=dev).to(torch.bfloat16)
        for w in ("q_norm", "k_norm"):
            st[w] = (1.0 + 0.1 * torch.randn(d, generator=gen, device=dev)).to(torch.bfloat16) if case["norm"] else None
        first = int(torch.randint(0, rows + 32, (1,), generator=gen, device=dev))
        st["pos_rows"] = torch.arange(first, first + rows, dtype=torch.int32, device=dev)
        st["kv_rows"] = _paged(rows, pages, gen)[0]
        width, kept = (d // 2, torch.uint8) if bits == 4 else (d, torch.int8)
        for c in "kv":
            st["cache_" + c] = torch.zeros(Hk, st["stride"], width, dtype=kept, device=dev)
            st[c + "_scale"] = torch.zeros(Hk, st["stride"], device=dev)
            st[c + "_out"] = torch.empty(rows, Hk, d, dtype=torch.bfloat16, device=dev)
        st["q_rot"] = torch.empty(rows, Hq * d, dtype=torch.bfloat16, device=dev)
        return st
    if kind == "read":
        rows, pages = case["rows"], -(-case["rows"] // PAGE) + 3
        st["stride"] = pages * PAGE
        st["cache_k"], st["k_scale"], st["cache_v"], st["v_scale"] = _random_pool(st["stride"], Hk, d, case["bits"], gen)
        st["kv_rows"] = _paged(rows, pages, gen)[0]
        for c in "kv":
            st[c + "_out"] = torch.empty(rows, Hk, d, dtype=torch.bfloat16, device=dev)
        return st
    Hq = case["Hq"]
    seqs, per = (1, case["rows"]) if kind == "prefill" else (case["seqs"], case["per"])
    ctx = case["base"] + case["rows"] if kind == "prefill" else case["ctx"]
    pages = seqs * -(-ctx // PAGE) + 3
    st["stride"], st["ctx"], st["seqs"], st["per"] = pages * PAGE, ctx, seqs, per
    st["cache_k"], st["k_scale"], st["cache_v"], st["v_scale"] = _random_pool(st["stride"], Hk, d, 4, gen)
    st["tables"] = _paged(ctx, pages, gen)[:seqs].contiguous()
    # the sessions of a batch have lengths between half the longest and the longest
    ends = torch.randint(max(per, ctx // 2), ctx + 1, (seqs,), generator=gen, device=dev)
    ends[0] = ctx
    pos = ends[:, None] - per + torch.arange(per, device=dev)
    if case.get("empty"):
        pos[-1] = -1
    st["row_pos"] = pos.reshape(-1).to(torch.int32)
    st["row_pt"] = (st["tables"].data_ptr() + 4 * ctx * (torch.arange(seqs * per, device=dev) // per)).to(torch.int64)
    st["q"] = (2.0 * torch.randn(seqs * per, Hq * d, generator=gen, device=dev)).to(torch.bfloat16)
    st["scale"] = 1.0 / 128 if d == 128 else 0.125
    st["out"] = torch.empty_like(st["q"])
    return st


# ---- the plain form -------------------------------------------------------------------------------------
def _pack(c):
    u = (c + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _values(cache, scale, rows, bits):
    """float32 values [Hk, *rows.shape, d] of the given pool rows."""
    c = cache[:, rows]
    if bits == 4:
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2).float() - 8
    return c.float() * scale[:, rows][..., None]


def _normed(x, w):
    # in 64 bits: the codes of K are decided by where a value lies between two of them
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _quantised(x, bits):
    s = (x.abs().amax(-1) / LEVELS[bits]).float()
    t = x.abs() / s.double()[..., None]
    c = torch.where(s[..., None] > 0, torch.floor(t + 0.5), 0.0).clamp(max=LEVELS[bits]) * torch.sign(x)
    return c.to(torch.int8), s


def _plain_write(st):
    c = st["case"]
    rows, Hq, Hk, d, bits = c["rows"], c["Hq"], c["Hk"], c["d"], c["bits"]
    q, k, v = st["qkv"].view(rows, Hq + 2 * Hk, d).double().split((Hq, Hk, Hk), 1)
    pos, kv_rows = st["pos_rows"].long(), st["kv_rows"].long()
    cos, sin = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
    q = _rotated(_normed(q, st["q_norm"]), cos, sin).to(torch.bfloat16).view(rows, Hq * d)
    k = _rotated(_normed(k, st["k_norm"]), cos, sin)
    codes_k, sk = _quantised(k, bits)
    codes_v, sv = _quantised(v, bits)
    for n, codes, s in (("k", codes_k, sk), ("v", codes_v, sv)):
        st["cache_" + n][:, kv_rows] = (_pack(codes) if bits == 4 else codes).transpose(0, 1)
        st[n + "_scale"][:, kv_rows] = s.transpose(0, 1)
    return [q, *_plain_read(st), st["k_scale"], st["v_scale"]]


def _plain_read(st):
    bits, rows = st["case"]["bits"], st["kv_rows"].long()
    return [_values(st[c], st[s], rows, bits).transpose(0, 1).to(torch.bfloat16).contiguous()
            for c, s in (("cache_k", "k_scale"), ("cache_v", "v_scale"))]


def _plain_attention(st):
    c = st["case"]
    Hq, Hk, d, seqs, per, ctx = c["Hq"], c["Hk"], c["d"], st["seqs"], st["per"], st["ctx"]
    G = Hq // Hk
    rows = st["tables"].long()
    k = _values(st["cache_k"], st["k_scale"], rows, 4)  # [Hk, seqs, ctx, d]
    q = st["q"].float().view(seqs, per, Hk, G, d).permute(2, 0, 1, 3, 4).reshape(Hk, seqs, per * G, d)
    logits = (q @ k.transpose(-1, -2)).view(Hk, seqs, per, G, ctx) * st["scale"]
    del k
    pos, t = st["row_pos"].view(seqs, per, 1, 1), torch.arange(ctx, device=q.device)
    seen = (t <= pos) & (t > pos - (c.get("window") or ctx + 1))
    logits = logits.masked_fill_(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp_(logits.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = p.sum(-1, keepdim=True)
    v = _values(st["cache_v"], st["v_scale"], rows, 4)
    o = (p.view(Hk, seqs, per * G, ctx) @ v).view(Hk, seqs, per, G, d) / torch.where(total > 0, total, 1.0)
    return o.permute(1, 2, 0, 3, 4).reshape(seqs * per, Hq * d).to(torch.bfloat16)


# ---- the framework's calls ------------------------------------------------------------------------------
def _read(k, st):
    c = st["case"]
    _done(k.kv_read_paged(st["cache_k"], st["cache_v"], st["k_scale"], st["v_scale"], st["kv_rows"], c["bits"], c["Hk"],
                          c["d"], st["stride"], st["k_out"], st["v_out"]))
    return [st["k_out"], st["v_out"]]


def _write(k, st):
    c = st["case"]
    _done(k.qk_norm_rope_kv_paged(st["qkv"], st["q_norm"], st["k_norm"], EPS, st["cos"], st["sin"], st["pos_rows"],
                                  st["kv_rows"], c["Hq"], c["Hk"], c["d"], st["stride"], st["max_pos"], c["bits"],
                                  st["q_rot"], st["cache_k"], st["cache_v"], st["k_scale"], st["v_scale"]))
    return [st["q_rot"], *_read(k, st), st["k_scale"], st["v_scale"]]


def _decode(k, st):
    c = st["case"]
    if "scratch" not in st:  # a decode loop keeps it
        need = k.attn_decode_int4_scratch_bytes(st["seqs"] * st["per"], st["per"], c["Hq"], c["Hk"], c["d"], st["ctx"])
        st["scratch"] = torch.empty(max(need, 16), dtype=torch.uint8, device=st["q"].device)
    _done(k.attn_decode_int4_paged(st["q"], st["cache_k"], st["cache_v"], st["k_scale"], st["v_scale"], st["row_pos"],
                                   c["Hq"], c["Hk"], c["d"], st["stride"], st["ctx"], st["scale"], st["out"],
                                   rows_per_group=st["per"], row_pt=st["row_pt"], window=c["window"],
                                   scratch=st["scratch"]))
    return st["out"]


def _prefill(k, st):
    c = st["case"]
    _done(k.prefill_attention_int4(st["q"], st["scale"], c["Hq"], c["Hk"], c["d"], c["base"], st["stride"], st["out"],
                                   st["cache_k"], st["cache_v"], st["k_scale"], st["v_scale"], pt=st["tables"][0]))
    return st["out"]


def _done(rc):
    if rc != 0:
        raise RuntimeError(f"the call returned {rc}")


def run(state):
    kind = state["case"]["kind"]
    if own:
        import granite4_b200  # noqa: F401
        from granite4_b200 import kernels
        return {"write": _write, "read": _read, "decode": _decode, "prefill": _prefill}[kind](kernels, state)
    if kind == "write":
        return _plain_write(state)
    if kind == "read":
        return _plain_read(state)
    return _plain_attention(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------
def work(case):
    kind, Hk, d = case["kind"], case["Hk"], case["d"]

    def pool_row(bits):  # codes and scales of K and V, all heads
        return 2 * Hk * (d * bits // 8 + 4)
    if kind == "write":
        Hq, rows, bits = case["Hq"], case["rows"], case["bits"]
        out = 2 * Hq * d + 2 * pool_row(bits) + 2 * 2 * Hk * d  # q_rot, pool written and read, values
        return {"bytes": rows * (2 * (Hq + 2 * Hk) * d + 4 * d + 12 + out), "flops": rows * (Hq + 2 * Hk) * d * 10}
    if kind == "read":
        return {"bytes": case["rows"] * (4 + pool_row(case["bits"]) + 4 * Hk * d), "flops": case["rows"] * 2 * Hk * d}
    Hq = case["Hq"]
    if kind == "prefill":
        rows, ctx = case["rows"], case["base"] + case["rows"]
        pairs = rows * case["base"] + rows * (rows + 1) // 2
        return {"bytes": ctx * (pool_row(4) + 4) + 4 * rows * Hq * d, "flops": 4 * pairs * Hq * d}
    # lengths are spread over [ctx / 2, ctx], the first is ctx
    seqs, per, ctx = case["seqs"], case["per"], case["ctx"]
    others = seqs - 1 - (1 if case["empty"] else 0)
    if case["window"]:
        w = min(case["window"], ctx)
        mean = min(w, 0.75 * ctx)
        seen = w + others * mean
    else:
        seen = ctx + others * 0.75 * ctx
    return {"bytes": seen * (pool_row(4) + 4) + seqs * per * (4 * Hq * d + 12), "flops": 4 * seen * per * Hq * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------
def _unpack64(cache, scale, rows, bits):
    """[n, Hk, d] values of pool rows, from the bytes' meaning."""
    picked = cache[:, rows].long()
    if bits == 4:
        d = 2 * picked.shape[-1]
        codes = torch.empty(*picked.shape[:-1], d, dtype=torch.float64, device=picked.device)
        codes[..., 0::2], codes[..., 1::2] = (picked % 16 - 8).double(), (picked // 16 - 8).double()
    else:
        codes = picked.double()
    return (codes * scale[:, rows].double().unsqueeze(-1)).transpose(0, 1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, Hk, d = case["kind"], case["Hk"], case["d"]
    if kind == "read":
        rows = st["kv_rows"].long()
        return [_unpack64(st["cache_k"], st["k_scale"], rows, case["bits"]),
                _unpack64(st["cache_v"], st["v_scale"], rows, case["bits"])]
    if kind == "write":
        n, Hq, top = case["rows"], case["Hq"], LEVELS[case["bits"]]
        x = st["qkv"].double().view(n, Hq + 2 * Hk, d)
        half = d // 2
        cos, sin = (st[t].double()[st["pos_rows"].long()].view(n, 1, half) for t in ("cos", "sin"))
        turned = []
        for part, w in ((x[:, :Hq], st["q_norm"]), (x[:, Hq:Hq + Hk], st["k_norm"])):
            if w is not None:
                part = part / torch.sqrt(part.pow(2).sum(-1, keepdim=True) / d + EPS) * w.double()
            # the pair (a, b) as a complex number, turned by the angle
            z = torch.complex(part[..., :half], part[..., half:]) * torch.complex(cos, sin)
            turned.append(torch.cat((z.real, z.imag), -1))
        values, scales = [], []
        for y in (turned[1], x[:, Hq + Hk:]):
            s = (y.abs().max(-1).values / top).float().double()
            ratio = torch.where(s.unsqueeze(-1) > 0, y / s.unsqueeze(-1), 0.0)
            code = torch.clamp(torch.trunc(ratio + torch.copysign(torch.tensor(0.5, device=y.device, dtype=y.dtype), ratio)), -top, top)
            values.append(code * s.unsqueeze(-1))
            pool = torch.zeros(Hk, st["stride"], dtype=torch.float64, device=y.device)
            pool[:, st["kv_rows"].long()] = s.t()
            scales.append(pool)
        return [turned[0].reshape(n, Hq * d), *values, *scales]
    Hq = case["Hq"]
    group, seqs, per = Hq // Hk, st["seqs"], st["per"]
    q = st["q"].double().view(seqs, per, Hk, group, d)
    pos = st["row_pos"].view(seqs, per).tolist()
    out = torch.zeros(seqs, per, Hk, group, d, dtype=torch.float64, device=q.device)
    for s in range(seqs):
        last = max(pos[s])
        if last < 0:
            continue
        first = max(0, min(pos[s]) + 1 - case["window"]) if case.get("window") else 0
        rows = st["tables"][s, first:last + 1].long()
        k, v = (_unpack64(st["cache_" + c], st[c + "_scale"], rows, 4) for c in "kv")
        where = torch.arange(first, last + 1, device=q.device)
        for j0 in range(0, per, 256):
            js = slice(j0, min(j0 + 256, per))
            at = torch.tensor(pos[s][js], device=q.device).view(-1, 1)
            hidden = where > at
            if case.get("window"):
                hidden |= where <= at - case["window"]
            for h in range(Hk):
                w = torch.einsum("pgd,td->pgt", q[s, js, h], k[:, h]) * st["scale"]
                w = torch.softmax(w.masked_fill(hidden.unsqueeze(1), -math.inf), -1)
                out[s, js, h] = torch.einsum("pgt,td->pgd", w, v[:, h])
    return out.view(seqs * per, Hq * d)
