"""The operators of the 4-bit KV cache: writing it, reading it back, and attention over it.

The cache holds keys and values in MXFP4: for every head row of D values, D/2 bytes of E2M1 nibbles (element 2j in the
low nibble) and D/32 E8M0 codes, value +-{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^(code - 127).  Pages of `page` positions,
head-major: kq, vq u8 (n_pages, Hkv, page, D/2), ks, vs u8 (n_pages, Hkv, page, D/32).  Sequence b is page b, or the
pages that an int32 table (B, max_pages) lists (-1: none).  Token m of sequence b sits at position dpos[b] + m; a
sequence whose positions are negative is an empty slot of the batch: it writes nothing and its output rows are zeros.

  attn   softmax(q K^T / sqrt(D)) V over positions 0 .. dpos[b] + m
  write  k, v -> MXFP4 rows at dpos[b] + m, read back as the values that the cache then stands for (a prompt's own
         attention reads these, so that it agrees with the steps that come after)
  read   rows of a context as bf16, fp16 or fp32
"""
import math

import torch

own = False   # True: run() calls this library's kernels, False: the plain form

DEV = "cuda"
MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token early in a conversation, 32 query and 4 kv heads: bound by latency
        _attn("attn one token, 500", B=1, M=1, Hkv=4, G=8, S=4096, ctx=500),
        # one token over a long document
        _attn("attn one token, 32000", B=1, M=1, Hkv=4, G=8, S=32768, ctx=32000),
        # speculative verify over a long document: one token and eight drafts
        _attn("attn nine tokens, 23001", B=1, M=9, Hkv=4, G=8, S=23296, ctx=23001),
        # a server's step: sequences of all lengths up to 8192, some slots empty
        _attn("attn 48 sequences", B=48, M=1, Hkv=4, G=8, S=8192, ctx=8192, page=64, ragged=True, out="bf16"),
        # the same over long contexts
        _attn("attn 32 long sequences", B=32, M=1, Hkv=4, G=8, S=32768, ctx=32768, page=128, ragged=True),
        # a small model's heads: 15 query and 5 kv heads of 64, fp16, the smallest pages
        _attn("attn odd heads", B=7, M=3, Hkv=5, G=3, D=64, S=1360, ctx=1350, page=16, ragged=True, q="fp16"),
        # a piece of a long prompt over what is written so far
        _attn("attn prompt piece", B=1, M=512, Hkv=4, G=8, S=8192, ctx=8192, out="bf16"),
        # the new token of every sequence of a batch
        _write("write 48 tokens", B=48, M=1, Hkv=4, S=8192, page=64),
        # a whole prompt
        _write("write prompt of 8000", B=1, M=8000, Hkv=4, S=8192),
        # a small model's heads, fp16, drafts of several tokens that cross pages
        _write("write odd heads", B=13, M=33, Hkv=5, D=64, S=1360, page=16, x="fp16"),
        # one conversation's context
        _read("read 4097", B=1, n=4097, Hkv=4, S=8192),
        # the contexts of a batch, for a library's attention
        _read("read 16 contexts", B=16, n=4000, Hkv=4, S=4096, page=64),
    ]


def _attn(name, B, M, Hkv, G, S, ctx, D=128, page=0, ragged=False, q="bf16", out="fp32"):
    return {"name": name, "op": "attn", "B": B, "M": M, "Hkv": Hkv, "G": G, "D": D, "S": S, "ctx": ctx, "page": page,
            "ragged": ragged, "x": q, "out": out}


def _write(name, B, M, Hkv, S, D=128, page=0, x="bf16"):
    return {"name": name, "op": "write", "B": B, "M": M, "Hkv": Hkv, "D": D, "S": S, "page": page, "x": x}


def _read(name, B, n, Hkv, S, D=128, page=0, out="bf16"):
    return {"name": name, "op": "read", "B": B, "n": n, "Hkv": Hkv, "D": D, "S": S, "page": page, "out": out}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "attn", "piece", "write", "read"])
    D, Hkv = rng.choice([64, 128, 128]), rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([0, 0, 16, 32, 64, 128])
    if op == "attn":      # steps of one to sixteen tokens, of one to many sequences
        B = rng.choice([1, _log(rng, 1, 64)])
        M = rng.choice([1, _log(rng, 1, 16)])
        ctx = _log(rng, M, 32768)
        ctx = max(M, min(ctx, 1900000 // (B * Hkv)))
        S = _room(rng, ctx, page)
        c = _attn("", B, M, Hkv, rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16]), S, ctx, D, page, rng.random() < 0.6,
                  rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["fp32", "bf16"]))
    elif op == "piece":   # pieces of a prompt
        B, M, G = rng.choice([1, 1, 2]), _log(rng, 17, 640), rng.choice([1, 4, 5, 8])
        ctx = min(M + _log(rng, 1, 8192), (1 << 27) // (B * Hkv * G * M))
        ctx = max(M, ctx)
        c = _attn("", B, M, Hkv, G, _room(rng, ctx, page), ctx, D, page, rng.random() < 0.3,
                  rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["fp32", "bf16"]))
    elif op == "write":
        B = rng.choice([1, _log(rng, 1, 64)])
        M = _log(rng, 1, 8192 // B)
        c = _write("", B, M, Hkv, _room(rng, M + _log(rng, 1, 4096), page), D, page, rng.choice(["bf16", "fp16", "fp32"]))
    else:
        B = rng.choice([1, _log(rng, 1, 32)])
        n = _log(rng, 1, 200000 // (B * Hkv))
        c = _read("", B, n, Hkv, _room(rng, n, page), D, page, rng.choice(["bf16", "fp16", "fp32"]))
    del c["name"]
    return c


def _room(rng, n, page):
    """Positions of a cache that holds n: a multiple of 16, or of the page."""
    step = page or 16
    return (n + rng.randrange(0, n + 1) // 2 + step - 1) // step * step


# ------------------------------------------------------------------ what a pass works on
def _lens(case):
    """Positions of each sequence after the step: one of them full, the others spread over the range; every sixteenth
    slot of a ragged batch is empty."""
    B, M, ctx = case["B"], case["M"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    g = 0.6180339887498949
    return [0 if i % 16 == 3 else M + int((ctx - M) * ((1.0 if i == 0 else (i * g) % 1.0))) for i in range(B)]


def _rand(shape, gen):
    """Keys or values as they come: a channel scale that is log-normal, so that blocks differ, on normal values."""
    x = torch.randn(shape, generator=gen, device=DEV)
    return x * torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device=DEV))


def _fill(n, page, Hkv, D, gen):
    """A cache of n pages and its content."""
    q = torch.empty((n, Hkv, page, D // 2), dtype=torch.uint8, device=DEV)
    s = torch.empty((n, Hkv, page, D // 32), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (Hkv * page * D))
    for i in range(0, n, step):
        m = min(step, n - i)
        q[i:i + m], s[i:i + m] = _quantize(_rand((m, page, Hkv, D), gen).transpose(1, 2))
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    B, Hkv, D, S, page = case["B"], case["Hkv"], case["D"], case["S"], case["page"]
    st = {"case": case, "pages": None}
    n, P = (B, S) if not page else (B * (S // page) + 3, page)
    if page:   # a pool whose pages are handed out in no order; pages past a sequence's end are not handed out
        perm = torch.randperm(n, generator=gen, device=DEV)[:B * (S // page)].view(B, S // page).to(torch.int32)
        if case["op"] == "attn":
            used = torch.tensor([(x + page - 1) // page for x in _lens(case)], device=DEV)
            perm = torch.where(torch.arange(S // page, device=DEV) < used[:, None], perm, -1).to(torch.int32)
        st["pages"] = perm.contiguous()
    kq, ks = _fill(n, P, Hkv, D, gen)
    vq, vs = _fill(n, P, Hkv, D, gen)
    st["cache"] = (kq, ks, vq, vs)
    if case["op"] == "attn":
        M, Hq = case["M"], Hkv * case["G"]
        st["dpos"] = torch.tensor([x - M for x in _lens(case)], dtype=torch.int32, device=DEV)
        st["q"] = (1.5 * torch.randn((B, M, Hq, D), generator=gen, device=DEV)).to(DT[case["x"]])
    elif case["op"] == "write":
        M = case["M"]
        st["dpos"] = torch.randint(0, S - M + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
        st["k"] = _rand((B, M, Hkv, D), gen).to(DT[case["x"]])
        st["v"] = _rand((B, M, Hkv, D), gen).to(DT[case["x"]])
    else:
        st["start"] = torch.randint(0, S - case["n"] + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    case, cache, pages = st["case"], st["cache"], st["pages"]
    if own:
        from moe_fused_inference_amd import kv4
        if case["op"] == "attn":
            return kv4.attn_decode4(st["q"], cache, st["dpos"], pages=pages, dtype=DT[case["out"]])
        if case["op"] == "write":
            kv4.kv4_write(st["k"], st["v"], cache, st["dpos"], pages=pages)
            return kv4.kv4_read(cache, case["M"], start=st["dpos"], pages=pages, dtype=torch.bfloat16)
        return kv4.kv4_read(cache, case["n"], start=st["start"], pages=pages, dtype=DT[case["out"]])
    if case["op"] == "attn":
        return _plain_attn(st["q"], cache, st["dpos"], pages, DT[case["out"]])
    if case["op"] == "write":
        _plain_write(st["k"], st["v"], cache, st["dpos"], pages)
        return _plain_read(cache, case["M"], st["dpos"], pages, torch.bfloat16)
    return _plain_read(cache, case["n"], st["start"], pages, DT[case["out"]])


def _quantize(x):
    """x (..., D) -> nibbles u8 (..., D/2), codes u8 (..., D/32)."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(b.abs().amax(-1) / 6)          # amax / 6 = m 2^e, m in [1/2, 1)
    e = torch.where(m > 0.5, e, e - 1)                # the smallest 2^e that is not below it
    e = torch.where(m == 0, 0, e).clamp(-127, 127)
    t = torch.ldexp(b, -e[..., None])
    a = t.abs()
    c = ((a >= 0.25).to(torch.uint8) + (a >= 0.75) + (a >= 1.25) + (a >= 1.75) + (a >= 2.5) + (a >= 3.5) + (a >= 5)
         + 8 * (t < 0).to(torch.uint8))
    c = c.reshape(*x.shape[:-1], -1, 2)
    return c[..., 0] | (c[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(q, s):
    """nibbles (..., D/2), codes (..., D/32) -> fp32 (..., D)."""
    mags = torch.tensor(MAGS + tuple(-v for v in MAGS), device=q.device)
    v = mags[torch.stack((q & 15, q >> 4), -1).long()].reshape(*s.shape, 32)
    return torch.ldexp(v, (s.int() - 127)[..., None]).reshape(*q.shape[:-1], -1)


def _rows(dpos, M, cache, pages):
    """(page, row in it, there) of positions dpos[b] .. dpos[b] + M - 1."""
    page = cache[0].shape[2]
    pos = dpos.long()[:, None] + torch.arange(M, device=dpos.device)
    B, top = dpos.numel(), page * (pages.shape[1] if pages is not None else 1)
    there = (pos >= 0) & (pos < top)
    pos = pos.clamp(0, top - 1)
    if pages is None:
        return torch.arange(B, device=dpos.device)[:, None].expand_as(pos), pos, there
    pid = pages.long().gather(1, pos // page)
    there &= (pid >= 0) & (pid < cache[0].shape[0])
    return pid.clamp(0, cache[0].shape[0] - 1), pos % page, there


def _plain_write(k, v, cache, dpos, pages):
    pid, row, there = _rows(dpos, k.shape[1], cache, pages)
    pid, row = pid[there], row[there]
    for x, q, s in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        q[pid, :, row], s[pid, :, row] = _quantize(x[there])


def _plain_read(cache, n, start, pages, dtype):
    pid, row, there = _rows(start, n, cache, pages)
    k, v = (_values(q[pid, :, row], s[pid, :, row]) * there[..., None, None]
            for q, s in ((cache[0], cache[1]), (cache[2], cache[3])))
    return k.to(dtype), v.to(dtype)


def _plain_attn(q, cache, dpos, pages, dtype):
    B, M, Hq, D = q.shape
    if pages is not None:   # each sequence's pages side by side
        there = (pages >= 0) & (pages < cache[0].shape[0])
        at = torch.where(there, pages, 0).long()
        cache = [c[at].transpose(1, 2).flatten(2, 3) for c in cache]
    k, v = _values(cache[0], cache[1]), _values(cache[2], cache[3])     # (B, Hkv, S, D)
    Hkv, S = k.shape[1], k.shape[2]
    x = q.float().view(B, M, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = torch.matmul(x, k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, M, S) / math.sqrt(D)
    pos = torch.arange(S, device=q.device)
    seen = pos <= dpos[:, None, None] + torch.arange(M, device=q.device)[:, None]      # (B, M, S)
    if pages is not None:
        seen &= there.repeat_interleave(S // pages.shape[1], 1)[:, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38))        # a row that sees nothing: all zeros
    o = torch.matmul(p.view(B, Hkv, -1, S), v).view(B, Hkv, -1, M, D)
    o = o / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, M, Hq, D).to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    row = Hkv * (D // 2 + D // 32)                       # bytes of a position's keys, or values
    if case["op"] == "attn":
        M, Hq, lens = case["M"], Hkv * case["G"], [x for x in _lens(case) if x]
        seen = sum(M * x - M * (M - 1) // 2 for x in lens)
        return {"bytes": 2 * row * sum(lens) + B * M * Hq * D * (size[case["x"]] + size[case["out"]]),
                "flops": 4 * D * Hq * seen}
    if case["op"] == "write":
        T = B * case["M"]
        return {"bytes": 2 * T * (Hkv * D * (size[case["x"]] + 2) + row), "flops": 2 * T * Hkv * D * 8}
    T = B * case["n"]
    return {"bytes": 2 * T * (row + Hkv * D * size[case["out"]]), "flops": 2 * T * Hkv * D}


# ------------------------------------------------------------------ the definition, in 64 bits
def _decode64(q, s):
    """E2M1 by its fields: exponent e, mantissa m: e = 0: m / 2, else (1 + m / 2) 2^(e - 1)."""
    n = torch.empty((*q.shape, 2), dtype=torch.float64, device=q.device)
    for j, c in enumerate((q.int() % 16, q.int() // 16)):
        e, m = (c // 2) % 4, (c % 2).double()
        n[..., j] = torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2.0, (e - 1).double())) * (1 - 2 * (c // 8))
    n = n.flatten(-2).unflatten(-1, (-1, 32))
    return (n * torch.pow(2.0, s.double() - 127)[..., None]).flatten(-2)


def _sequence64(x, b, pages, upto):
    """Positions 0 .. upto - 1 of sequence b of a tensor (n_pages, Hkv, page, .), as (Hkv, upto, .)."""
    if pages is None:
        return x[b, :, :upto]
    ids = pages[b, :(upto + x.shape[2] - 1) // x.shape[2]].long()
    return x[ids].transpose(0, 1).flatten(1, 2)[:, :upto]


def _round64(x):
    """The nearest MXFP4 values of x (..., D) with the smallest block scale that clips nothing, ties away from zero."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 6))                     # corrected where log2 rounds across a power of two
    e = torch.where(torch.pow(2.0, e - 1) * 6 >= top, e - 1, e)
    e = torch.where(torch.pow(2.0, e) * 6 < top, e + 1, e)
    scale = torch.where(top > 0, torch.pow(2.0, e.clamp(-127, 127)), 1.0)
    grid = torch.tensor(MAGS, dtype=torch.float64, device=x.device)
    mids = (grid[1:] + grid[:-1]) / 2
    return (torch.sign(b) * grid[torch.bucketize((b / scale).abs(), mids, right=True)] * scale).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    cache, pages, B = st["cache"], st["pages"], case["B"]
    if case["op"] == "write":
        return _round64(st["k"]), _round64(st["v"])
    if case["op"] == "read":
        got = []
        for q, s in ((cache[0], cache[1]), (cache[2], cache[3])):
            rows = []
            for b, at in enumerate(st["start"].tolist()):
                v = _decode64(_sequence64(q, b, pages, at + case["n"])[:, at:], _sequence64(s, b, pages, at + case["n"])[:, at:])
                rows.append(v.transpose(0, 1))
            got.append(torch.stack(rows))
        return tuple(got)
    M, G, D, Hkv = case["M"], case["G"], case["D"], case["Hkv"]
    o = torch.zeros((B, M, Hkv, G, D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case)):
        if not n:
            continue
        k, v = (_decode64(_sequence64(q, b, pages, n), _sequence64(s, b, pages, n))
                for q, s in ((cache[0], cache[1]), (cache[2], cache[3])))
        late = torch.arange(n, device=DEV) > n - M + torch.arange(M, device=DEV)[:, None]
        for h in range(Hkv):
            x = st["q"][b].double().view(M, Hkv, G, D)[:, h].transpose(0, 1)            # (G, M, D)
            w = (x @ k[h].T) * D ** -0.5
            o[b, :, h] = (torch.softmax(w.masked_fill(late, -math.inf), -1) @ v[h]).transpose(0, 1)
    return o.view(B, M, Hkv * G, D)
