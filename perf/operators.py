"""Cases of the decode step's attention operators: per-head norm and rotation,
the quantised paged cache (written and read back), attention over that cache
and attention with a prefix that the whole batch shares.

`run` computes an operator in its plain form (elementary torch operations in
32 bits) or, where `own` is true, by the framework's public entry points.

Cache layout (uint8 [pages, kv_heads, page_size / 16, block bytes]): a block
holds 16 tokens of one head, 16 rows of K, 16 rows of V (a row is head_dim *
bits / 8 bytes; int4: low nibble = even element), then 16 fp16 scales of K and
16 of V.  Rows are stored permuted inside their block, see `_positions`.
"""
import functools

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one token of one sequence through the norm and rotation: a launch's latency
        dict(name="rope 1 token", op="rope", tokens=1, q_heads=32, kv_heads=8, head_dim=128,
             rotary=128, pairs="halves", dtype="f16"),
        # a prompt's chunk, q and k as strided slices of one fused projection
        dict(name="rope 8192 tokens", op="rope", tokens=8192, q_heads=64, kv_heads=8,
             head_dim=128, rotary=128, pairs="halves", dtype="bf16"),
        # a decode batch's new tokens, appended and read back
        dict(name="append 16 int8", op="append", tokens=16, kv_heads=8, head_dim=128, bits=8,
             page=64, dtype="f16"),
        # a prompt's chunk quantised to 4 bits and read back
        dict(name="append 8192 int4", op="append", tokens=8192, kv_heads=8, head_dim=128, bits=4,
             page=64, dtype="bf16"),
        # an odd number of small-head tokens gathered from small pages
        dict(name="read 515 int8", op="read", tokens=515, kv_heads=4, head_dim=64, bits=8, page=16,
             dtype="bf16"),
        # a long context brought back to 16 bits
        dict(name="read 32768 int8", op="read", tokens=32768, kv_heads=8, head_dim=128, bits=8,
             page=64, dtype="f16"),
        # the first words of one conversation: latency
        dict(name="decode 1x77 int8", op="attention", batch=1, new=1, q_heads=32, kv_heads=8,
             head_dim=128, bits=8, page=16, len_min=77, len_max=77, window=0, dtype="f16"),
        # an ordinary ragged serving batch, an empty and a one-token sequence in it
        dict(name="decode 16 ragged int8", op="attention", batch=16, new=1, q_heads=64, kv_heads=8,
             head_dim=128, bits=8, page=64, len_min=0, len_max=4096, window=0, dtype="f16"),
        # several proposed tokens of a sequence checked at once, in a sliding window
        dict(name="verify 8x4 window int8", op="attention", batch=8, new=4, q_heads=32, kv_heads=4,
             head_dim=64, bits=8, page=32, len_min=100, len_max=4001, window=1024, dtype="bf16"),
        # a full server: long contexts in 4 bits
        dict(name="decode 64 long int4", op="attention", batch=64, new=1, q_heads=64, kv_heads=8,
             head_dim=128, bits=4, page=64, len_min=4096, len_max=8192, window=0, dtype="f16"),
        # a system prompt in front of a few short conversations
        dict(name="shared 1000 x16 int8", op="shared", batch=16, new=1, q_heads=32, kv_heads=8,
             head_dim=128, bits=8, page=16, prefix=1000, len_min=1, len_max=300, window=0,
             dtype="f16"),
        # a long document that a full batch asks about
        dict(name="shared 16384 x64 int8", op="shared", batch=64, new=1, q_heads=64, kv_heads=8,
             head_dim=128, bits=8, page=64, prefix=16384, len_min=1, len_max=1024, window=0,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attention", "attention", "attention", "shared",
                     "shared"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rope":
        dim = rng.choice([64, 80, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8])
        rotary = rng.choice([dim, dim, 32])
        return dict(op=op, tokens=_log(rng, 1, 8192) * 128 // max(dim, 128) or 1,
                    q_heads=heads * rng.choice([1, 4, 7, 8]), kv_heads=heads, head_dim=dim,
                    rotary=rotary, pairs=rng.choice(["halves", "neighbours"]), dtype=dtype)
    dim, heads = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    bits, page = rng.choice([8, 4]), rng.choice([16, 32, 64, 128])
    if op in ("append", "read"):
        most = (8192 if op == "append" else 32768) * 1024 // (heads * dim)
        return dict(op=op, tokens=_log(rng, 1, min(most, 65536)), kv_heads=heads, head_dim=dim,
                    bits=bits, page=page, dtype=dtype)
    new = rng.choice([1, 1, 1, 2, 3, 5, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    batch = _log(rng, 1, 64)
    per_token = heads * (dim * bits // 4 + 4)
    if op == "attention":
        len_max = _log(rng, 1, min(65536, 400_000_000 // (batch * per_token)))
        c = dict(window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))
    else:
        work = batch * new * group * heads * dim
        c = dict(prefix=_log(rng, 1, max(1, min(16384, 64 * 64 * 128 * 16384 // work))), window=0)
        len_max = _log(rng, 1, 1024)
    return dict(op=op, batch=batch, new=new, q_heads=heads * group, kv_heads=heads, head_dim=dim,
                bits=bits, page=page, len_min=rng.choice([0, 1, len_max // 2, len_max]),
                len_max=len_max, dtype=dtype, **c)


def _lengths(case):
    """The lengths of the batch, spread over [len_min, len_max] with both ends in it."""
    b, lo, hi = case["batch"], case["len_min"], case["len_max"]
    return [hi if b == 1 else lo + round((hi - lo) * i / (b - 1)) for i in range(b)]


def work(case):
    dim, kv = case["head_dim"], case["kv_heads"]
    if case["op"] == "rope":
        values = case["tokens"] * (case["q_heads"] + kv) * dim
        return {"bytes": 4 * values + case["tokens"] * (4 * case["rotary"] + 8) + 4 * dim,
                "flops": 8 * values}
    cached = kv * (dim * case["bits"] // 4 + 4)  # bytes of one token
    if case["op"] in ("append", "read"):
        values = case["tokens"] * kv * 2 * dim
        trips = 2 if case["op"] == "append" else 1
        return {"bytes": trips * (2 * values + case["tokens"] * cached) + 8 * case["tokens"],
                "flops": 4 * trips * values}
    rows, seen, read = case["new"] * case["q_heads"], 0, 0
    for n in _lengths(case):
        first = max(0, n - case["new"] + 1 - case["window"]) if case["window"] else 0
        read += n - first
        for i in range(case["new"]):
            at = n - case["new"] + i
            seen += max(0, min(at + 1, case["window"] or at + 1))
    prefix = case.get("prefix", 0)
    read += prefix
    seen += prefix * case["batch"] * case["new"]
    q = case["batch"] * rows * dim
    return {"bytes": read * cached + 4 * q + 4 * case["batch"] * rows
            + 4 * (read // case["page"] + case["batch"]),
            "flops": 4 * seen * case["q_heads"] * dim}


# --------------------------------------------------------- the cache's layout
@functools.lru_cache(None)
def _positions(row):
    """[16 * row] place inside its block part of each byte of 16 rows of `row` bytes."""
    j = torch.arange(16, device="cuda")[:, None]
    b = torch.arange(row, device="cuda")[None]
    chunk = b >> 4
    if row >= 128:
        chunk = chunk ^ (j & 7)
    elif row == 64:
        chunk = chunk ^ ((j >> 1) & 2)
        j = j ^ ((j >> 1) & 1)
    else:
        j = j ^ ((j >> 2) & 1)
    return (j * row + chunk * 16 + (b & 15)).reshape(-1)


def _unpack(part, row, bits):
    """uint8 [..., 16 * row] as stored -> fp32 [..., 16, head_dim] whole values."""
    part = part.index_select(-1, _positions(row)).unflatten(-1, (16, row))
    if bits == 8:
        return part.view(torch.int8).float()
    nibbles = torch.stack((part & 15, part >> 4), -1).flatten(-2)
    return (nibbles ^ 8).float() - 8


def _values(blocks, dim, bits):
    """uint8 [..., block bytes] -> the fp32 K and V [..., 16, dim] that they stand for."""
    row = dim * bits // 8
    scales = blocks[..., 32 * row:].contiguous().view(torch.float16).float()
    k = _unpack(blocks[..., :16 * row], row, bits) * scales[..., :16, None]
    v = _unpack(blocks[..., 16 * row:32 * row], row, bits) * scales[..., 16:, None]
    return k, v


def _quantise(x, bits):
    """fp32 [..., dim] -> whole values (int8) and the fp16 scale [...]."""
    top = 127 if bits == 8 else 7
    x = torch.nan_to_num(x)
    scale = (x.abs().amax(-1) / top).clamp(max=65504).half()
    inverse = torch.where(scale == 0, 0.0, 1.0 / scale.float())
    q = torch.round(x * inverse[..., None]).clamp(-top, top)
    return q.to(torch.int8), scale


def _bytes(q, bits):
    """int8 whole values [..., dim] -> uint8 [..., row]."""
    if bits == 8:
        return q.view(torch.uint8)
    q = q.view(torch.uint8).unflatten(-1, (-1, 2)) & 15
    return q[..., 0] | (q[..., 1] << 4)


def _blocks(k, v, bits):
    """fp32 K and V [..., 16, dim] -> uint8 [..., block bytes]."""
    parts, scales = [], []
    for x in (k, v):
        q, scale = _quantise(x, bits)
        b = _bytes(q, bits)
        inverse = torch.argsort(_positions(b.shape[-1]))
        parts.append(b.flatten(-2).index_select(-1, inverse))
        scales.append(scale.view(torch.uint8))
    return torch.cat(parts + scales, -1)


# ------------------------------------------------------------------ the inputs
def _filled_pages(pages, case, g):
    """A cache whose every token is written: K with a few strong channels, as real keys have."""
    dim, heads = case["head_dim"], case["kv_heads"]
    strong = 1 + 3 * (torch.rand(heads, 1, 1, dim, device="cuda", generator=g) > 0.95)
    row = dim * case["bits"] // 8
    out = torch.empty(pages, heads, case["page"] // 16, 32 * row + 64, dtype=torch.uint8,
                      device="cuda")
    step = max(1, (1 << 27) // (heads * case["page"] * dim))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        shape = (n, heads, case["page"] // 16, 16, dim)
        k = torch.randn(shape, device="cuda", generator=g) * strong
        v = torch.randn(shape, device="cuda", generator=g) + 0.1
        out[a:a + n] = _blocks(k, v, case["bits"])
    return out


@functools.lru_cache(None)
def _ext(name):
    from cudalab_b200.build import build
    return build(name)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, dim, kv = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    st = {"case": case}

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["op"] == "rope":
        n, heads = case["tokens"], case["q_heads"]
        qkv = normal(n, heads + 2 * kv, dim).to(dtype)  # one fused projection's output
        st["q"], st["k"] = qkv[:, :heads], qkv[:, heads:heads + kv]
        st["q_weight"] = (1 + 0.2 * normal(dim)).to(dtype)
        st["k_weight"] = (1 + 0.2 * normal(dim)).to(dtype)
        half = case["rotary"] // 2
        most = max(4096, n)
        angle = torch.arange(most, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda") / half)
        st["table"] = torch.cat((angle.cos(), angle.sin()), 1).contiguous()
        first = torch.randint(0, most - n + 1, (1,), device="cuda", generator=g)
        st["positions"] = torch.arange(n, device="cuda") + first
        return st

    page = case["page"]
    if case["op"] in ("append", "read"):
        n = case["tokens"]
        pages = -(-n // page) + 3
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(n, device="cuda") + page // 2  # starts inside a page
        st["slots"] = order[at // page] * page + at % page
        if case["op"] == "append":
            row = dim * case["bits"] // 8
            st["pages"] = torch.zeros(pages, kv, page // 16, 32 * row + 64, dtype=torch.uint8,
                                      device="cuda")
            st["k"], st["v"] = normal(n, kv, dim).to(dtype), normal(n, kv, dim).to(dtype)
        else:
            st["pages"] = _filled_pages(pages, case, g)
        return st

    batch, lengths = case["batch"], _lengths(case)
    width = max(1, -(-max(lengths) // page))
    shared = -(-case.get("prefix", 0) // page)
    order = torch.randperm(batch * width + shared, device="cuda", generator=g)
    st["pages"] = _filled_pages(len(order), case, g)
    st["table"] = order[:batch * width].view(batch, width).int()
    mixed = torch.randperm(batch, device="cuda", generator=g)
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")[mixed]
    if case["op"] == "shared":
        st["prefix"] = order[batch * width:].int()
    shape = (batch, case["q_heads"], dim)
    st["q"] = normal(*(shape if case["new"] == 1 else (batch, case["new"]) + shape[1:])).to(dtype)
    if own:
        st["workspace"] = _ext("kvattention").workspace("cuda")
    return st


# -------------------------------------------------------------- the plain forms
def _rope_plain(x, weight, st, case):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = case["rotary"] // 2
    row = st["table"][st["positions"]][:, None]
    c, s = row[..., :half], row[..., half:]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if case["pairs"] == "halves":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned, rest), -1).to(DTYPES[case["dtype"]])


def _append_plain(st, case):
    page, row = case["page"], case["head_dim"] * case["bits"] // 8
    slots = st["slots"]
    block, j = slots % page // 16, slots % 16
    at = slots // page
    for x, first in ((st["k"], 0), (st["v"], 1)):
        q, scale = _quantise(x.float(), case["bits"])
        # [tokens, 1, row] places of a token's bytes, [tokens, 1, 2] of its scale's
        place = _positions(row).view(16, row)[j][:, None] + first * 16 * row
        heads = torch.arange(case["kv_heads"], device="cuda")[None, :, None]
        where = (at[:, None, None], heads, block[:, None, None])
        st["pages"][where + (place,)] = _bytes(q, case["bits"])
        two = torch.arange(2, device="cuda") + (32 * row + 32 * first + 2 * j)[:, None, None]
        st["pages"][where + (two,)] = scale[..., None].view(torch.uint8)


def _read_plain(st, case):
    page, slots = case["page"], st["slots"]
    at, block, j = slots // page, slots % page // 16, slots % 16
    row = case["head_dim"] * case["bits"] // 8
    data = st["pages"][at, :, block]  # [tokens, heads, block bytes]
    place = _positions(row).view(16, row)[j][:, None].expand(-1, case["kv_heads"], -1)
    out = []
    for first in (0, 1):
        b = data.gather(-1, place + first * 16 * row)
        if case["bits"] == 8:
            x = b.view(torch.int8).float()
        else:
            x = (torch.stack((b & 15, b >> 4), -1).flatten(-2) ^ 8).float() - 8
        two = torch.arange(2, device="cuda") + (32 * row + 32 * first + 2 * j)[:, None, None]
        scale = data.gather(-1, two.expand(-1, case["kv_heads"], -1)).view(torch.float16)
        out.append((x * scale.float()).to(DTYPES[case["dtype"]]))
    return tuple(out)


def _attention_plain(st, case):
    dim, kv, new = case["head_dim"], case["kv_heads"], case["new"]
    batch = case["batch"]
    q = st["q"].float().view(batch, new, kv, -1, dim) * dim ** -0.5
    blocks = st["pages"][st["table"].long()]  # [batch, width, heads, blocks, bytes]
    k, v = _values(blocks, dim, case["bits"])
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(batch, kv, -1, dim)
    v = v.permute(0, 2, 1, 3, 4, 5).reshape(batch, kv, -1, dim)
    scores = torch.einsum("bqhgd,bhnd->bhqgn", q, k)
    j = torch.arange(k.shape[2], device="cuda")
    at = st["lengths"][:, None] - new + torch.arange(new, device="cuda")  # [batch, new]
    seen = j <= at[..., None]
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    scores = scores.masked_fill(~seen[:, None, :, None], float("-inf"))
    if case["op"] == "shared":
        pk, pv = _values(st["pages"][st["prefix"].long()], dim, case["bits"])
        pk = pk.permute(1, 0, 2, 3, 4).reshape(kv, -1, dim)[:, :case["prefix"]]
        pv = pv.permute(1, 0, 2, 3, 4).reshape(kv, -1, dim)[:, :case["prefix"]]
        front = torch.einsum("bqhgd,hnd->bhqgn", q, pk)
        scores = torch.cat((front, scores), -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).squeeze(-1)
    p = torch.where(total == 0, 0.0, p / total)
    if case["op"] == "shared":
        n = case["prefix"]
        out = torch.einsum("bhqgn,hnd->bqhgd", p[..., :n], pv)
        out = out + torch.einsum("bhqgn,bhnd->bqhgd", p[..., n:], v)
    else:
        out = torch.einsum("bhqgn,bhnd->bqhgd", p, v)
    shape = st["q"].shape
    return (out.to(st["q"].dtype).reshape(shape),
            lse.permute(0, 2, 1, 3).reshape(shape[:-1]).contiguous())


def run(st):
    case = st["case"]
    if case["op"] == "rope":
        if own:
            return _ext("qknorm_rope").forward(
                st["q"], st["k"], st["q_weight"], st["k_weight"], st["table"], st["positions"],
                eps=EPS, interleaved=case["pairs"] == "neighbours")
        return (_rope_plain(st["q"], st["q_weight"], st, case),
                _rope_plain(st["k"], st["k_weight"], st, case))
    if case["op"] in ("append", "read"):
        if own:
            cache = _ext("kvcache")
            if case["op"] == "append":
                cache.write(st["k"], st["v"], st["pages"], st["slots"])
            return cache.read(st["pages"], st["slots"], case["head_dim"], DTYPES[case["dtype"]])
        if case["op"] == "append":
            _append_plain(st, case)
        return _read_plain(st, case)
    if own:
        attend = _ext("kvattention")
        if case["op"] == "shared":
            return attend.forward_shared(st["q"], st["pages"], st["prefix"], case["prefix"],
                                         st["table"], st["lengths"], workspace=st["workspace"],
                                         return_lse=True)
        return attend.forward(st["q"], st["pages"], st["table"], st["lengths"],
                              window=case["window"], workspace=st["workspace"], return_lse=True)
    return _attention_plain(st, case)


# ------------------------------------------------------------ the definition
def _token(pages, slots, case):
    """fp64 K and V [tokens, heads, dim] of single tokens, byte by byte."""
    page, dim, bits = case["page"], case["head_dim"], case["bits"]
    row = dim * bits // 8
    data = pages[slots // page, :, (slots % page) // 16].double()  # [tokens, heads, bytes]
    j = slots % 16
    out = []
    for part in (0, 1):
        x = torch.empty(len(slots), data.shape[1], dim, dtype=torch.float64, device="cuda")
        for c in range(max(1, row // 16)):  # 16 bytes at a time
            if row >= 128:
                start = j * row + 16 * (c // 8 * 8 + (c % 8 ^ (j % 8)))
            elif row == 64:
                start = (j ^ (j // 2 % 2)) * 64 + 16 * (c ^ (2 * (j // 4 % 2)))
            else:
                start = (j ^ (j // 4 % 2)) * 32 + 16 * c
            start = start + part * 16 * row
            b = data.gather(2, (start[:, None] + torch.arange(16, device="cuda"))[:, None]
                            .expand(-1, data.shape[1], -1))
            if bits == 8:
                x[..., 16 * c:16 * c + 16] = torch.where(b > 127, b - 256, b)
            else:
                low, high = b % 16, torch.floor(b / 16)
                x[..., 32 * c:32 * c + 32:2] = torch.where(low > 7, low - 16, low)
                x[..., 32 * c + 1:32 * c + 32:2] = torch.where(high > 7, high - 16, high)
        at = 32 * row + 32 * part + 2 * j
        lo = data.gather(2, at[:, None, None].expand(-1, data.shape[1], 1))
        hi = data.gather(2, at[:, None, None].expand(-1, data.shape[1], 1) + 1)
        e, m = torch.floor(hi / 4) % 32, hi % 4 * 256 + lo  # fp16 scales are not negative
        scale = torch.where(e == 0, m * 2.0 ** -24, (1024 + m) * torch.exp2(e - 25))
        out.append(x * scale)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    dim = case["head_dim"]
    if case["op"] == "rope":
        out = []
        for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            half = case["rotary"] // 2
            i = torch.arange(half, device="cuda")
            a, b = (i, i + half) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., a], x[..., b])
            t = st["table"][st["positions"]].double()
            z = z * torch.complex(t[:, :half], t[:, half:])[:, None]
            y = x.clone()
            y[..., a], y[..., b] = z.real, z.imag
            out.append(y)
        return tuple(out)
    if case["op"] == "append":
        top, out = (127 if case["bits"] == 8 else 7), []
        for x in (st["k"].double(), st["v"].double()):
            s = (x.abs().amax(-1, keepdim=True) / top).half().double()
            out.append((torch.round(x / s)).clamp(-top, top) * s)
        return tuple(out)
    if case["op"] == "read":
        return tuple(_token(st["pages"], st["slots"], case))
    kv, new, page = case["kv_heads"], case["new"], case["page"]
    q = st["q"].double().view(case["batch"], new, kv, -1, dim) / dim ** 0.5
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:-1], float("-inf"), dtype=torch.float64, device="cuda")

    def slots(pages, n):
        j = torch.arange(n, device="cuda")
        return pages.long()[j // page] * page + j % page

    if case["op"] == "shared":
        pk, pv = _token(st["pages"], slots(st["prefix"], case["prefix"]), case)
    for b, n in enumerate(st["lengths"].tolist()):
        k, v = _token(st["pages"], slots(st["table"][b], n), case)
        if case["op"] == "shared":
            k, v = torch.cat((pk, k)), torch.cat((pv, v))
        before = k.shape[0] - n
        for i in range(new):
            end = before + max(0, n - new + i + 1)
            begin = max(0, end - case["window"]) if case["window"] else 0
            if end > begin:
                s = torch.einsum("hgd,nhd->hgn", q[b, i], k[begin:end])
                lse[b, i] = s.logsumexp(-1)
                p = (s - lse[b, i][..., None]).exp()
                out[b, i] = torch.einsum("hgn,nhd->hgd", p, v[begin:end])
    return out.view(st["q"].shape), lse.view(st["q"].shape[:-1])
