"""The operators of serving from a paged cache, as a list of cases that can be timed and compared.

Four operators, as one pass over a ragged batch of sequences calls them, one layer after the other:
  rope    heads of queries and keys normalised and rotated, `ops.rope_heads`
  write   the same, keys and values going into the pages of their sequences, `ops.rope_to_pages`; pages of 8 bits are read back
          (`ops.read_pages`), so that what they hold is compared as the values it stands for
  read    whole sequences out of their pages, `ops.read_pages`
  attend  attention of each sequence's new tokens over everything it has in the pages, `ops.paged_attention`

The path has inference only.  A case is a dict of plain values; `draw` makes more of the same ranges.  With `own` false the
operators are computed from elementary torch operations, in 32 bits (angles in 64).
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}
EPS = 1e-6
THETA = 10000.0
FACTOR = 1.1                 # on cosines and sines, as scalings for long contexts ask for
MOST_CODE, LEAST_EXPONENT, MOST_EXPONENT = 448.0, -32, 8
MAX_SCORES = 0.8e9           # of a drawn attention with heads of 128, every sequence as long as the longest: the largest listed has as many
MAX_ROWS = 70000             # tokens that a drawn case writes or reads


def _rope(name, tokens, heads, kv_heads, head_dim, rotary, first, interleaved=False, norm=False, dtype="float16"):
    case = {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary, "first": first,
            "interleaved": interleaved, "norm": norm, "dtype": dtype}
    return dict(case, name=name) if name else case


def _write(name, seqs, new, past, ragged, heads, kv_heads, head_dim, page, pages="float16", interleaved=False, norm=False, dtype="float16"):
    case = {"kind": "write", "seqs": seqs, "new": new, "past": past, "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "pages": pages, "interleaved": interleaved, "norm": norm, "dtype": dtype}
    return dict(case, name=name) if name else case


def _read(name, seqs, past, ragged, kv_heads, head_dim, page, pages="float16", dtype="float16"):
    case = {"kind": "read", "seqs": seqs, "new": 0, "past": past, "ragged": ragged, "heads": kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "pages": pages, "dtype": dtype}
    return dict(case, name=name) if name else case


def _attend(name, seqs, new, past, ragged, heads, kv_heads, head_dim, page, pages="float16"):
    case = {"kind": "attend", "seqs": seqs, "new": new, "past": past, "ragged": ragged, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "pages": pages, "dtype": "float16"}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decoded token, the heads of the framework's default configuration: the smallest call, where launch and latency count
        _rope("rope_1", 1, 32, 32, 128, 128, 2000),
        # a prompt chunk far into a long context, shared key heads, norms on queries and keys
        _rope("rope_norm_4096", 4096, 32, 8, 128, 128, 500000, norm=True),
        # odd sizes: 777 fp32 rows, heads of 96 of which 40 values are rotated, neighbouring pairs
        _rope("rope_partial_fp32", 777, 12, 4, 96, 40, 3, interleaved=True, dtype="float32"),
        # a decode step of 64 sequences
        _write("write_64x1", 64, 1, 2000, True, 32, 8, 128, 16),
        # prompts on their way into pages of 8 bits, and read back
        _write("write_e4m3_4x2048", 4, 2048, 0, False, 32, 8, 128, 64, pages="e4m3", norm=True),
        # a batch of sequences handed to a path with a contiguous cache
        _read("read_ragged_16", 16, 2048, True, 32, 128, 16),
        # one long document out of pages of 8 bits
        _read("read_e4m3_65536", 1, 65536, False, 8, 128, 256, pages="e4m3"),
        # one short sequence, one token: latency
        _attend("decode_1x600", 1, 1, 600, False, 32, 32, 128, 16),
        # a decode step of 64 sequences of very different lengths
        _attend("decode_64_ragged", 64, 1, 6000, True, 32, 8, 128, 16),
        # a decode step over long contexts in 8 bits
        _attend("decode_e4m3_4x100000", 4, 1, 100000, False, 32, 8, 128, 128, pages="e4m3"),
        # chunks and single tokens in one pass: heads of 64, seven queries a key head, 8 bits
        _attend("mixed_e4m3_8_ragged", 8, 500, 3000, True, 14, 2, 64, 32, pages="e4m3"),
        # a chunk of a long prompt over what is there already: the largest pass
        _attend("chunk_4096_over_4096", 1, 4096, 4096, False, 32, 8, 128, 64),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    return min(kv * rng.choice([1, 1, 2, 4, 4, 5, 7, 8]), 64) // kv * kv, kv


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attend", "attend", "attend"])
    heads, kv = _heads(rng)
    head_dim = rng.choice([64, 128, 128, 256])
    page, pages = rng.choice([16, 32, 64, 128, 256]), rng.choice(["float16", "e4m3"])
    dtype = rng.choice(["float16", "float16", "float32"])
    interleaved, norm, ragged = rng.random() < 0.4, rng.random() < 0.5, rng.random() < 0.6
    if kind == "rope":
        head_dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        rotary = head_dim if rng.random() < 0.6 else 2 * rng.randint(4, head_dim // 2)
        return _rope(None, _log_int(rng, 1, 8192), heads, kv, head_dim, rotary, _log_int(rng, 1, 1000000), interleaved, norm, dtype)
    if kind == "write":
        seqs, new = _log_int(rng, 1, 64), _log_int(rng, 1, 4096)
        while seqs * new > 8192:
            seqs, new = _log_int(rng, 1, 64), _log_int(rng, 1, 4096)
        return _write(None, seqs, new, min(_log_int(rng, 1, 4096), 65536 // seqs), ragged, heads, kv, head_dim, page, pages, interleaved, norm, dtype)
    if kind == "read":
        seqs, past = _log_int(rng, 1, 32), _log_int(rng, 1, 65536)
        while seqs * past * kv * head_dim > MAX_ROWS * 8 * 128:
            seqs, past = _log_int(rng, 1, 32), _log_int(rng, 1, 65536)
        return _read(None, seqs, past, ragged, kv, head_dim, page, pages, dtype)
    head_dim = rng.choice([64, 128, 128, 128, 256])
    while True:
        seqs, new, past = _log_int(rng, 1, 64), rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 2048)]), _log_int(rng, 1, 100000)
        if heads * seqs * new * (past + new) * max(1, head_dim // 128) <= MAX_SCORES and seqs * (past + new) * kv * head_dim <= 400000 * 8 * 128:
            return _attend(None, seqs, new, past, ragged, heads, kv, head_dim, page, pages)


def _lengths(case):
    """(new, length) of every sequence: all alike, or, ragged, of any size up to the case's, every third of a single token.  The
    first has the full sizes."""
    rng = random.Random(case["seqs"] * 7919 + case["new"] * 31 + case["past"])
    both = []
    for i in range(case["seqs"]):
        new, past = case["new"], case["past"]
        if case["ragged"] and i > 0:
            new = 0 if new == 0 else 1 if i % 3 == 0 else _log_int(rng, 1, new)
            past = _log_int(rng, 1, past) if past else 0
        both.append((new, past + new))
    return both


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    state = {"case": case}
    rotary = case.get("rotary", hd)
    if case["kind"] in ("rope", "write"):
        state["frequencies"] = THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
        state["norms"] = tuple(1.0 + 0.1 * normal(hd) for _ in range(2)) if case["norm"] else (None, None)
    if case["kind"] == "rope":
        qkv = normal(case["tokens"], heads + 2 * kv, hd)  # one product's rows: queries, keys and values side by side
        state["q"], state["k"] = qkv[:, :heads], qkv[:, heads:heads + kv]
        state["positions"] = case["first"] + torch.arange(case["tokens"], device="cuda")
        return state
    page, lengths = case["page"], _lengths(case)
    per_seq = [-(-length // page) for _, length in lengths]
    count, widest = sum(per_seq), max(per_seq)
    total = count + 3                                       # a pool with pages that are nobody's, used in any order
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed))[:count]
    table = torch.zeros((len(lengths), widest), dtype=torch.int32)
    at = 0
    for i, n in enumerate(per_seq):
        table[i, :n] = order[at:at + n]
        at += n
    state["table"] = table.cuda()
    new = torch.tensor([n if case["kind"] != "read" else length for n, length in lengths])
    state["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).cuda()
    state["lengths"] = torch.tensor([length for _, length in lengths], dtype=torch.int32).cuda()
    state["most_new"], state["tokens"] = int(new.max()), int(new.sum())
    shape = (total, kv, page, hd)
    if case["pages"] == "float16":
        state["pages"] = (normal(*shape, dtype=torch.float16), normal(*shape, dtype=torch.float16), None, None)
    else:
        codes = [(100.0 * torch.randn(shape, generator=gen, device="cuda")).clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
        exponents = [torch.randint(119, 122, shape[:3], generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
        state["pages"] = (*codes, *exponents)
    if case["kind"] == "write":
        qkv = normal(state["tokens"], heads + 2 * kv, hd)
        state["q"], state["k"], state["v"] = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    elif case["kind"] == "attend":
        state["q"] = normal(state["tokens"], heads, hd)
    return state


def _normed(x, weight):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, positions, frequencies, interleaved):
    angle = positions.double()[:, None, None] * frequencies
    cos, sin = (FACTOR * angle.cos()).float(), (FACTOR * angle.sin()).float()
    r = 2 * frequencies.numel()
    lo, hi = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    lo, hi = lo * cos - hi * sin, hi * cos + lo * sin
    turned = torch.stack([lo, hi], dim=-1).flatten(-2) if interleaved else torch.cat([lo, hi], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _places(state):
    """For every token: its sequence, its index there, and the page and the row of that page that are its own."""
    starts, lengths, page = state["starts"].long(), state["lengths"].long(), state["case"]["page"]
    row = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    at = lengths[seq] - (starts[seq + 1] - starts[seq]) + row - starts[seq]
    return seq, at, state["table"].long()[seq, at // page], at % page


def _quantised(x):
    """Codes and biased exponents of rows of 8 bits: x = code * 2^exponent, the exponent the least that holds the row."""
    most = x.abs().amax(-1)
    part, exponent = torch.frexp(most / MOST_CODE)
    exponent = torch.where(most > 0, exponent - (part == 0.5).int(), LEAST_EXPONENT).clamp(LEAST_EXPONENT, MOST_EXPONENT)
    bound = torch.where(exponent == MOST_EXPONENT, 240.0, MOST_CODE)[..., None]
    codes = torch.minimum(torch.maximum(x * torch.exp2(-exponent.float())[..., None], -bound), bound).to(torch.float8_e4m3fn)
    return codes, (exponent + 127).to(torch.uint8)


def _value(codes, exponents):
    return codes.float() if exponents is None else codes.float() * torch.exp2(exponents.float() - 127)[..., None]


def _plain_read(state, dtype):
    _, _, page, row = _places(state)
    k, v, ke, ve = state["pages"]
    return tuple(_value(t[page, :, row], None if e is None else e[page, :, row]).to(dtype) for t, e in ((k, ke), (v, ve)))


def _plain_write(state):
    case = state["case"]
    _, at, page, row = _places(state)
    q, k = (_rotated(_normed(state[n], w), at, state["frequencies"], case["interleaved"]) for n, w in zip("qk", state["norms"]))
    for x, codes, exponents in ((k, state["pages"][0], state["pages"][2]), (state["v"].float(), state["pages"][1], state["pages"][3])):
        if exponents is None:
            codes[page, :, row] = x.to(codes.dtype)
        else:
            c, e = _quantised(x)
            codes.view(torch.uint8)[page, :, row] = c.view(torch.uint8)
            exponents[page, :, row] = e
    return q.to(state["q"].dtype)


def _plain_attend(state):
    case = state["case"]
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    starts, lengths, table = state["starts"].long(), state["lengths"].long(), state["table"].long()
    B, n, longest = case["seqs"], state["most_new"], table.shape[1] * case["page"]
    k, v = ((_value(t[table], None if e is None else e[table])).permute(0, 2, 1, 3, 4).reshape(B, kv, longest, hd)
            for t, e in ((state["pages"][0], state["pages"][2]), (state["pages"][1], state["pages"][3])))
    new = starts[1:] - starts[:-1]
    token = torch.arange(n, device="cuda")
    row = (starts[:-1, None] + token).clamp(max=state["tokens"] - 1)
    q = state["q"].float()[row].view(B, n, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, heads // kv * n, hd)
    last = lengths[:, None] - new[:, None] + token                                      # the last key that a token sees
    key = torch.arange(longest, device="cuda")
    hidden = (key > last[..., None]) | (key >= lengths[:, None, None])                  # [B, n, longest]
    v = v.masked_fill((key >= lengths[:, None])[:, None, :, None], 0.0)
    scores = (q @ k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(hd)).view(B, kv, heads // kv, n, longest)
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(B, kv, -1, longest) @ v).view(B, kv, heads // kv, n, hd) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, heads * hd)
    seq, at, _, _ = _places(state)
    return out[seq, at - lengths[seq] + new[seq]].to(torch.float16)


@torch.no_grad()
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        from ternaryllm_amd import ops
        if kind in ("rope", "write"):
            how = {"factor": FACTOR, "interleaved": case["interleaved"], "q_norm": state["norms"][0], "k_norm": state["norms"][1], "eps": EPS}
        if kind == "rope":
            return ops.rope_heads(state["q"], state["k"], state["positions"], state["frequencies"], **how)
        pages = ops.Pages(*state["pages"])
        batch = ops.PageBatch(state["table"], state["starts"], state["lengths"], state["most_new"])
        if kind == "write":
            q = ops.rope_to_pages(state["q"], state["k"], state["v"], pages, batch, state["frequencies"], **how)
            if case["pages"] == "float16":
                return q, pages.k, pages.v
            return (q, *ops.read_pages(pages, batch, state["tokens"]))
        if kind == "read":
            return ops.read_pages(pages, batch, state["tokens"], DTYPES[case["dtype"]])
        return ops.paged_attention(state["q"], pages, batch)
    if kind == "rope":
        return tuple(_rotated(_normed(state[n], w), state["positions"], state["frequencies"], case["interleaved"]).to(state[n].dtype)
                     for n, w in zip("qk", state["norms"]))
    if kind == "write":
        q = _plain_write(state)
        return (q, *state["pages"][:2]) if case["pages"] == "float16" else (q, *_plain_read(state, torch.float16))
    return _plain_read(state, DTYPES[case["dtype"]]) if kind == "read" else _plain_attend(state)


def work(case):
    """Bytes: every input and every output once, of the pages the rows that are read or written.  Operations: the two products of
    the attention over the keys that each token sees, and a handful for each rotated value."""
    heads, kv, hd, kind = case["heads"], case["kv_heads"], case["head_dim"], case["kind"]
    es = 2 if case["dtype"] == "float16" else 4
    if kind == "rope":
        return {"bytes": case["tokens"] * ((heads + kv) * hd * 2 * es + 8) + case["rotary"] * 4 + (2 * hd * es if case["norm"] else 0),
                "flops": case["tokens"] * (heads + kv) * hd * (7 if case["norm"] else 3)}
    lengths = _lengths(case)
    row = 2 * kv * (hd * 2 if case["pages"] == "float16" else hd + 1)          # a token's key and value rows in the pages
    table = sum(-(-length // case["page"]) for _, length in lengths) * 4 + len(lengths) * 8
    if kind == "read":
        tokens = sum(length for _, length in lengths)
        return {"bytes": tokens * (row + 2 * kv * hd * es) + table, "flops": tokens * 2 * kv * hd}
    tokens = sum(new for new, _ in lengths)
    if kind == "write":
        back = 0 if case["pages"] == "float16" else tokens * (row + 2 * kv * hd * 2)
        return {"bytes": tokens * ((2 * heads + 2 * kv) * hd * es + row) + back + table + hd * 4 + (2 * hd * es if case["norm"] else 0),
                "flops": tokens * (heads + kv) * hd * (7 if case["norm"] else 3)}
    pairs = sum(new * length - new * (new - 1) // 2 for new, length in lengths)
    return {"bytes": sum(length for _, length in lengths) * row + 2 * tokens * heads * hd * 2 + table, "flops": 4 * pairs * heads * hd}


def _exact_rope(x, weight, positions, frequencies, interleaved):
    """x [tokens, heads, head_dim] normalised and rotated: the pairs as complex numbers times factor * exp(i angle)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    half = frequencies.numel()
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    turn = torch.polar(torch.full((), FACTOR, dtype=torch.float64, device="cuda"), positions.double()[:, None] * frequencies)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_held(x, e4m3):
    """What a row of a page stands for once x has been put into it: fp16, or the nearest of the 8-bit numbers (ties to the even
    one) times the row's power of two."""
    if not e4m3:
        return x.half()
    most = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(most, LEAST_EXPONENT)
    for power in range(LEAST_EXPONENT, MOST_EXPONENT):
        e = torch.where(most > MOST_CODE * 2.0 ** power, power + 1.0, e)
    y = x / torch.exp2(e)
    bound = torch.where(e == MOST_EXPONENT, 240.0, 448.0)
    y = torch.minimum(torch.maximum(y, -bound), bound)
    binade = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(binade - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def exact(case, seed):
    state = prepare(case, seed)
    kind, kv, hd = case["kind"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        return tuple(_exact_rope(state[n], w, state["positions"], state["frequencies"], case["interleaved"]) for n, w in zip("qk", state["norms"]))
    page, lengths, table = case["page"], _lengths(case), state["table"].tolist()
    k, v, ke, ve = state["pages"]

    def rows(seq, first, last, which):
        """Rows first .. last - 1 of a sequence as 64-bit values, page by page."""
        codes, exponents = (k, ke) if which == 0 else (v, ve)
        ids = torch.tensor(table[seq][first // page:-(-last // page)], device="cuda", dtype=torch.long)
        x = codes[ids].double()
        if exponents is not None:
            x = x * torch.pow(2.0, exponents[ids].double() - 127)[..., None]
        return x.transpose(1, 2).reshape(-1, kv, hd)[first % page:first % page + last - first]

    if kind == "read":
        return tuple(torch.cat([rows(i, 0, length, which) for i, (_, length) in enumerate(lengths)]) for which in (0, 1))
    if kind == "write":
        at = torch.cat([torch.arange(length - new, length, device="cuda") for new, length in lengths])
        q, key = (_exact_rope(state[n], w, at, state["frequencies"], case["interleaved"]) for n, w in zip("qk", state["norms"]))
        held = [_exact_held(x, case["pages"] == "e4m3") for x in (key, state["v"].double())]
        if case["pages"] == "e4m3":
            return (q, *held)
        first = 0
        for i, (new, length) in enumerate(lengths):
            for j in range(new):
                spot = length - new + j
                for codes, x in ((k, held[0]), (v, held[1])):
                    codes[table[i][spot // page], :, spot % page] = x[first + j]
            first += new
        return q, k, v
    group, first, out = case["heads"] // kv, 0, []
    for i, (new, length) in enumerate(lengths):
        keys, values = rows(i, 0, length, 0), rows(i, 0, length, 1)
        seen = torch.arange(length, device="cuda") <= torch.arange(length - new, length, device="cuda")[:, None]
        q = state["q"][first:first + new].double()
        heads = []
        for h in range(case["heads"]):
            s = q[:, h] @ keys[:, h // group].t().contiguous() / math.sqrt(hd)
            heads.append(torch.softmax(torch.where(seen, s, -math.inf), dim=-1) @ values[:, h // group].contiguous())
        out.append(torch.stack(heads, 1).reshape(new, -1))
        first += new
    return torch.cat(out)
