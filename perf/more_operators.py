"""The operators of many continuations of one prompt and of what they are worth, as a list of cases that can be timed and compared.

Three operators:
  share    attention of new tokens over a paged cache in which groups of sequences begin with the same tokens, whose keys and values are
           read once for a group, `ops.paged_attention(..., prefix=ops.PagePrefix(...))`
  loss     softmax cross entropy of hidden rows through a ternary head, no logits kept, `ops.cross_entropy`
  distill  the divergence of a ternary head's distribution from a teacher's, of which the top logits are known, `ops.distillation`

A loss is a pass that rates tokens, or a training step, which returns the gradients of the rows and of the head's column scales too.  A case
is a dict of plain values; `draw` makes more of the same ranges.  With `own` false the operators are computed from elementary torch
operations in 32 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}
IGNORED = -100               # the target of a row that counts for nothing
SPARSITY = 0.8               # of a head, the framework's default
SPREAD = 3.0                 # of logits: hidden rows of this size give distributions as peaked as a model's
MOST_COST = 4096 * 4096 * 32000      # rows * K * vocabulary of a drawn loss, of 16-bit rows: the largest listed
MOST_WEIGHTS = 4096 * 32000
MOST_SCORES = 256 * 32 * 16684       # scores of a drawn attention with heads of 128: the largest listed


def _share(name, groups, seqs, new, prefix, past, heads, kv_heads, head_dim, page, pages="float16"):
    case = {"kind": "share", "groups": groups, "seqs": seqs, "new": new, "prefix": prefix, "past": past, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "pages": pages}
    return dict(case, name=name) if name else case


def _loss(name, rows, K, vocab, step, dtype="float16"):
    case = {"kind": "loss", "rows": rows, "K": K, "vocab": vocab, "step": step, "dtype": dtype}
    return dict(case, name=name) if name else case


def _distill(name, rows, K, vocab, top, temperature, step, dtype="float16"):
    case = {"kind": "distill", "rows": rows, "K": K, "vocab": vocab, "top": top, "temperature": temperature, "step": step, "dtype": dtype}
    return dict(case, name=name) if name else case


def listed():
    return [
        # four answers to one short prompt, the heads of the framework's default configuration: the smallest call, where launches and latency count
        _share("share_4_over_512", 1, 4, 1, 512, 100, 32, 32, 128, 16),
        # a decode step of 64 samples of one long prompt, shared key heads
        _share("share_64_over_8192", 1, 64, 1, 8192, 500, 32, 8, 128, 64),
        # five prompts with thirteen drafts of three tokens each: heads of 64, seven queries a key head, a prefix that ends inside a page
        _share("share_5x13_over_5000", 5, 13, 3, 5000, 700, 14, 2, 64, 32),
        # many samples of a long document in pages of 8 bits: the largest pass over a prefix
        _share("share_e4m3_256_over_16384", 1, 256, 1, 16384, 300, 32, 8, 128, 128, pages="e4m3"),
        # one candidate's last token rated: latency
        _loss("rate_1", 1, 2048, 32000, False),
        # sixteen tokens rated through the head of the default configuration
        _loss("rate_16", 16, 4096, 32000, False),
        # odd sizes, fp32 rows: a training step
        _loss("step_fp32_333x1000x7777", 333, 1000, 7777, True, "float32"),
        # a training step of a small model
        _loss("step_1024x1024", 1024, 1024, 32000, True),
        # a training step of the default configuration's head: the largest product
        _loss("step_4096x4096", 4096, 4096, 32000, True),
        # a short answer compared with a teacher's eight likeliest tokens
        _distill("distill_40_of_8", 40, 2048, 32000, 8, 1.0, True),
        # odd sizes, a soft teacher of fifty tokens
        _distill("distill_fp32_777x1111x5003", 777, 1111, 5003, 50, 2.0, True, "float32"),
        # a batch of a distillation run
        _distill("distill_2048_of_32", 2048, 4096, 32000, 32, 2.0, True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["share", "loss", "distill"])
    if kind == "share":
        kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
        heads = min(kv * rng.choice([1, 1, 2, 4, 4, 5, 7, 8]), 64) // kv * kv
        head_dim, page, pages = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256]), rng.choice(["float16", "e4m3"])
        while True:
            groups, seqs, new = rng.choice([1, 1, 2, rng.randint(3, 8)]), _log_int(rng, 2, 256), rng.choice([1, 1, 1, rng.randint(2, 8)])
            prefix, past = _log_int(rng, 1, 65536), _log_int(rng, 1, 2048)
            scores = groups * seqs * new * heads * (prefix + past + new) * max(1, head_dim // 128)
            if scores <= MOST_SCORES and groups * (prefix + seqs * (past + new)) * kv * head_dim <= 400000 * 8 * 128:
                return _share(None, groups, seqs, new, prefix, past, heads, kv, head_dim, page, pages)
    dtype, step = rng.choice(["float16", "float16", "float32"]), rng.random() < 0.7
    while True:
        rows, K, vocab = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 1000, 130000)
        if rng.random() < 0.6:
            K, vocab = K // 64 * 64, vocab // 64 * 64
        if rows * K * vocab * (3 if dtype == "float32" else 1) <= MOST_COST and K * vocab <= MOST_WEIGHTS and rows * vocab <= MOST_WEIGHTS:
            break
    if kind == "loss":
        return _loss(None, rows, K, vocab, step, dtype)
    return _distill(None, rows, K, vocab, _log_int(rng, 1, 128), rng.choice([1.0, 1.0, 2.0, 4.0]), step, dtype)


# ---------------------------------------------------------------- what a program has in hand
_heads = {}


def _head(K, vocab):
    """A random ternary head [K, vocab], one for each size as a program keeps its model: dense (8 bits, for the plain form), the weights' count in each
    column, and, for the framework, packed."""
    if (K, vocab) not in _heads:
        gen = torch.Generator(device="cuda").manual_seed(K * 131 + vocab)
        r = torch.rand((K, vocab), generator=gen, device="cuda")
        dense = (r >= (SPARSITY + 1) / 2).to(torch.int8) - ((r >= SPARSITY) & (r < (SPARSITY + 1) / 2)).to(torch.int8)
        _heads[K, vocab] = {"dense": dense, "count": dense.abs().sum(0, dtype=torch.int32)}
    held = _heads[K, vocab]
    if own and "weight" not in held:
        from ternaryllm_amd import ops, packing
        held["weight"] = ops.DeviceWeight(packing.PackedWeight.from_dense(held["dense"].cpu().int()), "cuda")
        held["back"] = ops.BackWeight(held["weight"])
    return held


def _lengths(case):
    """(group, length beyond the prefix, new tokens among it) of every sequence: the first of the full sizes, others of any up to them."""
    rng = random.Random(case["groups"] * 7919 + case["seqs"] * 31 + case["past"])
    rows = []
    for g in range(case["groups"]):
        for i in range(case["seqs"]):
            past, new = (case["past"], case["new"]) if i == 0 else (_log_int(rng, 1, case["past"]), rng.randint(1, case["new"]))
            rows.append((g, past + new, new))
    return rows


def _prepare_share(case, gen, seed):
    heads, kv, hd, page, prefix = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["prefix"]
    rows = _lengths(case)
    whole, rest = prefix // page, prefix % page                     # the prefix's pages, and its tokens in a page that each sequence has a copy of
    per_seq = [-(-(rest + length) // page) for _, length, _ in rows]
    count = case["groups"] * whole + sum(per_seq)
    total = count + 3                                               # a pool with pages that are nobody's, used in any order
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed))[:count].tolist()
    table = torch.zeros((len(rows), whole + max(per_seq)), dtype=torch.int32)
    shape = (total, kv, page, hd)
    if case["pages"] == "float16":
        pages = [torch.randn(shape, generator=gen, device="cuda").half() for _ in range(2)] + [None, None]
    else:
        pages = [(100.0 * torch.randn(shape, generator=gen, device="cuda")).clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
        pages += [torch.randint(119, 122, shape[:3], generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
    for i, ((g, _, _), n) in enumerate(zip(rows, per_seq)):
        table[i, :whole] = torch.tensor(order[g * whole:(g + 1) * whole], dtype=torch.int32)
        at = case["groups"] * whole + sum(per_seq[:i])
        table[i, whole:whole + n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        if rest and i % case["seqs"]:
            first = int(table[i - i % case["seqs"], whole])
            for t in pages:
                if t is not None:
                    t.view(torch.uint8 if t.element_size() == 1 else t.dtype)[int(table[i, whole]), :, :rest] = \
                        t.view(torch.uint8 if t.element_size() == 1 else t.dtype)[first, :, :rest]
    new = torch.tensor([n for _, _, n in rows])
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)])
    state = {"case": case, "pages": tuple(pages), "table": table.cuda(), "starts": starts.int().cuda(), "tokens": int(new.sum()), "most_new": int(new.max()),
             "lengths": torch.tensor([prefix + length for _, length, _ in rows], dtype=torch.int32).cuda()}
    state["groups"] = torch.arange(0, len(rows) + 1, case["seqs"], dtype=torch.int32).cuda()
    state["shared"] = torch.full((len(rows),), prefix, dtype=torch.int32, device="cuda")
    # one product's rows: queries, keys and values side by side
    state["q"] = torch.randn((state["tokens"], heads + 2 * kv, hd), generator=gen, device="cuda").half()[:, :heads]
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "share":
        return _prepare_share(case, gen, seed)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    head = _head(case["K"], vocab)
    state = {"case": case, "head": head}
    # rows as they come out of a norm; a column's scale makes up for how many weights it has
    state["x"] = (SPREAD * torch.randn((rows, case["K"]), generator=gen, device="cuda")).to(dtype).requires_grad_(case["step"])
    jitter = 1.0 + 0.1 * torch.randn(vocab, generator=gen, device="cuda")
    state["scale"] = (jitter * torch.rsqrt(head["count"].clamp(min=1).float())).to(dtype).requires_grad_(case["step"])
    state["grad"] = 0.5 + torch.rand(rows, generator=gen, device="cuda")       # of the rows' losses: what each of them weighs
    padding = (torch.rand(rows, generator=gen, device="cuda") < 0.1) & (torch.arange(rows, device="cuda") > 0)
    if case["kind"] == "loss":
        state["targets"] = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").masked_fill_(padding, IGNORED)
        return state
    # the likeliest first: distinct tokens (a stride that divides nothing spreads them), rows of padding have no teacher
    top = case["top"]
    first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
    state["ids"] = (first + torch.arange(top, device="cuda") * (vocab // (top + 1))) % vocab
    teacher = (SPREAD * torch.randn((rows, top), generator=gen, device="cuda")).sort(dim=1, descending=True).values
    state["teacher"] = teacher.masked_fill_(padding[:, None], -math.inf)
    return state


# ---------------------------------------------------------------- the plain forms
def _value(codes, exponents):
    return codes.float() if exponents is None else codes.float() * torch.exp2(exponents.float() - 127)[..., None]


def _plain_share(state):
    case = state["case"]
    heads, kv, hd, page, prefix = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["prefix"]
    k, v, ke, ve = state["pages"]
    group, n = heads // kv, state["most_new"]
    starts, lengths, table = state["starts"].long(), state["lengths"].long(), state["table"].long()
    whole, rest = prefix // page, prefix % page
    columns = table.shape[1] - whole
    out = torch.empty((state["tokens"], heads * hd), dtype=torch.float16, device="cuda")
    for g in range(case["groups"]):
        first, last = g * case["seqs"], (g + 1) * case["seqs"]
        B = case["seqs"]
        token = torch.arange(n, device="cuda")
        new = starts[first + 1:last + 1] - starts[first:last]
        row = (starts[first:last, None] + token).clamp(max=state["tokens"] - 1)                                     # [B, n]
        q = state["q"][row].float().view(B, n, kv, group, hd).permute(2, 0, 3, 1, 4).mul(1 / math.sqrt(hd))        # [kv, B, group, n, hd]
        # the prefix, once for the group
        ids = table[first, :whole + (rest > 0)]
        pk, pv = (_value(t[ids], None if e is None else e[ids]).transpose(0, 1).reshape(kv, -1, hd)[:, :prefix] for t, e in ((k, ke), (v, ve)))
        s1 = q.reshape(kv, B * group * n, hd) @ pk.transpose(1, 2).contiguous()
        m1 = s1.amax(-1, keepdim=True)
        s1.sub_(m1).exp_()
        l1, o1 = s1.sum(-1, keepdim=True), s1 @ pv
        # what each sequence has of its own
        ids = table[first:last, whole:]
        ok, ov = (_value(t[ids], None if e is None else e[ids]).permute(2, 0, 1, 3, 4).reshape(kv, B, columns * page, hd)
                  for t, e in ((k, ke), (v, ve)))
        key = whole * page + torch.arange(columns * page, device="cuda")
        seen = lengths[first:last, None] - new[:, None] + token                                                     # the last key a token sees
        hidden = (key < prefix) | (key > seen[..., None]) | (key >= lengths[first:last, None, None])               # [B, n, keys]
        ov = ov.masked_fill((key >= lengths[first:last, None])[None, :, :, None], 0.0)
        s2 = (q.reshape(kv, B, group * n, hd) @ ok.transpose(2, 3).contiguous()).view(kv, B, group, n, -1)
        s2.masked_fill_(hidden[None, :, None], -math.inf)
        m2 = s2.amax(-1, keepdim=True)
        s2.sub_(m2).exp_()
        l2, o2 = s2.sum(-1, keepdim=True), (s2.view(kv, B, group * n, -1) @ ov).view(kv, B, group, n, hd)
        m1, l1, o1 = (t.view(kv, B, group, n, -1) for t in (m1, l1, o1))
        m = torch.maximum(m1, m2)
        w1, w2 = (m1 - m).exp(), (m2 - m).exp()
        y = ((o1 * w1 + o2 * w2) / (l1 * w1 + l2 * w2)).permute(1, 3, 0, 2, 4).reshape(B, n, heads * hd)
        there = token < new[:, None]
        out[row[there]] = y[there].half()
    return out


def _plain_loss(state):
    case = state["case"]
    x, w, s = state["x"].float(), state["head"]["dense"].float(), state["scale"].float()
    heat = case.get("temperature", 1.0)
    raw = x @ w
    z = raw * s / heat
    most = z.amax(-1, keepdim=True)
    lse = (z - most).exp_().sum(-1, keepdim=True).log() + most
    if case["kind"] == "loss":
        valid = state["targets"] != IGNORED
        ids, share = state["targets"].clamp(min=0)[:, None], valid.float()[:, None]
        loss = torch.where(valid, (lse - z.gather(1, ids))[:, 0], 0.0)
    else:
        t = state["teacher"] / heat
        top = t.amax(-1, keepdim=True)
        valid = top[:, 0] > -math.inf
        e = (t - top.masked_fill(~valid[:, None], 0.0)).exp()
        ids, share = state["ids"], e / e.sum(-1, keepdim=True).masked_fill(~valid[:, None], 1.0)
        known = torch.where(share > 0, share * share.log(), 0.0).sum(-1)
        loss = torch.where(valid, heat * heat * (known - (share * z.gather(1, ids)).sum(-1) + lse[:, 0]), 0.0)
    if not case["step"]:
        return loss
    dz = z.sub_(lse).exp_().scatter_add_(1, ids, -share).mul_((state["grad"] * heat * valid)[:, None])
    dx = (dz * s) @ w.t().contiguous()
    return loss, dx.to(state["x"].dtype), (dz * raw).sum(0).to(state["scale"].dtype)


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_share(state) if case["kind"] == "share" else _plain_loss(state)
    from ternaryllm_amd import ops
    if case["kind"] == "share":
        with torch.no_grad():
            batch = ops.PageBatch(state["table"], state["starts"], state["lengths"], state["most_new"])
            return ops.paged_attention(state["q"], ops.Pages(*state["pages"]), batch, prefix=ops.PagePrefix(state["groups"], state["shared"]))
    head, back = state["head"], state["head"]["back"] if case["step"] else None
    if case["kind"] == "loss":
        loss = ops.cross_entropy(head["weight"], state["x"], state["targets"], state["scale"], ignore=IGNORED, back=back)
    else:
        loss = ops.distillation(head["weight"], state["x"], state["ids"], state["teacher"], state["scale"], temperature=case["temperature"], back=back)
    if not case["step"]:
        return loss
    dx, ds = torch.autograd.grad(loss, (state["x"], state["scale"]), state["grad"])
    return loss.detach(), dx, ds


def work(case):
    """Bytes: every input and every output once, of the pages a prefix once for its group, of a head two bits a weight.  Operations: of an attention the
    two products over the keys that each row sees; of a loss the product of the logits, and of a step the two gradients' as well."""
    if case["kind"] == "share":
        heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        rows = _lengths(case)
        row = 2 * kv * (hd * 2 if case["pages"] == "float16" else hd + 1)
        tokens, own_keys = sum(new for _, _, new in rows), sum(length for _, length, _ in rows)
        table = sum(-(-(case["prefix"] + length) // case["page"]) for _, length, _ in rows) * 4 + len(rows) * 12
        pairs = sum(new * (case["prefix"] + length) - new * (new - 1) // 2 for _, length, new in rows)
        return {"bytes": (case["groups"] * case["prefix"] + own_keys) * row + 2 * tokens * heads * hd * 2 + table, "flops": 4 * pairs * heads * hd}
    rows, K, vocab, es = case["rows"], case["K"], case["vocab"], 2 if case["dtype"] == "float16" else 4
    bytes_ = rows * K * es + K * vocab // 4 + vocab * es + rows * 4 + (rows * 8 if case["kind"] == "loss" else rows * case["top"] * 12)
    if case["step"]:
        bytes_ += rows * K * es + vocab * es + rows * 4
    return {"bytes": bytes_, "flops": 2 * rows * K * vocab * (2 if case["step"] else 1)}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_share(case, state):
    heads, kv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    k, v, ke, ve = state["pages"]
    table, first, out = state["table"].tolist(), 0, []
    for i, (_, length, new) in enumerate(_lengths(case)):
        length += case["prefix"]
        ids = torch.tensor(table[i][:-(-length // page)], device="cuda")

        def rows(codes, exponents):
            x = codes[ids].double()
            if exponents is not None:
                x = x * torch.pow(2.0, exponents[ids].double() - 127)[..., None]
            return x.permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, :length]

        keys, values = rows(k, ke), rows(v, ve)
        q = state["q"][first:first + new].double().view(new, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)
        s = (q @ keys.transpose(1, 2).contiguous()).view(kv, heads // kv, new, length) / math.sqrt(hd)
        seen = torch.arange(length, device="cuda") <= torch.arange(length - new, length, device="cuda")[:, None]
        p = torch.softmax(torch.where(seen, s, -math.inf), dim=-1)
        y = (p.view(kv, -1, length) @ values).view(kv, heads // kv, new, hd)
        out.append(y.permute(2, 0, 1, 3).reshape(new, heads * hd))
        first += new
    return torch.cat(out)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "share":
            return _exact_share(case, state)
        w, s = state["head"]["dense"].double(), state["scale"].double()
        back = w.t().contiguous()
        heat = case.get("temperature", 1.0)
        losses, dxs, ds = [], [], torch.zeros_like(s)
        for m in range(0, case["rows"], 512):                       # some rows at a time
            x = state["x"][m:m + 512].double()
            raw = x @ w
            logs = torch.log_softmax(raw * s / heat, dim=-1)
            target = torch.zeros_like(raw)                          # the distribution that is wanted
            if case["kind"] == "loss":
                t = state["targets"][m:m + 512]
                for i in range(t.numel()):
                    if int(t[i]) != IGNORED:
                        target[i, t[i]] = 1.0
            else:
                soft = torch.softmax(state["teacher"][m:m + 512].double() / heat, dim=-1).nan_to_num(0.0)
                target.scatter_add_(1, state["ids"][m:m + 512], soft)
            counts = target.sum(-1) > 0
            gap = torch.special.xlogy(target, target) - target * logs
            losses.append(heat * heat * gap.sum(-1))
            if case["step"]:
                dz = (logs.exp() * counts[:, None] - target) * (heat * state["grad"][m:m + 512].double())[:, None]
                dxs.append((dz * s) @ back)
                ds += (dz * raw).sum(0)
    loss = torch.cat(losses)
    return (loss, torch.cat(dxs), ds) if case["step"] else loss
