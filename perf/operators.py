"""Cases of the batched serving operators: a paged key/value cache, the attention
that reads it (with and without a prefix that the whole batch shares) and sampling.

They are what one decode step of many sequences runs between its matrix products,
and what the prompts of such a batch run before it. Head counts and widths are
those of this repository's two topologies (7B: 32 heads of 128, 1B: 15 heads of
128) and of grouped-query layouts; a vocabulary of 512 is this repository's own.

    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU
    run(state)           one pass: plain torch, or with `own` the library's operators
    work(case)           bytes and operations the pass cannot do without
    exact(case, seed)    the same outputs in 64 bits
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BASES = 512              # vocabulary of this repository's models
SCRATCH = 256 << 20      # the workspace that a serving loop keeps
THETA = 10000.0


def listed():
    return [
        # One base of one generated sequence, 7B: the append of its decode step.
        dict(name="append_one", op="append", sequences=1, tokens=1, context=4001, heads=32,
             kv_heads=32, head_dim=128, page=64, rotary=128, interleaved=False, scale=128.0,
             source="f32", cache="bf16"),
        # A decode step of a large batch with grouped heads, far positions, a
        # quarter of each head rotated in neighbouring pairs.
        dict(name="append_batch", op="append", sequences=192, tokens=1, context=130000, heads=32,
             kv_heads=8, head_dim=128, page=16, rotary=32, interleaved=True, scale=1.0,
             source="bf16", cache="bf16"),
        # Prompts of ragged lengths entering the cache together, 7B heads.
        dict(name="append_prompts", op="append", sequences=8, tokens=2048, context=3000, heads=32,
             kv_heads=32, head_dim=128, page=64, rotary=128, interleaved=False, scale=16.0,
             source="f32", cache="bf16"),
        # The attention of one sequence's decode step after a prompt of about a
        # thousand bases, 7B.
        dict(name="decode_one", op="attention", sequences=1, tokens=1, context=1040, shared=0,
             heads=32, kv_heads=32, head_dim=128, page=64, cache="bf16"),
        # A decode step of sequences of very different lengths, grouped heads.
        dict(name="decode_batch", op="attention", sequences=64, tokens=1, context=8190, shared=0,
             heads=32, kv_heads=8, head_dim=128, page=16, cache="bf16"),
        # Prompts entering together, some with a cached beginning, 1B heads.
        dict(name="prompts", op="attention", sequences=4, tokens=1531, context=5003, shared=0,
             heads=15, kv_heads=15, head_dim=128, page=32, cache="f16"),
        # A chunk of one long prompt on what is cached of it, grouped heads.
        dict(name="prompt_chunk", op="attention", sequences=1, tokens=4096, context=16384,
             shared=0, heads=32, kv_heads=8, head_dim=128, page=64, cache="bf16"),
        # Continuations sampled from one long region, a decode step, 7B heads.
        dict(name="continuations", op="attention", sequences=24, tokens=1, context=300,
             shared=16384, heads=32, kv_heads=32, head_dim=128, page=64, cache="bf16"),
        # Variants of the bases behind one region, scored together.
        dict(name="variants", op="attention", sequences=48, tokens=33, context=33, shared=8192,
             heads=32, kv_heads=8, head_dim=128, page=16, cache="bf16"),
        # One base of one generated sequence, sampled.
        dict(name="sample_base", op="sample", rows=1, vocab=BASES, logits="f32"),
        # One base for each of many continuations.
        dict(name="sample_bases", op="sample", rows=2048, vocab=BASES, logits="f32"),
        # A decode step's tokens over a large vocabulary.
        dict(name="sample_batch", op="sample", rows=128, vocab=131072, logits="bf16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "shared", "shared", "sample"])
    if op == "sample":
        rows = _log_int(rng, 1, 2048)
        vocab = rng.choice([BASES, _log_int(rng, 200, 131072), _log_int(rng, 20000, 131072)])
        return dict(op="sample", rows=min(rows, 128 * 131072 // vocab), vocab=vocab,
                    logits=rng.choice(["f32", "bf16", "f16"]))
    heads, kv_heads, head_dim = rng.choice([(32, 32, 128), (15, 15, 128), (32, 8, 128),
                                            (28, 4, 128), (16, 2, 64), (16, 16, 64)])
    case = dict(op=op, sequences=_log_int(rng, 1, 192), tokens=1, context=0, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64, 128]),
                cache=rng.choice(["bf16", "bf16", "f16"]))
    if op == "append":
        if rng.random() < 0.5:
            case["tokens"] = _log_int(rng, 2, 8192 // case["sequences"])
        case["context"] = case["tokens"] + _log_int(rng, 1, 130000) - 1
        case["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
        case["interleaved"] = rng.choice([True, False])
        case["scale"] = rng.choice([1.0, 16.0, 128.0])
        case["source"] = rng.choice(["f32", "f32", case["cache"]])
        return case
    case.update(op="attention", shared=0)
    keys = 64 * 8192 // case["sequences"]  # cached keys of a sequence, at most
    if op == "shared":
        case["shared"] = case["page"] * _log_int(rng, 4, 16384 // case["page"])
        case["tokens"] = rng.choice([1, 1, _log_int(rng, 1, max(1, 1536 // case["sequences"]))])
        case["context"] = case["tokens"] + _log_int(rng, 1, min(512, keys)) - 1
        return case
    if rng.random() < 0.5:
        case["context"] = _log_int(rng, 16, min(keys, 16384))
        return case
    case["sequences"] = _log_int(rng, 1, 16)
    case["tokens"] = _log_int(rng, 2, 4096 // case["sequences"])
    case["context"] = case["tokens"] + rng.choice([0, _log_int(rng, 1, 8192)])
    return case


# ------------------------------------------------------------------ sizes
def _ragged(case):
    """New tokens and cached keys (behind the shared prefix) of each sequence: the
    first has the most, the others are spread over the logarithm."""
    rng = random.Random("%d %d %d" % (case["sequences"], case["tokens"], case["context"]))
    counts, own_keys = [case["tokens"]], [case["context"]]
    for _ in range(1, case["sequences"]):
        n = _log_int(rng, max(1, case["tokens"] // 16), case["tokens"])
        counts.append(n)
        own_keys.append(_log_int(rng, max(n, case["context"] // 16), case["context"]))
    return counts, own_keys


def _pages(case):
    return [-(-n // case["page"]) for n in _ragged(case)[1]]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    return generator


def _normal(generator, *shape, std=1.0):
    return torch.randn(*shape, generator=generator, device=DEVICE) * std


def _table(case, seed, shared_pages, lengths):
    """A page table as an allocator leaves it: a sequence's pages lie anywhere in the
    pool, entries behind its last key hold -1. An append needs only the pages that it
    writes to, so the pool of an append case holds those of its last tokens alone."""
    counts, own_keys = _ragged(case)
    page, first = case["page"], []
    for n, keys in zip(counts, own_keys):
        first.append((keys - n) // page if case["op"] == "append" else 0)
    pages = [-(-keys // page) - f for keys, f in zip(own_keys, first)]
    total = shared_pages + sum(pages)
    order = list(range(total))
    random.Random(seed).shuffle(order)
    shared, rest = order[:shared_pages], order[shared_pages:]
    width = shared_pages + max(f + n for f, n in zip(first, pages))
    rows, at = [], 0
    for f, n in zip(first, pages):
        row = shared + [-1] * f + rest[at:at + n]
        rows.append(row + [-1] * (width - len(row)))
        at += n
    return (torch.tensor(rows, dtype=torch.int32, device=DEVICE),
            torch.tensor(shared, dtype=torch.int32, device=DEVICE), total)


def _batch(case, seed):
    counts, own_keys = _ragged(case)
    shared = case.get("shared", 0)
    start = [0]
    for n in counts:
        start.append(start[-1] + n)
    lengths = [shared + n for n in own_keys]
    table, shared_table, total = _table(case, seed, shared // case["page"], lengths)
    return dict(start=torch.tensor(start, dtype=torch.int32, device=DEVICE),
                lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
                table=table, shared_table=shared_table, rows=start[-1], pages=total,
                most=max(counts), longest=max(lengths))


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(g, rows, vocab, std=2.5).to(TYPES[case["logits"]])
        pick = torch.randint(0, 4, (rows,), generator=g, device=DEVICE)
        spread = torch.rand(rows, generator=g, device=DEVICE)
        most = max(4, min(vocab, 64))
        top_k = torch.where(pick % 2 == 0, (2 + spread * (most - 2)).to(torch.int32), 0)
        return dict(logits=logits, top_k=top_k.to(torch.int32),
                    temperature=0.5 + torch.rand(rows, generator=g, device=DEVICE),
                    top_p=torch.where(pick >= 1, 0.8 + 0.19 * spread, 1.0),
                    min_p=torch.where(pick == 3, 0.02 * spread, 0.0),
                    uniform=torch.rand(rows, generator=g, device=DEVICE))
    s = _batch(case, seed)
    heads, kv, dim, kind = case["heads"], case["kv_heads"], case["head_dim"], TYPES[case["cache"]]
    pool = (s["pages"], kv, case["page"], dim)
    if case["op"] == "append":
        s["projected"] = _normal(g, s["rows"], (heads + 2 * kv) * dim).to(TYPES[case["source"]])
        s["inv_freq"] = THETA ** (-torch.arange(0, case["rotary"], 2, device=DEVICE,
                                                dtype=torch.float64) / case["rotary"])
        s["inv_freq"] = s["inv_freq"].float()
        s["keys"], s["values"] = (torch.zeros(pool, dtype=kind, device=DEVICE) for _ in range(2))
    else:
        s["query"] = _normal(g, s["rows"], heads, dim, std=1.5).to(kind)
        s["keys"], s["values"] = (torch.randn(pool, generator=g, device=DEVICE, dtype=kind)
                                  for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    heads, dim = case.get("heads"), case.get("head_dim")
    if case["op"] == "sample":
        s["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device=DEVICE)
        s["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device=DEVICE)
    elif case["op"] == "append":
        s["query"] = torch.empty(s["rows"], heads, dim, dtype=TYPES[case["cache"]], device=DEVICE)
    else:
        s["out"] = torch.empty_like(s["query"])
        s["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device=DEVICE)
    return s


# ------------------------------------------------------------ plain forms
def _positions(s):
    """Sequence and position of every row: the last rows of a sequence's length."""
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["start"][1:].long(), row, right=True)
    return seq, s["lengths"].long()[seq] - s["start"].long()[seq + 1] + row


def _rotate(x, angle, interleaved):
    """The first 2 * pairs elements of each head [rows, heads, dim] rotated."""
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    pairs = angle.shape[1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    case = s["case"]
    heads, kv, kind = case["heads"], case["kv_heads"], TYPES[case["cache"]]
    x = s["projected"].float().view(s["rows"], heads + 2 * kv, case["head_dim"])
    seq, pos = _positions(s)
    angle = (pos.double() / case["scale"])[:, None] * s["inv_freq"].double()
    turned = _rotate(x[:, :heads + kv], angle, case["interleaved"]).to(kind)
    page, slot = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["keys"][page, :, slot] = turned[:, heads:]
    s["values"][page, :, slot] = x[:, heads + kv:].to(kind)
    return [turned[:, :heads], s["keys"], s["values"]]


def _own_keys(s, pool, shared_pages):
    """Cached rows behind the shared prefix [sequences, kv_heads, keys, dim], F32."""
    table = s["table"][:, shared_pages:].long().clamp_min(0)
    x = pool[table].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4]).float()


def _plain_attention(s):
    case, q = s["case"], s["query"]
    kv, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    group, sequences, most = case["heads"] // kv, case["sequences"], s["most"]
    shared_pages = case["shared"] // page
    seq, pos = _positions(s)
    slot = torch.arange(s["rows"], device=DEVICE) - s["start"].long()[seq]
    # The rows of a sequence side by side: [sequences, kv_heads, most * group, dim].
    rows = torch.zeros(sequences, most, case["heads"], dim, device=DEVICE)
    rows[seq, slot] = q.float() * dim ** -0.5
    seen = torch.full((sequences, most), -1, dtype=torch.long, device=DEVICE)
    seen[seq, slot] = pos
    rows = rows.view(sequences, most, kv, group, dim).transpose(1, 2)
    rows = rows.reshape(sequences, kv, most * group, dim)
    keys, values = (_own_keys(s, s[name], shared_pages) for name in ("keys", "values"))
    score = torch.matmul(rows, keys.transpose(2, 3).contiguous())
    at = case["shared"] + torch.arange(keys.shape[2], device=DEVICE)
    hidden = (at > seen[:, :, None]).repeat_interleave(group, 1)[:, None]
    score.masked_fill_(hidden, -math.inf)
    peak = score.amax(3, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    if shared_pages:
        # The prefix's keys once for the rows of all sequences.
        every = rows.transpose(0, 1).reshape(kv, -1, dim)
        prefix = [s[name][s["shared_table"].long()].transpose(0, 1).reshape(kv, -1, dim).float()
                  for name in ("keys", "values")]
        first = torch.matmul(every, prefix[0].transpose(1, 2).contiguous())
        apart = first.amax(2).view(kv, sequences, -1).transpose(0, 1)[..., None]
        peak = torch.maximum(peak, apart)
        first = (first - peak.transpose(0, 1).reshape(kv, -1, 1)).exp_()
    score = score.sub_(peak).exp_()
    total, out = score.sum(3, keepdim=True), torch.matmul(score, values)
    if shared_pages:
        total += first.sum(2).view(kv, sequences, -1).transpose(0, 1)[..., None]
        out += torch.matmul(first, prefix[1]).view(kv, sequences, -1, dim).transpose(0, 1)
    out = out / total
    out = out.view(sequences, kv, most, group, dim).transpose(1, 2)
    return out.reshape(sequences, most, case["heads"], dim)[seq, slot].to(q.dtype)


def _plain_sample(s):
    logits, order = s["logits"].float().sort(dim=1, descending=True, stable=True)
    weight = logits.double() / s["temperature"].double()[:, None]
    weight = (weight - weight[:, :1]).exp()
    rank = torch.arange(logits.shape[1], device=DEVICE)
    limit = s["top_k"][:, None]
    weight = torch.where((limit > 0) & (rank >= limit), 0.0, weight)
    before = weight.cumsum(1) - weight
    total = weight.sum(1, keepdim=True)
    top_p = s["top_p"].double()[:, None]
    keep = ((top_p >= 1) | (before < top_p * total)) & (weight >= s["min_p"].double()[:, None])
    weight = weight * keep
    ahead = weight.cumsum(1)
    # Weights behind the last one kept are zero: that one is the last index to win.
    drawn = (ahead <= s["uniform"].double()[:, None] * ahead[:, -1:]).sum(1, keepdim=True)
    last = (weight > 0).sum(1, keepdim=True) - 1
    return order.gather(1, torch.minimum(drawn, last))[:, 0].to(torch.int32)


# -------------------------------------------------------- the operators
def _library():
    path = os.path.join(os.getcwd(), "evo.cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from evo_hip import native
    return native


def _dtype(native, tensor):
    return {torch.float32: native.DTYPE_F32, torch.bfloat16: native.DTYPE_BF16,
            torch.float16: native.DTYPE_F16}[tensor.dtype]


def _cache(native, s):
    case, keys = s["case"], s["keys"]
    return native.PagedCache(dtype=_dtype(native, keys), key_pages=keys.data_ptr(),
                             value_pages=s["values"].data_ptr(), pages=s["pages"],
                             page_size=case["page"], kv_heads=case["kv_heads"],
                             head_dim=case["head_dim"])


def _sequences(native, s):
    case = s["case"]
    shared = case.get("shared", 0)
    return native.PagedBatch(sequences=case["sequences"], tokens=s["rows"], max_tokens=s["most"],
                             max_length=s["longest"], token_start=s["start"].data_ptr(),
                             lengths=s["lengths"].data_ptr(), page_table=s["table"].data_ptr(),
                             table_stride=s["table"].stride(0), shared_length=shared,
                             shared_table=s["shared_table"].data_ptr() if shared else None)


def _own_append(s):
    native, case = _library(), s["case"]
    native.call("evo_hip_paged_append", ctypes.byref(_cache(native, s)),
                ctypes.byref(_sequences(native, s)), _dtype(native, s["projected"]),
                s["projected"].data_ptr(), s["projected"].stride(0), case["heads"], 0,
                s["inv_freq"].data_ptr(), case["rotary"], int(case["interleaved"]), case["scale"],
                s["query"].data_ptr(), s["query"].stride(0),
                torch.cuda.current_stream().cuda_stream)
    return [s["query"], s["keys"], s["values"]]


def _own_attention(s):
    native, case = _library(), s["case"]
    native.call("evo_hip_paged_attention", ctypes.byref(_cache(native, s)),
                ctypes.byref(_sequences(native, s)), s["query"].data_ptr(), s["query"].stride(0),
                case["heads"], case["head_dim"] ** -0.5, s["out"].data_ptr(), s["out"].stride(0),
                s["scratch"].data_ptr(), SCRATCH, torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_sample(s):
    native, case, logits = _library(), s["case"], s["logits"]
    native.call("evo_hip_sample", _dtype(native, logits), logits.data_ptr(), case["rows"],
                case["vocab"], logits.stride(0), s["temperature"].data_ptr(),
                s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(),
                s["uniform"].data_ptr(), s["tokens"].data_ptr(), s["scratch"].data_ptr(), SCRATCH,
                torch.cuda.current_stream().cuda_stream)
    return s["tokens"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "sample": _own_sample}[op](state)
    return {"append": _plain_append, "attention": _plain_attention,
            "sample": _plain_sample}[op](state)


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "sample":
        size = 4 if case["logits"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 24),
                "flops": 4 * case["rows"] * case["vocab"]}
    counts, own_keys = _ragged(case)
    heads, kv, dim, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(counts)
    if case["op"] == "append":
        size = 4 if case["source"] == "f32" else 2
        return {"bytes": rows * (heads + 2 * kv) * dim * (size + 2),
                "flops": 3 * rows * (heads + kv) * case["rotary"]}
    cached = case["shared"] + sum(own_keys)
    seen = sum(n * (case["shared"] + keys) - n * (n - 1) // 2
               for n, keys in zip(counts, own_keys))
    return {"bytes": 4 * cached * kv * dim + 4 * rows * heads * dim,
            "flops": 4 * seen * heads * dim}


# ------------------------------------------------------------------ exact
def _exact_append(case, s):
    counts, own_keys = _ragged(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["projected"].double()
    query = x[:, :heads * dim].reshape(-1, heads, dim).clone()
    key = x[:, heads * dim:(heads + kv) * dim].reshape(-1, kv, dim).clone()
    value = x[:, (heads + kv) * dim:].reshape(-1, kv, dim)
    pos = torch.cat([torch.arange(keys - n, keys) for n, keys in zip(counts, own_keys)])
    half = case["rotary"] // 2
    for i in range(half):
        low, high = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
        angle = (pos.double() / case["scale"] * float(s["inv_freq"][i])).to(DEVICE)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        for z in (query, key):
            pair = torch.complex(z[:, :, low], z[:, :, high]) * turn
            z[:, :, low], z[:, :, high] = pair.real, pair.imag
    keys, values = s["keys"].double(), s["values"].double()
    table, row = s["table"].cpu(), 0
    for i, (n, length) in enumerate(zip(counts, own_keys)):
        where = torch.arange(length - n, length)
        into = table[i, where // page].long().to(DEVICE), slice(None), (where % page).to(DEVICE)
        keys[into], values[into] = key[row:row + n], value[row:row + n]
        row += n
    return [query, keys, values]


def _exact_attention(case, s):
    counts, own_keys = _ragged(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table, parts, row = s["table"].cpu(), [], 0
    for i, (n, keys) in enumerate(zip(counts, own_keys)):
        length = case["shared"] + keys
        pages = table[i, :-(-length // page)].long().to(DEVICE)
        out = torch.empty(n, heads, dim, dtype=torch.float64, device=DEVICE)
        for h in range(kv):
            k, v = (s[name][pages, h].reshape(-1, dim)[:length].double()
                    for name in ("keys", "values"))
            for g in range(heads // kv):
                head = h * (heads // kv) + g
                score = s["query"][row:row + n, head].double() @ k.t() / math.sqrt(dim)
                if n > 1:
                    hidden = torch.ones(n, length, dtype=torch.bool, device=DEVICE)
                    score[hidden.triu(length - n + 1)] = -math.inf
                out[:, head] = torch.softmax(score, 1) @ v
        parts.append(out)
        row += n
    return torch.cat(parts)


def _exact_sample(case, s):
    found = []
    rows = zip(s["logits"].double(), s["temperature"].tolist(), s["top_k"].tolist(),
               s["top_p"].tolist(), s["min_p"].tolist(), s["uniform"].tolist())
    for logits, temperature, top_k, top_p, min_p, uniform in rows:
        order = torch.sort(logits, descending=True, stable=True).indices
        if top_k:
            order = order[:top_k]
        share = torch.softmax(logits[order] / temperature, 0)
        if top_p < 1:
            order = order[:int((share.cumsum(0) - share < top_p).sum())]
            share = share[:len(order)]
        share = share[share >= min_p * share[0]]
        reached = share.cumsum(0) > uniform * share.sum()
        found.append(order[:len(share)][reached][0])
    return torch.stack(found).to(torch.int32)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return _exact_sample(case, s)
