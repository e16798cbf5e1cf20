"""Cases of three operators of a step of many requests: low-rank adapters beside a
shared projection, the paged append of heads that are normalized first, and what a
row of logits says of given tokens.

Widths are those of this repository's two topologies (7B: width 4096, inner 11264,
32 heads of 128; 1B: width 1920, 15 heads of 128) and of grouped-query layouts; a
vocabulary of 512 is this repository's own.

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
EPS = 1e-6


def listed():
    return [
        # One base of one generated sequence, 7B heads: the append of its decode step.
        dict(name="heads_one", op="heads", sequences=1, tokens=1, context=4001, heads=32,
             kv_heads=32, head_dim=128, page=64, rotary=128, interleaved=False, scale=128.0,
             per_head=False, inside=True, source="f32", cache="bf16"),
        # A decode step of a large batch with grouped heads, far positions, a
        # quarter of each head rotated in neighbouring pairs, scales for each head.
        dict(name="heads_batch", op="heads", sequences=192, tokens=1, context=130000, heads=32,
             kv_heads=8, head_dim=128, page=16, rotary=32, interleaved=True, scale=1.0,
             per_head=True, inside=False, source="bf16", cache="bf16"),
        # Prompts of ragged lengths entering the cache together, 7B heads.
        dict(name="heads_prompts", op="heads", sequences=8, tokens=2048, context=3000, heads=32,
             kv_heads=32, head_dim=128, page=64, rotary=128, interleaved=False, scale=16.0,
             per_head=False, inside=True, source="f32", cache="bf16"),
        # One base of one request, on the attention projection of 7B.
        dict(name="adapters_one", op="adapters", rows=1, width=4096, out=12288, rank=16,
             adapters=8, used=1, runs=False, mixed=False, planes=2),
        # A decode step of a batch whose requests have adapters of their own, some
        # share one and some have none, 7B's attention projection.
        dict(name="adapters_decode", op="adapters", rows=96, width=4096, out=12288, rank=16,
             adapters=64, used=40, runs=False, mixed=False, planes=2),
        # A larger batch on few adapters of high rank, in BF16, 7B's MLP.
        dict(name="adapters_shared", op="adapters", rows=512, width=4096, out=11264, rank=64,
             adapters=6, used=6, runs=False, mixed=False, planes=1),
        # Short prompts of ragged lengths, ranks that differ and are odd, 1B.
        dict(name="adapters_short", op="adapters", rows=301, width=1920, out=5760, rank=24,
             adapters=16, used=9, runs=True, mixed=True, planes=2),
        # Prompts of several requests, 7B's attention projection.
        dict(name="adapters_prompts", op="adapters", rows=4096, width=4096, out=12288, rank=64,
             adapters=8, used=6, runs=True, mixed=False, planes=2),
        # One generated base with its alternatives.
        dict(name="logprobs_base", op="logprobs", rows=1, vocab=BASES, logits="f32", top=4),
        # A sequence scored base by base.
        dict(name="logprobs_record", op="logprobs", rows=8192, vocab=BASES, logits="f32", top=4),
        # The tokens of a few requests over a large vocabulary of odd size.
        dict(name="logprobs_few", op="logprobs", rows=5, vocab=100003, logits="f16", top=20),
        # A prompt scored over a large vocabulary, with alternatives.
        dict(name="logprobs_prompt", op="logprobs", rows=256, vocab=131072, logits="bf16", top=5),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["heads", "adapters", "adapters", "logprobs"])
    if op == "logprobs":
        rows = _log_int(rng, 1, 8192)
        vocab = rng.choice([BASES, _log_int(rng, 200, 131072), _log_int(rng, 20000, 262144)])
        logits = rng.choice(["f32", "bf16", "f16"])
        most = 256 * 131072 // (2 if logits == "f32" else 1)
        return dict(op="logprobs", rows=max(1, min(rows, most // vocab)), vocab=vocab,
                    logits=logits, top=rng.choice([0, 1, 5, 20, _log_int(rng, 1, 64)]))
    if op == "adapters":
        width, out = rng.choice([(4096, 12288), (4096, 4096), (4096, 11264), (11264, 4096),
                                 (1920, 5760), (8 * _log_int(rng, 32, 1024),
                                                _log_int(rng, 300, 12000))])
        rank = 8 * _log_int(rng, 1, 16)
        rows = min(_log_int(rng, 1, 4096), 4096 * 64 // rank)
        adapters = _log_int(rng, 1, 64)
        return dict(op="adapters", rows=rows, width=width, out=out, rank=rank, adapters=adapters,
                    used=_log_int(rng, 1, adapters), runs=rng.random() < 0.5,
                    mixed=rng.random() < 0.4, planes=rng.choice([1, 2]))
    heads, kv_heads, head_dim = rng.choice([(32, 32, 128), (15, 15, 128), (32, 8, 128),
                                            (28, 4, 128), (16, 2, 64), (16, 16, 64)])
    case = dict(op="heads", sequences=_log_int(rng, 1, 192), tokens=1, context=0, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64, 128]),
                cache=rng.choice(["bf16", "bf16", "f16"]), per_head=rng.random() < 0.3,
                inside=rng.random() < 0.5)
    if rng.random() < 0.5:
        case["tokens"] = _log_int(rng, 2, 8192 // case["sequences"])
    case["context"] = case["tokens"] + _log_int(rng, 1, 130000) - 1
    case["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
    case["interleaved"] = rng.choice([True, False])
    case["scale"] = rng.choice([1.0, 16.0, 128.0])
    case["source"] = rng.choice(["f32", "f32", case["cache"]])
    return case


# ------------------------------------------------------------------ sizes
def _ragged(case):
    """New tokens and cached keys of each sequence: the first has the most, the others
    are spread over the logarithm."""
    rng = random.Random("%d %d %d" % (case["sequences"], case["tokens"], case["context"]))
    counts, keys = [case["tokens"]], [case["context"]]
    for _ in range(1, case["sequences"]):
        n = _log_int(rng, max(1, case["tokens"] // 16), case["tokens"])
        counts.append(n)
        keys.append(_log_int(rng, max(n, case["context"] // 16), case["context"]))
    return counts, keys


def _adapter_of_rows(case):
    """The adapter of each row (-1: none), and each adapter's rank. In runs: the rows of
    a request lie side by side; otherwise each row is a request's newest token."""
    rng = random.Random("%d %d %d" % (case["rows"], case["rank"], case["adapters"]))
    used = rng.sample(range(case["adapters"]), case["used"])
    pick = used + [-1] if case["rows"] > 1 else used
    of_rows = []
    if case["runs"]:
        most = max(1, case["rows"] // 4)
        while len(of_rows) < case["rows"]:
            of_rows += [rng.choice(pick)] * _log_int(rng, max(1, most // 16), most)
        of_rows = of_rows[:case["rows"]]
    else:
        of_rows = [rng.choice(pick) for _ in range(case["rows"])]
    ranks = [rng.randint(1, case["rank"]) if case["mixed"] else case["rank"]
             for _ in range(case["adapters"])]
    return of_rows, ranks


# ------------------------------------------------------------------ inputs
def _gen(seed):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    return generator


def _normal(generator, *shape, std=1.0):
    return torch.randn(*shape, generator=generator, device=DEVICE) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _heads_inputs(case, seed, g):
    """A page table as an allocator leaves it: a sequence's pages lie anywhere in the
    pool, which holds those that the append writes to; other entries hold -1."""
    counts, lengths = _ragged(case)
    page = case["page"]
    first = [(keys - n) // page for n, keys in zip(counts, lengths)]
    pages = [-(-keys // page) - f for keys, f in zip(lengths, first)]
    order = list(range(sum(pages)))
    random.Random(seed).shuffle(order)
    width, rows, at = max(f + n for f, n in zip(first, pages)), [], 0
    for f, n in zip(first, pages):
        row = [-1] * f + order[at:at + n]
        rows.append(row + [-1] * (width - len(row)))
        at += n
    start = [0]
    for n in counts:
        start.append(start[-1] + n)
    heads, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    s = dict(start=_ints(start), lengths=_ints(lengths), table=_ints(rows), rows=start[-1],
             pages=len(order), most=max(counts), longest=max(lengths))
    # A head's size varies from token to token and from head to head.
    x = _normal(g, s["rows"], heads + 2 * kv, dim)
    x *= (0.7 * _normal(g, s["rows"], heads + 2 * kv, 1)).exp_()
    s["projected"] = x.view(s["rows"], -1).to(TYPES[case["source"]])
    s["query_scale"], s["key_scale"] = (
        1 + _normal(g, n if case["per_head"] else 1, dim, std=0.2) for n in (heads, kv))
    s["inv_freq"] = (THETA ** (-torch.arange(0, case["rotary"], 2, device=DEVICE,
                                             dtype=torch.float64) / case["rotary"])).float()
    pool = (s["pages"], kv, page, dim)
    s["keys"], s["values"] = (torch.zeros(pool, dtype=TYPES[case["cache"]], device=DEVICE)
                              for _ in range(2))
    return s


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "heads":
        return _heads_inputs(case, seed, g)
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(g, rows, vocab, std=2.5)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
        # Most given tokens are among the likely ones; one row in eight knows its token.
        row = torch.arange(rows, device=DEVICE)
        logits[row, tokens] += 6.0 * torch.rand(rows, generator=g, device=DEVICE)
        logits[row[::8], tokens[::8]] += 24.0
        # One row in five allows a part of the vocabulary only.
        allowed = torch.rand(vocab, generator=g, device=DEVICE) < 0.6
        allowed[:64] = True
        logits[1::5] = logits[1::5].masked_fill(~allowed, -math.inf)
        tokens[1::5] %= 64
        return dict(logits=logits.to(TYPES[case["logits"]]), tokens=tokens.to(torch.int32))
    rows, width, out, rank = (case[n] for n in ("rows", "width", "out", "rank"))
    of_rows, ranks = _adapter_of_rows(case)
    x = _normal(g, rows, width)
    high = x.to(torch.bfloat16)
    s = dict(high=high, low=(x - high.float()).to(torch.bfloat16) if case["planes"] == 2 else None,
             down=_normal(g, case["adapters"], rank, width, std=width ** -0.5).to(torch.bfloat16),
             up=_normal(g, case["adapters"], out, rank, std=rank ** -0.5).to(torch.bfloat16),
             scales=0.25 + torch.rand(case["adapters"], generator=g, device=DEVICE),
             shared=_normal(g, rows, out), of_rows=_ints(of_rows), ranks=_ints(ranks))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "heads":
        s["query"] = torch.empty(s["rows"], case["heads"], case["head_dim"],
                                 dtype=TYPES[case["cache"]], device=DEVICE)
        return s
    s["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device=DEVICE)
    if case["op"] == "adapters":
        of_rows, ranks = _adapter_of_rows(case)
        # The rows of each adapter that is met, and its rank, as a scheduler has them.
        s["groups"] = [(a, ranks[a], torch.tensor([i for i, b in enumerate(of_rows) if a == b],
                                                  device=DEVICE))
                       for a in sorted(set(of_rows)) if a >= 0]
        s["out"] = torch.empty_like(s["shared"])
        return s
    rows, top = case["rows"], case["top"]
    for name in ("logprob", "entropy"):
        s[name] = torch.empty(rows, device=DEVICE)
    s["rank"] = torch.empty(rows, dtype=torch.int32, device=DEVICE)
    s["top_tokens"] = torch.empty(rows, top, dtype=torch.int32, device=DEVICE)
    s["top_logprobs"] = torch.empty(rows, top, device=DEVICE)
    return s


def _found(case):
    """Names of the outputs for a row of logits."""
    return ("logprob", "entropy", "rank") + (("top_tokens", "top_logprobs") if case["top"] else ())


# ------------------------------------------------------------ plain forms
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


def _plain_heads(s):
    case = s["case"]
    heads, kv, kind = case["heads"], case["kv_heads"], TYPES[case["cache"]]
    x = s["projected"].float().view(s["rows"], heads + 2 * kv, case["head_dim"])
    turned = x[:, :heads + kv]
    mean = turned.square().mean(-1, keepdim=True)
    size = (mean + EPS).sqrt() if case["inside"] else mean.sqrt() + EPS
    scale = torch.cat([s["query_scale"].expand(heads, -1), s["key_scale"].expand(kv, -1)])
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["start"][1:].long(), row, right=True)
    pos = s["lengths"].long()[seq] - s["start"].long()[seq + 1] + row
    angle = (pos.double() / case["scale"])[:, None] * s["inv_freq"].double()
    turned = _rotate(turned / size * scale, angle, case["interleaved"]).to(kind)
    page, slot = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["keys"][page, :, slot] = turned[:, heads:]
    s["values"][page, :, slot] = x[:, heads + kv:].to(kind)
    return [turned[:, :heads], s["keys"], s["values"]]


def _plain_adapters(s):
    x = s["high"].float()
    if s["low"] is not None:
        x = x + s["low"].float()
    out = s["shared"].clone()
    for a, rank, rows in s["groups"]:
        inner = x[rows] @ s["down"][a, :rank].float().t()
        out[rows] += (inner @ s["up"][a, :, :rank].float().t()) * s["scales"][a]
    return out


def _plain_logprobs(s):
    logits, order = s["logits"].float().sort(dim=1, descending=True, stable=True)
    away = logits - logits[:, :1]
    # The first token's weight is 1: the others' sum keeps what a sure token leaves.
    weight = away[:, 1:].double().exp()
    others = weight.sum(1, keepdim=True)
    log_total = others.log1p()
    spread = (weight * away[:, 1:].double().clamp_min(-1e4)).sum(1)
    rank = (order == s["tokens"].long()[:, None]).to(torch.int32).argmax(1, keepdim=True)
    top = s["case"]["top"]
    found = {"logprob": (away.gather(1, rank) - log_total)[:, 0].float(),
             "entropy": (log_total - spread[:, None] / (1 + others))[:, 0].float(),
             "rank": rank[:, 0].to(torch.int32)}
    if top:
        found["top_tokens"] = order[:, :top].to(torch.int32)
        found["top_logprobs"] = (away[:, :top] - log_total).float()
    return found


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


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_heads(s):
    native, case, keys = _library(), s["case"], s["keys"]
    cache = native.PagedCache(dtype=_dtype(native, keys), key_pages=keys.data_ptr(),
                              value_pages=s["values"].data_ptr(), pages=s["pages"],
                              page_size=case["page"], kv_heads=case["kv_heads"],
                              head_dim=case["head_dim"])
    batch = native.PagedBatch(sequences=case["sequences"], tokens=s["rows"],
                              max_tokens=s["most"], max_length=s["longest"],
                              token_start=s["start"].data_ptr(), lengths=s["lengths"].data_ptr(),
                              page_table=s["table"].data_ptr(),
                              table_stride=s["table"].stride(0))
    native.call("evo_hip_paged_append_normed", ctypes.byref(cache), ctypes.byref(batch),
                _dtype(native, s["projected"]), s["projected"].data_ptr(),
                s["projected"].stride(0), case["heads"], 0, s["query_scale"].data_ptr(),
                s["key_scale"].data_ptr(), case["head_dim"] if case["per_head"] else 0, EPS,
                int(case["inside"]), s["inv_freq"].data_ptr(), case["rotary"],
                int(case["interleaved"]), case["scale"], s["query"].data_ptr(),
                s["query"].stride(0), _stream())
    return [s["query"], s["keys"], s["values"]]


def _own_adapters(s):
    native, case = _library(), s["case"]
    pool = native.Adapters(adapters=case["adapters"], rank=case["rank"], in_width=case["width"],
                           out_width=case["out"], down=s["down"].data_ptr(),
                           up=s["up"].data_ptr(), scales=s["scales"].data_ptr(),
                           ranks=s["ranks"].data_ptr() if case["mixed"] else None)
    native.call("evo_hip_adapter_linear", ctypes.byref(pool), s["of_rows"].data_ptr(),
                s["high"].data_ptr(), None if s["low"] is None else s["low"].data_ptr(),
                s["high"].stride(0), case["rows"], s["shared"].data_ptr(), s["out"].data_ptr(),
                s["out"].stride(0), s["scratch"].data_ptr(), SCRATCH, _stream())
    return s["out"]


def _own_logprobs(s):
    native, case, logits = _library(), s["case"], s["logits"]
    top = case["top"]
    native.call("evo_hip_token_logprobs", _dtype(native, logits), logits.data_ptr(), case["rows"],
                case["vocab"], logits.stride(0), s["tokens"].data_ptr(), s["logprob"].data_ptr(),
                s["rank"].data_ptr(), s["entropy"].data_ptr(), top,
                s["top_tokens"].data_ptr() if top else None,
                s["top_logprobs"].data_ptr() if top else None, s["scratch"].data_ptr(), SCRATCH,
                _stream())
    return {name: s[name] for name in _found(case)}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"heads": _own_heads, "adapters": _own_adapters,
                "logprobs": _own_logprobs}[op](state)
    return {"heads": _plain_heads, "adapters": _plain_adapters,
            "logprobs": _plain_logprobs}[op](state)


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["logits"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 8 * case["top"]),
                "flops": 6 * case["rows"] * case["vocab"]}
    if case["op"] == "heads":
        rows = sum(_ragged(case)[0])
        heads, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
        size = 4 if case["source"] == "f32" else 2
        return {"bytes": rows * (heads + 2 * kv) * dim * (size + 2),
                "flops": rows * (heads + kv) * (4 * dim + 3 * case["rotary"])}
    of_rows, ranks = _adapter_of_rows(case)
    both = case["width"] + case["out"]
    met = [a for a in of_rows if a >= 0]
    return {"bytes": case["rows"] * 8 * case["out"] + len(met) * 2 * case["planes"] *
            case["width"] + sum(2 * ranks[a] * both for a in set(met)),
            "flops": sum(2 * ranks[a] * both for a in met)}


# ------------------------------------------------------------------ exact
def _exact_heads(case, s):
    counts, lengths = _ragged(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["projected"].double()
    parts = {"query": x[:, :heads * dim].reshape(-1, heads, dim),
             "key": x[:, heads * dim:(heads + kv) * dim].reshape(-1, kv, dim)}
    value = x[:, (heads + kv) * dim:].reshape(-1, kv, dim)
    pos = torch.cat([torch.arange(keys - n, keys) for n, keys in zip(counts, lengths)])
    half = case["rotary"] // 2
    for name in parts:
        z = parts[name]
        size = torch.linalg.vector_norm(z, dim=2, keepdim=True) / math.sqrt(dim)
        size = torch.hypot(size, torch.full_like(size, math.sqrt(EPS))) if case["inside"] \
            else size + EPS
        z = z * s[name + "_scale"].double() / size
        for i in range(half):
            low, high = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
            angle = (pos.double() / case["scale"] * float(s["inv_freq"][i])).to(DEVICE)
            turn = torch.polar(torch.ones_like(angle), angle)[:, None]
            pair = torch.complex(z[:, :, low], z[:, :, high]) * turn
            z[:, :, low], z[:, :, high] = pair.real, pair.imag
        parts[name] = z
    keys, values = s["keys"].double(), s["values"].double()
    table, row = s["table"].cpu(), 0
    for i, (n, length) in enumerate(zip(counts, lengths)):
        where = torch.arange(length - n, length)
        into = table[i, where // page].long().to(DEVICE), slice(None), (where % page).to(DEVICE)
        keys[into], values[into] = parts["key"][row:row + n], value[row:row + n]
        row += n
    return [parts["query"], keys, values]


def _exact_adapters(case, s):
    of_rows, ranks = _adapter_of_rows(case)
    of_rows = torch.tensor(of_rows, device=DEVICE)
    x = s["high"].double() + (0 if s["low"] is None else s["low"].double())
    out = s["shared"].double()
    for a in range(case["adapters"]):
        rows = (of_rows == a).nonzero()[:, 0]
        if len(rows):
            both = s["up"][a, :, :ranks[a]].double(), s["down"][a, :ranks[a]].double()
            out[rows] += float(s["scales"][a]) * torch.mm(torch.mm(x[rows], both[1].t()),
                                                          both[0].t())
    return out


def _exact_logprobs(case, s):
    found = {n: [] for n in _found(case)}
    step = max(1, (1 << 24) // case["vocab"])
    for first in range(0, case["rows"], step):
        logits = s["logits"][first:first + step].double()
        tokens = s["tokens"][first:first + step, None].long()
        # Relative to the row's first token; log1p keeps what a sure token leaves.
        first_of_row = torch.max(logits, 1, keepdim=True)
        away = logits - first_of_row.values
        others = away.exp().scatter_(1, first_of_row.indices, 0.0).sum(1, keepdim=True)
        share = away - others.log1p()
        chosen = share.gather(1, tokens)
        found["logprob"].append(chosen[:, 0])
        found["entropy"].append(-(share.exp() * share.clamp_min(-1e300)).sum(1))
        index = torch.arange(case["vocab"], device=DEVICE)
        before = (share > chosen) | ((share == chosen) & (index < tokens))
        found["rank"].append(before.sum(1))
        if case["top"]:
            order = torch.sort(logits, dim=1, descending=True, stable=True).indices
            found["top_tokens"].append(order[:, :case["top"]])
            found["top_logprobs"].append(share.gather(1, order[:, :case["top"]]))
    found = {name: torch.cat(parts) for name, parts in found.items()}
    return {name: x if x.is_floating_point() else x.to(torch.int32) for name, x in found.items()}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"heads": _exact_heads, "adapters": _exact_adapters,
            "logprobs": _exact_logprobs}[case["op"]](case, s)
