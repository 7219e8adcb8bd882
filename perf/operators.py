"""The serving operators on device pointers, case by case: attention over packed prompts, attention of drafted token
trees over a paged K/V cache, and the cache's own steps (update, compact, write).

run() computes a case in plain torch operations where `own` is false and through huggingfaceeacp_b200.native where it is
true. Prompts and drafted rows are views of one fused [rows, q | k | v] projection, as a decoder layer leaves them.
"""
import math

import torch

own = False

PAGE = 64  # positions of a page (HF_PAGE_ROWS)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTHS = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # A handful of chat turns of 3 to 40 tokens on the engine's own heads (8 of 256 over one): latency.
        {"name": "packed_short_f16", "op": "packed", "type": "f16", "heads": 8, "kv_heads": 1, "width": 256,
         "sequences": 6, "shortest": 3, "longest": 41},
        # The engine's type and heads at about its 2048-row prefill block, several prompts in one block.
        {"name": "packed_block_f32", "op": "packed", "type": "f32", "heads": 8, "kv_heads": 1, "width": 256,
         "sequences": 4, "shortest": 100, "longest": 1001},
        # Two long documents, the longest prompts that a server admits at once.
        {"name": "packed_long_bf16", "op": "packed", "type": "bf16", "heads": 32, "kv_heads": 8, "width": 128,
         "sequences": 2, "shortest": 8191, "longest": 8191},
        # The ordinary decode step of a batch: one token a sequence, caches of 500 to 8000 tokens.
        {"name": "tree_decode_bf16", "op": "tree", "type": "bf16", "heads": 32, "kv_heads": 8, "width": 128,
         "sequences": 64, "shortest": 500, "longest": 8000, "nodes": 1, "branch": 1},
        # A batch of 16 with trees of 15 drafted tokens on the engine's heads and cache type.
        {"name": "tree_draft_f32", "op": "tree", "type": "f32", "heads": 8, "kv_heads": 1, "width": 256,
         "sequences": 16, "shortest": 100, "longest": 2048, "nodes": 15, "branch": 2},
        # One conversation with a wide tree over a short cache: latency.
        {"name": "tree_one_f16", "op": "tree", "type": "f16", "heads": 32, "kv_heads": 8, "width": 128,
         "sequences": 1, "shortest": 777, "longest": 777, "nodes": 63, "branch": 4},
        # One decode step's bookkeeping for 16 sequences: each grows by a token, one ends, one forks.
        {"name": "update_step_f32", "op": "update", "type": "f32", "layers": 18, "kv_width": 256, "pages": 256,
         "sequences": 16, "shortest": 10, "longest": 600, "releases": 1, "forks": 1, "grow": 1},
        # Beam search over a batch: 32 forks of long sequences that grow at once, so each copies its last page.
        {"name": "update_beams_bf16", "op": "update", "type": "bf16", "layers": 32, "kv_width": 1024, "pages": 1500,
         "sequences": 96, "shortest": 200, "longest": 2000, "releases": 8, "forks": 32, "grow": 4},
        # A small pool after a few retirements.
        {"name": "compact_small_f32", "op": "compact", "type": "f32", "layers": 18, "kv_width": 256, "pages": 96,
         "sequences": 12, "shortest": 50, "longest": 400},
        # A large pool, half empty, packed before a part of it is given back.
        {"name": "compact_large_bf16", "op": "compact", "type": "bf16", "layers": 32, "kv_width": 1024, "pages": 900,
         "sequences": 40, "shortest": 100, "longest": 1100},
        # The accepted rows of 64 drafted trees of one layer, picked by index.
        {"name": "write_accepted_f32", "op": "write", "type": "f32", "layers": 18, "kv_width": 256, "sequences": 64,
         "shortest": 1, "longest": 5, "before": 700, "drafted": 15},
        # A packed admission batch's keys and values of one layer.
        {"name": "write_prompts_bf16", "op": "write", "type": "bf16", "layers": 2, "kv_width": 1024, "sequences": 24,
         "shortest": 20, "longest": 1500, "before": 0, "drafted": 0},
    ]


HEADS = [(8, 1, 256), (32, 8, 128), (16, 16, 64), (12, 4, 96), (20, 4, 128), (9, 3, 64), (7, 1, 80), (16, 8, 256)]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = {}
    for c in listed():
        w, best = work(c), top.setdefault(c["op"], {"bytes": 0, "flops": 0})
        top[c["op"]] = {k: max(best[k], w[k]) for k in best}
    while True:
        op = rng.choice(["packed", "packed", "tree", "tree", "update", "compact", "write"])
        case = {"op": op, "type": rng.choice(["f32", "bf16", "f16"])}
        if op in ("packed", "tree"):
            case["heads"], case["kv_heads"], case["width"] = rng.choice(HEADS)
            case["sequences"] = _log(rng, 1, 48)
            case["longest"] = _log(rng, 1, 8000)
            case["shortest"] = rng.randint(0 if op == "tree" else 1, case["longest"])
            if op == "tree":
                case["nodes"] = rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, 64)])
                case["branch"] = rng.choice([1, 2, 3, 5])
        else:
            case["layers"] = rng.choice([2, 18, 26, 32])
            case["kv_width"] = rng.choice([64, 256, 512, 1024])
            case["sequences"] = _log(rng, 2, 96)
            case["longest"] = _log(rng, 2, 2000)
            case["shortest"] = rng.randint(1, case["longest"])
            if op == "update":
                n = case["sequences"]
                case["releases"] = rng.randint(0, n // 4)
                case["forks"] = rng.randint(0, (n - case["releases"]) // 3)
                case["grow"] = rng.choice([1, 1, rng.randint(2, 70)])
            if op != "write":
                case["pages"] = int(_pages_needed(case) * rng.uniform(1.05, 2.2)) + 2
            else:
                case["before"] = rng.choice([0, rng.randint(1, 1500)])
                case["drafted"] = 0 if case["before"] == 0 else rng.choice([0, case["longest"] + rng.randint(1, 40)])
        w = work(case)
        heavy = op == "packed" and case["sequences"] * case["longest"] ** 2 * case["heads"] > 2 * 8192 ** 2 * 32
        cache = op in ("update", "compact", "write") and _pool_bytes(case) > 8e9
        if not heavy and not cache and all(w[k] <= top[op][k] for k in w):
            return case


# ---- sizes, from the case alone ------------------------------------------------------------------------------------


def _lengths(case, count=None):
    """Lengths spread over [shortest, longest], more short than long ones, the first the longest."""
    count = case["sequences"] if count is None else count
    span = case["longest"] - case["shortest"]
    return [case["longest"] if i == 0 else case["shortest"] + int((span + 1) * (((i * 0.6180339887 + 0.37) % 1) ** 1.6))
            for i in range(count)]


def _parents(case):
    return [(i - 1) // case["branch"] if i else -1 for i in range(case["nodes"])]


def _depths(case):
    depths = []
    for p in _parents(case):
        depths.append(1 if p < 0 else depths[p] + 1)
    return depths


def _held(length):
    return -(-length // PAGE)


def _live(case):
    """The sequences that hold tokens before the call; the others of an update are the forks' targets."""
    return case["sequences"] - case.get("forks", 0)


def _pages_needed(case):
    lengths = _lengths(case, _live(case))
    return sum(_held(n) for n in lengths) + case["sequences"] * (1 + _held(case.get("grow", 0) + PAGE - 1))


def _table_stride(case):
    return _held(case["longest"] + case.get("grow", 0)) + 3


def _pool_bytes(case):
    pages = case["pages"] if "pages" in case else sum(_held(n + case["before"]) for n in _lengths(case)) + 3
    return 2 * case["layers"] * pages * PAGE * case["kv_width"] * WIDTHS[case["type"]]


def work(case):
    e = WIDTHS[case["type"]]
    if case["op"] == "packed":
        lengths = _lengths(case)
        h, kv, d, rows = case["heads"], case["kv_heads"], case["width"], sum(lengths)
        return {"bytes": rows * (2 * h + 2 * kv) * d * e + 4 * len(lengths),
                "flops": 4 * h * d * sum(n * (n + 1) // 2 for n in lengths)}
    if case["op"] == "tree":
        lengths, rows = _lengths(case), case["sequences"] * case["nodes"]
        h, kv, d = case["heads"], case["kv_heads"], case["width"]
        return {"bytes": rows * (2 * h + 2 * kv) * d * e + 2 * kv * d * e * sum(lengths)
                + 4 * (sum(_held(n) for n in lengths) + 2 * len(lengths) + rows),
                "flops": 4 * h * d * (case["nodes"] * sum(lengths) + case["sequences"] * sum(_depths(case)))}
    if case["op"] == "write":
        rows = sum(_lengths(case))
        return {"bytes": 4 * rows * case["kv_width"] * e + 8 * case["sequences"], "flops": 0}
    row = 2 * case["layers"] * case["kv_width"] * e  # one position of every layer, keys and values
    lengths = _lengths(case, _live(case))
    if case["op"] == "update":
        copied, touched = _update_work(case, lengths)
        return {"bytes": 2 * copied * row + 4 * (2 * touched + 2 * case["sequences"] + case["pages"]), "flops": 0}
    live = sum(_held(n) for n in lengths)
    moved = live - live * live // case["pages"]  # as many as a random placing moves on average
    return {"bytes": 2 * moved * PAGE * row + 4 * (2 * live + case["sequences"] + 2 * case["pages"]), "flops": 0}


def _update_work(case, lengths):
    """(rows copied, table entries touched) of an update: a fork's last page is copied when it is partly filled."""
    kept = list(range(case["releases"], len(lengths)))
    touched = sum(_held(lengths[i]) for i in range(case["releases"]))
    copied = 0
    for i in range(case["forks"]):
        n = lengths[kept[i % len(kept)]]
        touched += _held(n)
        copied += n % PAGE
    return copied, touched + case["sequences"]


# ---- inputs --------------------------------------------------------------------------------------------------------


class State:
    pass


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    return _int([0] + torch.tensor(lengths, dtype=torch.int64).cumsum(0).tolist())


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    s = State()
    s.case, s.op, s.dtype = dict(case), case["op"], TYPES[case["type"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    if s.op in ("packed", "tree"):
        h, kv, d = case["heads"], case["kv_heads"], case["width"]
        s.lengths = _lengths(case)
        rows_of = s.lengths if s.op == "packed" else [case["nodes"]] * case["sequences"]
        s.rows = sum(rows_of)
        s.offsets = _offsets(rows_of)
        qkv = _normal(g, s.rows, (h + 2 * kv) * d, dtype=s.dtype)
        s.q, s.k, s.v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], 1))
        s.stride = qkv.stride(0)
        s.out = torch.empty(s.rows, h, d, dtype=s.dtype, device="cuda")
        s.scale = 1.0 / math.sqrt(d)
    if s.op == "tree":
        held = [_held(n) for n in s.lengths]
        s.pages, s.table_stride, s.layers, s.kv_width = sum(held) + 5, max(held) + 2, 1, kv * d
        _book(s, case["sequences"], s.lengths, host)
        s.parents = _int(_parents(case) * case["sequences"])
    elif s.op == "write":
        lengths = _lengths(case)
        s.layers, s.kv_width, s.layer = case["layers"], case["kv_width"], case["layers"] // 2
        full = [n + case["before"] for n in lengths]
        s.pages, s.table_stride = sum(_held(n) for n in full) + 3, max(_held(n) for n in full) + 1
        _book(s, case["sequences"], full, host)
        s.offsets, s.rows = _offsets(lengths), sum(lengths)
        drafted = case["drafted"]
        source = drafted * case["sequences"] if drafted else s.rows
        kvs = _normal(g, source, 2 * s.kv_width, dtype=s.dtype)
        s.k, s.v = kvs.split(s.kv_width, 1)
        s.index = None
        if drafted:  # of each tree an ascending choice of its rows
            s.index = _int([i * drafted + int(x) for i, n in enumerate(lengths)
                            for x in sorted(torch.randperm(drafted, generator=host)[:n].tolist())])
    elif s.op in ("update", "compact"):
        s.layers, s.kv_width = case["layers"], case["kv_width"]
        s.pages, s.table_stride = case["pages"], _table_stride(case)
        lengths = _lengths(case, _live(case)) + [0] * case.get("forks", 0)
        _book(s, case["sequences"], lengths, host)
        if s.op == "update":
            kept = list(range(case["releases"], _live(case)))
            s.release = _int(list(range(case["releases"])))
            s.forks = _int([[kept[i % len(kept)], _live(case) + i] for i in range(case["forks"])]).reshape(-1, 2)
            s.grow = _int([0] * case["releases"] + [case["grow"]] * (case["sequences"] - case["releases"]))
    if s.op != "packed":
        pool = (s.layers, s.pages, PAGE, s.kv_width)
        if s.op == "tree":
            s.keys, s.values = _normal(g, *pool, dtype=s.dtype), _normal(g, *pool, dtype=s.dtype)
        else:  # what is only moved needs no distribution: values of 11 bits that each type holds
            s.keys, s.values = (torch.randint(-1024, 1024, pool, generator=g, device="cuda", dtype=torch.int16).to(s.dtype)
                                for _ in range(2))
    if own:
        _plan(s)
    return s


def _book(s, sequences, lengths, host):
    """table | lengths | refs | result in one buffer: distinct pages in a random order, the book kept to begin each pass from."""
    order = torch.randperm(s.pages, generator=host, dtype=torch.int64)
    table = torch.full((sequences, s.table_stride), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        table[i, : _held(n)] = order[at : at + _held(n)].to(torch.int32)
        at += _held(n)
    refs = torch.zeros(s.pages, dtype=torch.int32)
    refs[order[:at]] = 1
    book = torch.cat([table.reshape(-1), torch.tensor(lengths, dtype=torch.int32), refs, torch.zeros(3, dtype=torch.int32)])
    s.book0 = book.cuda()
    s.book = s.book0.clone()
    a, b, c = sequences * s.table_stride, sequences, s.pages
    s.table = s.book[:a].view(sequences, s.table_stride)
    s.length, s.refs, s.result = s.book[a : a + b], s.book[a + b : a + b + c], s.book[a + b + c :]


def _plan(s):
    from huggingfaceeacp_b200 import native

    c = s.case
    dtype = {"f32": native.F32, "bf16": native.BF16, "f16": native.F16}[c["type"]]
    size = 0
    if s.op != "packed":
        s.cache = native.PageCache(dtype, s.layers, s.pages, s.kv_width, c["sequences"], s.table_stride, s.keys.data_ptr(),
                                   s.values.data_ptr(), s.table.data_ptr(), s.length.data_ptr(), s.refs.data_ptr())
        size = s.cache.workspace_bytes
    if s.op == "packed":
        s.plan = native.PackedAttention(dtype, c["heads"], c["kv_heads"], c["width"], scale=s.scale)
        size = s.plan.workspace_bytes(c["sequences"], s.rows)
    elif s.op == "tree":
        s.plan = native.TreeAttention(dtype, c["heads"], c["kv_heads"], c["width"], scale=s.scale)
        size = s.plan.workspace_bytes(c["sequences"], s.rows, c["nodes"], c["longest"])
    s.workspace = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")


# ---- the passes ----------------------------------------------------------------------------------------------------


def run(s):
    return {"packed": _packed, "tree": _tree, "update": _update, "compact": _compact, "write": _write}[s.op](s)


def _room(s):
    return {"workspace": s.workspace.data_ptr(), "workspace_bytes": s.workspace.numel(),
            "stream": torch.cuda.current_stream().cuda_stream}


def _packed(s):
    if own:
        s.plan.run(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(), s.offsets.data_ptr(),
                   s.case["sequences"], s.rows, q_stride=s.stride, k_stride=s.stride, v_stride=s.stride, **_room(s))
        return s.out
    begin, count = s.offsets[:-1, None].long(), (s.offsets[1:] - s.offsets[:-1])[:, None]
    at = torch.arange(s.case["longest"], device="cuda")
    there = at < count  # [B, L]: rows of the padded batch that exist
    rows = torch.where(there, begin + at, 0)
    kv, group = s.case["kv_heads"], s.case["heads"] // s.case["kv_heads"]
    q = s.q[rows].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4)  # [B, KV, G, L, D]
    k = s.k[rows].float().permute(0, 2, 3, 1)[:, :, None]  # [B, KV, 1, D, L]
    v = s.v[rows].float().permute(0, 2, 1, 3)[:, :, None]  # [B, KV, 1, L, D]
    scores = (q * s.scale) @ k
    scores.masked_fill_(at[None, :] > at[:, None], -math.inf)  # causal: a row that exists sees no row past its sequence
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (scores @ v) / scores.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, L, H, D]
    return out.reshape(-1, *out.shape[2:])[there.reshape(-1)].to(s.dtype)


def _tree(s):
    c = s.case
    if own:
        s.plan.run(s.cache, 0, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(), s.offsets.data_ptr(),
                   s.parents.data_ptr(), s.rows, c["nodes"], c["longest"], q_stride=s.stride, k_stride=s.stride,
                   v_stride=s.stride, **_room(s))
        return s.out
    b, n, kv, d = c["sequences"], c["nodes"], c["kv_heads"], c["width"]
    at = torch.arange(c["longest"], device="cuda")
    page = s.table[:, at // PAGE].clamp(min=0).long()  # [B, L]
    keys, values = (x[0].view(s.pages, PAGE, kv, d)[page, at % PAGE] for x in (s.keys, s.values))  # [B, L, KV, D]
    k = torch.cat([keys, s.k.unflatten(0, (b, n))], 1).float().permute(0, 2, 3, 1)  # [B, KV, D, L + N]
    v = torch.cat([values, s.v.unflatten(0, (b, n))], 1).float().permute(0, 2, 1, 3)
    node = torch.arange(n, device="cuda")
    step = (s.parents.view(b, n)[:, :, None] == node).float() + torch.eye(n, device="cuda")
    path = torch.linalg.matrix_power(step, n) > 0  # [B, N, N]: j on the path from i up
    seen = torch.cat([(at < s.length[:, None])[:, None].expand(b, n, -1), path], 2)  # [B, N, L + N]
    q = s.q.float().unflatten(0, (b, n)).unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4)  # [B, KV, G, N, D]
    scores = (q.flatten(2, 3) * s.scale) @ k  # [B, KV, G N, L + N]
    scores = scores.unflatten(2, (-1, n)).masked_fill_(~seen[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (scores.flatten(2, 3) @ v).unflatten(2, (-1, n)) / scores.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(b * n, c["heads"], d).to(s.dtype)


def _cache_out(s):
    return {"table": s.table, "lengths": s.length, "refs": s.refs, "result": s.result, "keys": s.keys, "values": s.values}


def _update(s):
    s.book.copy_(s.book0)
    if own:
        s.cache.update(release=s.release.data_ptr(), releases=s.release.numel(), forks=s.forks.data_ptr(),
                       fork_count=s.forks.shape[0], grow=s.grow.data_ptr(), result=s.result.data_ptr(), **_room(s))
        return _cache_out(s)
    table, length, refs = s.table, s.length, s.refs
    gone = s.release.long()
    rows = table[gone]
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).int().flatten())
    table[gone] = -1
    length[gone] = 0
    source, target = s.forks[:, 0].long(), s.forks[:, 1].long()
    rows = table[source]
    table[target] = rows
    length[target] = length[source]
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).int().flatten())
    # Growth: a sequence copies its partly filled last page while another still holds it, in the sequences' order.
    held = (length + PAGE - 1) // PAGE
    grows = s.grow > 0
    last = table.gather(1, (held - 1).clamp(min=0)[:, None].long())[:, 0]
    open_ = grows & (length % PAGE != 0)
    same = (last[:, None] == last[None, :]) & open_[None, :]
    holders = refs[last.clamp(min=0).long()] - torch.tril(same, -1).sum(1)
    copies = open_ & (holders > 1)
    grown = length + s.grow.clamp(min=0)
    new = (grown + PAGE - 1) // PAGE - held
    need = new + copies
    first = need.cumsum(0) - need
    free = refs == 0
    order = torch.argsort(~free, stable=True)  # the free pages first, ascending
    room, wanted = free.sum(), need.sum()
    past = (grown > s.table_stride * PAGE).sum()
    fits = (wanted <= room) & (past == 0)
    copies, grows = copies & fits, grows & fits
    column = torch.arange(s.table_stride, device="cuda")
    rank = column - held[:, None]
    fresh = (rank >= 0) & (rank < new[:, None]) & grows[:, None]
    entry = first[:, None] + copies[:, None] + rank
    table.copy_(torch.where(fresh, order[entry.clamp(0, s.pages - 1)].int(), table))
    to = order[first.clamp(0, s.pages - 1)].int()
    at = (column == held[:, None] - 1) & copies[:, None]
    table.copy_(torch.where(at, to[:, None], table))
    refs.index_add_(0, last.clamp(min=0).long(), -copies.int())
    taken = torch.arange(s.pages, device="cuda") < wanted * fits
    refs[order] += taken.int()
    used = length % PAGE
    which = copies.nonzero()[:, 0]
    rows = (torch.arange(PAGE, device="cuda") < used[which, None])[None, :, :, None]
    for pool in (s.keys, s.values):
        pool[:, to[which].long()] = torch.where(rows, pool[:, last[which].long()], pool[:, to[which].long()])
    length.copy_(torch.where(grows, grown, length))
    s.result[0] = (refs == 0).sum()
    s.result[1] = (wanted - room).clamp(min=0)
    s.result[2] = past
    return _cache_out(s)


def _compact(s):
    s.book.copy_(s.book0)
    if own:
        s.cache.compact(live=s.result.data_ptr(), **_room(s))
        return _cache_out(s)
    live = s.refs > 0
    count = live.sum()
    page = torch.arange(s.pages, device="cuda")
    leaves, hole = live & (page >= count), ~live & (page < count)
    source, target = leaves.nonzero()[:, 0], hole.nonzero()[:, 0]  # both ascending, and as many
    renamed = page.clone()
    renamed[source] = target
    s.table.copy_(torch.where(s.table >= 0, renamed[s.table.clamp(min=0).long()].int(), s.table))
    s.refs[target] = s.refs[source]
    s.refs[source] = 0
    for pool in (s.keys, s.values):
        pool[:, target] = pool[:, source]
    s.result[0] = count
    return _cache_out(s)


def _write(s):
    if own:
        s.cache.write(s.layer, s.k.data_ptr(), s.v.data_ptr(), s.offsets.data_ptr(), s.rows, source_rows=s.k.shape[0],
                      index=0 if s.index is None else s.index.data_ptr(), k_stride=s.k.stride(0), v_stride=s.v.stride(0),
                      stream=torch.cuda.current_stream().cuda_stream)
        return {"keys": s.keys, "values": s.values}
    row = torch.arange(s.rows, device="cuda")
    sequence = torch.searchsorted(s.offsets[1:], row, right=True)
    position = s.length[sequence] - s.offsets[1:][sequence] + row
    at = s.table[sequence, position // PAGE].long() * PAGE + position % PAGE
    for pool, rows in ((s.keys, s.k), (s.values, s.v)):
        pool[s.layer].view(-1, s.kv_width)[at] = rows if s.index is None else rows[s.index.long()]
    return {"keys": s.keys, "values": s.values}


# ---- in 64 bits, sequence by sequence ------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] not in ("packed", "tree"):
        return None  # copies and whole numbers
    s = prepare(case, seed)
    group = case["heads"] // case["kv_heads"]
    parents = _parents(case) if s.op == "tree" else None
    out = torch.zeros(s.rows, case["heads"], case["width"], dtype=torch.float64, device="cuda")
    start = 0
    for i, length in enumerate(s.lengths):
        n = length if parents is None else len(parents)
        k, v = (x[start : start + n].double() for x in (s.k, s.v))
        if parents is None:
            seen = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
        else:
            pages = s.table[i, : _held(length)].long()
            cached = [x[0, pages].reshape(-1, case["kv_heads"], case["width"])[:length].double() for x in (s.keys, s.values)]
            k, v = torch.cat([cached[0], k]), torch.cat([cached[1], v])
            path = torch.zeros(n, n, dtype=torch.bool)
            for j in range(n):
                up = j
                while up >= 0:
                    path[j, up] = True
                    up = parents[up]
            seen = torch.cat([torch.ones(n, length, dtype=torch.bool), path], 1).cuda()
        for h in range(case["heads"]):
            scores = s.q[start : start + n, h].double() @ k[:, h // group].T / math.sqrt(case["width"])
            weights = torch.softmax(torch.where(seen, scores, -math.inf), 1)
            out[start : start + n, h] = weights @ v[:, h // group]
        start += n
    return out
