"""Serving operators around the paged KV pool, as measurable cases.

Three families, each one pass of the operator as a serving program calls it:

- "shared": `shared_prefix_attn`, the attention of a batch whose requests share
  a long prefix (one system prompt or document, many continuations), the prefix
  attended once for all of a group's rows;
- "alibi": `paged_attn_alibi`, paged attention with a bias that falls linearly
  with the distance between query and key, one slope a query head;
- "tables": `extend_block_tables`, block tables, token map and slots of a
  scheduler step made on the GPU from the requests' lengths.

With `own` false, `run` computes the same in elementary torch operations in 32
bits; with `own` true it calls the framework. The metadata of an attention
batch is made in `prepare`, as a program makes it once and uses it in all
layers. Sequence lengths are part of the case (drawn from its "lengths"
number); values, pool placement and slot order are made from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

MAX_ROWS = 8192        # rows of one batch's metadata
MAX_CONTEXT = 32768
GEOMETRIES = [         # (query heads, kv heads, head_dim) of the configurations and tests
    (32, 8, 128), (32, 8, 128), (64, 8, 128), (8, 2, 128), (14, 2, 64), (16, 8, 256), (8, 8, 128), (24, 8, 128),
    (32, 8, 64),
]


def _attention(family, name=None, **fields):
    # `groups` sets of `seqs` requests in all, each set behind one prefix of prefix_lo .. prefix_hi tokens (0: none);
    # every request has own_lo .. own_hi cached tokens of its own behind it and new_lo .. new_hi new tokens.
    case = {
        "family": family, "seqs": 1, "groups": 1, "prefix_lo": 0, "prefix_hi": 0, "own_lo": 0, "own_hi": 0,
        "new_lo": 1, "new_hi": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128, "softcap": 0.0,
        "window": -1, "lengths": 1,
    }
    assert set(fields) <= set(case), set(fields) - set(case)
    case.update(fields)
    return case if name is None else {"name": name, **case}


def _tables(name=None, **fields):
    # `seqs` requests with cached_lo .. cached_hi tokens get new_lo .. new_hi more; the first `forks` of them start
    # with the pages of one parent request. `requests` rows of `context` tokens in the tables.
    case = {
        "family": "tables", "seqs": 1, "forks": 0, "cached_lo": 0, "cached_hi": 0, "new_lo": 1, "new_hi": 1,
        "page": 16, "requests": 64, "context": 4096, "lengths": 1,
    }
    assert set(fields) <= set(case), set(fields) - set(case)
    case.update(fields)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # Four continuations of one short prompt on a small model: launches and host work are what counts.
        _attention("shared", "shared_smallest", seqs=4, prefix_lo=512, prefix_hi=512, own_lo=0, own_hi=63, q_heads=8,
                   kv_heads=2),
        # A server's ordinary decode batch behind one system prompt.
        _attention("shared", "shared_batch", seqs=64, prefix_lo=4096, prefix_hi=4096, own_lo=32, own_hi=1023),
        # Many readers of one long document: the largest.
        _attention("shared", "shared_document", seqs=256, prefix_lo=32000, prefix_hi=32000, own_lo=16, own_hi=700),
        # Six prompts of a small model with ragged sets of requests behind them, four draft tokens each to verify.
        _attention("shared", "shared_drafts_d64", seqs=45, groups=6, prefix_lo=300, prefix_hi=5000, own_lo=0,
                   own_hi=900, new_lo=4, new_hi=4, q_heads=14, kv_heads=2, head_dim=64, page=16),
        # Wide heads with logit softcap and a sliding window that ends inside the prefix, token-granular map.
        _attention("shared", "shared_d256_window", seqs=48, groups=2, prefix_lo=3000, prefix_hi=6000, own_lo=100,
                   own_hi=3000, q_heads=16, head_dim=256, page=1, softcap=50.0, window=4096),
        # Four short conversations, one query head a kv head.
        _attention("alibi", "alibi_smallest", seqs=4, own_lo=1, own_hi=511, q_heads=8, kv_heads=8),
        # An ordinary decode batch.
        _attention("alibi", "alibi_decode", seqs=64, own_lo=511, own_hi=4095),
        # Eight prompts' chunks of 512 tokens, 2048 tokens in the cache.
        _attention("alibi", "alibi_prefill", seqs=8, own_lo=2048, own_hi=2048, new_lo=512, new_hi=512),
        # Decode rows of a small model on a long, ragged cache with small pages.
        _attention("alibi", "alibi_long_d64", seqs=17, own_lo=2000, own_hi=20000, q_heads=14, kv_heads=2, head_dim=64,
                   page=16),
        # A decode step of a full server: one new token a request, a page now and then.
        _tables("tables_decode", seqs=256, cached_lo=128, cached_hi=4000, requests=512, context=4608),
        # Conversations that start from one 8192-token prompt's pages.
        _tables("tables_fork", seqs=64, forks=64, cached_lo=8192, cached_hi=8192, new_lo=5, new_hi=300, requests=128,
                context=16384),
        # New prompts: the largest.
        _tables("tables_prompts", seqs=48, new_lo=1000, new_hi=32000, page=128, requests=256, context=32768),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    cases = listed()
    most = {f: {k: max(work(c)[k] for c in cases if c["family"] == f) for k in ("bytes", "flops")}
            for f in ("shared", "alibi", "tables")}
    while True:
        family = rng.choice(["shared", "shared", "shared", "alibi", "alibi", "tables"])
        number = rng.randrange(1 << 20)
        if family == "tables":
            page = rng.choice([1, 16, 16, 64, 128])
            f = {"seqs": _log(rng, 1, 512), "page": page, "lengths": number}
            kind = rng.choice(["decode", "prompts", "fork"])
            context = _log(rng, 64, MAX_CONTEXT)
            f["new_hi"] = rng.choice([1, 1, 4]) if kind == "decode" else _log(rng, 2, max(2, context // 2))
            f["new_lo"] = 1 if kind == "decode" else int(f["new_hi"] * rng.choice([0.0, 0.1, 0.8]))
            room = context - f["new_hi"]
            f["cached_hi"] = rng.randint(0, room)
            f["cached_lo"] = int(f["cached_hi"] * rng.choice([0.0, 0.3, 0.9]))
            if kind == "fork":
                f["cached_lo"] = f["cached_hi"] = f["cached_hi"] // page * page
                f["forks"] = rng.randint(1, f["seqs"])
            f["context"] = context
            f["requests"] = f["seqs"] + rng.randint(1, 100)
            case = _tables(**f)
            if case["requests"] * context > 1 << 24:
                continue
        else:
            q_heads, kv_heads, head_dim = rng.choice(GEOMETRIES)
            f = {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([1, 16, 16, 128]),
                 "lengths": number}
            if rng.random() < 0.25:
                f["softcap"] = rng.choice([30.0, 50.0])
            if rng.random() < 0.25:
                f["window"] = rng.choice([128, 1024, 4096, 1000])
            f["seqs"] = _log(rng, 1, 256)
            kind = rng.choice(["decode", "decode", "drafts", "chunks"])
            if kind == "drafts":
                f["new_lo"] = f["new_hi"] = rng.randint(2, 7)
            if kind == "chunks":
                f["seqs"] = _log(rng, 1, 8)
                f["new_hi"] = _log(rng, 8, 1024)
                f["new_lo"] = max(1, int(f["new_hi"] * rng.choice([0.2, 0.6, 1.0])))
            if family == "shared":
                f["groups"] = rng.randint(1, min(8, f["seqs"]))
                f["prefix_hi"] = _log(rng, 16, MAX_CONTEXT)
                f["prefix_lo"] = int(f["prefix_hi"] * rng.choice([0.3, 0.7, 1.0]))
                f["own_hi"] = _log(rng, 1, 2048)
            else:
                f["own_hi"] = _log(rng, 16, MAX_CONTEXT)
            f["own_lo"] = int(f["own_hi"] * rng.choice([0.05, 0.25, 0.9]))
            case = _attention(family, **f)
            if case["seqs"] * case["new_hi"] > MAX_ROWS:
                continue
        w = work(case)
        if w["bytes"] <= most[family]["bytes"] and w["flops"] <= most[family]["flops"]:
            return case


def _sequences(case):
    """Attention: [(group, prefix, own cached tokens, new tokens)], a group's requests side by side."""
    rng = random.Random(case["lengths"])
    groups = case["groups"]
    prefix = [rng.randint(case["prefix_lo"], case["prefix_hi"]) for _ in range(groups)]
    cuts = sorted(rng.sample(range(1, case["seqs"]), groups - 1))
    seqs = []
    for s in range(case["seqs"]):
        g = sum(1 for c in cuts if c <= s)
        seqs.append((g, prefix[g], rng.randint(case["own_lo"], case["own_hi"]), rng.randint(case["new_lo"], case["new_hi"])))
    return seqs


def _lengths(case):
    """Tables: [(cached tokens, new tokens)]; a parent's row, when there are forks, comes behind the others."""
    rng = random.Random(case["lengths"])
    return [(rng.randint(case["cached_lo"], case["cached_hi"]), rng.randint(case["new_lo"], case["new_hi"]))
            for _ in range(case["seqs"])]


def work(case):
    if case["family"] == "tables":
        seqs, page = _lengths(case), case["page"]
        rows = sum(n for _, n in seqs)
        copied = sum(c for c, _ in seqs[:case["forks"]])
        taken = sum(-(-(c + n) // page) - -(-c // page) for c, n in seqs)
        # Lengths and requests in, pages in and into the tables, tokens into the map; a row's slot, request and
        # position; the parent's entries read once, written into every fork.
        pages = copied // page
        read = len(seqs) * 24 + taken * 8 + (seqs[0][0] + seqs[0][0] // page) * 4 * (case["forks"] > 0)
        return {"bytes": read + len(seqs) * 8 + (taken + pages) * 4 + (rows + copied) * 4 + rows * 12,
                "flops": 0}
    window = case["window"] if case["window"] > 0 else 1 << 30
    rows = keys = pairs = 0
    first_of = {}
    for g, prefix, cached, n in _sequences(case):
        start = prefix + cached  # position of the first new token
        low = max(0, start + 1 - window)
        prefix = _shared_tokens(case, prefix)
        rows += n
        keys += start + n - max(prefix, low)
        first_of[g] = (prefix, min(low, first_of.get(g, (0, low))[1]))
        # Keys that row i sees: min(start + i + 1, window).
        full = min(n, max(0, start + n - window))
        ramp = n - full
        pairs += ramp * (start + 1) + ramp * (ramp - 1) // 2 + full * window
    keys += sum(max(0, prefix - low) for prefix, low in first_of.values())
    q_width, kv_width = case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    # Keys and values once (a shared prefix once for its group), queries and outputs once, the new rows read and
    # written once, one table entry a page.
    return {"bytes": keys * kv_width * 4 + rows * q_width * 4 + rows * kv_width * 8 + 4 * (keys // case["page"] + 2 * rows),
            "flops": 4 * q_width * pairs}


def _slopes(heads):
    """A geometric sequence of slopes, 2^(-8 i / n) for the n heads of the next power of two, every other one first."""
    n = 1 << (heads - 1).bit_length()
    steps = [2.0 ** (-8.0 * (i + 1) / n) for i in range(n)]
    return (steps[1::2] + steps[0::2])[:heads] if n != heads else steps


def _place(case, seed):
    """(token map [sequences, context] int32, slots): tokens in blocks scattered over the pool; a group's requests
    share the whole pages of their prefix and hold copies of its last, partial page."""
    seqs, page = _sequences(case), case["page"]
    rng = np.random.default_rng(seed)
    whole = {g: prefix // page for g, prefix, _, _ in seqs}
    need = sum(whole.values()) + sum(-(-(prefix + cached + n) // page) - prefix // page + 1 for _, prefix, cached, n in seqs)
    blocks = rng.permutation(need + 1).astype(np.int64)
    context = max(prefix + cached + n for _, prefix, cached, n in seqs)
    mapping = np.full((len(seqs), context), -1, dtype=np.int32)
    at, head = 0, {}
    for s, (g, prefix, cached, n) in enumerate(seqs):
        end = prefix + cached + n
        if g not in head:
            head[g] = blocks[at:at + whole[g]]
            at += whole[g]
        mine = -(-end // page) - whole[g]
        table = np.concatenate([head[g], blocks[at:at + mine]])
        at += mine
        tokens = np.arange(end)
        mapping[s, :end] = table[tokens // page] * page + tokens % page
    return mapping, len(blocks) * page


def _shared_tokens(case, prefix):
    """Tokens of a prefix that a group's requests hold in the same slots: its whole pages."""
    return prefix // case["page"] * case["page"]


def prepare(case, seed):
    return _prepare_tables(case, seed) if case["family"] == "tables" else _prepare_attention(case, seed)


def _prepare_attention(case, seed):
    seqs, d = _sequences(case), case["head_dim"]
    q_heads, kv_heads = case["q_heads"], case["kv_heads"]
    mapping, slots = _place(case, seed)
    news = [n for _, _, _, n in seqs]
    starts = [prefix + cached for _, prefix, cached, _ in seqs]
    requests = np.repeat(np.arange(len(seqs)), news)
    positions = np.concatenate([np.arange(p, p + n) for p, n in zip(starts, news)])
    locations = mapping[requests, positions].astype(np.int64)
    rows = len(positions)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)

    pool = normal(1, 2, kv_heads, slots, d)
    group_rows, group_prefix = [], []
    for g, prefix, _, n in seqs:
        if g == len(group_rows):
            group_rows.append(0)
            group_prefix.append(_shared_tokens(case, prefix))
        group_rows[g] += n
    state = {
        "case": case, "pool": pool, "query": normal(rows, q_heads * d), "key": normal(rows, kv_heads * d),
        "value": normal(rows, kv_heads * d), "scale": float(np.float32(1 / math.sqrt(d))),
        "slopes": torch.tensor(_slopes(q_heads), dtype=torch.float32, device="cuda"),
        "group_rows": group_rows, "group_prefix": group_prefix, "where": (mapping, positions, locations),
    }
    if own:
        import gaudirt_amd

        gaudirt_amd.load_extension()
        state["views"] = gaudirt_amd.kv_pool_views(pool, 0)
        state["metadata"] = torch.classes.gaudirt.PagedMetadata(
            torch.from_numpy(locations), torch.from_numpy(requests), torch.from_numpy(positions),
            torch.from_numpy(mapping), slots)
    else:
        state["mapping"] = torch.from_numpy(mapping).cuda()
        state["positions"] = torch.from_numpy(positions).cuda()
        state["locations"] = torch.from_numpy(locations).cuda()
        state["seqs"] = [(p, n) for p, n in zip(starts, news)]
    return state


def _prepare_tables(case, seed):
    """A pool with `requests` table rows, the batch's rows among them; pages of cached tokens in scattered order."""
    seqs, page = _lengths(case), case["page"]
    rng = np.random.default_rng(seed)
    width = -(-case["context"] // page)
    rows = rng.permutation(case["requests"] - 1)[:len(seqs)]  # the last row is the parent's
    parent = case["requests"] - 1
    total = sum(-(-(c + n) // page) for c, n in seqs) + width + 1
    pages = rng.permutation(np.arange(1, total + 1))
    tables = np.full((case["requests"], width), -1, dtype=np.int32)
    at = 0

    def cached(row, tokens):
        nonlocal at
        count = -(-tokens // page)
        tables[row, :count] = pages[at:at + count]
        at += count

    forks = case["forks"]
    if forks:
        cached(parent, seqs[0][0])
    for row, (c, _) in list(zip(rows, seqs))[forks:]:
        cached(row, c)
    tokens = np.arange(case["context"])
    held = tables[:, tokens // page]
    mapping = np.where(held >= 0, held * page + (tokens % page).astype(np.int32), -1).astype(np.int32)
    filled = {parent: seqs[0][0]} if forks else {}
    filled.update({int(r): c for r, (c, _) in list(zip(rows, seqs))[forks:]})
    for r, c in filled.items():
        mapping[r, c:] = -1

    def put(a, dtype):
        return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dtype)

    parents = np.full(len(seqs), -1)
    parents[:forks] = parent
    if own:
        import gaudirt_amd

        gaudirt_amd.load_extension()
    return {
        "case": case, "tables": put(tables, torch.int32), "mapping": put(mapping, torch.int32),
        "requests": put(rows, torch.int32), "prefixes": put([c for c, _ in seqs], torch.int64),
        "lengths": put([n for _, n in seqs], torch.int64), "free_pages": put(pages[at:], torch.int64),
        "free_head": torch.zeros(1, dtype=torch.int32, device="cuda"), "parents": put(parents, torch.int32),
        "slots": (total + 1) * page, "rows": sum(n for _, n in seqs),
    }


def run(state):
    case = state["case"]
    if case["family"] == "tables":
        return (_own_tables if own else _plain_tables)(state)
    if not own:
        return _plain_attention(state)
    key_pool, value_pool = state["views"]
    common = state["query"], state["key"], state["value"], key_pool, value_pool, state["metadata"]
    rest = case["head_dim"], state["scale"], case["softcap"], case["window"]
    if case["family"] == "shared":
        out = torch.ops.gaudirt.shared_prefix_attn(*common, state["group_rows"], state["group_prefix"], *rest)
    else:
        out = torch.ops.gaudirt.paged_attn_alibi(*common, state["slopes"], *rest)
    return {"out": out, "pool": state["pool"]}


def _plain_attention(state):
    """New rows into the pool, then every request's rows over its keys, in 32 bits."""
    case, pool = state["case"], state["pool"]
    d, q_heads, kv_heads = case["head_dim"], case["q_heads"], case["kv_heads"]
    group, softcap, window = q_heads // kv_heads, case["softcap"], case["window"]
    pool[0, 0][:, state["locations"]] = state["key"].view(-1, kv_heads, d).transpose(0, 1)
    pool[0, 1][:, state["locations"]] = state["value"].view(-1, kv_heads, d).transpose(0, 1)
    query = state["query"].float().view(-1, kv_heads, group, d)
    out = torch.empty_like(state["query"])
    first = 0
    for s, (start, n) in enumerate(state["seqs"]):
        slots = state["mapping"][s, :start + n].long()
        low = max(0, start + 1 - window) if window > 0 else 0  # no row sees a key before this one
        slots = slots[low:]
        at = torch.arange(low, start + n, device="cuda")
        position = state["positions"][first:first + n]
        distance = (at[None, :] - position[:, None]).float()  # 0 at the row's own key, negative before it
        hidden = at[None, :] > position[:, None]
        if window > 0:
            hidden |= at[None, :] <= position[:, None] - window
        for h in range(kv_heads):
            k, v = pool[0, 0, h][slots].float(), pool[0, 1, h][slots].float()
            q = query[first:first + n, h]
            score = (q.reshape(n * group, d) @ k.t().contiguous()).view(n, group, -1) * state["scale"]
            if softcap > 0:
                score = softcap * torch.tanh(score / softcap)
            if case["family"] == "alibi":
                slopes = state["slopes"][h * group:(h + 1) * group]
                score = score + slopes[None, :, None] * distance[:, None, :]
            score = score.masked_fill(hidden[:, None, :], -math.inf)
            weight = torch.exp(score - score.amax(dim=2, keepdim=True))
            weight = weight / weight.sum(dim=2, keepdim=True)
            result = (weight.view(n * group, -1) @ v).view(n, group, d)
            out.view(-1, kv_heads, group, d)[first:first + n, h] = result.to(out.dtype)
        first += n
    return {"out": out, "pool": pool}


def _own_tables(state):
    return dict(zip(("locations", "row_requests", "positions", "seq_lens", "counts", "tables", "mapping"), (
        *torch.ops.gaudirt.extend_block_tables(
            state["tables"], state["mapping"], state["requests"], state["prefixes"], state["lengths"],
            state["free_pages"], state["free_head"], state["parents"], state["case"]["page"], state["slots"],
            state["rows"]),
        state["tables"], state["mapping"])))


def _plain_tables(state):
    """The same from scans and gathers; every sequence's pages come from the free list in batch order."""
    page, tables, mapping = state["case"]["page"], state["tables"], state["mapping"]
    requests, prefixes, lengths = state["requests"].long(), state["prefixes"], state["lengths"]
    parents = state["parents"].long()
    end = prefixes + lengths
    held = (prefixes + page - 1) // page
    need = (end + page - 1) // page - held
    first_page = need.cumsum(0) - need
    first_row = lengths.cumsum(0) - lengths
    width, context = tables.shape[1], mapping.shape[1]
    # A fork's cached tokens are its parent's.
    entry = torch.arange(width, device="cuda")
    token = torch.arange(context, device="cuda")
    forked = (parents >= 0)[:, None]
    source = parents.clamp(min=0)
    mine = torch.where(forked & (entry < held[:, None]), tables[source], tables[requests])
    tokens = torch.where(forked & (token < prefixes[:, None]), mapping[source], mapping[requests])
    # New pages behind the held ones, new tokens behind the cached ones.
    order = entry - held[:, None]
    new = (order >= 0) & (order < need[:, None])
    taken = (state["free_head"].long() + first_page)[:, None] + order
    mine = torch.where(new, state["free_pages"][taken.clamp(0, len(state["free_pages"]) - 1)].int(), mine)
    slot = mine[:, token // page] * page + (token % page).int()
    tokens = torch.where((token >= prefixes[:, None]) & (token < end[:, None]), slot, tokens)
    tables[requests] = mine
    mapping[requests] = tokens
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(first_row, row, right=True) - 1
    position = prefixes[seq] + row - first_row[seq]
    counts = torch.stack([lengths.sum(), state["free_head"][0] + need.sum(), 0 * need.sum(), 0 * need.sum() - 1]).int()
    return {"locations": mapping[requests[seq], position], "row_requests": requests[seq].int(),
            "positions": position.int(), "seq_lens": end, "counts": counts, "tables": tables, "mapping": mapping}


def exact(case, seed):
    return _exact_tables(case, seed) if case["family"] == "tables" else _exact_attention(case, seed)


def _exact_tables(case, seed):
    """Request by request on the host."""
    state = prepare(case, seed)
    page = case["page"]
    tables, mapping = state["tables"].cpu().numpy().copy(), state["mapping"].cpu().numpy().copy()
    free = state["free_pages"].cpu().numpy()
    parents = state["parents"].tolist()
    locations, requests, positions, taken = [], [], [], 0
    for row, parent, prefix, n in zip(state["requests"].tolist(), parents, state["prefixes"].tolist(),
                                      state["lengths"].tolist()):
        held = -(-prefix // page)
        if parent >= 0:
            tables[row, :held] = tables[parent, :held]
            mapping[row, :prefix] = mapping[parent, :prefix]
        for entry in range(held, -(-(prefix + n) // page)):
            tables[row, entry] = free[taken]
            taken += 1
        at = np.arange(prefix, prefix + n)
        slots = tables[row, at // page] * page + at % page
        mapping[row, at] = slots
        locations.append(slots)
        positions.append(at)
        requests.append(np.full(n, row))
    return {
        "locations": torch.from_numpy(np.concatenate(locations).astype(np.int32)),
        "row_requests": torch.from_numpy(np.concatenate(requests).astype(np.int32)),
        "positions": torch.from_numpy(np.concatenate(positions).astype(np.int32)),
        "seq_lens": torch.from_numpy(np.array([c + n for c, n in _lengths(case)], dtype=np.int64)),
        "counts": torch.tensor([state["rows"], taken, 0, -1], dtype=torch.int32),
        "tables": torch.from_numpy(tables), "mapping": torch.from_numpy(mapping),
    }


def _exact_attention(case, seed):
    """Head by head in 64 bits, a softmax over the keys that each row may see."""
    state = prepare(case, seed)
    seqs, d = _sequences(case), case["head_dim"]
    kv_heads, q_heads = case["kv_heads"], case["q_heads"]
    group = q_heads // kv_heads
    mapping, positions, locations = state["where"]
    slots_of = torch.from_numpy(mapping).cuda().long()
    keys, values = state["pool"][0, 0], state["pool"][0, 1]
    locations = torch.from_numpy(locations).cuda()
    for pool, new in ((keys, state["key"]), (values, state["value"])):
        for h in range(kv_heads):
            pool[h].index_copy_(0, locations, new[:, h * d:(h + 1) * d].contiguous())
    query = state["query"].double()
    out = torch.zeros(query.shape, dtype=torch.float64, device="cuda")
    slopes = torch.tensor(_slopes(q_heads), dtype=torch.float32).double().tolist()
    row = 0
    for s, (_, prefix, cached, n) in enumerate(seqs):
        start, end = prefix + cached, prefix + cached + n
        low = max(0, start - case["window"] + 1) if case["window"] > 0 else 0
        at = torch.arange(low, end, device="cuda")
        where = torch.arange(start, end, device="cuda")[:, None]
        seen = at <= where
        if case["window"] > 0:
            seen &= at > where - case["window"]
        for h in range(kv_heads):
            k = keys[h].index_select(0, slots_of[s, low:end]).double().t().contiguous()
            v = values[h].index_select(0, slots_of[s, low:end]).double()
            for j in range(h * group, (h + 1) * group):
                columns = slice(j * d, (j + 1) * d)
                score = (query[row:row + n, columns].contiguous() @ k) * state["scale"]
                if case["softcap"] > 0:
                    score = torch.tanh(score / case["softcap"]) * case["softcap"]
                if case["family"] == "alibi":
                    score = score - slopes[j] * (where - at).double()
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                out[row:row + n, columns] = torch.softmax(score, dim=1) @ v
        row += n
    return {"out": out, "pool": None}
