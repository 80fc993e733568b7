"""Performance cases of the operators for drafted tokens over blocks of KV memory.

Three kinds of work, each over the range of sizes it is used at:

* ``attention``  attention of drafted trees (or chains, or single tokens) over a blocked or slotted
                 KV cache: ``kernels.tree_attn``;
* ``tables``     the block tables, slot maps, positions and tree masks of a step, from the
                 requests' lengths: ``kernels.block_tables``;
* ``commit``     the walk along the tree that the target model agrees with, and the move of its K/V
                 rows to the end of the context: ``kernels.tree_commit``.

Layouts.  Rows of all requests lie one after the other; request b has rows ``row_start[b]`` to
``row_start[b + 1] - 1``, one per node of its tree.  Node 0 is the token that the request feeds next, the
parent of node i is a node before it.  Position p of request b is cached in block
``tables[b, p // block]`` at offset ``p % block``; planes are ``[blocks, kv heads, block, head dim]``, so a
slotted cache is one whose blocks are its slots.  Free blocks lie in a ring: ``pool`` is
``[head, count, 0, status, ids...]``.
"""

from __future__ import annotations

import importlib

import torch

own = False
DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
VOCAB = 151936


# ---- the cases ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one user, one token after a short prompt: the least there is
        {"name": "attention-1x1-300", "kind": "attention", "type": "fp16", "heads": 14, "kv_heads": 2, "dim": 64,
         "requests": 1, "shortest": 300, "longest": 300, "nodes": 1, "block": 64, "tree": False},
        # one user, a wide tree over a conversation
        {"name": "attention-1x48-4096", "kind": "attention", "type": "fp16", "heads": 14, "kv_heads": 2, "dim": 64,
         "requests": 1, "shortest": 4096, "longest": 4096, "nodes": 48, "block": 16, "tree": True},
        # a full serving batch on KV slots, a small tree each (block 0: one block per request)
        {"name": "attention-64x8-1500", "kind": "attention", "type": "fp16", "heads": 14, "kv_heads": 2, "dim": 64,
         "requests": 64, "shortest": 200, "longest": 1500, "nodes": 8, "block": 0, "tree": True},
        # plain decode of long rows over small blocks
        {"name": "attention-16x1-8192", "kind": "attention", "type": "fp16", "heads": 14, "kv_heads": 2, "dim": 64,
         "requests": 16, "shortest": 8192, "longest": 8192, "nodes": 1, "block": 16, "tree": False},
        # few users with contexts of any length (the first without any tree node but its own) in odd blocks
        {"name": "attention-5x23-777", "kind": "attention", "type": "bf16", "heads": 14, "kv_heads": 2, "dim": 64,
         "requests": 5, "shortest": 0, "longest": 777, "nodes": 23, "block": 24, "tree": True},
        # large trees over long documents, the widest heads
        {"name": "attention-8x64-16384", "kind": "attention", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "requests": 8, "shortest": 12000, "longest": 16384, "nodes": 64, "block": 32, "tree": True},
        # one user's next token
        {"name": "tables-1x1", "kind": "tables", "requests": 1, "shortest": 300, "longest": 300, "rows": 1,
         "block": 16, "tree": False, "admit": False},
        # a serving batch's next trees
        {"name": "tables-64x16", "kind": "tables", "requests": 64, "shortest": 200, "longest": 2000, "rows": 16,
         "block": 16, "tree": True, "admit": False},
        # prompts are admitted, and the requests end
        {"name": "tables-admit-256x2048", "kind": "tables", "requests": 256, "shortest": 0, "longest": 0,
         "rows": 2048, "block": 16, "tree": False, "admit": True},
        # a full serving batch on KV slots
        {"name": "commit-64x8", "kind": "commit", "type": "fp16", "layers": 24, "kv_heads": 2, "dim": 64,
         "requests": 64, "shortest": 20, "longest": 200, "nodes": 8, "block": 0},
        # large trees of a few users, a cache of more and wider heads
        {"name": "commit-4x64", "kind": "commit", "type": "bf16", "layers": 32, "kv_heads": 8, "dim": 128,
         "requests": 4, "shortest": 100, "longest": 700, "nodes": 64, "block": 16},
    ]


def _log(rng, low: int, high: int) -> int:
    """A size between ``low`` and ``high``, spread over the logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng) -> dict:
    kind = rng.choice(["attention"] * 6 + ["tables"] * 2 + ["commit"] * 2)
    if kind == "tables":
        requests, admit = _log(rng, 1, 500), rng.random() < 0.4
        longest = 0 if admit else _log(rng, 1, 8000)
        return {"kind": kind, "requests": requests, "shortest": longest // rng.choice((1, 2, 5)), "longest": longest,
                "rows": _log(rng, 2, min(2048, 400000 // requests)) if admit else _log(rng, 1, 64),
                "block": rng.choice((16, 32, 64, 24)), "tree": not admit and rng.random() < 0.6, "admit": admit}
    heads, kv_heads, dim = rng.choice(((14, 2, 64), (14, 2, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128)))
    kind_type, nodes = rng.choice(("fp16", "bf16")), _log(rng, 1, 64)
    block = rng.choice((0, 16, 32, 64, 24))
    if kind == "commit":
        requests, longest = _log(rng, 1, 64), _log(rng, 1, 300)
        return {"kind": kind, "type": kind_type, "layers": rng.choice((2, 12, 24)), "kv_heads": kv_heads, "dim": dim,
                "requests": requests, "shortest": longest // rng.choice((1, 2, 5)), "longest": longest, "nodes": nodes,
                "block": block}
    requests = _log(rng, 1, 64)
    longest = _log(rng, 1, min(32768, 1_000_000 // (requests * kv_heads * dim // 128)))
    return {"kind": kind, "type": kind_type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "requests": requests,
            "shortest": longest // rng.choice((1, 2, 5)), "longest": longest,
            "nodes": min(nodes, max(1, 8192 // (requests * 8))), "block": block, "tree": rng.random() < 0.7}


def _ragged(count: int, shortest: int, longest: int) -> list[int]:
    """Sizes from ``shortest`` to ``longest`` in no particular order; the first is the longest."""
    return [longest - int((longest - shortest) * ((i * 0.618034) % 1.0)) for i in range(count)]


def _sizes(case: dict) -> tuple[list[int], list[int], int]:
    """(cached tokens per request, new rows per request, tokens per block)"""
    lengths = _ragged(case["requests"], case["shortest"], case["longest"])
    if case["shortest"] < case["longest"] and case["requests"] > 1:
        lengths[1] = case["shortest"]
    most = case.get("nodes", case.get("rows"))
    new = _ragged(case["requests"], 1 + most // 2, most)
    return lengths, new, case["block"] or -(-(case["longest"] + most) // 64) * 64


# ---- inputs ------------------------------------------------------------------------------
def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(new: list[int]) -> list[int]:
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _node_numbers(new: list[int]) -> torch.Tensor:
    """For every row, the number of its node in its tree."""
    starts = _ints(_starts(new)[:-1]).long()
    counts = _ints(new).long()
    return torch.arange(sum(new), device=DEVICE) - torch.repeat_interleave(starts, counts, output_size=sum(new))


def _parents(new: list[int], gen) -> torch.Tensor:
    """A parent among the four nodes before each (-1: node 0 has none)."""
    node = _node_numbers(new)
    back = 1 + (torch.rand(node.numel(), device=DEVICE, generator=gen) * node.clamp(max=4)).floor().long()
    return (node - back).clamp(min=-1).to(torch.int32)


def _block_tables(lengths, new, block, gen, spare: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Tables whose blocks lie in any order, and the ids that are left."""
    counts = [-(-(n + m) // block) for n, m in zip(lengths, new)]
    ids = torch.randperm(sum(counts) + spare, device=DEVICE, generator=gen).to(torch.int32)
    width = max(counts)
    place = _ints(_starts(counts)[:-1]).long()[:, None] + torch.arange(width, device=DEVICE)
    live = torch.arange(width, device=DEVICE) < _ints(counts)[:, None]
    return torch.where(live, ids[place.clamp(max=ids.numel() - 1)], 0).to(torch.int32), ids[sum(counts):]


def _tree_mask(parents: torch.Tensor, new: list[int]) -> torch.Tensor:
    """Bits of the nodes that every node sees (its ancestors and itself), 32 to a word."""
    most = max(new)
    reach = _ancestors(_padded(parents, new, most))
    words = -(-most // 32)
    reach = torch.nn.functional.pad(reach, (0, 32 * words - most))
    bits = (reach.view(len(new), most, words, 32).long() << torch.arange(32, device=DEVICE)).sum(-1)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    return bits[torch.arange(most, device=DEVICE) < _ints(new)[:, None]].contiguous()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    lengths, new, block = _sizes(case)
    state = {"kind": case["kind"], "block": block, "lengths": _ints(lengths), "most": max(new), "longest": max(lengths)}
    if case["kind"] == "tables":
        rows = sum(new)
        parents = _parents(new, gen)
        state.update(parents=parents if case["tree"] else None, new=_ints(new), max_rows=rows + 7, admit=case["admit"],
                     over=torch.full((len(new),), -1, dtype=torch.int32, device=DEVICE))
        tables, left = _block_tables(lengths, new, block, gen, spare=5)
        held = [-(-n // block) for n in lengths]
        # of the table, what the cached tokens fill is held; the rest is still in the ring, with the spare blocks
        columns = torch.arange(tables.shape[1], device=DEVICE)
        live = columns < _ints([-(-(n + m) // block) for n, m in zip(lengths, new)])[:, None]
        mine = columns < _ints(held)[:, None]
        free = torch.cat([tables[live & ~mine], left])
        ring = torch.zeros(sum(held) + free.numel(), dtype=torch.int32, device=DEVICE)
        ring[:free.numel()] = free
        state.update(tables=torch.where(mine, tables, 0).to(torch.int32), held=_ints(held),
                     pool=torch.cat([_ints([0, free.numel(), 0, 0]), ring]))
        return state
    dtype = TYPES[case["type"]]
    tables, left = _block_tables(lengths, new, block, gen, spare=2)
    blocks = int(sum(-(-(n + m) // block) for n, m in zip(lengths, new))) + 2
    state.update(tables=tables, row_start=_ints(_starts(new)), parents=_parents(new, gen))
    if case["kind"] == "attention":
        shape = (blocks, case["kv_heads"], block, case["dim"])
        state["k"], state["v"] = (torch.randn(shape, device=DEVICE, generator=gen, dtype=dtype) for _ in range(2))
        state["q"] = 1.5 * torch.randn(sum(new), case["heads"], case["dim"], device=DEVICE, generator=gen, dtype=dtype)
        state["mask"] = _tree_mask(state["parents"], new) if case["tree"] else None
        return state
    state["kv"] = torch.randn(case["layers"], 2, blocks, case["kv_heads"], block, case["dim"], device=DEVICE,
                              generator=gen, dtype=dtype)
    # the target agrees with the last child of four nodes in five
    rows = sum(new)
    tokens = torch.randint(0, VOCAB, (rows,), device=DEVICE, generator=gen)
    start_of = torch.arange(rows, device=DEVICE) - _node_numbers(new)
    child = torch.full((rows + 1,), -1, dtype=torch.long, device=DEVICE)
    parent_row = torch.where(state["parents"] < 0, rows, start_of + state["parents"])
    child.scatter_reduce_(0, parent_row, torch.arange(rows, device=DEVICE), "amax")
    agrees = (child[:rows] >= 0) & (torch.rand(rows, device=DEVICE, generator=gen) < 0.8)
    other = torch.randint(0, VOCAB, (rows,), device=DEVICE, generator=gen)
    state.update(tokens=tokens, targets=torch.where(agrees, tokens[child[:rows].clamp(min=0)], other))
    return state


# ---- plain forms -------------------------------------------------------------------------
def _padded(rows: torch.Tensor, new, most: int, fill: int = -1) -> torch.Tensor:
    """[requests, most]: the rows' values by request and node."""
    counts = new if isinstance(new, torch.Tensor) else _ints(new)
    starts = torch.cumsum(counts, 0) - counts
    node = torch.arange(most, device=DEVICE)
    place = (starts[:, None] + node).clamp(max=rows.numel() - 1)
    return torch.where(node < counts[:, None], rows[place], fill)


def _ancestors(parents: torch.Tensor) -> torch.Tensor:
    """[requests, n, n]: whether node j is node i or an ancestor of it (parents [requests, n], -1: none)."""
    n = parents.shape[1]
    node = torch.arange(n, device=DEVICE)
    reach = ((parents[:, :, None] == node) | (node[:, None] == node)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = ((reach @ reach) > 0).float()
    return reach > 0


def _plain_attention(s: dict) -> torch.Tensor:
    q, k, v, tables, block = s["q"], s["k"], s["v"], s["tables"].long(), s["block"]
    rows, heads, dim = q.shape
    kv_heads, start = k.shape[1], s["row_start"].long()
    new = start[1:] - start[:-1]
    requests, most = new.numel(), s["most"]
    node = torch.arange(most, device=DEVICE)
    live = node < new[:, None]
    row = (start[:-1, None] + node).clamp(max=rows - 1)
    # keys and values by position
    place = torch.arange(s["longest"] + most, device=DEVICE)
    at = tables[:, (place // block).clamp(max=tables.shape[1] - 1)]
    keys = k.transpose(1, 2)[at, place % block].float()          # [requests, places, kv heads, dim]
    values = v.transpose(1, 2)[at, place % block].float()
    # which of them a row sees
    length = s["lengths"].long()
    drafted = place - length[:, None]                              # number of the node that lies there
    if s["mask"] is None:
        sees = drafted[:, None] <= node[:, None]
    else:
        word = s["mask"][row].long()                               # [requests, most, words]
        number = drafted.clamp(min=0, max=32 * word.shape[2] - 1)[:, None].expand(-1, most, -1)
        sees = (word.gather(2, number // 32) >> (number % 32)) & 1 > 0
    sees = ((drafted < 0)[:, None] | sees) & (drafted < new[:, None])[:, None]
    queries = q[row].float().view(requests, most, kv_heads, heads // kv_heads, dim)
    score = torch.einsum("bnhgd,bshd->bhgns", queries, keys) * dim ** -0.5
    score = score.masked_fill(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    values = values.masked_fill((drafted >= new[:, None])[:, :, None, None], 0.0)
    out = torch.einsum("bhgns,bshd->bnhgd", weight, values)
    total = total.permute(0, 3, 1, 2, 4)
    out = torch.where(total > 0, out / total, 0.0).reshape(requests, most, heads, dim)
    return out[live].to(q.dtype)


def _plain_tables(s: dict, n_new: torch.Tensor):
    tables, held, pool, block = s["tables"], s["held"], s["pool"], s["block"]
    max_rows, most, parents = s["max_rows"], s["most"], s["parents"]
    requests, width = tables.shape
    length, ring = s["lengths"].long(), pool[4:]
    blocks = ring.numel()
    over, take = n_new < 0, n_new.clamp(min=0).long()
    want = (length + take + block - 1) // block
    need = torch.where(take > 0, (want - held).clamp(min=0), 0)
    head, count = pool[0].long(), pool[1].long()
    missing = need.sum() - count
    short = ((take > 0) & (want > width)).any()
    many = (take.sum() > max_rows) | (parents is not None and (take > most).any())
    status = torch.where(short, -1, torch.where(many, -2, missing.clamp(min=0)))
    fine = (status == 0).long()
    need, take = need * fine, take * fine
    # blocks that requests give back go behind those in the ring, new ones come from its head
    column = torch.arange(width, device=DEVICE)
    gone = torch.where(over, held, 0).long()
    back = (head + count + (torch.cumsum(gone, 0) - gone)[:, None] + column) % blocks
    back = torch.where(column < gone[:, None], back, blocks)
    older = ring.clone()
    ring.copy_(torch.cat([ring, ring[:1]]).scatter(0, back.view(-1), tables.view(-1))[:blocks])
    number = column - held[:, None]
    fresh = older[(head + (torch.cumsum(need, 0) - need)[:, None] + number) % blocks]
    tables.copy_(torch.where((number >= 0) & (number < need[:, None]), fresh, tables))
    held.copy_(torch.where(over, 0, held + need))
    pool[0] = (head + need.sum()) % blocks
    pool[1] = count - need.sum() + gone.sum()
    pool[3] = status
    # rows
    start = torch.nn.functional.pad(torch.cumsum(take, 0), (1, 0))
    row = torch.arange(max_rows, device=DEVICE)
    request = torch.searchsorted(start[1:], row, right=True).clamp(max=requests - 1)
    live = row < start[-1]
    node = row - start[request]
    place = length[request] + node
    slot = tables[request, (place // block).clamp(max=width - 1)].long() * block + place % block
    slot_map = torch.where(live, slot, -1)
    mask = None
    if parents is not None:
        padded = _padded(parents, take, most)
        reach = _ancestors(padded)[request, node.clamp(max=most - 1)] & live[:, None]
        node = reach.sum(-1) - 1
        words = -(-most // 32)
        bits = torch.nn.functional.pad(reach, (0, 32 * words - most)).view(max_rows, words, 32).long()
        bits = (bits << torch.arange(32, device=DEVICE)).sum(-1)
        mask = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    positions = torch.where(live, length[request] + node, 0).to(torch.int32)
    return start.to(torch.int32), slot_map, positions, mask


def _plain_commit(s: dict):
    kv, tables, block, start = s["kv"], s["tables"].long(), s["block"], s["row_start"].long()
    most, rows = s["most"], s["tokens"].numel()
    new = start[1:] - start[:-1]
    node = torch.arange(most, device=DEVICE)
    live = node < new[:, None]
    parents = _padded(s["parents"], new, most)
    tokens, targets = _padded(s["tokens"], new, most), _padded(s["targets"], new, most)
    right = (tokens == targets.gather(1, parents.clamp(min=0).long())) & (parents >= 0) & live
    # of siblings that are right, the first
    brothers = (parents[:, :, None] == parents[:, None, :]) & right[:, None, :] & (node[None, :] < node[:, None])
    right &= ~brothers.any(-1)
    right[:, 0] |= live[:, 0]
    reach = _ancestors(parents)
    kept = live & ~(reach & ~right[:, None, :]).any(-1)
    accepted = kept.sum(-1)
    path = torch.where(kept, node, most).sort(-1).values
    path = torch.where(node < accepted[:, None], path, -1)
    # (what is not moved is copied onto itself: row 0 never moves)
    moved = node < accepted[:, None]
    source = s["lengths"].long()[:, None] + torch.where(moved, path, 0)
    target = s["lengths"].long()[:, None] + torch.where(moved, node, 0)
    of, to = tables.gather(1, source // block).view(-1), tables.gather(1, target // block).view(-1)
    kv[:, :, to, :, target.view(-1) % block] = kv[:, :, of, :, source.view(-1) % block]
    last = (start[:-1] + path.amax(-1)).clamp(max=rows - 1)
    return path.to(torch.int32), accepted.to(torch.int32), s["targets"][last], (s["lengths"] + accepted).to(torch.int32), kv


# ---- one pass ----------------------------------------------------------------------------
def _kernels():
    importlib.import_module("__graft_entry__").load_package()
    return importlib.import_module("quic_cu_b200.kernels")


def _tables(s: dict, n_new: torch.Tensor):
    if not own:
        return _plain_tables(s, n_new)
    return _kernels().block_tables(s["tables"], s["held"], s["pool"], s["lengths"], n_new, s["block"], s["max_rows"],
                                   parents=s["parents"], max_new=s["most"])


def run(state: dict):
    s = state
    if s["kind"] == "tables":
        out = [_tables(s, s["new"])]
        if s["admit"]:
            out.append(_tables(s, s["over"]))
        return out, s["tables"], s["held"], s["pool"]
    if s["kind"] == "attention":
        if not own:
            return _plain_attention(s)
        return _kernels().tree_attn(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["row_start"], mask=s["mask"],
                                    max_new=s["most"], max_len=s["longest"])
    if not own:
        return _plain_commit(s)
    return (*_kernels().tree_commit(s["kv"], s["tables"], s["lengths"], s["row_start"], s["parents"], s["tokens"],
                                    s["targets"], s["most"]), s["kv"])


# ---- what a pass cannot do without -------------------------------------------------------
def work(case: dict) -> dict:
    lengths, new, block = _sizes(case)
    rows, cached = sum(new), sum(n + m for n, m in zip(lengths, new))
    blocks = sum(-(-(n + m) // block) for n, m in zip(lengths, new))
    if case["kind"] == "tables":
        before = sum(-(-n // block) for n in lengths)
        words = -(-max(new) // 32) if case["tree"] else 0
        # lengths, rows and blocks per request in, starts and blocks out; a slot (8) and a position (4) per row, its
        # parent and mask; a block is read in one place and written in another
        amount = 5 * 4 * len(new) + rows * 12 + rows * (4 + 4 * words if case["tree"] else 0) + 8 * (blocks - before)
        return {"bytes": amount + (8 * blocks if case["admit"] else 0), "flops": 0}
    if case["kind"] == "commit":
        # the tree and the tokens; the least that is moved is nothing: the path of a tree may be where it belongs
        return {"bytes": rows * (4 + 8 + 8) + len(new) * 24 + 4 * rows, "flops": 0}
    item = 2 * case["dim"]
    return {"bytes": cached * 2 * case["kv_heads"] * item + 2 * rows * case["heads"] * item + 4 * blocks,
            # every node sees the context and itself
            "flops": 4 * case["heads"] * case["dim"] * sum(m * (n + 1) for n, m in zip(lengths, new))}


# ---- in 64 bits --------------------------------------------------------------------------
def _walk(parents: list[int], i: int) -> list[int]:
    """Node i and its ancestors, from the root."""
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found[::-1]


def exact(case: dict, seed: int):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    lengths, new, block = _sizes(case)
    starts, tables, parents = _starts(new), s["tables"].cpu(), s["parents"].tolist()
    if case["kind"] == "commit":
        tokens, targets, kv = s["tokens"].tolist(), s["targets"].tolist(), s["kv"].double()
        after = kv.clone()
        for b, n in enumerate(new):
            tree, at = parents[starts[b]:starts[b] + n], 0
            for depth in range(n):
                source, target = lengths[b] + at, lengths[b] + depth
                after[:, :, int(tables[b, target // block]), :, target % block] = \
                    kv[:, :, int(tables[b, source // block]), :, source % block]
                nexts = [j for j in range(n) if tree[j] == at and tokens[starts[b] + j] == targets[starts[b] + at]]
                if not nexts:
                    break
                at = nexts[0]
        return None, None, None, None, after
    group, out = case["heads"] // case["kv_heads"], torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(new):
        ids = tables[b, : -(-(lengths[b] + n) // block)].to(DEVICE).long()
        q = s["q"][starts[b]:starts[b] + n].double()
        hidden = torch.ones(n, lengths[b] + n, dtype=torch.bool)
        hidden[:, :lengths[b]] = False
        tree = parents[starts[b]:starts[b] + n]
        for i in range(n):
            hidden[i, [lengths[b] + j for j in (_walk(tree, i) if case["tree"] else range(i + 1))]] = False
        hidden = hidden.to(DEVICE)
        for h in range(case["kv_heads"]):
            k, v = (s[name][ids, h].reshape(-1, case["dim"])[: lengths[b] + n].double() for name in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                logits = (q[:, g] @ k.T / case["dim"] ** 0.5).masked_fill_(hidden, -torch.inf)
                out[starts[b]:starts[b] + n, g] = torch.softmax(logits, -1) @ v
    return out
