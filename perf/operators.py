"""Measured cases of the paged-cache operators: cache_write, cache_read, tree_attention, verify_drafts.

One step of a serving loop that drafts tokens: the rows of the drafted tokens are quantised into a paged cache
(cache_write; cache_read gives rows back), the drafted tree attends to the cache (tree_attention, with the
single token as the tree of one node), and the drafts are held against the target's probabilities
(verify_drafts).  `run` computes them with elementary torch operations in 32 bits where `own` is false, and with
this library's kernels where it is true.
"""
import math
import os
import sys

import torch

own = False

SOURCE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CACHE = {"bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_MAX = {"i8": 127.0, "e4m3": 448.0}  # largest code of a quantised cache
LEAST_ROW = 2.0 ** -100  # a row whose largest magnitude is below this is stored as zeros
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1, "e4m3": 1}


def listed():
    return [
        # One decode step of a small batch: the rows of one new token per sequence, where the call's latency counts.
        dict(name="write-decode", op="write", rows=8, heads=8, dim=128, page=16, pages=512, source="bf16", cache="i8"),
        # The drafted trees of a batch, an odd number of rows and of heads, 16-bit rows kept in 16 bits.
        dict(name="write-drafts", op="write", rows=777, heads=5, dim=96, page=32, pages=128, source="f16", cache="f16"),
        # A long prompt written at once.
        dict(name="write-prompt", op="write", rows=32768, heads=8, dim=128, page=64, pages=640, source="bf16",
             cache="e4m3"),
        # A few rows back, as when an accepted branch moves to the places that follow the context.
        dict(name="read-branch", op="read", rows=61, heads=8, dim=128, page=16, pages=512, source="f32", cache="i8"),
        # The cache of whole sequences back in 16 bits, to be stored or sent elsewhere.
        dict(name="read-sequences", op="read", rows=50001, heads=8, dim=128, page=64, pages=1024, source="bf16",
             cache="e4m3"),
        # One token of one sequence after a short context: the smallest call of a decode loop.
        dict(name="attend-one", op="attend", batch=1, nodes=1, kv_heads=8, group=4, dim=128, page=16, context=1000,
             ragged=False, branch=1, source="bf16", cache="bf16"),
        # One token each of a ragged batch over an 8-bit cache: ordinary decoding.
        dict(name="attend-decode", op="attend", batch=32, nodes=1, kv_heads=8, group=4, dim=128, page=64, context=8192,
             ragged=True, branch=1, source="bf16", cache="i8"),
        # Small trees of a batch, odd sizes throughout.
        dict(name="attend-tree", op="attend", batch=7, nodes=13, kv_heads=5, group=3, dim=96, page=24, context=4099,
             ragged=True, branch=2, source="f16", cache="e4m3"),
        # A chain of drafted tokens after a very long context.
        dict(name="attend-long", op="attend", batch=1, nodes=8, kv_heads=8, group=4, dim=128, page=64, context=131072,
             ragged=False, branch=1, source="bf16", cache="i8"),
        # Wide trees with many query heads to a cache head: products bound it, not the cache.
        dict(name="attend-wide", op="attend", batch=4, nodes=64, kv_heads=8, group=8, dim=128, page=64, context=16384,
             ragged=True, branch=3, source="bf16", cache="bf16"),
        # A short chain against its drafter's probabilities.
        dict(name="verify-chain", op="verify", batch=4, nodes=5, vocab=32003, branch=1, source="bf16", draft=True,
             temperature=0.8),
        # A batch of trees whose drafted tokens are the drafter's first choices.
        dict(name="verify-tree", op="verify", batch=32, nodes=32, vocab=128256, branch=3, source="bf16", draft=False,
             temperature=1.0),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["write", "read", "attend", "attend", "attend", "verify"])
    if op in ("write", "read"):
        rows = spread(1, 32768)
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        return dict(op=op, rows=rows, heads=rng.randint(1, 8), dim=rng.choice([64, 80, 96, 128]), page=page,
                    pages=rows // page + rng.randint(2, 300), source=rng.choice(["bf16", "f16", "f32"]),
                    cache=rng.choice(["i8", "e4m3", "bf16", "f16"]))
    if op == "attend":
        source = rng.choice(["bf16", "f16"])
        case = dict(op="attend", batch=spread(1, 32), nodes=rng.choice([1, 1, spread(2, 64), spread(2, 64)]),
                    kv_heads=rng.randint(1, 8), group=rng.choice([1, 2, 3, 4, 5, 6, 8]),
                    dim=rng.choice([64, 80, 96, 128, 128]), page=rng.choice([8, 16, 24, 32, 64, 128]),
                    context=spread(16, 131072), ragged=rng.random() < 0.7, branch=rng.choice([1, 2, 3, 4]),
                    source=source, cache=rng.choice(["i8", "e4m3", source]))
        top = next(c for c in listed() if c["name"] == "attend-wide")
        limit = top["batch"] * top["context"] * top["kv_heads"]  # cache rows, and products below
        while (case["batch"] * case["context"] * case["kv_heads"] > limit
               or work(case)["flops"] > work(top)["flops"]):
            if case["batch"] > 1 and rng.random() < 0.5:
                case["batch"] -= (case["batch"] + 1) // 2
            else:
                case["context"] = case["context"] * 2 // 3 + 1
        return case
    case = dict(op="verify", batch=spread(1, 32), nodes=spread(2, 48), vocab=spread(2000, 200000),
                branch=rng.choice([1, 1, 2, 3]), source=rng.choice(["bf16", "f16", "f32"]), draft=rng.random() < 0.5,
                temperature=rng.choice([0.0, 0.6, 1.0, 1.3]))
    while case["batch"] * case["nodes"] * case["vocab"] > 32 * 32 * 128256 // (4 if case["draft"] else 2):
        if rng.random() < 0.5:
            case["vocab"] = case["vocab"] * 2 // 3 + 1
        else:
            case["batch"] -= case["batch"] // 3
            case["nodes"] -= case["nodes"] // 4
    return case


# ---- what follows from a case alone ----------------------------------------------------------------------------

def contexts(case):
    """Committed tokens of each sequence: a ragged batch falls off evenly to a quarter of the longest."""
    b, longest = case["batch"], case["context"]
    if not case["ragged"]:
        return [longest] * b
    return [max(1, longest - (longest * 3 * ((5 * i) % b)) // (4 * b)) for i in range(b)]


def parent_list(nodes, branch):
    """The drafted tree: node 0 is the root, every node has `branch` children while there are nodes (1: a chain)."""
    return [-1] + [(i - 1) // branch for i in range(1, nodes)]


def branches(case):
    """For each sequence the nodes of the branch that its target agrees with, the root first."""
    parents, n = parent_list(case["nodes"], case["branch"]), case["nodes"]
    found = []
    for b in range(case["batch"]):
        leaf = n - 1 - b % max(1, n // 2)
        path = [leaf]
        while path[-1] > 0:
            path.append(parents[path[-1]])
        path.reverse()
        found.append(path[:1 + (5 * b + 2) % len(path)])
    return found


def work(case):
    if case["op"] in ("write", "read"):
        values = 2 * case["rows"] * case["heads"] * case["dim"]
        scales = 2 * case["rows"] * case["heads"] * 4 if case["cache"] in CODE_MAX else 0
        source, code = SIZE[case["source"]], SIZE[case["cache"]]
        if case["op"] == "read":
            return {"bytes": values * (source + code) + scales + 8 * case["rows"], "flops": values}
        # The written rows come back in the pass, so they cross memory once more in each form.
        return {"bytes": 2 * (values * (source + code) + scales + 8 * case["rows"]), "flops": 5 * values}
    if case["op"] == "attend":
        rows = sum(c + case["nodes"] for c in contexts(case)) * case["kv_heads"]
        per_row = 2 * case["dim"] * SIZE[case["cache"]] + (8 if case["cache"] in CODE_MAX else 0)
        queries = case["batch"] * case["nodes"] * case["kv_heads"] * case["group"]
        return {"bytes": rows * per_row + queries * (2 * case["dim"] * SIZE[case["source"]] + 4),
                "flops": 4 * rows * case["nodes"] * case["group"] * case["dim"]}
    visited = sum(len(path) for path in branches(case))
    ends = case["batch"] * case["vocab"] * 4  # the race's row, and the drafter's where a child was turned down
    ends *= 0 if case["temperature"] == 0 else 2 if case["draft"] else 1
    return {"bytes": visited * case["vocab"] * SIZE[case["source"]] + ends, "flops": 4 * visited * case["vocab"]}


# ---- inputs ------------------------------------------------------------------------------------------------------

def seeded(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def row_values(gen, rows, heads, dim):
    """Rows as keys are: a few channels carry much more than the others."""
    channel = torch.exp(0.5 * normal(gen, 1, heads, dim))
    return normal(gen, rows, heads, dim) * channel


def filled_cache(gen, case, pages):
    """K and V of a cache in use: every row holds values and, where quantised, its scale."""
    shape, kind = (pages, case["page"], case.get("heads") or case["kv_heads"], case["dim"]), case["cache"]
    out = []
    for _ in range(2):
        if kind == "i8":
            code = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
        elif kind == "e4m3":
            code = (130.0 * normal(gen, *shape)).clamp_(-448, 448).to(torch.float8_e4m3fn)
        else:
            code = normal(gen, *shape).to(CACHE[kind])
        out.append(code)
    for code in out[:2]:
        if kind in CODE_MAX:
            size = 73.0 if kind == "i8" else 130.0  # a code's usual magnitude: rows of about unit variance
            out.append(torch.exp(0.3 * normal(gen, *shape[:3])) / size)
        else:
            out.append(None)
    return dict(zip(("k", "v", "k_scale", "v_scale"), out))


def prepare(case, seed):
    gen = seeded(seed)
    op, source = case["op"], SOURCE[case["source"]]
    if op in ("write", "read"):
        rows, places = case["rows"], case["page"] * case["pages"]
        # Whole pages in no order, filled from their starts, as an allocator gives them out.
        order = torch.randperm(case["pages"], generator=gen, device="cuda")
        at = torch.arange(rows, device="cuda")
        slots = order[at // case["page"]] * case["page"] + at % case["page"]
        if rows > 16:  # padding rows of a batch have no place
            slots[torch.randint(0, rows, (rows // 16,), generator=gen, device="cuda")] = -1
        state = dict(case=case, slots=slots, **filled_cache(gen, case, case["pages"]))
        assert int(slots.max()) < places
        if op == "write":
            state["key"] = row_values(gen, rows, case["heads"], case["dim"]).to(source)
            state["value"] = row_values(gen, rows, case["heads"], case["dim"]).to(source)
        return state
    if op == "attend":
        b, t = case["batch"], case["nodes"]
        lengths = contexts(case)
        width = -(-(max(lengths) + t) // case["page"])
        pages = b * width
        state = dict(case=case, **filled_cache(gen, case, pages))
        order = torch.randperm(pages, generator=gen, device="cuda")
        state["page_table"] = order.reshape(b, width).to(torch.int32)
        state["context"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        parents = parent_list(t, case["branch"])
        sees = [[False] * t for _ in range(t)]
        for i in range(t):
            j = i
            while j >= 0:
                sees[i][j] = True
                j = parents[j]
        state["mask"] = torch.tensor(sees, device="cuda").expand(b, t, t).contiguous()
        q = normal(gen, b, t, case["kv_heads"] * case["group"], case["dim"])
        state["q"] = (1.5 * q).to(source)
        return state
    b, t, vocab = case["batch"], case["nodes"], case["vocab"]
    parents = parent_list(t, case["branch"])
    state = dict(case=case, parents=torch.tensor(parents, dtype=torch.int32, device="cuda").expand(b, t).contiguous())
    # Siblings hold different tokens: a stride through the vocabulary from a start of the seed's choosing.
    start = torch.randint(0, vocab, (b, 1), generator=gen, device="cuda")
    tokens = (start + torch.arange(t, device="cuda") * (vocab // t)) % vocab
    state["tokens"] = tokens.to(torch.int32)
    logits = torch.empty(b, t, vocab, dtype=source, device="cuda").normal_(generator=gen).mul_(2.0)
    size = math.log(vocab) + 2.0  # of the log of a row's sum
    sequence, node, child = [], [], []
    for i, path in enumerate(branches(case)):
        for above, below in zip(path, path[1:]):
            sequence.append(i), node.append(above), child.append(below)
    if sequence:
        sequence, node, child = (torch.tensor(v, device="cuda") for v in (sequence, node, child))
        logits[sequence, node, tokens[sequence, child]] = size + 4.0
    state["logits"] = logits
    state["uniforms"] = torch.rand(b, t, generator=gen, device="cuda")
    state["race"] = torch.empty(b, vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-30).reciprocal_()
    state["draft"] = None
    if case["draft"]:
        q = normal(gen, b, t, vocab)
        above = state["parents"][:, 1:].long()
        q[torch.arange(b, device="cuda")[:, None], above, tokens[:, 1:]] = size + 2.0  # as they came from the drafter
        state["draft"] = torch.softmax(q, dim=2)
    return state


# ---- the plain forms: elementary operations in 32 bits ----------------------------------------------------------

def plain_rows(state, flat, inside, out_type):
    """Rows `flat` of the cache, K and V, as the values they stand for; rows that are not `inside` are zeros."""
    got = []
    for name in ("k", "v"):
        cache, scale = state[name], state[name + "_scale"]
        rows = cache.view(-1, *cache.shape[2:])[flat].float()
        if scale is not None:
            rows = rows * scale.view(-1, scale.shape[2])[flat].unsqueeze(2)
        got.append(torch.where(inside[:, None, None], rows, 0.0).to(out_type))
    return got


def plain_write(state):
    slots, kind = state["slots"], state["case"]["cache"]
    inside = slots >= 0
    flat = slots[inside]
    for name, rows in (("k", state["key"]), ("v", state["value"])):
        cache = state[name]
        x = rows[inside].float()
        if kind in CODE_MAX:
            top = CODE_MAX[kind]
            most = x.abs().amax(dim=2, keepdim=True)
            fine = torch.isfinite(most)
            live = fine & (most >= LEAST_ROW)
            code = torch.where(live, x * (torch.full_like(most, top) / most), 0.0)
            code = code.round().to(torch.int8) if kind == "i8" else code.clamp(-top, top).to(torch.float8_e4m3fn)
            scale = torch.where(live, most * (1.0 / top), torch.where(fine, 0.0, torch.nan))
            held = state[name + "_scale"]
            held.view(-1, held.shape[2])[flat] = scale.squeeze(2)
            cache.view(torch.int8).view(-1, *cache.shape[2:])[flat] = code.view(torch.int8)
        else:
            cache.view(-1, *cache.shape[2:])[flat] = x.to(cache.dtype)
    return plain_rows(state, slots.clamp_min(0), inside, SOURCE[state["case"]["source"]])


def plain_read(state):
    slots = state["slots"]
    return plain_rows(state, slots.clamp_min(0), slots >= 0, SOURCE[state["case"]["source"]])


def plain_attend(state):
    q, table, context, mask = state["q"], state["page_table"].long(), state["context"].long(), state["mask"]
    b, t, heads, dim = q.shape
    kv = state["k"].shape[2]

    def laid_out(name):  # [B, kv, L, dim]
        rows = state[name][table].float()
        if state[name + "_scale"] is not None:
            rows = rows * state[name + "_scale"][table].unsqueeze(4)
        return rows.view(b, -1, kv, dim).transpose(1, 2)

    k, v = laid_out("k"), laid_out("v")
    length = k.shape[2]
    # [B, kv, T * group, dim]: the query heads of a cache head together.
    rows = q.float().view(b, t, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, dim)
    scores = torch.matmul(rows, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    place = torch.arange(length, device=q.device)[None, :] - context[:, None]  # [B, L]: negative in the context
    drafted = (place >= 0) & (place < t)
    seen = mask.gather(2, place.clamp(0, t - 1)[:, None, :].expand(b, t, length))
    seen = (place < 0)[:, None, :] | (seen & drafted[:, None, :])  # [B, T, L]
    seen = seen[:, None, :, None, :].expand(b, kv, t, heads // kv, length).reshape(b, kv, -1, length)
    scores = scores.masked_fill(~seen, -torch.inf)
    most = scores.amax(dim=3, keepdim=True)
    weights = torch.exp(scores - most)
    total = weights.sum(dim=3, keepdim=True)
    out = torch.matmul(weights, v) / total
    lse = (most + torch.log(total)).squeeze(3)
    out = out.view(b, kv, t, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(b, t, heads, dim)
    lse = lse.view(b, kv, t, heads // kv).permute(0, 2, 1, 3).reshape(b, t, heads)
    return out.to(q.dtype), lse


def plain_verify(state):
    case, logits, draft = state["case"], state["logits"], state["draft"]
    tokens, parents = state["tokens"].long(), state["parents"].long()
    greedy = case["temperature"] == 0
    b, t, vocab = logits.shape
    x = logits.float()
    if not greedy:
        x = x * (1.0 / case["temperature"])
    most = x.amax(dim=2, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(dim=2, keepdim=True)
    logp = x - (most + torch.log(total))
    batch = torch.arange(b, device=x.device)
    at = torch.zeros(b, dtype=torch.long, device=x.device)
    count = torch.zeros(b, dtype=torch.long, device=x.device)
    path = torch.full((b, t), -1, dtype=torch.long, device=x.device)
    said = torch.full((b, t), -1, dtype=torch.long, device=x.device)
    logs = torch.zeros(b, t, device=x.device)
    p = e / total
    left = p[:, 0].clone()
    best = x.argmax(dim=2)
    # A node is tried only where its parent was taken and its elder siblings were not, so the nodes follow one
    # another; every step is over the whole batch.
    for i in range(1, t):
        tried = parents[:, i] == at
        token = tokens[:, i]
        if greedy:
            taken = tried & (best[batch, at] == token)
        else:
            q = draft[batch, at] if draft is not None else None
            qx = q[batch, token] if draft is not None else 1.0
            taken = tried & (state["uniforms"][:, i] * qx < left[batch, token])
            rest = (left - q).clamp_min(0.0) if draft is not None else left.scatter(1, token[:, None], 0.0)
            mass = rest.sum(dim=1, keepdim=True)
            rest = torch.where(mass > 0, rest / mass, p[batch, at])
            left = torch.where(taken[:, None], p[:, i], torch.where(tried[:, None], rest, left))
        slot = torch.where(taken, count, t - 1)
        logs[batch, slot] = torch.where(taken, logp[batch, at, token], logs[batch, slot])
        path[batch, slot] = torch.where(taken, i, path[batch, slot])
        said[batch, slot] = torch.where(taken, token, said[batch, slot])
        count = count + taken
        at = torch.where(taken, i, at)
    last = best[batch, at] if greedy else (left * state["race"]).argmax(dim=1)
    logs[batch, count] = logp[batch, at, last]
    said[batch, count] = last
    return count.to(torch.int32), path.to(torch.int32), said.to(torch.int32), logs


# ---- one pass ----------------------------------------------------------------------------------------------------

def framework():
    import_path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "t4a-cuda-kernels_b200")
    if import_path not in sys.path:
        sys.path.insert(0, import_path)
    import t4a_b200
    return t4a_b200


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"write": plain_write, "read": plain_read, "attend": plain_attend, "verify": plain_verify}[op](state)
    t4 = framework()
    if op in ("write", "read"):
        if op == "write":
            t4.cache_write(state["key"], state["value"], state["k"], state["v"], state["slots"],
                           k_scale=state["k_scale"], v_scale=state["v_scale"])
        return t4.cache_read(state["k"], state["v"], state["slots"], SOURCE[state["case"]["source"]],
                             k_scale=state["k_scale"], v_scale=state["v_scale"])
    if op == "attend":
        return t4.tree_attention(state["q"], state["k"], state["v"], state["page_table"], state["context"],
                                 mask=state["mask"], k_scale=state["k_scale"], v_scale=state["v_scale"])
    return t4.verify_drafts(state["logits"], state["tokens"], state["parents"], uniforms=state["uniforms"],
                            draft=state["draft"], race=state["race"], temperature=state["case"]["temperature"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact_write(state):
    kind, out = state["case"]["cache"], []
    for name in ("key", "value"):
        x = state[name].double()
        if kind == "i8":
            step = x.abs().amax(dim=2, keepdim=True) / 127
            x = torch.round(x / step) * step
        elif kind == "e4m3":
            step = x.abs().amax(dim=2, keepdim=True) / 448
            y = x / step
            # Four significant bits down to 2^-6, steps of 2^-9 below.
            unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
            x = torch.round(y / unit) * unit * step
        else:
            x = x.to(CACHE[kind]).double()
        out.append(x * (state["slots"] >= 0)[:, None, None])
    return out


def exact_read(state):
    out = []
    for name in ("k", "v"):
        x = state[name].double().flatten(0, 1)
        if state[name + "_scale"] is not None:
            x = x * state[name + "_scale"].double().flatten(0, 1).unsqueeze(-1)
        x = torch.cat([x, torch.zeros_like(x[:1])])  # the slot -1 is the row of zeros at the end
        out.append(x[state["slots"]])
    return out


def exact_attend(state):
    q, kv = state["q"].double(), state["k"].shape[2]
    group = q.shape[2] // kv
    out, lse = torch.zeros_like(q), q.new_zeros(q.shape[:3])
    for b, context in enumerate(state["context"].tolist()):
        t = q.shape[1]
        pages = state["page_table"][b].long()
        rows = {}
        for name in ("k", "v"):
            x = state[name][pages].double()
            if state[name + "_scale"] is not None:
                x = x * state[name + "_scale"][pages].double()[..., None]
            rows[name] = x.flatten(0, 1)[:context + t]
        for h in range(kv):
            queries = q[b, :, h * group:(h + 1) * group]
            s = torch.einsum("tgd,ld->tgl", queries, rows["k"][:, h]) / math.sqrt(q.shape[3])
            s[:, :, context:] = torch.where(state["mask"][b][:, None, :], s[:, :, context:], -math.inf)
            lse[b, :, h * group:(h + 1) * group] = torch.logsumexp(s, dim=2)
            out[b, :, h * group:(h + 1) * group] = torch.einsum("tgl,ld->tgd", torch.softmax(s, dim=2), rows["v"][:, h])
    return [out, lse]


def exact_verify(state):
    case = state["case"]
    temperature = case["temperature"] or 1.0
    b, t, _ = state["logits"].shape
    logs = torch.zeros(b, t, dtype=torch.float64, device="cuda")
    for i in range(b):
        parents, tokens = state["parents"][i].tolist(), state["tokens"][i].tolist()
        u = state["uniforms"][i].double().tolist()
        at, length = 0, 0
        while True:
            logp = torch.log_softmax(state["logits"][i, at].double() / temperature, dim=0)
            p, taken = logp.exp(), None
            for child in (c for c in range(t) if parents[c] == at):
                x = tokens[child]
                if case["temperature"] == 0:
                    if int(logp.argmax()) == x:
                        taken = child
                        break
                    continue
                if state["draft"] is not None:
                    q = state["draft"][i, at].double()
                    if u[child] * float(q[x]) < float(p[x]):
                        taken = child
                        break
                    p = torch.relu(p - q)
                else:
                    if u[child] < float(p[x]):
                        taken = child
                        break
                    p = p.clone()
                    p[x] = 0
                p = p / p.sum()
            if taken is None:
                break
            logs[i, length] = logp[tokens[taken]]
            at, length = taken, length + 1
        last = logp.argmax() if case["temperature"] == 0 else (p * state["race"][i].double()).argmax()
        logs[i, length] = logp[last]
    return [None, None, None, logs]


def exact(case, seed):
    return {"write": exact_write, "read": exact_read, "attend": exact_attend, "verify": exact_verify}[case["op"]](
        prepare(case, seed))
