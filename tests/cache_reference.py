"""Plain 64-bit implementations of the paged-cache operators, and random inputs for them."""
import math

import torch

CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rows_of(cache, scale):
    """[places, heads, dim] in 64 bits: the values that the cache's rows stand for."""
    x = cache.double().flatten(0, 1)
    return x if scale is None else x * scale.double().flatten(0, 1).unsqueeze(-1)


def attention(q, k, v, k_scale, v_scale, table, context, sees, live, scale):
    """(out, lse, spread, size): sees [batch, nodes, nodes]; live [batch]; spread is sum w |v| and size the
    largest scale * sum |q k|, the magnitudes that rounding errors go by."""
    batch, nodes, heads, dim = q.shape
    pages, page, kv, _ = k.shape
    group = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    spread, size = torch.zeros_like(out), torch.zeros_like(lse)
    kr, vr = rows_of(k, k_scale), rows_of(v, v_scale)
    for b in range(batch):
        places = table.shape[1] * page
        c = min(max(0, int(context[b])), places)
        n = min(int(live[b]), nodes)
        length = min(c + n, places)
        place = torch.arange(length, device=q.device)
        at = table[b, place // page].long() * page + place % page
        there = (at >= 0) & (at < pages * page)
        at = at.clamp(0, max(0, pages * page - 1))
        if n == 0 or length == 0:
            continue
        seen = there.expand(n, length).clone()
        seen[:, c:] &= sees[b, :n, :length - c].bool()
        some = seen.any(dim=1)
        for h in range(kv):
            o = slice(h * group, (h + 1) * group)
            qq, kk, vv = q[b, :n, o].double(), kr[at, h], vr[at, h]
            # Rows that nobody sees may hold anything.
            kk, vv = (torch.where(seen.any(dim=0)[:, None], x, 0.0) for x in (kk, vv))
            s = torch.where(seen[:, None, :], torch.einsum("ngd,ld->ngl", qq, kk) * scale, -math.inf)
            w = torch.where(some[:, None, None], torch.softmax(s, dim=2), 0.0)
            out[b, :n, o] = torch.einsum("ngl,ld->ngd", w, vv)
            lse[b, :n, o] = torch.logsumexp(s, dim=2)
            spread[b, :n, o] = torch.einsum("ngl,ld->ngd", w, vv.abs())
            size[b, :n, o] = torch.where(seen[:, None, :], torch.einsum("ngd,ld->ngl", qq.abs(), kk.abs()),
                                         0.0).amax(dim=2) * abs(scale)
    return out, lse, spread, size


def walk(logits, tokens, parents, uniforms, draft, race, temperature):
    """(count, path, said, logs) of one sequence, in 64 bits."""
    nodes = tokens.numel()
    vocab = logits.shape[1]
    path, said, logs = [], [], []
    at = 0
    while True:
        x = logits[at].double()
        x = torch.where(x.isnan(), -math.inf, x) / (temperature or 1.0)
        logp = torch.log_softmax(x, dim=0)
        p = logp.exp()
        r, best, taken = p, int(x.argmax()), None
        for c in range(at + 1, nodes):
            if int(parents[c]) != at:
                continue
            token = int(tokens[c])
            inside = 0 <= token < vocab
            if temperature == 0:
                hit = token == best
            else:
                q = draft[at].double() if draft is not None else None
                chance = (float(q[token]) if draft is not None else 1.0) if inside else 1.0
                hit = inside and float(uniforms[c]) * chance < float(r[token])
            if hit:
                taken = c
                break
            if temperature != 0:
                if draft is not None:
                    r = (r - q).clamp_min(0)
                else:
                    r = r.clone()
                    if inside:
                        r[token] = 0
                r = r / r.sum() if float(r.sum()) > 0 else p
        if taken is None:
            last = best if temperature == 0 else int((r * race.double()).argmax())
            said.append(last)
            logs.append(float(logp[last]))
            return len(path), path, said, logs
        path.append(taken)
        said.append(int(tokens[taken]))
        logs.append(float(logp[said[-1]]))
        at = taken


def random_cache(gen, pages, page, heads, dim, dtype, device="cuda"):
    """[k, v, k_scale, v_scale] of rows of about unit variance."""
    shape, out = (pages, page, heads, dim), []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device=device)
        if dtype == torch.int8:
            out.append((x * 42).round().clamp(-127, 127).to(dtype))
        elif dtype == torch.float8_e4m3fn:
            out.append((x * 130).clamp(-448, 448).to(dtype))
        else:
            out.append(x.to(dtype))
    for _ in range(2):
        size = {torch.int8: 42.0, torch.float8_e4m3fn: 130.0}.get(dtype)
        out.append(None if size is None else
                   torch.exp(0.5 * torch.randn(shape[:3], generator=gen, device=device)) / size)
    return out


def random_tree(rng, nodes):
    """Parents of a random tree and which nodes each node sees: itself and its ancestors."""
    parents = [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, nodes)]
    sees = torch.zeros(nodes, nodes, dtype=torch.bool)
    for i in range(nodes):
        j = i
        while j >= 0:
            sees[i, j] = True
            j = parents[j]
    return parents, sees
