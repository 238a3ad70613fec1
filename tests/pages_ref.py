"""The operators over a cache in pages in plain float64 and plain loops, on the CPU, for their tests."""
import math

import torch

BLOCK = 64
TOP = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ROWS = {"fp32": torch.float32, "bf16": torch.bfloat16}
E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest(u, cache):
    """the nearest of the type's values, half to even, none past its largest"""
    u = u.clamp(-TOP[cache], TOP[cache])
    if cache == "int8":
        return torch.round(u)
    mid = (E4M3[1:] + E4M3[:-1]) / 2
    i = torch.bucketize(u.abs().contiguous(), mid)
    tie = (i < 126) & (u.abs() == mid[i.clamp(max=125)]) & (i % 2 == 1)
    return torch.where(u.isnan(), u, torch.sign(u) * E4M3[i + tie.long()])


class Pool:
    """Pages in float64: codes [layers, pages, heads, blocks, 64, head size] of K and V, scales [layers, pages, heads, blocks]."""

    def __init__(self, layers, pages, h, page, hs, cache, g=None):
        shape = (layers, pages, h, page // BLOCK)
        self.cache, self.page, self.h, self.hs, self.pages = cache, page, h, hs, pages
        self.code, self.scale = [], []
        for _ in range(2):
            if g is None:
                c, s = torch.zeros(shape + (BLOCK, hs), dtype=torch.float64), torch.zeros(shape)
            else:
                c = nearest(torch.randn(shape + (BLOCK, hs), generator=g, dtype=torch.float64) * TOP[cache] / 4, cache)
                s = torch.exp(torch.randn(shape, generator=g)) * 0.02
            self.code.append(c)
            self.scale.append(s)

    def tensors(self, layout="plain", device="cuda", layers=True):
        """K, V and their scales as the operators take them; layouts: contiguous, heads before pages, a part of a wider pool"""
        out = []
        for side in range(2):
            c = self.code[side]
            layers_, pages, h, nb = c.shape[:4]
            c = c.reshape(layers_, pages, h, self.page, self.hs) if side == 0 else c.transpose(-1, -2)
            out.append(place(c.float().to(TYPES[self.cache]), layout, device))
        out += [place(s, layout, device) for s in self.scale]
        return out if layers else [x[0] for x in out]

    def values(self, side, layer=0):
        """[pages, heads, page, head size]"""
        c, s = self.code[side][layer], self.scale[side][layer]
        return (c * s.double()[..., None, None]).reshape(self.pages, self.h, self.page, self.hs)

    def compare(self, tensors, only=None):
        """whether the operators' tensors hold these codes and scales (of the pages in `only`)"""
        for side in range(2):
            c = tensors[side].view(torch.int8).cpu().view(TYPES[self.cache]).double()
            c = c if c.dim() == (5 if side == 0 else 6) else c.unsqueeze(0)
            c = c.reshape(self.code[side].shape) if side == 0 else c.transpose(-1, -2)
            s = tensors[2 + side].cpu()
            s = s if s.dim() == 4 else s.unsqueeze(0)
            pick = slice(None) if only is None else only
            assert same(c[:, pick], self.code[side][:, pick]), ("codes", side)
            assert same(s[:, pick], self.scale[side][:, pick]), ("scales", side)


def place(x, layout, device):
    bits = x.view(torch.int8) if x.element_size() == 1 else x
    if layout == "heads":  # heads before pages
        y = bits.transpose(1, 2).contiguous().to(device).transpose(1, 2)
    elif layout == "wide":  # every other page and head of a larger pool
        y = torch.full((x.shape[0], 2 * x.shape[1], 2 * x.shape[2]) + tuple(x.shape[3:]), 55, dtype=bits.dtype, device=device)
        y = y[:, 1::2, ::2]
        y.copy_(bits)
    else:
        y = bits.contiguous().to(device)
    return y.view(x.dtype) if x.element_size() == 1 else y


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def write(pool, k_rows, v_rows, table, pos, n, path=None, refs=None, layer=0):
    """rows [b, t, h, hs] into the pool, a block of a head after the other"""
    per, t = len(table[0]), k_rows.shape[1]
    for side, rows in enumerate((k_rows, v_rows)):
        for b in range(len(table)):
            blocks = {}
            for i in range(min(max(n[b], 0), t)):
                p = pos[b] + i
                if 0 <= p < per * pool.page:
                    src = i if path is None else path[b][i]
                    row = rows[b, src].double() if 0 <= src < t else torch.zeros(pool.h, pool.hs, dtype=torch.float64)
                    blocks.setdefault(p // BLOCK, []).append((p % BLOCK, row))
            for at, new in blocks.items():
                pg, blk = table[b][at * BLOCK // pool.page], at * BLOCK % pool.page // BLOCK
                if not 0 <= pg < pool.pages or (refs is not None and refs[pg] != 1):
                    continue
                for h in range(pool.h):
                    code, scale = pool.code[side][layer, pg, h, blk], pool.scale[side][layer, pg, h]
                    x = torch.stack([r[h] for _, r in new])
                    first = new[0][0]
                    want = float((x.abs().max() / TOP[pool.cache]).float())
                    s = float(scale[blk]) if first else 0.0
                    if not math.isfinite(want) or not math.isfinite(s):
                        scale[blk] = math.nan
                        code[first:first + len(new)] = 0.0
                        continue
                    sign = -1.0 if s < 0 else 1.0
                    s = abs(s)
                    if s == 0.0:
                        s = want
                        code[:first] = 0.0
                    else:
                        f = 1.0
                        while s < want:
                            s, f = s * 2.0, f * 0.5
                        if f != 1.0:
                            code[:first] = nearest(code[:first] * f, pool.cache)
                    scale[blk] = sign * s
                    code[first:first + len(new)] = nearest(x * sign / s, pool.cache) if s else 0.0


def read(pool, table, pos, n, t, layer=0):
    """rows [b, t, h, hs] of K and V, and which of them there are"""
    per = len(table[0])
    out = [torch.zeros(len(table), t, pool.h, pool.hs, dtype=torch.float64) for _ in range(2)]
    there = torch.zeros(len(table), t, dtype=torch.bool)
    val = [pool.values(0, layer), pool.values(1, layer)]
    for b in range(len(table)):
        for i in range(min(n[b], t)):
            p = pos[b] + i
            if 0 <= p < per * pool.page and 0 <= table[b][p // pool.page] < pool.pages:
                there[b, i] = True
                for side in range(2):
                    out[side][b, i] = val[side][table[b][p // pool.page], :, p % pool.page]
    return out[0], out[1], there


def fork(table, lens, refs, to, source, page):
    old, old_lens, b = [list(r) for r in table], list(lens), len(table)
    for i, x in enumerate(to):
        if not 0 <= x < b or x in to[i + 1:]:
            continue
        for e in old[x]:
            if 0 <= e < len(refs):
                refs[e] -= 1
        s = source[i]
        lens[x] = min(max(old_lens[s], 0), len(old[x]) * page) if 0 <= s < b else 0
        need = -(-lens[x] // page)
        table[x] = [old[s][j] if j < need and 0 <= old[s][j] < len(refs) else -1 for j in range(len(old[x]))]
        for e in table[x]:
            if e >= 0:
                refs[e] += 1


def reserve(pool, table, refs, lens, n, most):
    """(1, pages taken) or (0, pages wanted)"""
    page, per = pool.page, len(table[0])
    asked, fits = [], True
    for b in range(len(table)):
        nn, at = max(n[b], 0), max(lens[b], 0)
        if nn and (nn > most or at + nn > per * page):
            fits = False
        elif nn:
            asked += [(b, j) for j in range(at // page, (at + nn - 1) // page + 1)]
    has = {}
    for b, j in asked:
        e = table[b][j]
        if 0 <= e < len(refs) and refs[e] > 1:
            has.setdefault(e, []).append((b, j))
    need = []
    for b, j in asked:
        e = table[b][j]
        if not (0 <= e < len(refs)) or refs[e] <= 0:
            need.append((b, j, -1))
        elif refs[e] > 1 and not (len(has[e]) == refs[e] and has[e][-1] == (b, j)):
            need.append((b, j, e))
    free = [i for i, r in enumerate(refs) if r <= 0]
    if not fits or len(free) < len(need):
        return 0, len(need)
    for (b, j, e), new in zip(need, free):
        if e >= 0:
            refs[e] -= 1
            at = max(lens[b], 0) - j * page
            blocks = -(-at // BLOCK) if 0 < at < page else 0
            for x in pool.code + pool.scale:
                x[:, new, :, :blocks] = x[:, e, :, :blocks]
        table[b][j] = new
        refs[new] = 1
    return 1, len(need)


def compact(pool, table, refs):
    used = [i for i, r in enumerate(refs) if r > 0]
    u = len(used)
    far, hole = [i for i in used if i >= u], [i for i in range(u) if refs[i] <= 0]
    went = dict(zip(far, hole))
    for a, b in went.items():
        for x in pool.code + pool.scale:
            x[:, b] = x[:, a]
        refs[b], refs[a] = refs[a], 0
    for row in table:
        row[:] = [e if not u <= e < len(refs) else went.get(e, -1) for e in row]
    return u, len(far)


def accept(logits, tokens, coins, parents, n, probs, temperature):
    """(kept, path, next, logp) of one sequence; logits [t, vocab] and probs in float64.  The residuals one after another, as
    distributions."""
    t, v = logits.shape

    def target(r):
        x = logits[r]
        if x.isnan().any() or x.max() == math.inf or x.max() == -math.inf:
            return None
        if temperature == 0.0:
            return torch.nn.functional.one_hot(torch.nonzero(x == x.max())[0, 0], v).double()
        return torch.softmax(x / temperature, -1)

    path, logp = [-1] * t, [0.0] * t
    if n < 1:
        return 0, path, -1, logp
    parent = [i - 1 if parents is None else parents[i] for i in range(t)]
    for i in range(1, n):
        if 0 <= parent[i] < i:
            p = target(parent[i])
            ok = 0 <= tokens[i] < v
            logp[i] = -math.inf if not ok else math.nan if p is None else math.log(p[tokens[i]]) if p[tokens[i]] > 0 else -math.inf
    node, way = 0, [0]
    while True:
        p = target(node)
        if p is None:
            break
        left, gone, step = p, [], None
        for c in range(node + 1, n):
            if parent[c] != node or not 0 <= tokens[c] < v:
                continue
            x = tokens[c]
            q = 1.0 if probs is None else float(probs[node, x])
            if coins[c] * q < float(left[x]):
                step = c
                break
            if probs is None:
                gone.append(x)
                rest = p.clone()
                rest[gone] = 0.0
            else:
                rest = (left - probs[node]).clamp(min=0.0)
            left = rest / rest.sum() if rest.sum() > 0 else rest
        if step is None:
            break
        node = step
        way.append(node)
    path[:len(way)] = way
    if p is None:
        logp[0] = math.nan
        return len(way), path, -1, logp
    w = left if left.sum() > 0 else p
    c = torch.cumsum(w, 0)
    token = int(torch.nonzero(c > coins[0] * c[-1])[0, 0])
    logp[0] = math.log(p[token])
    return len(way), path, token, logp
