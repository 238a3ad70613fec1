"""Timed cases of the operators over a cache in pages: rows written into pages of 8 bits with a scale for each block of 64 tokens
and head, and read back (page_write, page_read), attention over such pages and over the newest tokens' own rows (page_attention),
pages shared, copied, freed and moved together (page_fork, page_reserve, page_compact), and drafted tokens kept or dropped against
the target's probabilities (draft_accept).

`run` computes them in plain torch where `own` is false, and calls the framework where it is true.  A page holds `page` positions
of every kv head: K as [page, head size], V as [page / 64, head size, 64], a scale for each 64 positions of either.  Head layouts
are those of the repository's configurations: Qwen2 0.5B (14 heads, 2 kv heads of 64, 24 layers), Qwen2 7B (28, 4 of 128, 28),
llama2.c 288 (6, 6 of 48, 6) and 768 (12, 12 of 64, 12)."""
import importlib.util
import math
import os

import numpy as np
import torch

own = False

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_package = None


def _own():
    global _package
    if _package is None:
        spec = importlib.util.spec_from_file_location(
            "llm_hip", os.path.join(_REPO, "local-llama-pynq-z2_amd", "__init__.py"))
        _package = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_package)
    return _package


HEADS = {"qwen2-0.5b": (14, 2, 64), "qwen2-7b": (28, 4, 128), "llama2c-288": (6, 6, 48), "llama2c-768": (12, 12, 64)}
LAYERS = {"qwen2-0.5b": 24, "qwen2-7b": 28, "llama2c-288": 6, "llama2c-768": 12}
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
BLOCK = 64


def listed():
    return [
        # one decode step's rows of a small model: latency
        dict(name="write_step_0p5b", kind="write", heads="qwen2-0.5b", cache="int8", rows="fp32", page=64, seqs=1, pos=700,
             new=1),
        # a prompt's second chunk: 2048 new rows, the whole prefix read back for the chunk's attention
        dict(name="write_chunk_7b", kind="write", heads="qwen2-7b", cache="int8", rows="fp32", page=128, seqs=1, pos=5021,
             new=2048),
        # a decode step early in a dialog: latency
        dict(name="step_0p5b_203", kind="attend", heads="qwen2-0.5b", cache="int8", rows="fp32", page=64, seqs=1, pos=203,
             new=1),
        # a batch of decode steps, lengths from nothing to 8190, 16-bit activations
        dict(name="step_batch_e4m3", kind="attend", heads="qwen2-7b", cache="e4m3", rows="bf16", page=64, seqs=32, pos=8190,
             new=1),
        # a drafted tree of one long sequence
        dict(name="tree_7b_int8", kind="attend", heads="qwen2-7b", cache="int8", rows="fp32", page=128, seqs=1, pos=12003,
             new=37),
        # whole trees of 64 for a batch of long sequences: the largest
        dict(name="tree_batch_int8", kind="attend", heads="qwen2-7b", cache="int8", rows="bf16", page=64, seqs=8, pos=16000,
             new=64),
        # four beams of one sequence take their parents' pages and make room for a token each: latency
        dict(name="fork_beams_0p5b", kind="fork", heads="qwen2-0.5b", page=64, seqs=4, beams=4, pos=700),
        # the same for a batch: the last pages of all layers copied
        dict(name="fork_batch_7b", kind="fork", heads="qwen2-7b", page=64, seqs=64, beams=4, pos=520),
        # a few dialogs end, the pool is moved together, others begin: latency
        dict(name="compact_0p5b", kind="compact", heads="qwen2-0.5b", page=64, seqs=6, pos=300),
        # half of a large batch ends
        dict(name="compact_7b", kind="compact", heads="qwen2-7b", page=64, seqs=48, pos=700),
        # a chain of five drafted by a smaller model for one dialog: latency
        dict(name="accept_chain", kind="accept", seqs=1, nodes=6, vocab=151936, logits="fp32", draft="fp32", tree=False,
             temperature=1.0),
        # trees of looked-up drafts for a batch
        dict(name="accept_trees", kind="accept", seqs=16, nodes=37, vocab=151936, logits="bf16", draft="", tree=True,
             temperature=0.75),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "attend", "attend", "attend", "fork", "compact", "accept", "accept"])
    if kind == "accept":
        vocab = rng.choice([_log(rng, 300, 152064), 32000, 151936])
        seqs = _log(rng, 1, 32)
        nodes = max(1, min(rng.randint(1, 64), 80_000_000 // (vocab * seqs)))
        return dict(kind=kind, seqs=seqs, nodes=nodes, vocab=vocab, logits=rng.choice(["fp32", "bf16"]),
                    draft=rng.choice(["", "fp32", "bf16"]), tree=rng.choice([False, True]),
                    temperature=rng.choice([1.0, 1.0, 0.75, 1.25, 0.0]))
    heads, page = rng.choice(list(HEADS)), rng.choice([64, 64, 128, 256])
    if kind == "fork":
        beams = rng.choice([1, 2, 4, 5])
        groups = _log(rng, 1, 16)
        return dict(kind=kind, heads=heads, page=page, seqs=beams * groups, beams=beams, pos=_log(rng, 1, 520))
    if kind == "compact":
        return dict(kind=kind, heads=heads, page=page, seqs=_log(rng, 2, 48), pos=_log(rng, 1, 512))
    seqs = rng.choice([1, 1, _log(rng, 1, 32)])
    shape = dict(kind=kind, heads=heads, cache=rng.choice(["int8", "e4m3"]), rows=rng.choice(["fp32", "bf16"]), page=page,
                 seqs=seqs)
    most = min(32768, 131072 // seqs)
    if kind == "write":
        new = _log(rng, 1, min(2048, 16384 // seqs))
        return dict(**shape, pos=rng.randint(0, min(most, 8192)), new=new)
    return dict(**shape, pos=_log(rng, 1, most) - 1, new=rng.choice([1, 1, rng.randint(1, 64)]))


# ---- inputs ------------------------------------------------------------------------------------------------------


def _lengths(case):
    """The committed length and the new rows of every sequence: the first has the case's own, the others less (none and
    one among them)."""
    lens, new = [case["pos"]], [case["new"]]
    for b in range(1, case["seqs"]):
        f = (b * 0.6180339887) % 1.0
        lens.append(0 if b == 3 else min(1, case["pos"]) if b == 5 else int(case["pos"] * f))
        new.append(case["new"] - (b * 7) % (1 + case["new"] // 3))
    return lens, new


def _round_e4m3(q):
    """float64 values within 448 to e4m3's, half to even: the distance of its values around q is q's power of two (at least
    2^-6), three bits further down"""
    step = ((((q.view(torch.int64) >> 52) & 2047).clamp(min=1023 - 6) - 3) << 52).view(torch.float64)
    return torch.round(q / step) * step


def _codes(x, s, cache):
    """codes of float64 values x at the scales s (float32, of x's shape or one to broadcast), the quotient in 64 bits"""
    s = s.double()
    q = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x)).clamp(-TOP[cache], TOP[cache])
    return torch.round(q).to(torch.int8) if cache == "int8" else _round_e4m3(q).float().to(torch.float8_e4m3fn)


def _bytes(x):
    return x.view(torch.int8)


def _rows(g, shape):
    """Rows as the path meets them: normal, some channels much larger than others."""
    ch = torch.exp(torch.randn(shape[-1], generator=g, device=g.device))
    return torch.randn(shape, generator=g, device=g.device) * ch


def _table(g, lens, page, room, n_pages, per):
    """A table of random pages for `lens` positions, -1 behind them, and the pages' counts."""
    dev = g.device
    need = (lens.long() + page - 1) // page
    have = torch.arange(per, device=dev) < need.unsqueeze(1)
    ids = torch.randperm(n_pages, generator=g, device=dev).int()
    table = torch.full((lens.numel(), per), -1, dtype=torch.int32, device=dev)
    table[have] = ids[:int(need.sum())]
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    refs[ids[:int(need.sum())].long()] = 1
    return table, refs


def _pool(g, case, n_pages):
    """Pages full of rows: codes and scales of K [pages, kv heads, page, head size] and V [.., page / 64, head size, 64]."""
    _, kv, hs = HEADS[case["heads"]]
    nb = case["page"] // BLOCK
    st = {}
    for name in ("k", "v"):
        x = _rows(g, (n_pages, kv, nb, BLOCK, hs))
        if name == "v":
            x = x * 0.1
        s = (x.double().abs().amax((-1, -2)) / TOP[case["cache"]]).float()
        c = _codes(x.double(), s[..., None, None], case["cache"])
        if name == "v":
            c = _bytes(c).transpose(-1, -2).contiguous().view(TYPES[case["cache"]])
        st[name] = c if name == "v" else c.view(n_pages, kv, case["page"], hs)
        st[name + "s"] = s
    return st


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    st = dict(case=case)
    if case["kind"] == "accept":
        return _prepare_accept(st, case, g)
    if case["kind"] in ("fork", "compact"):
        return _prepare_pages(st, case, g)
    heads, kv, hs = HEADS[case["heads"]]
    b, t, page = case["seqs"], case["new"], case["page"]
    lens, new = _lengths(case)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
    full = st["lens"] + (st["new"] if case["kind"] == "write" else 0)
    per = max(1, -(-(case["pos"] + t) // page))
    n_pages = int(((full.long() + page - 1) // page).sum()) + 3
    st["table"], st["refs"] = _table(g, full, page, t, n_pages, per)
    st.update(_pool(g, case, n_pages))
    rows = TYPES[case["rows"]]
    st["kr"] = _rows(g, (b, t, kv, hs)).to(rows)
    st["vr"] = (_rows(g, (b, t, kv, hs)) * 0.1).to(rows)
    if case["kind"] == "write":
        return st
    st["q"] = (torch.randn(b, t, heads, hs, generator=g, device=dev) * 0.7).to(rows)
    # the tree: node 0 is the root, the others hang on a node before them (half of them on the last: long paths)
    sees = torch.eye(t, dtype=torch.bool, device=dev).repeat(b, 1, 1)
    back = torch.rand(b, t, generator=g, device=dev)
    for i in range(1, t):
        p = torch.where(back[:, i] < 0.5, torch.full_like(back[:, i], i - 1), torch.floor((back[:, i] - 0.5) * 2.0 * i))
        sees[:, i] |= sees[torch.arange(b, device=dev), p.long().clamp(0, i - 1)]
    bits = torch.ones(t, dtype=torch.int64, device=dev) << torch.arange(t, device=dev)
    st["mask"] = (sees * bits).sum(-1)
    return st


def _prepare_pages(st, case, g):
    dev = g.device
    _, kv, hs = HEADS[case["heads"]]
    layers, page, b = LAYERS[case["heads"]], case["page"], case["seqs"]
    per = (case["pos"] + page) // page
    f = torch.arange(b, device=dev)
    if case["kind"] == "fork":
        # the beams of a group are as long as each other, and share what they had a step ago
        beams = case["beams"]
        lens = (case["pos"] - (f // beams * 37) % (1 + case["pos"] // 3)).int()
        first = f // beams * beams
        n_pages = b * per + b
        table, refs = _table(g, lens, page, 1, n_pages, per)
        old = torch.arange(per, device=dev) < (lens // page).unsqueeze(1)
        shared = torch.where(old, table[first], table)
        used = shared[shared >= 0].long()
        refs = torch.zeros_like(refs).index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
        st["table"], st["refs"], st["lens"] = shared, refs, lens
        pick = torch.floor(torch.rand(b, generator=g, device=dev) ** 2 * beams).int().clamp(0, beams - 1)
        st["to"], st["from"] = f.int(), first.int() + pick
        st["one"] = torch.ones(b, dtype=torch.int32, device=dev)
    else:
        lens = (case["pos"] - (f * 37) % (1 + case["pos"] // 3)).int()
        n_pages = b * per + 1
        st["table"], st["refs"] = _table(g, lens, page, 0, n_pages, per)
        st["lens"], st["full"] = lens, lens.clone()
        half = torch.rand(b, generator=g, device=dev).argsort() % 2  # they end in turn
        st["turn"], st["sets"], st["empty"], st["begin"] = 0, [], [], []
        for i in range(2):
            to = torch.nonzero(half == i).flatten().int()
            st["sets"].append(to)
            st["empty"].append(torch.full_like(to, -1))
            st["begin"].append(torch.where(half == i, lens, torch.zeros_like(lens)))
    for name in ("k", "v"):
        shape = (page, hs) if name == "k" else (page // BLOCK, hs, BLOCK)
        st[name] = torch.randint(-127, 128, (layers, n_pages, kv) + shape, generator=g, device=dev, dtype=torch.int8)
        st[name + "s"] = torch.rand(layers, n_pages, kv, page // BLOCK, generator=g, device=dev) * 0.05
    return st


def _prepare_accept(st, case, g):
    dev = g.device
    b, t, v = case["seqs"], case["nodes"], case["vocab"]
    x = torch.randn(b, t, v, generator=g, device=dev) * 2.0
    hot = torch.randint(0, v, (b, t, 4), generator=g, device=dev)
    x.scatter_add_(2, hot, 6.0 + 8.0 * torch.rand(b, t, 4, generator=g, device=dev))
    st["logits"] = x.to(TYPES[case["logits"]])
    # a token hangs on the one before it (a chain), or on one of the last few
    i = torch.arange(t, device=dev)
    back = torch.randint(1, 4, (b, t), generator=g, device=dev) if case["tree"] else torch.ones(b, t, dtype=torch.int64, device=dev)
    parents = torch.where(i > 0, (i - back).clamp(min=0), torch.full_like(back, -1))
    st["parents"] = parents.int() if case["tree"] else None
    at = parents.clamp(min=0)
    seq = torch.arange(b, device=dev).unsqueeze(1)
    # the draft's opinion: the target's, not quite
    y = x + torch.randn(b, t, v, generator=g, device=dev) * 0.7
    q = torch.softmax(y, -1)
    st["probs"] = q.to(TYPES[case["draft"]]) if case["draft"] else None
    drawn = torch.multinomial(q.view(b * t, v), 3, replacement=bool(case["draft"]), generator=g).view(b, t, 3)
    st["tokens"] = drawn[seq, at, i % 3].int()
    st["coins"] = torch.rand(b, t, generator=g, device=dev)
    st["n"] = (t - (torch.arange(b, device=dev) * 7) % (1 + t // 3)).int()
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _exponent(x):
    """x = m 2^e, m in [0.5, 1)"""
    return torch.frexp(x.double())


def _plain_write(st):
    case = st["case"]
    page, cache, top = case["page"], case["cache"], TOP[case["cache"]]
    _, kv, hs = HEADS[case["heads"]]
    dev, t = st["k"].device, case["new"]
    per = st["table"].shape[1]
    b, i = torch.nonzero(torch.arange(t, device=dev) < st["new"].unsqueeze(1), as_tuple=True)
    at = st["lens"].long()[b] + i
    pg = st["table"].long()[b, at // page]
    blk, off = at % page // BLOCK, at % BLOCK
    nth = at // BLOCK - st["lens"].long()[b] // BLOCK  # the blocks of a sequence that get rows
    most = (t + BLOCK - 1) // BLOCK + 1
    lens = st["lens"].long()
    tail = lens % BLOCK  # rows that the first of them has already
    where = (lens // page).clamp(max=per - 1)
    tpg = st["table"].long().gather(1, where.unsqueeze(1)).squeeze(1).clamp(min=0)
    tblk = lens % page // BLOCK
    keep = torch.arange(BLOCK, device=dev) < tail.unsqueeze(1)  # [seqs, 64]
    for name in ("k", "v"):
        pool, sc = st[name], st[name + "s"]
        x = st[name + "r"][b, i].double()  # [rows, kv, hs]
        amax = torch.zeros(case["seqs"] * most, kv, dtype=torch.float64, device=dev)
        amax.scatter_reduce_(0, (b * most + nth).unsqueeze(1).expand(-1, kv), x.abs().amax(-1), "amax")
        fresh = (amax / top).float().view(case["seqs"], most, kv)
        old = sc[tpg, :, tblk]  # [seqs, kv]
        old = torch.where((tail > 0).unsqueeze(1), old, torch.zeros_like(old))
        (m0, e0), (m1, e1) = _exponent(old), _exponent(fresh[:, 0])
        up = (e1 - e0 + (m1 > m0).int()).clamp(min=0)  # the least power of two that covers the new rows
        up = torch.where((old > 0) & (fresh[:, 0] > old), up, torch.zeros_like(up))
        grown = torch.where(old > 0, torch.ldexp(old.double(), up).float(), fresh[:, 0])
        s = torch.cat((grown.unsqueeze(1), fresh[:, 1:]), 1)  # [seqs, blocks, kv]
        bits = _bytes(pool)
        if name == "k":
            bits = bits.view(-1, kv, page // BLOCK, BLOCK, hs)
        else:
            bits = bits.transpose(-1, -2)
        had = bits[tpg, :, tblk].contiguous()  # [seqs, kv, 64, hs]
        val = had.double() if cache == "int8" else had.view(TYPES[cache]).double()
        val = val * torch.ldexp(torch.ones_like(old, dtype=torch.float64), -up)[..., None, None]
        val = _bytes(torch.round(val).to(torch.int8) if cache == "int8" else _round_e4m3(val).float().to(TYPES[cache]))
        took = (keep & (st["new"] > 0).unsqueeze(1)).view(-1, 1, BLOCK, 1)
        live = torch.nonzero((tail > 0) & (st["new"] > 0)).flatten()
        bits[tpg[live], :, tblk[live]] = torch.where(took, val, had)[live]
        bits[pg, :, blk, off] = _bytes(_codes(x, s[b, nth].unsqueeze(-1), cache))
        sc[pg, :, blk] = s[b, nth]
    # all of the sequences read back
    reach = torch.arange(case["pos"] + t, device=dev)
    k, v = _gathered(st, case["pos"] + t)
    have = (reach < (lens + st["new"]).unsqueeze(1))[..., None, None]
    k, v = (torch.where(have, x.permute(0, 2, 1, 3), torch.zeros((), device=dev)).contiguous() for x in (k, v))
    return k, v, st["ks"], st["vs"]


def _gathered(st, end):
    """The values of K and V of the first `end` positions, [seqs, kv heads, positions, head size]."""
    case = st["case"]
    _, kv, hs = HEADS[case["heads"]]
    b, page = case["seqs"], case["page"]
    pages = -(-end // page)
    ids = st["table"][:, :pages].long().clamp(min=0)
    k = _bytes(st["k"])[ids].view(TYPES[case["cache"]]).float().view(b, pages, kv, page // BLOCK, BLOCK, hs)
    v = _bytes(st["v"])[ids].view(TYPES[case["cache"]]).float().transpose(-1, -2)
    return tuple((x * st[s][ids][..., None, None]).permute(0, 2, 1, 3, 4, 5).reshape(b, kv, pages * page, hs)[:, :, :end]
                 for x, s in ((k, "ks"), (v, "vs")))


def _plain_attend(st):
    case = st["case"]
    heads, kv, hs = HEADS[case["heads"]]
    b, t, end = case["seqs"], case["new"], case["pos"]
    dev = st["q"].device
    k, v = _gathered(st, end)
    k = torch.cat((k, st["kr"].float().permute(0, 2, 1, 3)), 2)
    v = torch.cat((v, st["vr"].float().permute(0, 2, 1, 3)), 2)
    q = st["q"].float().view(b, t, kv, heads // kv, hs).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hs)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hs))  # [b, kv, group t, end + t]
    step = torch.arange(t, device=dev)
    live = step < st["new"].unsqueeze(1)  # [b, t]
    before = (torch.arange(end, device=dev) < st["lens"].unsqueeze(1)).unsqueeze(1).expand(b, t, end)
    bit = ((st["mask"].unsqueeze(-1) >> step) & 1 != 0) & live.unsqueeze(1)
    sees = (torch.cat((before, bit), 2) & live.unsqueeze(-1)).unsqueeze(1).unsqueeze(1)
    s = s.view(b, kv, heads // kv, t, end + t).masked_fill(~sees, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z > 0, z, torch.ones_like(z))).view(b, kv, -1, end + t)
    o = torch.matmul(p, v).view(b, kv, heads // kv, t, hs).permute(0, 3, 1, 2, 4).reshape(b, t, heads, hs)
    return o.to(st["q"].dtype)


def _plain_fork(table, lens, refs, to, source, page):
    to, src = to.long(), source.long()
    there = src >= 0
    length = torch.where(there, lens[src.clamp(min=0)], torch.zeros_like(lens[to]))
    need = ((length.long() + page - 1) // page).unsqueeze(1)
    new = torch.where(torch.arange(table.shape[1], device=table.device) < need, table[src.clamp(min=0)], -torch.ones_like(table[to]))
    old = table[to]
    for x, by in ((old, -1), (new, 1)):
        used = x[x >= 0].long()
        refs.index_add_(0, used, torch.full_like(used, by, dtype=torch.int32))
    table[to] = new
    lens[to] = length


def _plain_reserve(st, n, most):
    """Room for n[b] positions behind lens[b] (at most `most`): new pages, and own copies of shared ones."""
    case, table, refs = st["case"], st["table"], st["refs"]
    page, dev = case["page"], st["table"].device
    b, per = table.shape
    lens = st["lens"].long()
    j = (lens // page).unsqueeze(1) + torch.arange((most + page - 1) // page + 1, device=dev)
    touched = (j <= ((lens + n - 1) // page).unsqueeze(1)) & (n > 0).unsqueeze(1)
    j = j.clamp(max=per - 1)
    e = table.long().gather(1, j)
    valid = touched & (e >= 0)
    e = e.clamp(min=0)
    shared = valid & (refs[e] > 1)
    seq = torch.arange(b, device=dev).unsqueeze(1).expand_as(e)
    claims = torch.zeros_like(refs).index_add_(0, e[shared], torch.ones_like(e[shared], dtype=torch.int32))
    last = torch.full_like(refs, -1, dtype=torch.int64).scatter_reduce_(0, e[shared], seq[shared], "amax")
    keep = shared & (claims[e] == refs[e]) & (last[e] == seq)  # all who have it want it: the last one keeps it
    need = touched & (~valid | (shared & ~keep))
    free = torch.nonzero(refs == 0).flatten()
    total = need.sum()
    rank = (need.flatten().cumsum(0) - 1).view_as(e)
    new = free[rank.clamp(min=0, max=max(free.numel() - 1, 0))]
    # of the first page the positions before lens, in whole blocks
    copied = need[:, 0] & valid[:, 0] & (lens % page > 0)
    blocks = torch.arange(page // BLOCK, device=dev) * BLOCK < (lens % page).unsqueeze(1)
    s, blk = torch.nonzero(copied.unsqueeze(1) & blocks, as_tuple=True)
    _, kv, hs = HEADS[case["heads"]]
    for name in ("k", "v"):
        pool = st[name].view(st[name].shape[0], -1, kv, page // BLOCK, BLOCK * hs)
        pool[:, new[s, 0], :, blk] = pool[:, e[s, 0], :, blk]
        st[name + "s"][:, new[s, 0], :, blk] = st[name + "s"][:, e[s, 0], :, blk]
    left = e[shared & need]
    refs.index_add_(0, left, torch.full_like(left, -1, dtype=torch.int32))
    refs[new[need]] = 1
    table[seq[need], j[need]] = new[need].int()
    return torch.stack((torch.ones_like(total), total)).int()


def _plain_compact(st):
    table, refs = st["table"], st["refs"]
    used = refs > 0
    count = used.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    hole = torch.nonzero(~used & (ids < count)).flatten()
    far = torch.nonzero(used & (ids >= count)).flatten()
    for name in ("k", "v", "ks", "vs"):
        st[name][:, hole] = st[name][:, far]
    ids[far] = hole
    table.copy_(torch.where(table >= 0, ids[table.long().clamp(min=0)].int(), table))
    refs[hole] = refs[far]
    refs[far] = 0
    return torch.stack((count, torch.ones_like(count) * far.numel())).int()


def _plain_accept(st):
    case = st["case"]
    b, t, v = st["logits"].shape
    dev = st["logits"].device
    x = st["logits"].double()
    temp = float(np.float32(case["temperature"]))
    best = x.argmax(-1)  # (of the inputs here the first of equal ones)
    best = (x == x.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1) if temp == 0.0 else best
    seq, node = torch.arange(b, device=dev), torch.arange(t, device=dev)
    if temp == 0.0:
        lp = torch.full_like(x, -math.inf).scatter_(2, best.unsqueeze(-1), 0.0)
    else:
        y = x / temp
        e = y - y.amax(-1, keepdim=True)
        lp = e - torch.log(torch.exp(e).sum(-1, keepdim=True))
    n = st["n"].long()
    parents = node.expand(b, t) - 1 if st["parents"] is None else st["parents"].long()
    tok = st["tokens"].long()
    logp = lp[seq.unsqueeze(1), parents.clamp(min=0), tok]
    logp = torch.where((node > 0) & (node < n.unsqueeze(1)), logp, torch.zeros_like(logp))
    q = st["probs"]
    cur, kept = torch.zeros_like(n), (n > 0).long()
    path = torch.full((b, t), -1, dtype=torch.int64, device=dev)
    path[:, 0] = torch.where(n > 0, torch.zeros_like(n), path[:, 0])
    a, z = torch.zeros(b, dtype=torch.float64, device=dev), torch.ones(b, dtype=torch.float64, device=dev)
    out = torch.zeros(b, v, dtype=torch.bool, device=dev)  # tokens that were turned down after the current node
    for i in range(1, t):
        asked = (parents[:, i] == cur) & (i < n)
        p = torch.exp(lp[seq, cur, tok[:, i]])
        if q is None:
            w = torch.where(out[seq, tok[:, i]], torch.zeros_like(p), p)
            takes = asked & (st["coins"][:, i].double() * z < w)
        else:
            qi = q[seq, cur, tok[:, i]].double()
            w = (p - a * qi).clamp(min=0.0)
            takes = asked & (st["coins"][:, i].double() * qi * z < w)
        no = asked & ~takes
        if q is None:
            out[seq, tok[:, i]] |= no
            z = torch.where(no, (z - w).clamp(min=0.0), z)
            out &= ~takes.unsqueeze(1)
        else:
            a = torch.where(no, a + z, a)
            later = (parents[:, i + 1:] == cur.unsqueeze(1)).any(1) & no if i + 1 < t else torch.zeros_like(no)
            r = torch.nonzero(later).flatten()  # only those that another token is held against
            left = (torch.exp(lp[r, cur[r]]) - a[r].unsqueeze(1) * q[r, cur[r]].double()).clamp(min=0.0).sum(-1)
            z = z.index_copy(0, r, left)
        a, z = torch.where(takes, torch.zeros_like(a), a), torch.where(takes, torch.ones_like(z), z)
        cur = torch.where(takes, torch.full_like(cur, i), cur)
        path[seq, kept.clamp(max=t - 1)] = torch.where(takes, cur, path[seq, kept.clamp(max=t - 1)])
        kept = kept + takes.long()
    p = torch.exp(lp[seq, cur])
    w = torch.where(out, torch.zeros_like(p), p) if q is None else (p - a.unsqueeze(1) * q[seq, cur].double()).clamp(min=0.0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    c = w.cumsum(-1)
    drawn = (c > (st["coins"][:, 0].double() * c[:, -1]).unsqueeze(1)).to(torch.uint8).argmax(-1)
    logp[:, 0] = lp[seq, cur, drawn]
    return kept.int(), path.int(), drawn.int(), logp.float()


def _plain_fork_step(st):
    _plain_fork(st["table"], st["lens"], st["refs"], st["to"], st["from"], st["case"]["page"])
    got = _plain_reserve(st, st["one"].long(), 1)
    return [st[x] for x in ("table", "lens", "refs")] + [got] + [st[x] for x in ("k", "v", "ks", "vs")]


def _plain_compact_step(st):
    i = st["turn"]
    st["turn"] = 1 - i
    _plain_fork(st["table"], st["lens"], st["refs"], st["sets"][i], st["empty"][i], st["case"]["page"])
    moved = _plain_compact(st)
    got = _plain_reserve(st, st["begin"][i].long(), st["case"]["pos"])
    st["lens"].copy_(st["full"])
    return [st[x] for x in ("table", "lens", "refs")] + [moved, got] + [st[x] for x in ("k", "v", "ks", "vs")]


def run(state):
    case = state["case"]
    if not own:
        return {"write": _plain_write, "attend": _plain_attend, "fork": _plain_fork_step, "compact": _plain_compact_step,
                "accept": _plain_accept}[case["kind"]](state)
    P = _own()
    st = state
    if case["kind"] == "accept":
        return P.draft_accept(st["logits"], st["tokens"], st["coins"], parents=st["parents"], n=st["n"], probs=st["probs"],
                              temperature=case["temperature"])
    pool = (st["k"], st["v"], st["ks"], st["vs"])
    if case["kind"] == "write":
        P.page_write(st["kr"], st["vr"], *pool, st["table"], st["lens"], st["new"], refs=st["refs"])
        end = case["pos"] + case["new"]
        k, v = P.page_read(*pool, st["table"], torch.zeros_like(st["lens"]), end, st["lens"] + st["new"])
        return k, v, st["ks"], st["vs"]
    if case["kind"] == "attend":
        return P.page_attention(st["q"], *pool, st["table"], st["lens"], k_rows=st["kr"], v_rows=st["vr"], n=st["new"],
                                mask=st["mask"], max_len=case["pos"])
    if case["kind"] == "fork":
        P.page_fork(st["table"], st["lens"], st["refs"], st["to"], st["from"], case["page"])
        got = P.page_reserve(*pool, st["table"], st["refs"], st["lens"], st["one"], max_n=1)
        return [st["table"], st["lens"], st["refs"], got] + list(pool)
    i = st["turn"]
    st["turn"] = 1 - i
    P.page_fork(st["table"], st["lens"], st["refs"], st["sets"][i], st["empty"][i], case["page"])
    moved = P.page_compact(*pool, st["table"], st["refs"])
    got = P.page_reserve(*pool, st["table"], st["refs"], st["lens"], st["begin"][i], max_n=case["pos"])
    st["lens"].copy_(st["full"])
    return [st["table"], st["lens"], st["refs"], moved, got] + list(pool)


def work(case):
    if case["kind"] == "accept":
        # every row's logits, and one of the draft's rows for each sequence
        rows = sum(case["nodes"] - (b * 7) % (1 + case["nodes"] // 3) for b in range(case["seqs"]))
        size = {"fp32": 4, "bf16": 2, "": 0}
        return {"bytes": case["vocab"] * (rows * size[case["logits"]] + case["seqs"] * size[case["draft"]])
                + 24 * case["seqs"] * case["nodes"], "flops": 3 * rows * case["vocab"]}
    heads, kv, hs = HEADS[case["heads"]]
    page = case["page"]
    block = 2 * kv * (BLOCK * hs + 4)  # of K and V
    if case["kind"] in ("fork", "compact"):
        layers, b, per = LAYERS[case["heads"]], case["seqs"], (case["pos"] + page) // page
        ints = 4 * (2 * b * per + 4 * b)
        if case["kind"] == "fork":
            # beams that share a parent: all but one copy its last page (three parents of four taken by about two)
            lens = [case["pos"] - (i // case["beams"] * 37) % (1 + case["pos"] // 3) for i in range(b)]
            blocks = sum(-(-(n % page) // BLOCK) for n in lens) * (case["beams"] - 1) / (2 * case["beams"])
            return {"bytes": ints + 2 * layers * block * blocks, "flops": b * per}
        lens = [case["pos"] - (i * 37) % (1 + case["pos"] // 3) for i in range(b)]
        pages = sum(-(-n // page) for n in lens)
        # half of the pages go, and half of what stays lies behind its place
        return {"bytes": ints + 2 * layers * block * (page // BLOCK) * pages / 4, "flops": b * per}
    lens, new = _lengths(case)
    act = 4 if case["rows"] == "fp32" else 2
    if case["kind"] == "write":
        blocks = sum(-(-(n + c) // BLOCK) for n, c in zip(lens, new))
        fresh = sum(-(-(n % BLOCK + c) // BLOCK) for n, c in zip(lens, new))
        back = case["seqs"] * (case["pos"] + case["new"])
        return {"bytes": 2 * sum(new) * kv * hs * act + block * (blocks + fresh) + 2 * back * kv * hs * 4,
                "flops": 2 * kv * hs * (4 * sum(new) + back)}
    return {"bytes": sum(2 * n * kv * hs + 8 * kv * (-(-n // BLOCK)) + 2 * c * (heads + kv) * hs * act + 8 * c
                         for n, c in zip(lens, new)),
            "flops": sum(4 * heads * hs * c * (n + 1) for n, c in zip(lens, new))}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------


E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def _nearest(u, cache):
    """the nearest of the type's values, half to even"""
    u = u.clamp(-TOP[cache], TOP[cache])
    if cache == "int8":
        return torch.round(u)
    every = E4M3.to(u.device)
    mid = (every[1:] + every[:-1]) / 2.0
    i = torch.bucketize(u.abs().contiguous(), mid)
    tie = (i < 126) & (u.abs() == mid[i.clamp(max=125)]) & (i % 2 == 1)
    return torch.sign(u) * every[i + tie.long()]


def _exact_write(st):
    case = st["case"]
    lens, new = _lengths(case)
    page, cache = case["page"], case["cache"]
    _, kv, hs = HEADS[case["heads"]]
    end = case["pos"] + case["new"]
    table = st["table"].tolist()
    got, scales = [], []
    for name in ("k", "v"):
        code = st[name].float().double()
        code = code.view(-1, kv, page // BLOCK, BLOCK, hs) if name == "k" else code.transpose(-1, -2)
        sc = st[name + "s"].double()
        out = torch.zeros(case["seqs"], end, kv, hs, dtype=torch.float64, device=code.device)
        for b, (n, c) in enumerate(zip(lens, new)):
            for first in range(0, n + c, BLOCK):
                pg, blk = table[b][first // page], first % page // BLOCK
                lo, hi = max(n, first), min(n + c, first + BLOCK)
                if lo < hi:  # rows of this block
                    x = st[name + "r"][b, lo - n:hi - n].double().permute(1, 0, 2)
                    want = (x.abs().amax((1, 2)) / TOP[cache]).float().double()
                    for h in range(kv):
                        s, w = float(sc[pg, h, blk]) if lo > first else 0.0, float(want[h])
                        if s > 0.0:
                            while s < w:
                                s *= 2.0
                                code[pg, h, blk] /= 2.0
                            code[pg, h, blk, :lo - first] = _nearest(code[pg, h, blk, :lo - first], cache)
                        else:
                            s = w
                        sc[pg, h, blk] = s
                        code[pg, h, blk, lo - first:hi - first] = _nearest(x[h] / s, cache) if s > 0.0 else 0.0
                m = min(n + c - first, BLOCK)
                out[b, first:first + m] = (code[pg, :, blk, :m] * sc[pg, :, blk][:, None, None]).permute(1, 0, 2)
        got.append(out)
        scales.append(sc)
    return got + scales


def _exact_attend(st):
    case = st["case"]
    heads, kv, hs = HEADS[case["heads"]]
    lens, new = _lengths(case)
    page = case["page"]
    out = torch.zeros(case["seqs"], case["new"], heads, hs, dtype=torch.float64, device=st["q"].device)
    for b, (n, c) in enumerate(zip(lens, new)):
        ids = st["table"][b, :-(-n // page)].long()
        for h in range(kv):
            g = slice(h * (heads // kv), (h + 1) * (heads // kv))
            k = st["k"].view(torch.int8)[ids, h].view(st["k"].dtype).float().double().view(-1, BLOCK, hs)
            v = st["v"].view(torch.int8)[ids, h].view(st["v"].dtype).float().double().view(-1, hs, BLOCK).transpose(1, 2)
            k = (k * st["ks"][ids, h].double().view(-1, 1, 1)).reshape(-1, hs)[:n]
            v = (v * st["vs"][ids, h].double().view(-1, 1, 1)).reshape(-1, hs)[:n]
            k = torch.cat((k, st["kr"][b, :c, h].double()))
            v = torch.cat((v, st["vr"][b, :c, h].double()))
            s = torch.tensordot(st["q"][b, :c, g].double(), k, dims=([2], [1])) / math.sqrt(hs)  # [c, group, n + c]
            seen = torch.ones(c, n + c, dtype=torch.bool, device=s.device)
            for j in range(c):
                seen[:, n + j] = (st["mask"][b, :c] >> j) & 1 != 0
            s[~seen.unsqueeze(1).expand_as(s)] = -math.inf
            out[b, :c, g] = torch.tensordot(torch.softmax(s, -1), v, dims=([2], [0]))
    return out


def _exact_accept(st):
    case = st["case"]
    b, t, v = st["logits"].shape
    temp = float(np.float32(case["temperature"]))
    kept, drawn = [], []
    path = torch.full((b, t), -1, dtype=torch.int32)
    logp = torch.zeros(b, t, dtype=torch.float64)
    tokens, n = st["tokens"].tolist(), st["n"].tolist()
    parents = [[i - 1 for i in range(t)]] * b if st["parents"] is None else st["parents"].tolist()
    for s in range(b):
        def probabilities(r):
            x = st["logits"][s, r].double()
            if temp == 0.0:
                first = int(torch.nonzero(x == x.max())[0])
                return torch.nn.functional.one_hot(torch.tensor(first, device=x.device), v).double()
            return torch.softmax(x / temp, -1)
        for i in range(1, n[s]):
            p = probabilities(parents[s][i])[tokens[s][i]]
            logp[s, i] = torch.log(p)
        node, way, turned = 0, [0], []
        left = target = probabilities(0)
        coins = st["coins"][s].double().tolist()
        while True:
            step = None
            for c in (i for i in range(node + 1, n[s]) if parents[s][i] == node):
                x = tokens[s][c]
                q = 1.0 if st["probs"] is None else float(st["probs"][s, node, x])
                if coins[c] * q < float(left[x]):
                    step = c
                    break
                if st["probs"] is None:
                    turned.append(x)
                    rest = target.clone()
                    rest[turned] = 0.0
                else:
                    rest = (left - st["probs"][s, node].double()).clamp(min=0.0)
                left = rest / rest.sum() if float(rest.sum()) > 0.0 else rest
            if step is None:
                break
            node, turned = step, []
            way.append(node)
            left = target = probabilities(node)
        w = left if float(left.sum()) > 0.0 else target
        c = torch.cumsum(w, 0)
        token = int(torch.searchsorted(c, coins[0] * float(c[-1]), right=True))
        logp[s, 0] = torch.log(target[token])
        kept.append(len(way))
        path[s, :len(way)] = torch.tensor(way, dtype=torch.int32)
        drawn.append(token)
    return torch.tensor(kept, dtype=torch.int32), path, torch.tensor(drawn, dtype=torch.int32), logp


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # (whole numbers, and codes and scales that are copied as they are)
    st = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "accept": _exact_accept}[case["kind"]](st)
