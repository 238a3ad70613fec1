"""Timed cases of the operators on device memory: K and V rows written into a cache of 8 bits and read back (kv_write,
kv_read), attention for a tree of drafted tokens over a cache (tree_attention), and log probabilities of given tokens with
the entropy and the top alternatives (logprobs).

`run` computes them in plain torch in 32 bits where `own` is false, and calls the framework where it is true.  Head
layouts are those of the repository's configurations: Qwen2 0.5B (14 heads, 2 kv heads of 64), Qwen2 7B (28, 4 of 128),
llama2.c 288 (6, 6 of 48) and 768 (12, 12 of 64)."""
import importlib.util
import math
import os

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
BYTES = {"fp32": 4, "bf16": 2, "int8": 1, "e4m3": 1}
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one decode step's rows of a small model: latency
        dict(name="kv_step_0p5b", kind="kv", heads="qwen2-0.5b", cache="int8", rows="fp32", seqs=1, ctx=1024, pos=700,
             new=1, back=1),
        # a prompt's second chunk: 2048 new rows, the whole prefix read back for the chunk's attention
        dict(name="kv_chunk_7b", kind="kv", heads="qwen2-7b", cache="int8", rows="fp32", seqs=1, ctx=8192, pos=5021,
             new=2048, back=7069),
        # many sequences, ragged, 16-bit activations
        dict(name="kv_batch_e4m3", kind="kv", heads="qwen2-7b", cache="e4m3", rows="bf16", seqs=24, ctx=4096, pos=3001,
             new=129, back=517),
        # a decode step early in a dialog: latency
        dict(name="step_0p5b_203", kind="tree", heads="qwen2-0.5b", cache="int8", rows="fp32", seqs=1, ctx=1024,
             pos=203, new=1),
        # a decode step late in a long context
        dict(name="step_7b_32k", kind="tree", heads="qwen2-7b", cache="int8", rows="fp32", seqs=1, ctx=32768,
             pos=32701, new=1),
        # a batch of decode steps, lengths from nothing to 8192, 16-bit activations
        dict(name="step_batch_e4m3", kind="tree", heads="qwen2-7b", cache="e4m3", rows="bf16", seqs=32, ctx=8192,
             pos=8190, new=1),
        # a drafted tree over the framework's own fp32 cache
        dict(name="tree_0p5b_fp32", kind="tree", heads="qwen2-0.5b", cache="fp32", rows="fp32", seqs=1, ctx=4096,
             pos=2950, new=21),
        # a drafted tree over a long int8 cache
        dict(name="tree_7b_int8", kind="tree", heads="qwen2-7b", cache="int8", rows="fp32", seqs=1, ctx=16384,
             pos=12003, new=37),
        # whole trees of 64 for a batch: the largest
        dict(name="tree_batch_bf16", kind="tree", heads="qwen2-7b", cache="bf16", rows="bf16", seqs=8, ctx=16384,
             pos=16000, new=64),
        # one step's logits with its alternatives: latency
        dict(name="logprobs_step_65536", kind="logprobs", rows=1, vocab=65536, given=1, top=20, type="fp32",
             temperature=1.0),
        # a drafted tree's logits: a few rows, several children each
        dict(name="logprobs_tree_bf16", kind="logprobs", rows=37, vocab=151936, given=4, top=5, type="bf16",
             temperature=0.7),
        # a text scored, every position's logits
        dict(name="logprobs_text_151936", kind="logprobs", rows=1021, vocab=151936, given=1, top=10, type="fp32",
             temperature=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["kv", "tree", "tree", "tree", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice([_log(rng, 300, 152064), _log(rng, 300, 152064), 32000, 65536, 151936])
        return dict(kind=kind, rows=_log(rng, 1, min(1021, 90_000_000 // vocab)), vocab=vocab, given=rng.randint(1, 6),
                    top=rng.choice([1, 5, 20, rng.randint(1, 32)]), type=rng.choice(["fp32", "bf16"]),
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.3]))
    heads, seqs = rng.choice(list(HEADS)), rng.choice([1, 1, _log(rng, 1, 32)])
    ctx = _log(rng, 64, min(32768, 131072 // seqs))
    shape = dict(heads=heads, cache=rng.choice(["int8", "int8", "e4m3", "bf16", "fp32"]), rows=rng.choice(["fp32", "bf16"]),
                 seqs=seqs, ctx=ctx)
    if kind == "kv":
        new = _log(rng, 1, min(ctx, 2048))
        pos = rng.randint(0, ctx - new)
        return dict(kind=kind, **shape, pos=pos, new=new, back=rng.randint(new, pos + new))
    new = rng.choice([1, 1, rng.randint(1, 64)])
    new = min(new, ctx // 2)
    return dict(kind=kind, **shape, pos=rng.randint(0, ctx - new), new=new)


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


def _rows(g, shape):
    """Rows as the path meets them: normal, some channels much larger than others."""
    ch = torch.exp(torch.randn(shape[-1], generator=g, device=g.device))
    return torch.randn(shape, generator=g, device=g.device) * ch


def _quantize(x, cache):
    """Codes and scales of rows (the last dimension), the quotient in 64 bits."""
    if cache in ("fp32", "bf16"):
        return x.to(TYPES[cache]), None
    top = 127.0 if cache == "int8" else 448.0
    x = x.double()
    s = (x.abs().amax(-1) / top).float()
    q = x / torch.where(s > 0, s, torch.ones_like(s)).double().unsqueeze(-1)
    q = torch.where((s > 0).unsqueeze(-1), q, torch.zeros_like(q))
    if cache == "int8":
        return torch.round(q).clamp(-127, 127).to(torch.int8), s
    # the distance of e4m3's values around q: its power of two (at least 2^-6), three bits further down
    step = ((((q.view(torch.int64) >> 52) & 2047).clamp(min=1023 - 6) - 3) << 52).view(torch.float64)
    return (torch.round(q / step) * step).clamp(-448, 448).float().to(torch.float8_e4m3fn), s


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    st = dict(case=case)
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        x = torch.randn(n, v, generator=g, device=dev) * 2.5
        hot = torch.randint(0, v, (n, 8), generator=g, device=dev)
        x.scatter_add_(1, hot, torch.rand(n, 8, generator=g, device=dev) * 9.0)
        st["logits"] = x.to(TYPES[case["type"]])
        given = torch.randint(0, v, (n, case["given"]), generator=g, device=dev)
        given[:, :1] = hot[:, :1]
        st["tokens"] = given.int()
        return st
    heads, kv, hs = HEADS[case["heads"]]
    b, t, ctx = case["seqs"], case["new"], case["ctx"]
    lens, new = _lengths(case)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
    for name in ("k", "v"):
        x = _rows(g, (b, kv, ctx, hs))
        if name == "v":
            x = x * 0.1
        st[name], st[name + "s"] = _quantize(x, case["cache"])
    rows = TYPES[case["rows"]]
    if case["kind"] == "kv":
        st["kr"] = _rows(g, (b, t, kv, hs)).to(rows)
        st["vr"] = (_rows(g, (b, t, kv, hs)) * 0.1).to(rows)
        st["from"] = (st["lens"] + st["new"] - case["back"]).clamp(min=0)
        st["count"] = st["lens"] + st["new"] - st["from"]
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


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales.unsqueeze(-1)


def _plain_kv(st):
    case = st["case"]
    dev, t, ctx = st["k"].device, case["new"], case["ctx"]
    step = torch.arange(t, device=dev)
    b, i = torch.nonzero(step < st["new"].unsqueeze(1), as_tuple=True)
    at = (st["lens"].long()[b] + i)
    out = []
    back = torch.arange(case["back"], device=dev)
    have = (back < st["count"].unsqueeze(1))
    where = (st["from"].long().unsqueeze(1) + back).clamp(max=ctx - 1)
    seq = torch.arange(case["seqs"], device=dev).unsqueeze(1)
    for name in ("k", "v"):
        codes, s = _quantize(st[name + "r"][b, i], case["cache"])
        store = st[name] if s is None or case["cache"] == "int8" else st[name].view(torch.int8)
        store[b, :, at] = codes if store is st[name] else codes.view(torch.int8)
        if s is not None:
            st[name + "s"][b, :, at] = s
        got = store[seq, :, where]  # [seqs, back, kv, hs]
        got = _values(got if store is st[name] else got.view(torch.float8_e4m3fn),
                      None if s is None else st[name + "s"][seq, :, where])
        out.append(torch.where(have[:, :, None, None], got, torch.zeros_like(got)))
    return out + [x for x in (st["ks"], st["vs"]) if x is not None]


def _plain_tree(st):
    case = st["case"]
    heads, kv, hs = HEADS[case["heads"]]
    b, t, end = case["seqs"], case["new"], case["pos"] + case["new"]
    dev = st["q"].device
    k = _values(st["k"][:, :, :end], None if st["ks"] is None else st["ks"][:, :, :end])
    v = _values(st["v"][:, :, :end], None if st["vs"] is None else st["vs"][:, :, :end])
    q = st["q"].float().view(b, t, kv, heads // kv, hs).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hs)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(hs))  # [b, kv, group t, end]
    at = torch.arange(end, device=dev)
    lens = st["lens"].long().view(b, 1, 1)
    node = at.view(1, 1, end) - lens  # [b, 1, end]
    bit = (st["mask"].unsqueeze(-1) >> node.clamp(0, 63)) & 1
    sees = (node < 0) | ((node < st["new"].view(b, 1, 1)) & (bit != 0))
    live = torch.arange(t, device=dev) < st["new"].unsqueeze(1)  # [b, t]
    sees = (sees & live.unsqueeze(-1)).unsqueeze(1).unsqueeze(1)
    s = s.view(b, kv, heads // kv, t, end).masked_fill(~sees, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z > 0, z, torch.ones_like(z))).view(b, kv, -1, end)
    o = torch.matmul(p, v).view(b, kv, heads // kv, t, hs).permute(0, 3, 1, 2, 4).reshape(b, t, heads, hs)
    return o.to(st["q"].dtype)


def _plain_logprobs(st):
    case = st["case"]
    x = st["logits"].float()
    y = x / case["temperature"]
    m = y.amax(-1, keepdim=True)
    e = torch.exp(y - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    entropy = torch.log(z.squeeze(-1)) - (e / z * (y - m)).sum(-1)
    logp = torch.gather(y, 1, st["tokens"].long()) - lse
    top = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]
    return logp, entropy, top.int(), torch.gather(y, 1, top) - lse, lse.squeeze(-1)


def run(state):
    case = state["case"]
    if not own:
        return {"kv": _plain_kv, "tree": _plain_tree, "logprobs": _plain_logprobs}[case["kind"]](state)
    P = _own()
    if case["kind"] == "kv":
        P.kv_write(state["kr"], state["vr"], state["k"], state["v"], state["lens"], state["new"],
                   k_scale=state["ks"], v_scale=state["vs"])
        k, v = P.kv_read(state["k"], state["v"], state["from"], case["back"], state["count"],
                         k_scale=state["ks"], v_scale=state["vs"])
        return [k, v] + [x for x in (state["ks"], state["vs"]) if x is not None]
    if case["kind"] == "tree":
        return P.tree_attention(state["q"], state["k"], state["v"], state["lens"], state["new"], state["mask"],
                                k_scale=state["ks"], v_scale=state["vs"], max_len=case["pos"])
    return P.logprobs(state["logits"], state["tokens"], case["top"], temperature=case["temperature"])


def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * BYTES[case["type"]] + case["rows"] * (8 * case["given"] + 8 * case["top"] + 8),
                "flops": 5 * n}
    heads, kv, hs = HEADS[case["heads"]]
    lens, new = _lengths(case)
    row = kv * (hs * BYTES[case["cache"]] + (4 if case["cache"] in ("int8", "e4m3") else 0))
    act = BYTES[case["rows"]]
    if case["kind"] == "kv":
        back = sum(min(n + c, case["back"]) for n, c in zip(lens, new))
        old = sum(max(0, min(n + c, case["back"]) - c) for n, c in zip(lens, new))
        return {"bytes": 2 * (sum(new) * (kv * hs * act + row) + old * row + back * kv * hs * 4),
                "flops": 2 * kv * hs * (4 * sum(new) + back)}
    return {"bytes": sum(2 * (n + c) * row + 2 * c * heads * hs * act + 8 * c for n, c in zip(lens, new)),
            "flops": sum(4 * heads * hs * c * (n + 1) for n, c in zip(lens, new))}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        x = st["logits"].double()
        rows = torch.arange(x.shape[0], device=x.device).unsqueeze(1)
        lse = torch.logsumexp(x / case["temperature"], -1)
        lp = x / case["temperature"] - lse.unsqueeze(-1)
        entropy = -(torch.exp(lp) * lp).sum(-1)
        order = torch.argsort(-x, dim=-1, stable=True)[:, :case["top"]]
        return lp[rows, st["tokens"].long()], entropy, order.int(), lp[rows, order], lse
    heads, kv, hs = HEADS[case["heads"]]
    lens, new = _lengths(case)
    if case["kind"] == "kv":
        out = []
        top = {"int8": 127.0, "e4m3": 448.0}.get(case["cache"])
        scales = []
        for name in ("k", "v"):
            val = st[name].float().double()
            sc = None if top is None else st[name + "s"].double()
            if sc is not None:
                val = val * sc.unsqueeze(-1)
            got = torch.zeros(case["seqs"], case["back"], kv, hs, dtype=torch.float64, device=val.device)
            for b, (n, c) in enumerate(zip(lens, new)):
                x = st[name + "r"][b, :c].double().permute(1, 0, 2)  # [kv, c, hs]
                if top is None:
                    val[b, :, n:n + c] = x.to(TYPES[case["cache"]]).double()
                else:
                    # the scale is held in 32 bits, and a code is the nearest of the type's values
                    s = (x.abs().max(-1)[0] / top).float().double()
                    u = x / s.unsqueeze(-1)
                    if case["cache"] == "int8":
                        u = torch.round(u)
                    else:
                        every = torch.arange(127, dtype=torch.uint8, device=u.device).view(torch.float8_e4m3fn).double()
                        mid = (every[1:] + every[:-1]) / 2.0
                        i = torch.bucketize(u.abs().contiguous(), mid)
                        tie = (i < 126) & (u.abs() == mid[i.clamp(max=125)]) & (i % 2 == 1)
                        u = torch.sign(u) * every[i + tie.long()]
                    val[b, :, n:n + c] = u * s.unsqueeze(-1)
                    sc[b, :, n:n + c] = s
                m = min(n + c, case["back"])
                got[b, :m] = val[b, :, n + c - m:n + c].permute(1, 0, 2)
            out.append(got)
            scales += [] if sc is None else [sc]
        return out + scales
    out = torch.zeros(case["seqs"], case["new"], heads, hs, dtype=torch.float64, device=st["q"].device)
    for b, (n, c) in enumerate(zip(lens, new)):
        for h in range(kv):
            g = slice(h * (heads // kv), (h + 1) * (heads // kv))
            k, v = (st[x][b, h, :n + c].float().double() * (1.0 if st[x + "s"] is None else
                                                            st[x + "s"][b, h, :n + c].double().unsqueeze(-1))
                    for x in ("k", "v"))
            q = st["q"][b, :c, g].double()
            s = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(hs)  # [c, group, n + c]
            seen = torch.ones(c, n + c, dtype=torch.bool, device=q.device)
            for j in range(c):
                seen[:, n + j] = (st["mask"][b, :c] >> j) & 1 != 0
            s[~seen.unsqueeze(1).expand_as(s)] = -math.inf
            out[b, :c, g] = torch.tensordot(torch.softmax(s, -1), v, dims=([2], [0]))
    return out
