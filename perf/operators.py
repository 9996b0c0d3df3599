"""Cases of the speculative-decoding operators: what is timed and compared, in a plain form and in the framework's.

One speculative step drafts a tree of tokens, rotates and appends its keys and values (``rope_append``), attends
from every node to the cached context and its own ancestors (``tree_attention``), walks the tree against the
target's distributions (``verify_tree``) and moves the accepted path's keys and values into place (``commit_path``).

``own`` false: ``run`` computes an operator with elementary torch operations in 32 bits.  ``own`` true: ``run`` calls
``nurostream_b200.spec``.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one decoded token of the 64-head / 8-kv-head, 64-wide fp32 model that the framework decodes
        dict(name="rope token", op="rope", B=1, T=1, hq=64, hkv=8, hd=64, rot=64, inter=False, tree=False, len=2048,
             ctx=2112, dt="f32", cache="f32"),
        # a batch of drafted trees, part of the head rotated in pairs of neighbours, some sequences with fewer nodes
        dict(name="rope trees", op="rope", B=16, T=33, hq=64, hkv=8, hd=128, rot=64, inter=True, tree=True, len=900,
             ctx=1024, dt="bf16", cache="bf16"),
        # two prompts written into the cache (a chain of tokens, no tree)
        dict(name="rope prompts", op="rope", B=2, T=2049, hq=64, hkv=8, hd=128, rot=128, inter=False, tree=False,
             len=1001, ctx=4096, dt="bf16", cache="bf16"),
        # one decoded token of the fp32 model's full-attention layer
        dict(name="attn token", op="attn", B=1, T=1, hq=64, hkv=8, hd=64, tree=False, len=2048, ctx=2112, window=0,
             sinks=True, dt="f32"),
        # a drafted tree in the same layer
        dict(name="attn tree", op="attn", B=1, T=16, hq=64, hkv=8, hd=64, tree=True, len=2048, ctx=2112, window=0,
             sinks=True, dt="f32"),
        # a served batch of uneven contexts with trees of an odd size, 16-bit cache
        dict(name="attn ragged", op="attn", B=8, T=27, hq=64, hkv=8, hd=64, tree=True, len=8191, ctx=8256, window=0,
             sinks=True, dt="bf16"),
        # one long context, a chain of four drafts after the last token
        dict(name="attn long", op="attn", B=1, T=5, hq=64, hkv=8, hd=128, tree=False, len=131071, ctx=131200, window=0,
             sinks=False, dt="bf16"),
        # the largest trees over long contexts
        dict(name="attn big trees", op="attn", B=8, T=64, hq=64, hkv=8, hd=128, tree=True, len=16384, ctx=16512,
             window=0, sinks=False, dt="bf16"),
        # one sequence's chain of drafts copied from its own text (no draft distribution), fp32 logits
        dict(name="verify chain", op="verify", B=1, T=8, V=201088, tree=False, draft=False, dt="f32"),
        # a served batch of trees drawn from a draft model's distributions
        dict(name="verify trees", op="verify", B=16, T=32, V=201088, tree=True, draft=True, dt="bf16"),
        # the accepted path of one sequence, all layers of the fp32 model
        dict(name="commit one", op="commit", L=36, B=1, T=16, hkv=8, hd=64, len=500, ctx=640, dt="f32"),
        # the accepted paths of a served batch
        dict(name="commit batch", op="commit", L=36, B=8, T=64, hkv=8, hd=128, len=500, ctx=640, dt="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "verify", "commit"])
    if op == "rope":
        tree = rng.random() < 0.5
        B = _log(rng, 1, 16)
        T = _log(rng, 1, 64) if tree else max(1, _log(rng, 1, 4098) // B)
        hkv = rng.choice([1, 2, 4, 8])
        hd = rng.choice([64, 80, 96, 128])
        n = _log(rng, 1, 2000)
        return dict(op=op, B=B, T=T, hq=hkv * rng.randint(1, 8), hkv=hkv, hd=hd, rot=rng.choice([hd, hd // 2]),
                    inter=rng.random() < 0.5, tree=tree, len=n, ctx=n + T + rng.randint(1, 64),
                    dt=rng.choice(["f32", "f16", "bf16"]), cache=rng.choice(["f32", "f16", "bf16"]))
    if op == "attn":
        dt = rng.choice(["f32", "f16", "bf16"])
        hkv, rep, hd = rng.choice([1, 2, 4, 8]), rng.randint(1, 8), rng.choice([64, 80, 96, 128])
        B, T = _log(rng, 1, 16), _log(rng, 1, 64)
        # no more work than an eighth of the largest listed case (fp32: a sixty-fourth), nor a longer context than the longest
        most = 8 * 64 * 64 * 16384 * 128 // (64 if dt == "f32" else 8)
        n = max(1, min(_log(rng, 1, 131071), most // (B * T * hkv * rep * hd), (1 << 28) // (B * hkv * hd)))
        return dict(op=op, B=B, T=T, hq=hkv * rep, hkv=hkv, hd=hd, tree=rng.random() < 0.7, len=n,
                    ctx=n + T + rng.randint(1, 64), window=rng.choice([0, 0, 128, _log(rng, 1, 4096)]),
                    sinks=rng.random() < 0.5, dt=dt)
    if op == "verify":
        V = rng.choice([_log(rng, 1000, 201088), 201088])
        B = _log(rng, 1, 16)
        return dict(op=op, B=B, T=_log(rng, 1, 32), V=V, tree=rng.random() < 0.6, draft=rng.random() < 0.5,
                    dt=rng.choice(["f32", "f16", "bf16"]))
    n = _log(rng, 1, 500)
    T = _log(rng, 2, 64)
    return dict(op=op, L=rng.choice([1, 24, 36, 48]), B=_log(rng, 1, 8), T=T, hkv=rng.choice([2, 4, 8]),
                hd=rng.choice([64, 80, 128]), len=n, ctx=n + T + rng.randint(0, 32), dt=rng.choice(["f32", "f16", "bf16"]))


# ------------------------------------------------------------------------------------------------ inputs


def _lens(case):
    """Uneven contexts: from the case's length down to half of it."""
    B, n = case["B"], case["len"]
    return [n - (n * b) // (2 * B) for b in range(B)]


def _nodes(case):
    """Used nodes of each sequence's tree: every third sequence of a batch has fewer."""
    T = case["T"]
    return [T if b % 3 != 2 else max(1, T - T // 4) for b in range(case["B"])]


def _parents(case, gen):
    """Trees in topological order: node 0 is the root, each other node hangs on one of the six before it; -2: unused."""
    if not case["tree"]:
        return None
    B, T = case["B"], case["T"]
    t = torch.arange(T)
    back = (torch.rand(B, T, generator=gen) * t.clamp(max=6)).long().clamp(max=5)
    p = torch.where(t > 0, t - 1 - back, t - 1)
    used = t < torch.tensor(_nodes(case))[:, None]
    return torch.where(used, p, p.new_full((), -2)).to(torch.int32).to(_DEV)


def _randn(gen, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=gen, device=_DEV) * scale).to(dt)


def prepare(case, seed):
    cpu, gen = torch.Generator().manual_seed(seed), torch.Generator(device=_DEV).manual_seed(seed)
    s = dict(case)
    if case["op"] == "verify":
        return _prepare_verify(s, cpu, gen)
    s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=_DEV)
    if case["op"] == "commit":
        L, B, T = case["L"], case["B"], case["T"]
        dt = _DT[case["dt"]]
        s["k"] = _randn(gen, (L, B, case["hkv"], case["ctx"], case["hd"]), dt)
        s["v"] = _randn(gen, (L, B, case["hkv"], case["ctx"], case["hd"]), dt)
        s["caches"] = [(s["k"][i], s["v"][i]) for i in range(L)]
        # a path: node 0, then about a third of the others in ascending order
        keep = torch.rand(B, T, generator=cpu) < 0.35
        keep[:, 0] = True
        order = torch.argsort((~keep).int() * T + torch.arange(T), dim=1)
        n = keep.sum(1, keepdim=True)
        s["path"] = torch.where(torch.arange(T) < n, order, -1).to(torch.int32).to(_DEV)
        s["n_acc"] = (n[:, 0] - 1).to(torch.int32).to(_DEV)
        return s
    B, T, hq, hkv, hd = case["B"], case["T"], case["hq"], case["hkv"], case["hd"]
    dt = _DT[case["dt"]]
    s["parents"] = _parents(case, cpu)
    if case["op"] == "rope":
        half = case["rot"] // 2
        inv = 150000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        inv = torch.where(torch.arange(half) < half // 2, inv, inv / 32.0)  # long-context scaling of the slow half
        a = torch.arange(case["ctx"], dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = (1.35 * a.cos()).float().to(_DEV), (1.35 * a.sin()).float().to(_DEV)
        qkv = _randn(gen, (B, T, hq + 2 * hkv, hd), dt)
        s["q"], s["k"], s["v"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:]
        s["kc"] = _randn(gen, (B, hkv, case["ctx"], hd), _DT[case["cache"]])
        s["vc"] = _randn(gen, (B, hkv, case["ctx"], hd), _DT[case["cache"]])
        s["out"] = torch.empty((B, T, hq, hd), dtype=dt, device=_DEV)
        return s
    s["q"] = _randn(gen, (B, T, hq, hd), dt, 1.5)
    s["kc"] = _randn(gen, (B, hkv, case["ctx"], hd), dt)
    s["vc"] = _randn(gen, (B, hkv, case["ctx"], hd), dt)
    s["sk"] = _randn(gen, (hq,), torch.float32) if case["sinks"] else None
    s["out"] = torch.empty_like(s["q"])
    return s


def _prepare_verify(s, cpu, gen):
    B, T, V = s["B"], s["T"], s["V"]
    s["parents"] = par = _parents(s, cpu)
    t = torch.arange(T, device=_DEV)
    p = (t - 1).expand(B, T) if par is None else par.long()
    # peaked next-token logits: a few dozen likely tokens above a broad floor; the draft's are near the target's
    z = torch.randn(B, T, V, generator=gen, device=_DEV) * 1.5
    z += 18.0 * torch.rand(B, T, V, generator=gen, device=_DEV) * (torch.rand(B, T, V, generator=gen, device=_DEV) < 60.0 / V)
    s["logits"] = z.to(_DT[s["dt"]])
    temp = torch.tensor([(0.7, 1.0, 0.0, 1.3)[b % 4] for b in range(B)], device=_DEV)
    s["temp"] = temp
    d = torch.softmax((z + 0.7 * torch.randn(B, T, V, generator=gen, device=_DEV)) / temp.clamp(min=0.7)[:, None, None], -1)
    s["draft"] = d if s["draft"] else None
    # each node's children: draws without replacement from the draft's distribution at that node, in order
    noise = torch.empty(B, T, V, device=_DEV).exponential_(generator=gen)
    top = (d / noise).topk(min(6, V), -1).indices
    older = (p[:, :, None] == p[:, None, :]) & (t[None, :] < t[:, None])
    rank = older.sum(-1)
    b = torch.arange(B, device=_DEV)[:, None]
    s["tokens"] = top[b, p.clamp(min=0), rank.clamp(max=top.shape[-1] - 1)].to(torch.int32).contiguous()
    s["u"] = torch.rand(B, T, generator=gen, device=_DEV)
    s["race"] = torch.empty(B, V, device=_DEV).exponential_(generator=gen)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _ancestors(parents, B, T):
    """(B, T, T) truth: node t sees node s (itself and its ancestors); unused nodes see and are seen by nothing."""
    if parents is None:
        return torch.ones(T, T, dtype=torch.bool, device=_DEV).tril().expand(B, T, T)
    t = torch.arange(T, device=_DEV)
    step = (parents[:, :, None] == t).float() + torch.eye(T, device=_DEV)
    return (torch.linalg.matrix_power(step, T) > 0) & (parents >= -1)[:, :, None]


def _turn(x, cos, sin, rot, inter):
    x = x.float()
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    c, d = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((c, d), -1).flatten(-2) if inter else torch.cat((c, d), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_rope(s):
    B, T = s["B"], s["T"]
    t = torch.arange(T, device=_DEV)
    if s["parents"] is None:
        depth, used = t.expand(B, T), torch.ones(B, T, dtype=torch.bool, device=_DEV)
    else:
        depth, used = _ancestors(s["parents"], B, T).sum(-1) - 1, s["parents"] >= -1
    pos = (s["lens"][:, None] + depth.clamp(min=0)).long()
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    u = used[:, :, None, None]
    q = torch.where(u, _turn(s["q"], cos, sin, s["rot"], s["inter"]), 0.0)
    k = _turn(s["k"], cos, sin, s["rot"], s["inter"])
    b, slot = torch.arange(B, device=_DEV)[:, None], (s["lens"][:, None] + t).long()
    kc, vc = s["kc"], s["vc"]
    kc[b, :, slot] = torch.where(u, k.to(kc.dtype), kc[b, :, slot])
    vc[b, :, slot] = torch.where(u, s["v"].float().to(vc.dtype), vc[b, :, slot])
    return q.to(s["q"].dtype), kc, vc


def _plain_attn(s):
    B, T, hq, hkv, hd = s["B"], s["T"], s["hq"], s["hkv"], s["hd"]
    span, rep = s["len"] + T, hq // hkv
    k, v = s["kc"][:, :, :span].float(), s["vc"][:, :, :span].float()
    q = s["q"].float().view(B, T, hkv, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, hkv, T * rep, hd)
    x = (q @ k.transpose(-1, -2)) / math.sqrt(hd)
    anc = _ancestors(s["parents"], B, T)
    depth = anc.sum(-1) - 1
    j, n = torch.arange(span, device=_DEV), s["lens"][:, None, None]
    node = (j - n).clamp(0, T - 1).long()
    seen = torch.where(j < n, (depth >= 0)[:, :, None], anc.gather(2, node.expand(B, T, span)) & (j < n + T))
    if s["window"]:
        at = torch.where(j < n, j, n + depth[:, None, :].gather(2, node))
        seen = seen & (n + depth[:, :, None] - at < s["window"])
    seen = seen[:, None, :, None].expand(B, 1, T, rep, span).reshape(B, 1, T * rep, span)
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    if s["sk"] is not None:
        sk = s["sk"].view(1, hkv, 1, rep).expand(B, hkv, T, rep).reshape(B, hkv, T * rep, 1)
        m = torch.maximum(m, sk)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(x - m)
    den = e.sum(-1, keepdim=True)
    if s["sk"] is not None:
        den = den + torch.exp(sk - m)
    o = (e @ v) / torch.where(den == 0, 1.0, den)
    o = o.view(B, hkv, T, rep, hd).permute(0, 2, 1, 3, 4).reshape(B, T, hq, hd)
    return o.to(s["q"].dtype)


def _plain_verify(s):
    B, T, V = s["B"], s["T"], s["V"]
    b, t = torch.arange(B, device=_DEV), torch.arange(T, device=_DEV)
    par = (t - 1).expand(B, T) if s["parents"] is None else s["parents"].long()
    tok, greedy = s["tokens"].long(), s["temp"] == 0

    def at(n):
        """The target's distribution at node n: softmax of logits / temperature, or all on the largest logit."""
        x = s["logits"][:, n].float()
        e = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, s["temp"])[:, None])
        hot = (torch.arange(V, device=_DEV) == x.argmax(-1, keepdim=True)).float()
        return torch.where(greedy[:, None], hot, e / e.sum(-1, keepdim=True))

    r = at(0)
    q = s["draft"][:, 0].float() if s["draft"] is not None else None
    cur, n = torch.zeros(B, dtype=torch.long, device=_DEV), torch.zeros(B, dtype=torch.long, device=_DEV)
    path = torch.full((B, T), -1, dtype=torch.long, device=_DEV)
    path[:, 0] = 0
    for c in range(1, T):
        here, x = par[:, c] == cur, tok[:, c:c + 1]
        hot = torch.arange(V, device=_DEV) == x
        one = hot.float() if q is None else q
        one = torch.where(greedy[:, None], hot.float(), one)
        qx, rx = one.gather(1, x)[:, 0], r.gather(1, x)[:, 0]
        yes = here & (s["u"][:, c] * qx < rx)
        no = here & ~yes
        w = (r - one).clamp(min=0)
        z = w.sum(-1, keepdim=True)
        r = torch.where((no[:, None]) & (z > 0), w / z, r)
        r = torch.where(yes[:, None], at(c), r)
        if q is not None:
            left = 1.0 - qx[:, None]
            q = torch.where(no[:, None], torch.where(hot | (left <= 0), 0.0, q / left), q)
            q = torch.where(yes[:, None], s["draft"][:, c].float(), q)
        n = n + yes
        path = torch.where(yes[:, None] & (t == n[:, None]), c, path)
        cur = torch.where(yes, c, cur)
    nxt = torch.where(greedy, r.argmax(-1), (r / s["race"]).argmax(-1))
    return path.to(torch.int32), n.to(torch.int32), nxt.to(torch.int32)


def _plain_commit(s):
    B, T = s["B"], s["T"]
    b, t = torch.arange(B, device=_DEV)[:, None], torch.arange(T, device=_DEV)
    live = (t <= s["n_acc"][:, None])
    to = (s["lens"][:, None] + t).long()
    frm = torch.where(live, s["lens"][:, None] + s["path"], to).long()
    for x in (s["k"], s["v"]):
        x[:, b, :, to] = x[:, b, :, frm]
    return s["k"], s["v"], s["lens"] + 1 + s["n_acc"]


def run(s):
    if own:
        from nurostream_b200 import spec
        if s["op"] == "rope":
            q = spec.rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["kc"], s["vc"], s["lens"], s["parents"],
                                 rotary_dim=s["rot"], interleaved=s["inter"], q_out=s["out"])
            return q, s["kc"], s["vc"]
        if s["op"] == "attn":
            return spec.tree_attention(s["q"], s["kc"], s["vc"], s["lens"], s["parents"], sinks=s["sk"],
                                       window=s["window"], out=s["out"])
        if s["op"] == "verify":
            return spec.verify_tree(s["tokens"], s["logits"], s["u"], s["race"], s["parents"], draft_probs=s["draft"],
                                    temperature=s["temp"])
        return s["k"], s["v"], spec.commit_path(s["caches"], s["lens"], s["path"], s["n_acc"])
    return {"rope": _plain_rope, "attn": _plain_attn, "verify": _plain_verify, "commit": _plain_commit}[s["op"]](s)


# ------------------------------------------------------------------------------------------------ work


def work(case):
    B, T = case["B"], case["T"]
    if case["op"] == "rope":
        n = B * T * (case["hq"] + 2 * case["hkv"]) * case["hd"]
        kv = B * T * 2 * case["hkv"] * case["hd"]
        return {"bytes": n * _SIZE[case["dt"]] + (n - kv) * _SIZE[case["dt"]] + kv * _SIZE[case["cache"]]
                + B * T * case["rot"] * 4, "flops": 3 * B * T * (case["hq"] + case["hkv"]) * case["rot"]}
    if case["op"] == "attn":
        # every cached key and value in reach once, queries and outputs once; products with the keys each row sees
        w = case["window"]
        keys = sum(min(n, w - 1) if w else n for n in _lens(case)) + B * T
        e = _SIZE[case["dt"]]
        return {"bytes": keys * 2 * case["hkv"] * case["hd"] * e + 2 * B * T * case["hq"] * case["hd"] * e,
                "flops": 4 * keys * T * case["hq"] * case["hd"]}
    if case["op"] == "verify":
        # the rows of the nodes that the walk stands on (about one accepted draft and the root here; each row's
        # logits, and the draft's row beside it where there is one), and the race of the last
        rows = min(T, 2)
        return {"bytes": B * case["V"] * (rows * (_SIZE[case["dt"]] + (4 if case["draft"] else 0)) + 4),
                "flops": 5 * B * case["V"] * rows}
    n = B * (T / 3.0)
    return {"bytes": 4 * case["L"] * n * case["hkv"] * case["hd"] * _SIZE[case["dt"]], "flops": 0}


# ------------------------------------------------------------------------------------------------ 64 bits


def _depth_list(case, parents):
    """Depth and ancestor set of every used node, one sequence after another (None: an unused node)."""
    out = []
    for b in range(case["B"]):
        p = list(range(-1, case["T"] - 1)) if parents is None else parents[b].tolist()
        seen = []
        for t, up in enumerate(p):
            seen.append(None if up < -1 else {t} | (seen[up] if up >= 0 else set()))
        out.append(seen)
    return out


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    lens = s["lens"].tolist()
    if case["op"] == "commit":
        path, n_acc = s["path"].tolist(), s["n_acc"].tolist()
        k, v = s["k"].double(), s["v"].double()
        for x, src in ((k, s["k"]), (v, s["v"])):
            for b in range(case["B"]):
                for i in range(n_acc[b] + 1):
                    x[:, b, :, lens[b] + i] = src[:, b, :, lens[b] + path[b][i]].double()
        return k, v, None
    if case["op"] == "rope":
        return _exact_rope(case, s, lens)
    trees = _depth_list(case, s["parents"])
    B, T, hkv, hd = case["B"], case["T"], case["hkv"], case["hd"]
    rep = case["hq"] // hkv
    out = torch.zeros(B, T, case["hq"], hd, dtype=torch.float64, device=_DEV)
    for b in range(B):
        n = lens[b]
        see = torch.zeros(T, n + T, dtype=torch.bool)
        for t, up in enumerate(trees[b]):
            if up is None:
                continue
            lo = max(0, n + len(up) - 1 - case["window"] + 1) if case["window"] else 0
            see[t, lo:n] = True
            for a in up:
                see[t, n + a] = not case["window"] or len(up) - len(trees[b][a]) < case["window"]
        see = see.to(_DEV)
        for g in range(hkv):
            keys, vals = s["kc"][b, g, :n + T].double(), s["vc"][b, g, :n + T].double()
            for h in range(g * rep, (g + 1) * rep):
                x = (s["q"][b, :, h].double() @ keys.T) * hd ** -0.5
                x = x.masked_fill(~see, -math.inf)
                if case["sinks"]:
                    x = torch.cat((x, s["sk"][h].double().expand(T, 1)), 1)
                pr = torch.softmax(x, -1)[:, :n + T]
                out[b, :, h] = torch.where(see.any(1, keepdim=True), torch.nan_to_num(pr) @ vals, 0.0)
    return out


def _exact_rope(case, s, lens):
    B, T, r, h = case["B"], case["T"], case["rot"], case["rot"] // 2
    even = torch.arange(r, device=_DEV).view(h, 2) if case["inter"] else torch.arange(r, device=_DEV).view(2, h).T
    first, second = even[:, 0], even[:, 1]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    kc, vc = s["kc"].double(), s["vc"].double()
    qo = torch.zeros_like(q)
    if s["parents"] is None:
        up = [[t + 1 for t in range(T)]] * B
    else:
        up = [[0 if a is None else len(a) for a in seq] for seq in _depth_list(case, s["parents"])]
    for b in range(B):
        live = torch.tensor([t for t in range(T) if up[b][t]], device=_DEV)
        at = torch.tensor([lens[b] + up[b][t] - 1 for t in range(T) if up[b][t]], device=_DEV)
        c, d = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
        for x, kind in ((q, "q"), (k, "k")):
            y = x[b, live].clone()
            y[..., first] = x[b, live][..., first] * c - x[b, live][..., second] * d
            y[..., second] = x[b, live][..., second] * c + x[b, live][..., first] * d
            if kind == "q":
                qo[b, live] = y
            else:
                kc[b, :, lens[b] + live] = y.transpose(0, 1)
        vc[b, :, lens[b] + live] = v[b, live].transpose(0, 1)
    return qo, kc, vc
