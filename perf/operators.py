"""What the speculative-decoding operators are timed on: cases, inputs, and their plain forms.

``run`` computes one pass: with ``own`` false in elementary torch operations (32 bits; 64 where a comparison decides
which token comes out), with ``own`` true by the calls a user makes of ``maple_flash_dgx_spark_b200.kernels``.  The
sizes are the benchmark architecture's (48 layers, 32 query and 4 KV heads of 128, vocabulary 151936) and its
workloads' (one sequence of some hundred positions, 64 sequences of 8192, one of 65536).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_ES = {"bf16": 2, "f32": 4}
VOCAB = 151936


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # the smallest plan, one sequence with a short draft: latency
        {"name": "plan-1x8", "op": "plan", "B": 1, "N": 8, "chain": False},
        # the plan of a full server batch with the largest trees
        {"name": "plan-256x64", "op": "plan", "B": 256, "N": 64, "chain": False},
        # one user, a chain of four drafted tokens after a short prompt: latency
        {"name": "attn-chain-1x600", "op": "attn", "B": 1, "N": 5, "H": 32, "Hkv": 4, "D": 128, "T": 640, "len": 600,
         "window": 0, "dtype": "bf16", "chain": True, "ragged": False},
        # sixteen users at different points of their answers, a sliding-window layer, an odd tree
        {"name": "attn-window-16x4000", "op": "attn", "B": 16, "N": 13, "H": 32, "Hkv": 4, "D": 128, "T": 4096,
         "len": 4000, "window": 512, "dtype": "bf16", "chain": False, "ragged": True},
        # the batch-64 decode workload with a tree of eight: bound by the cache's bytes
        {"name": "attn-tree-64x8192", "op": "attn", "B": 64, "N": 8, "H": 32, "Hkv": 4, "D": 128, "T": 8192,
         "len": 8150, "window": 0, "dtype": "bf16", "chain": False, "ragged": False},
        # the long-context workload with the largest tree: bound by the products
        {"name": "attn-tree-1x65536", "op": "attn", "B": 1, "N": 64, "H": 32, "Hkv": 4, "D": 128, "T": 65536,
         "len": 65440, "window": 0, "dtype": "bf16", "chain": False, "ragged": False},
        # a small fp32 model with heads of 64, ragged
        {"name": "attn-f32-4x1500", "op": "attn", "B": 4, "N": 17, "H": 16, "Hkv": 2, "D": 64, "T": 1536, "len": 1500,
         "window": 0, "dtype": "f32", "chain": False, "ragged": True},
        # greedy decoding of one user with a looked-up draft
        {"name": "verify-greedy-1x5", "op": "verify", "B": 1, "N": 5, "V": VOCAB, "dtype": "bf16", "top_k": 1,
         "top_p": 1.0, "temperature": 1.0, "draft": "none", "chain": True, "replacement": False},
        # sampled decoding of sixteen users, trees of 24 tokens picked by a draft's scores
        {"name": "verify-tree-16x24", "op": "verify", "B": 16, "N": 24, "V": VOCAB, "dtype": "bf16", "top_k": 20,
         "top_p": 0.95, "temperature": 1.0, "draft": "none", "chain": False, "replacement": False},
        # the batch-64 workload, chains drawn from a draft model's probabilities
        {"name": "verify-draft-64x8", "op": "verify", "B": 64, "N": 8, "V": VOCAB, "dtype": "bf16", "top_k": 50,
         "top_p": 0.9, "temperature": 0.8, "draft": "f32", "chain": True, "replacement": False},
        # one user's accepted rows of all 48 layers
        {"name": "commit-1x8", "op": "commit", "B": 1, "N": 8, "L": 48, "Hkv": 4, "D": 128, "T": 640, "len": 600,
         "dtype": "bf16"},
        # sixteen users' accepted rows of all 48 layers, larger trees
        {"name": "commit-16x32", "op": "commit", "B": 16, "N": 32, "L": 48, "Hkv": 4, "D": 128, "T": 512, "len": 470,
         "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "attn", "attn", "attn", "verify", "verify", "commit"])
    if op == "plan":
        return {"op": op, "B": _spread(rng, 1, 256), "N": _spread(rng, 1, 64), "chain": rng.random() < 0.2}
    if op == "attn":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        D = rng.choice([64, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 2, 4, 5, 8])
        N, length = _spread(rng, 1, 64), _spread(rng, 1, 65000)
        most = (8 if dtype == "bf16" else 1) << 26  # cache elements of one K or V, and rows times keys
        B = _spread(rng, 1, max(1, min(64, most // (Hkv * (length + 200) * D), (most // 4) // (H * N * (length + 200)))))
        return {"op": op, "B": B, "N": N, "H": H, "Hkv": Hkv, "D": D, "T": length + N + rng.randrange(0, 100),
                "len": length, "window": rng.choice([0, 0, 0, _spread(rng, 16, 2048)]), "dtype": dtype,
                "chain": rng.random() < 0.3, "ragged": rng.random() < 0.5}
    if op == "verify":
        N = _spread(rng, 1, 64)
        V = rng.choice([VOCAB, _spread(rng, 1000, VOCAB)])
        draft = rng.choice(["none", "f32", "bf16"])
        B = _spread(rng, 1, max(1, min(64, 512 * VOCAB // (N * V))))
        return {"op": op, "B": B, "N": N, "V": V, "dtype": rng.choice(["bf16", "f32"]),
                "top_k": rng.choice([1, _spread(rng, 2, 64), _spread(rng, 2, 64)]),
                "top_p": round(rng.uniform(0.5, 1.0), 3), "temperature": round(rng.uniform(0.3, 1.5), 3),
                "draft": draft, "chain": rng.random() < 0.4, "replacement": rng.random() < 0.3}
    N = _spread(rng, 1, 64)
    length = _spread(rng, 1, 2000)
    Hkv, D, dtype = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice(["bf16", "bf16", "f32"])
    L = _spread(rng, 1, 64)
    B = _spread(rng, 1, max(1, min(32, (1 << 29) // (L * Hkv * (length + 200) * D * _ES[dtype]))))
    return {"op": op, "B": B, "N": N, "L": L, "Hkv": Hkv, "D": D, "T": length + N + rng.randrange(0, 100),
            "len": length, "dtype": dtype}


# ------------------------------------------------- sizes fixed by a case --
def _lens(case):
    """Cached positions of each sequence (fixed by the case, so that its work is)."""
    if not case.get("ragged"):
        return [case["len"]] * case["B"]
    r = random.Random(case["B"] * 7919 + case["len"])
    return [max(1, min(case["len"], int(case["len"] * r.uniform(0.05, 1.0)))) for _ in range(case["B"])]


def _trees(case, seed):
    """Parents [B][N]: chains or random trees with about a third of the nodes on the trunk; ragged cases end some
    sequences' trees early (padding: -2)."""
    r = random.Random(seed * 1000003 + 17)
    rows = []
    for _ in range(case["B"]):
        n = case["N"] if not case.get("ragged") else r.randint(max(1, case["N"] // 2), case["N"])
        rows.append([-1] + [i - 1 if case.get("chain") or r.random() < 0.3 else r.randrange(max(0, i - 12), i)
                            for i in range(1, n)] + [-2] * (case["N"] - n))
    return rows


def _kept(case):
    """How many nodes of each sequence are accepted (fixed by the case), the root among them."""
    r = random.Random(case["B"] * 31 + case["N"])
    return [r.randint(1, min(case["N"], 8)) for _ in range(case["B"])]


def work(case):
    B, N = case["B"], case["N"]
    if case["op"] == "plan":
        return {"bytes": B * N * 16, "flops": B * N}
    if case["op"] == "attn":
        es, W = _ES[case["dtype"]], case["window"]
        keys = [min(n, W) + N if W else n + N for n in _lens(case)]  # rows of K and of V that some node sees
        kv = 2 * sum(keys) * case["Hkv"] * case["D"] * es
        qo = 2 * B * N * case["H"] * case["D"] * es
        return {"bytes": kv + qo + B * (8 + 8 * N), "flops": 4 * case["H"] * N * sum(keys) * case["D"]}
    if case["op"] == "verify":
        probs = 0 if case["draft"] == "none" else B * N * case["top_k"] * _ES[case["draft"]]
        return {"bytes": B * N * case["V"] * _ES[case["dtype"]] + probs + B * N * (4 + 8 + 4) + B * N * 12,
                "flops": B * N * case["V"]}
    rows = sum(_kept(case)) - B  # the root stays in its place
    return {"bytes": max(2 * rows * case["L"] * 2 * case["Hkv"] * case["D"] * _ES[case["dtype"]], 1) + B * N * 4,
            "flops": 0}


# ----------------------------------------------------------------- inputs --
def _masks(parents):
    """Ancestor masks (python whole numbers, as signed 64-bit words) of each tree."""
    rows = []
    for row in parents:
        m = []
        for i, p in enumerate(row):
            m.append(0 if p < -1 else (1 << i) | (m[p] if p >= 0 else 0))
        rows.append([v - (1 << 64) if v >> 63 else v for v in m])
    return rows


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    B, N = case["B"], case["N"]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.empty(*shape, device=dev, dtype=dtype).normal_(0.0, scale, generator=g)

    st = {"case": case}
    if case["op"] != "commit":
        trees = _trees(case, seed)
        st["parents"] = torch.tensor(trees, dtype=torch.int32, device=dev)
    if case["op"] == "attn":
        dt, D = _DT[case["dtype"]], case["D"]
        # queries and keys leave an RMS norm (unit variance); a trained model's q.k spreads wider than chance
        st["q"] = normal(B, N, case["H"], D, scale=2.0, dtype=dt)
        st["k"] = normal(B, case["Hkv"], case["T"], D, dtype=dt)
        st["v"] = normal(B, case["Hkv"], case["T"], D, dtype=dt)
        st["seqlen"] = torch.tensor(_lens(case), dtype=torch.int64, device=dev)
        rows = list(range(B))
        random.Random(seed + 5).shuffle(rows)  # a server's slots are permuted as sequences leave
        st["row_map"] = torch.tensor(rows, dtype=torch.int32, device=dev)
        st["mask"] = torch.tensor(_masks(trees), dtype=torch.int64, device=dev)
        st["scale"] = D ** -0.5
    elif case["op"] == "verify":
        V, T = case["V"], case["temperature"]
        st["logits"] = normal(B, N, V, scale=2.5, dtype=_DT[case["dtype"]])
        st["uniform"] = torch.rand(B, N, device=dev, generator=g)
        tokens = torch.zeros(B, N, dtype=torch.int64, device=dev)
        draft = torch.empty(B, N, V, device=dev, dtype=_DT[case["draft"]]) if case["draft"] != "none" else None
        for b in range(B):
            par = st["parents"][b].clamp(min=0).long()
            # the draft's view of each node: the target's logits, blurred
            score = st["logits"][b].float() / T
            score.add_(torch.randn(N, V, device=dev, generator=g), alpha=0.3)
            gumbel = torch.empty(N, V, device=dev).exponential_(generator=g).log_().neg_()
            if draft is not None:
                top = torch.topk(score, min(40, V), dim=-1).values[:, -1:]
                draft[b] = torch.softmax(score.masked_fill(score < top, float("-inf")), -1).to(draft.dtype)
                seen = draft[b].float().log()
                tokens[b] = (seen[par] + gumbel).argmax(-1)
            else:
                tokens[b] = (2.0 * score[par] + 0.5 * gumbel).argmax(-1)
        st["tokens"], st["draft"] = tokens, draft
    elif case["op"] == "commit":
        shape = (case["L"], 2, B, case["Hkv"], case["T"], case["D"])
        st["cache"] = normal(*shape, dtype=_DT[case["dtype"]])
        if own:  # the layers' caches, looked over once when the cache is made
            from maple_flash_dgx_spark_b200 import kernels

            st["rows"] = kernels.CacheRows([st["cache"][i, 0] for i in range(case["L"])],
                                           [st["cache"][i, 1] for i in range(case["L"])])
        r = random.Random(seed * 13 + 1)
        kept = _kept(case)
        path = [[0] + sorted(r.sample(range(1, N), n - 1)) + [-1] * (N - n) for n in kept]
        st["path"] = torch.tensor(path, dtype=torch.int32, device=dev)
        st["n_path"] = torch.tensor(kept, dtype=torch.int32, device=dev)
        st["seqlen"] = torch.full((B,), case["len"], dtype=torch.int64, device=dev)
    return st


# ------------------------------------------------------------ plain forms --
def _popcount(m):
    bits = (m.unsqueeze(-1) >> torch.arange(64, device=m.device)) & 1
    return bits.sum(-1)


def _plain_plan(st):
    par = st["parents"].long()
    B, N = par.shape
    ids = torch.arange(N, device=par.device)
    see = torch.eye(N, dtype=torch.bool, device=par.device).expand(B, N, N) & (par >= -1)[:, :, None]
    up = torch.where(par >= 0, par, ids)
    for _ in range(6):  # ancestors within 2, 4, .. 64 steps
        see = see | torch.gather(see, 1, up[:, :, None].expand(B, N, N))
        up = torch.gather(up, 1, up)
    mask = (see.long() << ids).sum(-1)
    depth = (see.sum(-1) - 1).clamp(min=0).int()
    return mask, depth


def _visible(mask, seqlen, n_keys, window):
    """[B, N, n_keys]: whether node i sees key t (cached positions, then the nodes)."""
    B, N = mask.shape
    t = torch.arange(n_keys, device=mask.device)[None, None, :]
    s = seqlen[:, None, None]
    j = (t - s).clamp(0, N - 1).expand(B, N, n_keys)
    depth = _popcount(mask) - 1
    pos = s + depth[:, :, None]
    node = ((mask[:, :, None] >> j) & 1 == 1) & (t >= s) & (t < s + N)
    key_pos = torch.where(t < s, t, s + torch.gather(depth[:, None, :].expand(B, N, N), 2, j))
    vis = ((t < s) | node) & (mask != 0)[:, :, None]
    return vis & (key_pos > pos - window) if window else vis


def _plain_attn(st):
    c = st["case"]
    B, N, H, Hkv, D = c["B"], c["N"], c["H"], c["Hkv"], c["D"]
    n_keys = min(c["T"], c["len"] + N)
    row = st["row_map"].long()
    k, v = st["k"][row, :, :n_keys].float(), st["v"][row, :, :n_keys].float()
    q = st["q"].float().reshape(B, N, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st["scale"]).reshape(B, Hkv, H // Hkv, N, n_keys)
    s.masked_fill_(~_visible(st["mask"], st["seqlen"], n_keys, c["window"])[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, -1, n_keys), v).reshape(B, Hkv, H // Hkv, N, D) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(st["q"].dtype)


def _plain_verify(st):
    c = st["case"]
    B, N, V = c["B"], c["N"], c["V"]
    K, dev = min(c["top_k"], V), st["logits"].device
    val, ids = torch.sort(st["logits"].reshape(B * N, V), dim=-1, descending=True, stable=True)
    val, ids = val[:, :K].double().reshape(B, N, K), ids[:, :K].reshape(B, N, K)
    temperature, top_p = (float(np.float32(c[x])) for x in ("temperature", "top_p"))  # fp32 arguments
    w = ((val - val[..., :1]) * (1.0 / temperature)).exp()
    w = w / w.sum(-1, keepdim=True)
    before = w.cumsum(-1) - w
    w = torch.where(before <= top_p, w, 0.0)
    w = w / w.sum(-1, keepdim=True)
    q_all = None if st["draft"] is None else torch.gather(st["draft"], 2, ids).double()
    at = torch.arange(B, device=dev)
    cur = torch.zeros(B, dtype=torch.int64, device=dev)
    p, idp = w[:, 0], ids[:, 0]
    q = q_all[:, 0] if q_all is not None else None
    par, tok, u = st["parents"].long(), st["tokens"], st["uniform"].double()
    live = par[:, 0] >= -1
    path = torch.full((B, N), -1, dtype=torch.int32, device=dev)
    out = torch.full((B, N), -1, dtype=torch.int64, device=dev)
    path[:, 0] = torch.where(live, 0, -1)
    n_path = live.int()
    left = torch.ones(B, dtype=torch.float64, device=dev)  # draft probability of the tokens not yet refused
    # whether an earlier sibling carries the same token: refused then, and drawn without replacement not there to draw
    twin = (par[:, :, None] == par[:, None, :]) & (tok[:, :, None] == tok[:, None, :])
    again = twin.tril(-1).any(-1) if not c["replacement"] else torch.zeros_like(par, dtype=torch.bool)
    for i in range(1, N):
        child = live & (par[:, i] == cur)
        x = tok[:, i]
        hit = idp == x[:, None]
        px = (p * hit).sum(-1)
        if q is None:
            qx, qn = torch.ones_like(px), hit.double()
        else:
            raw = torch.where(again[:, i], 0.0, st["draft"][at, cur, x].double())
            qx, qn = (raw / left).clamp(max=1), (q / left[:, None]).clamp(max=1)
        take = child & (u[:, i] * qx < px)
        drop = child & ~take
        rest = (p - qn).clamp(min=0)
        total = rest.sum(-1, keepdim=True)
        rest = torch.where(total > 0, rest / total.clamp(min=1e-300), p)
        p = torch.where(drop[:, None], rest, p)
        if q is not None and not c["replacement"]:
            q = torch.where(drop[:, None] & hit, 0.0, q)
            left = torch.where(drop, (left - raw).clamp(min=1e-30), left)
        cur = torch.where(take, i, cur)
        p = torch.where(take[:, None], w[:, i], p)
        idp = torch.where(take[:, None], ids[:, i], idp)
        if q is not None:
            q = torch.where(take[:, None], q_all[:, i], q)
            left = torch.where(take, 1.0, left)
        out[at, (n_path.long() - 1).clamp(min=0)] = torch.where(take, x, out[at, (n_path.long() - 1).clamp(min=0)])
        path[at, n_path.long().clamp(max=N - 1)] = torch.where(take, i, path[at, n_path.long().clamp(max=N - 1)])
        n_path = n_path + take.int()
    cum = p.cumsum(-1)
    pick = (cum <= u[:, :1] * cum[:, -1:]).sum(-1)
    last = (torch.where(p > 0, torch.arange(K, device=dev), 0)).amax(-1)
    nxt = torch.gather(idp, 1, torch.minimum(pick, last)[:, None])[:, 0]
    end = (n_path.long() - 1).clamp(min=0)
    out[at, end] = torch.where(live, nxt, out[at, end])
    return path, n_path, out


def _plain_commit(st):
    c, cache = st["case"], st["cache"]
    d = torch.arange(c["N"], device=cache.device)
    src = torch.where(d < st["n_path"][:, None], st["path"].long(), d) + st["seqlen"][:, None]
    at = torch.arange(c["B"], device=cache.device)[:, None]
    cache[:, :, at, :, st["seqlen"][:, None] + d] = cache[:, :, at, :, src]
    return cache


def run(st):
    c = st["case"]
    if own:
        from maple_flash_dgx_spark_b200 import kernels

        if c["op"] == "plan":
            plan = kernels.tree_plan(st["parents"])
            return plan.mask, plan.depth
        if c["op"] == "attn":
            return kernels.tree_gqa_attn(st["q"], st["k"], st["v"], st["seqlen"], st["mask"], row_map=st["row_map"],
                                         scale=st["scale"], window=c["window"] or None)
        if c["op"] == "verify":
            return kernels.verify_tree(st["logits"], st["tokens"], st["parents"], st["uniform"],
                                       temperature=c["temperature"], top_p=c["top_p"], top_k=c["top_k"],
                                       draft_probs=st["draft"], replacement=c["replacement"])
        kernels.commit_tree(st["rows"], st["seqlen"], st["path"], st["n_path"])
        return st["cache"]
    return {"plan": _plain_plan, "attn": _plain_attn, "verify": _plain_verify, "commit": _plain_commit}[c["op"]](st)


# ------------------------------------------------------- exact, in 64 bits --
def exact(case, seed):
    """The attention by its definition in 64 bits, node by node; the rows moved one by one.  The other operators give
    whole numbers."""
    if case["op"] not in ("attn", "commit"):
        return None
    st = prepare(case, seed)
    if case["op"] == "commit":
        cache, path = st["cache"].double(), st["path"].tolist()
        for b, n in enumerate(st["n_path"].tolist()):
            for d in range(n):
                cache[:, :, b, :, case["len"] + d] = cache[:, :, b, :, case["len"] + path[b][d]].clone()
        return cache
    B, N, H, Hkv, D = case["B"], case["N"], case["H"], case["Hkv"], case["D"]
    if B * N > 2000:
        return None
    out = torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda")
    parents, W = st["parents"].tolist(), case["window"]
    for b, (n, row) in enumerate(zip(_lens(case), st["row_map"].tolist())):
        k, v = st["k"][row].double(), st["v"][row].double()
        depth = []
        for i, p in enumerate(parents[b]):
            depth.append(0 if p == -1 else depth[p] + 1 if p >= 0 else -1)
            if p < -1:
                continue
            line, j = [], i
            while j >= 0:
                if not W or depth[i] - depth[j] < W:
                    line.append(n + j)
                j = parents[b][j]
            first = max(0, n + depth[i] - W + 1) if W else 0
            keys = torch.tensor(list(range(first, n)) + line, device="cuda")
            qi = st["q"][b, i].double().reshape(Hkv, H // Hkv, D)
            p_ = torch.softmax(torch.einsum("hgd,htd->hgt", qi, k[:, keys]) * st["scale"], -1)
            out[b, i] = torch.einsum("hgt,htd->hgd", p_, v[:, keys]).reshape(H, D)
    return out
