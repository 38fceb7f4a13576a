"""Plain restatements in 64 bits of the speculative-decoding operators (tree
plan, tree attention, draft verification, commit), written from their
definitions, sequence by sequence and node by node; test infrastructure."""

from __future__ import annotations

import math

import numpy as np


def plan(parents):
    """(mask, depth, bad) of [B][N] parents."""
    B, N = len(parents), len(parents[0])
    mask, depth, bad = np.zeros((B, N), np.uint64), np.zeros((B, N), np.int32), False
    for b in range(B):
        line: list = []
        for i, p in enumerate(parents[b]):
            if p >= i:
                bad = True
            up = None if (p < -1 or p >= i) else set() if p < 0 else line[p]
            line.append(None if up is None else up | {i})
        for i, anc in enumerate(line):
            if anc is not None:
                mask[b, i] = sum(1 << j for j in anc)
                depth[b, i] = len(anc) - 1
    return mask.view(np.int64), depth, bad


def visible_keys(mask, s, i, n_nodes, window):
    """Slots that node i of a sequence with s positions sees."""
    bits = [int(m) & ((1 << n_nodes) - 1) for m in mask]
    if bits[i] == 0:
        return []
    pos = s + bin(bits[i]).count("1") - 1
    keys = [t for t in range(s) if not window or t > pos - window]
    for j in range(n_nodes):
        if (bits[i] >> j) & 1:
            at = s + bin(bits[j]).count("1") - 1
            if not window or at > pos - window:
                keys.append(s + j)
    return keys


def attention(q, k, v, seqlen, mask, row_map, scale, window):
    """(out, slack): torch float64 [B, N, H, D] and, for tolerances, per element
    sum_t p_t |v_t| and per row the largest sum_d |q_d k_d| * scale."""
    import torch

    B, N, H, D = q.shape
    Hkv = k.shape[1]
    out = torch.zeros(B, N, H, D, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    reach = torch.zeros(B, N, H, 1, dtype=torch.float64, device=q.device)
    mask = np.asarray(mask, dtype=np.int64).view(np.uint64)
    for b in range(B):
        row = b if row_map is None else int(row_map[b])
        s = int(seqlen[b])
        kd, vd = k[row].double(), v[row].double()
        for i in range(N):
            keys = visible_keys([int(m) for m in mask[b]], s, i, N, window)
            if not keys:
                continue
            at = torch.tensor(keys, device=q.device)
            qi = q[b, i].double().reshape(Hkv, H // Hkv, D)
            kk, vv = kd[:, at], vd[:, at]
            p = torch.softmax(torch.einsum("hgd,htd->hgt", qi, kk) * scale, -1)
            out[b, i] = torch.einsum("hgt,htd->hgd", p, vv).reshape(H, D)
            mass[b, i] = torch.einsum("hgt,htd->hgd", p, vv.abs()).reshape(H, D)
            reach[b, i] = (torch.einsum("hgd,htd->hgt", qi.abs(), kk.abs()).amax(-1) * scale).reshape(H, 1)
    return out, mass, reach


def sampler_weights(logits, temperature, top_p, top_k):
    """(ids, p): the sampler's distribution, ids in order of falling logits."""
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    order = np.argsort(-x, kind="stable")[: min(top_k, len(x))]
    v = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / float(np.float32(temperature))))
    w = w / w.sum()
    before, kept = 0.0, []
    for i, wi in enumerate(w):
        kept.append(wi if before <= float(np.float32(top_p)) else 0.0)
        before += wi
    kept = np.array(kept)
    return order.astype(np.int64), kept / kept.sum()


def verify(logits, tokens, parents, uniform, *, temperature, top_p, top_k, draft=None, replacement=False):
    """(path, n_path, ids) of numpy inputs, by the rejection rule."""
    B, N, V = logits.shape
    path, ids = np.full((B, N), -1, np.int32), np.full((B, N), -1, np.int64)
    n_path = np.zeros(B, np.int32)
    for b in range(B):
        if parents[b][0] < -1:
            continue
        cur, out, way = 0, [], [0]
        cand, p = sampler_weights(logits[b, 0], temperature, top_p, top_k)
        q = None if draft is None else draft[b, 0].astype(np.float64).copy()
        left = 1.0
        for c in range(1, N):
            if parents[b][c] != cur:
                continue
            x = int(tokens[b][c])
            at = np.nonzero(cand == x)[0]
            px = p[at[0]] if len(at) else 0.0
            if q is None:
                qx, qc = 1.0, (cand == x).astype(np.float64)
            else:
                qx = min(q[x] / left, 1.0) if 0 <= x < V else 0.0
                qc = np.minimum(q[cand] / left, 1.0)
            if float(uniform[b][c]) * qx < px:
                out.append(x)
                way.append(c)
                cur, left = c, 1.0
                cand, p = sampler_weights(logits[b, c], temperature, top_p, top_k)
                q = None if draft is None else draft[b, c].astype(np.float64).copy()
                continue
            rest = np.maximum(p - qc, 0.0)
            if rest.sum() > 0:
                p = rest / rest.sum()
            if q is not None and not replacement and 0 <= x < V:
                left = max(left - q[x], 1e-30)
                q[x] = 0.0
        target, cum, pick = float(uniform[b][0]) * math.fsum(p), 0.0, 0
        for w in p:
            cum += w
            pick += cum <= target
        out.append(int(cand[min(pick, int(np.nonzero(p)[0][-1]))]))
        path[b, : len(way)], ids[b, : len(out)], n_path[b] = way, out, len(way)
    return path, n_path, ids


def commit(cache, seqlen, path, n_path, row_map=None):
    """The cache [Bc, n_kv, T, D] after the move (numpy, a copy)."""
    out = cache.copy()
    for b in range(len(n_path)):
        row = b if row_map is None else int(row_map[b])
        for d in range(int(n_path[b])):
            out[row, :, seqlen[b] + d] = cache[row, :, seqlen[b] + path[b][d]]
    return out
