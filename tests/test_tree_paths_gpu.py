"""Speculative-decoding operators: the ways through their kernels that only
larger grids take (several items per CTA, joins by a second launch), arguments
at the edge of their types, and the cache's book-keeping around a step."""

from __future__ import annotations

import random

import numpy as np
import pytest

from tests import tree_reference as ref
from tests.test_tree_gpu import (K, attn_case, check_attention, clean_error_word, flags,  # noqa: F401
                                 prefill, run_attn, tiny, trees, verify_attn, verify_inputs)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


# -------------------------------------------------------------- attention --
def workspace(B, N, H, Hkv, D, T):
    """Bytes of partial results: 0 where one split or a cluster takes a row."""
    from maple_flash_dgx_spark_b200 import _lib

    return _lib.lib().maple_tree_gqa_workspace_bytes(B, N, H, Hkv, D, T, 0, 1)


def ragged_lens(seed, B, most):
    """Empty, single and odd lengths beside tile edges, then anything."""
    r = random.Random(seed)
    edge = [0, 1, 127, 128, 129, most]
    return [edge[b % 8] if b % 8 < 6 else r.randint(0, most) for b in range(B)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,H,groups", [(5, 24, 1),      # 15 rows: both warpgroups share a row tile
                                        (20, 56, 1),     # 140 rows: a row tile each, the second short
                                        (43, 48, 2)])    # 258 rows: two pairs of row tiles, three of them in use
@pytest.mark.parametrize("window", [0, 150])
def test_attention_several_items_per_cta(cuda, K, N, H, groups, D, window):
    """More row tiles than SMs, so that CTAs go on from item to item (tile rings,
    item slots and the queries' place used again) over sequences with no keys, a
    part of a tile and several, some of them padding."""
    B, Hkv, T = 48 if groups == 1 else 24, 8, 420
    assert B * Hkv * groups > 2 * 148 and workspace(B, N, H, Hkv, D, T) == 0
    c = attn_case(41, B, N, H, Hkv, D, T, ragged_lens(41, B, T - N), BF, ragged=True)
    c["mask"][[3, 17, 18]] = 0
    got = verify_attn(K, c, window)
    assert (got[[3, 17, 18]] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,N,H,Hkv,T", [(2, 5, 8, 2, 20000),       # one row tile
                                         (2, 26, 10, 2, 20000),     # 130 rows: a pair
                                         (2, 64, 10, 2, 20000),     # 320 rows: two pairs
                                         (1, 64, 32, 4, 30000),     # 512 rows
                                         (40, 3, 8, 4, 5100),       # several items per CTA and a join
                                         (40, 33, 16, 4, 5100)])
def test_attention_joined_by_a_second_launch(cuda, K, B, N, H, Hkv, D, T):
    """More splits than a cluster joins, of which sequences use none, one, some or
    all: partial sums in memory, over all row tiles and heads."""
    assert workspace(B, N, H, Hkv, D, T) > 0
    lens = [T - N, 1300] if B == 2 else [T - N] if B == 1 else ragged_lens(43, B, 900)
    if B > 2:
        lens[6], lens[7], lens[14] = T - N, 2600, 4001
    verify_attn(K, attn_case(43, B, N, H, Hkv, D, T, lens, BF, ragged=B > 2))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [512, 6000])
def test_attention_single_token_is_decode_bf16(cuda, K, D, T):
    """One node without a tree against ``decode_gqa_attn`` on the same caches:
    both round their weights (half a step of each, at most that of sum p |v|) and
    their outputs, and sum scores in fp32."""
    c = attn_case(45, 3, 1, 16, 2, D, T, [T - 1, 3, 77], BF)
    got = verify_attn(K, c)
    want = K.decode_gqa_attn(c["q"].transpose(1, 2).contiguous(), c["k"], c["v"], torch.tensor(c["lens"], device=cuda),
                             scale=c["scale"], window=None)
    exact, mass, reach = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], None, c["scale"], 0)
    inner = mass * (2.0 ** -8 + 2 * (D * 2.0 ** -24 * reach + 2.0 ** -20) + 2 * T * 2.0 ** -24)
    tol = 2 * (inner + 2.0 ** -8 * (exact.abs() + inner))
    assert ((got.double() - want.transpose(1, 2).double()).abs() <= tol + 1e-30).all()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 256), (F32, 128)])
@pytest.mark.parametrize("scale", [2.0 ** -116, -(2.0 ** -110), 1e-33, 0.0])
def test_attention_tiny_scales(cuda, K, dtype, D, scale):
    """Scales far below 1 with keys as far above it (both types reach 2^127):
    scores near 1; and a scale of 0, whose weights are all the same."""
    c = attn_case(46, 2, 6, 8, 2, D, 300, [250, 17], dtype)
    c["scale"] = scale
    c["k"] = c["k"] * (2.0 ** 113 if scale == 0 else 0.25 / abs(scale))
    got = run_attn(K, c)
    want, mass, reach = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], None, scale, 0)
    check_attention(got, want, mass, reach.abs(), dtype, 256)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 256), (F32, 128)])
@pytest.mark.parametrize("N", [1, 40])
@pytest.mark.parametrize("up", [3.0, 7.0, 7.9])
def test_attention_largest_value_behind_a_rising_maximum(cuda, K, dtype, D, N, up):
    """A key whose weight is 2^up times all that came before it, and with it the
    type's largest value: no partial product leaves fp32."""
    c = attn_case(47, 1, N, 4, 1, D, 5000, [4900], dtype)
    c["scale"] = 1.0
    c["q"] = torch.zeros_like(c["q"])
    c["q"][..., 0] = 1.0
    c["k"][..., 0] = 0.0
    for t in (300, 1700, 4800):
        c["k"][:, :, t, 0] = up * 0.6931
    c["v"][0, 0, 300, 1] = torch.finfo(dtype).max
    c["v"][0, 0, 300, 2] = -torch.finfo(dtype).max
    verify_attn(K, c)


# ------------------------------------------- arguments at their types' ends --
def test_whole_numbers_past_32_bits(cuda, K):
    """int64 parents, paths, counts and cache rows that int32 does not hold are
    out of range, not their low words."""
    big = 1 << 32
    plan = K.tree_plan(torch.tensor([[-1, 0, big, 1, -big - 1]], device=cuda))
    assert flags(cuda) == 2 and plan.mask.tolist() == [[1, 3, 0, 11, 0]]
    logits, tok, par, u, _ = verify_inputs(51, 1, 4, 50, chain=True)
    kw = dict(temperature=1.0, top_p=1.0, top_k=20)
    args = (logits, torch.from_numpy(tok).to(cuda))
    path, n, ids = K.verify_tree(*args, torch.tensor([[-1, big, big, big]], device=cuda), torch.zeros(1, 4, device=cuda), **kw)
    assert flags(cuda) == 2 and n.tolist() == [1] and path.tolist() == [[0, -1, -1, -1]]
    k, v = (torch.randn(2, 2, 20, 64, device=cuda).to(BF) for _ in range(2))
    keep = k.clone(), v.clone()
    rows, s = K.CacheRows([k], [v]), torch.tensor([4, 5], device=cuda)
    good, cnt = torch.tensor([[0, 2, -1], [0, 2, -1]], device=cuda), torch.tensor([2, 2], device=cuda)
    for path, n, row_map in ((good + torch.tensor([0, big, 0], device=cuda), cnt, None), (good, cnt + big, None),
                             (good, cnt, torch.tensor([big, big + 1], device=cuda))):
        K.commit_tree(rows, s, path, n, row_map=row_map)
        assert flags(cuda) == 2
        assert torch.equal(k, keep[0]) and torch.equal(v, keep[1])
    c = attn_case(52, 2, 3, 4, 2, 64, 40, [3, 4], BF, rows=[0, 1])
    got = K.tree_gqa_attn(c["q"], c["k"], c["v"], torch.tensor([3, 4], device=cuda), torch.from_numpy(c["mask"]).to(cuda),
                          row_map=torch.tensor([0, big + 1], device=cuda), scale=1.0)
    assert flags(cuda) == 2 and (got[1] == 0).all() and (got[0] != 0).any()


@pytest.mark.parametrize("n", [0, 1, 255, 256, 257, 300000])
def test_narrowing_saturates(cuda, K, n):
    g = torch.Generator().manual_seed(n)
    x = torch.randint(-(1 << 33), 1 << 33, (n, 2), generator=g)
    x[: n // 3] >>= 12
    ends = [v for e in (1 << 31, 1 << 32, 1 << 63) for v in (e - 2, e - 1, e, e + 1, -e - 1, -e, -e + 1)]
    ends = torch.tensor([v for v in ends if -(1 << 63) <= v < 1 << 63])
    x[: ends.numel(), 0] = ends[:n]
    want = x.clamp(-(1 << 31), (1 << 31) - 1).int()
    x = x.to(cuda)
    for got, w in ((K._as_int32(x, "narrow", 0), want), (K._as_int32(x[:, 0], "narrow", 0), want[:, 0]),
                   (K._as_int32(x[:, 1].int(), "narrow", 0), x[:, 1].int().cpu())):
        assert got.dtype == torch.int32 and got.is_contiguous() and torch.equal(got.cpu(), w)


def test_verify_node_0_with_a_parent_is_padding(cuda, K):
    """As in the plan: a parent that is not before its node makes it padding, and
    a sequence whose node 0 is padding draws nothing."""
    logits, tok, _, u, q = verify_inputs(53, 4, 5, 60, draft=F32)
    par = torch.tensor([[0, 0, 1, 0, 0], [3, 0, 0, 0, 0], [-1, 0, 1, 1, 2], [-2, 0, 1, 1, 2]], dtype=torch.int32, device=cuda)
    assert (K.tree_plan(par).mask[[0, 1, 3]] == 0).all() and flags(cuda) == 2
    for draft in (None, q):
        path, n, ids = K.verify_tree(logits, torch.from_numpy(tok).to(cuda), par, torch.zeros_like(torch.from_numpy(u)).to(cuda),
                                     temperature=1.0, top_p=1.0, top_k=20, draft_probs=draft)
        assert flags(cuda) == 2
        assert n[[0, 1, 3]].tolist() == [0, 0, 0] and int(n[2]) >= 1
        assert (path[[0, 1, 3]] == -1).all() and (ids[[0, 1, 3]] == -1).all()


# ------------------------------------------------------------- the caches --
def small_cache(cuda, batch=3, max_len=32, layers=2):
    from maple_flash_dgx_spark_b200.model import KVCache

    cache = KVCache(["full_attention"] * layers, None, n_kv=2, head_dim=64, max_len=max_len, batch=batch, dtype=BF, device=cuda)
    for t in cache.k + cache.v:
        t.normal_()
    return cache


@pytest.mark.parametrize("told", [False, True])
def test_refused_paths_leave_the_lengths(cuda, K, told):
    """A path that does not rise, or leaves the cache, moves nothing, so its
    sequence gets no longer either."""
    cache = small_cache(cuda, batch=5)
    lens = [3, 28, 5, 6, 7]
    cache.seqlen.copy_(torch.tensor(lens))
    cache.seen = list(lens)
    path = torch.tensor([[0, 2, 3, -1, -1], [0, 2, 4, -1, -1], [0, 3, 1, -1, -1], [-1] * 5, [0, 1, 2, 3, 4]],
                        dtype=torch.int32, device=cuda)
    n = torch.tensor([3, 3, 3, 0, 6], dtype=torch.int32, device=cuda)
    before = [t.clone() for t in cache.k + cache.v]
    cache.commit_tree(path, n, kept=[3, 0, 0, 0, 0] if told else None)
    assert flags(cuda) == 2
    assert cache.seqlen.tolist() == cache.seen == [6, 28, 5, 6, 7]
    for t, old in zip(cache.k + cache.v, before):
        assert torch.equal(t[1:], old[1:])
        assert torch.equal(t[0, :, [4, 5]], old[0, :, [5, 6]])


def test_commit_many_layers_reports_once(cuda, K):
    cache = small_cache(cuda, batch=2, layers=131)
    path, n = torch.tensor([[0, 2], [0, 1]], device=cuda), torch.tensor([2, 1], device=cuda)
    path[0, 1] = 1
    cache.commit_tree(path, n)
    assert cache.seqlen.tolist() == cache.seen == [2, 1]


def test_overlapping_caches_are_refused(cuda, K):
    """Rows move in place: no strides or views that let two of them share elements."""
    R = 30 * 64

    def view(strides, shift=0, base=torch.zeros(1 << 15, dtype=BF, device=cuda)):
        return base.as_strided((2, 2, 30, 64), (*strides, 64, 1), shift)

    def apart(strides):
        return view(strides, base=torch.zeros(1 << 15, dtype=BF, device=cuda))

    for k, v in ((view((R, R)), apart((R, R))),                             # head 1 of one is head 0 of the next
                 (view((R, 2 * R - 64)), apart((R, 2 * R - 64))),           # by a position
                 (view((2 * R, R)), view((2 * R, R), 64)),                  # two caches, a position apart
                 (view((2 * R, R)), view((2 * R, R), 2 * R))):              # one's second sequence, the other's first
        with pytest.raises(ValueError, match="overlap"):
            K.CacheRows([k], [v])
    K.CacheRows([view((3 * R, 2 * R))], [apart((3 * R, 2 * R))])            # rows 0, 2, 3 and 5
    K.CacheRows([view((4 * R, R))], [view((4 * R, R), 2 * R)])              # each in the other's gaps
    for perm in ((0, 1, 2), (1, 0, 2), (2, 0, 1), (1, 2, 0)):               # of (K or V, sequence, head)
        size = [(2, 3, 4)[p] for p in perm]
        both = torch.zeros(*size, 30, 64, dtype=BF, device=cuda).permute(*[perm.index(i) for i in range(3)], 3, 4)
        K.CacheRows([both[0]], [both[1]])


def one_tree(cuda, model, cache, batch, seed=5):
    g = torch.Generator().manual_seed(seed)
    tok = torch.randint(0, 512, (batch, 3), generator=g).to(cuda)
    par = torch.tensor([[-1, 0, 1]] * batch, dtype=torch.int32, device=cuda)
    model.forward_tree(tok, par, cache)
    n = torch.full((batch,), 2, dtype=torch.int32, device=cuda)
    return torch.tensor([[0, 1, -1]] * batch, dtype=torch.int32, device=cuda), n


def test_commit_goes_to_the_slots_of_the_step(cuda, K):
    """The commit of a tree step is refused for slots that had none in it, and
    changes nothing then."""
    model = tiny(cuda, BF)
    cache = model.make_cache(max_len=32, batch=3)
    cache.remap = True
    with cache.prefill_slot(1):
        path, n = one_tree(cuda, model, cache, 1)
    with pytest.raises(ValueError, match="slot"):
        cache.commit_tree(path, n)
    with cache.prefill_slot(2), pytest.raises(ValueError, match="slot"):
        cache.commit_tree(path, n)
    assert cache.seen == cache.seqlen.tolist() == [0, 0, 0]
    cache.swap_slots(1, 2)  # the sequence is in slot 2 now, with its length and its rows
    with cache.prefill_slot(1), pytest.raises(ValueError, match="slot"):
        cache.commit_tree(path, n)
    with cache.prefill_slot(2):
        cache.commit_tree(path, n)
        assert cache.seen == cache.seqlen.tolist() == [0, 0, 2]
    # a whole batch, committed slot by slot
    path, n = one_tree(cuda, model, cache, 2)
    with cache.prefill_slot(1):
        cache.commit_tree(path[1:], n[1:])
        with pytest.raises(ValueError, match="slot"):
            cache.commit_tree(path[1:], n[1:])  # a second time
    with cache.prefill_slot(0):
        cache.commit_tree(path[:1], n[:1])
    assert cache.seen == cache.seqlen.tolist() == [2, 2, 2]
    # two steps, each in a slot of its own, before their commits
    for slot in (0, 2):
        with cache.prefill_slot(slot):
            path, n = one_tree(cuda, model, cache, 1)
    with cache.prefill_slot(1), pytest.raises(ValueError, match="slot"):
        cache.commit_tree(path, n)
    for slot in (0, 2):
        with cache.prefill_slot(slot):
            cache.commit_tree(path, n)
    assert cache.seen == cache.seqlen.tolist() == [4, 2, 4]
    # one that was given up
    one_tree(cuda, model, cache, 2)
    cache.reset_identity()
    path, n = one_tree(cuda, model, cache, 3)
    cache.commit_tree(path, n, kept=[2, 2, 2])
    assert cache.seen == cache.seqlen.tolist() == [2, 2, 2]


# ------------------------------------------------------------ in the model --
def test_tokens_of_padding_are_not_looked_at(cuda, K):
    """Padding is the parents' alone: -1, as verify_tree fills its ids with, may
    stand there."""
    model = tiny(cuda, BF)
    cache = model.make_cache(max_len=32, batch=2)
    par = torch.tensor([[-1, 0, 0, 1], [-1, 0, -2, -2]], dtype=torch.int32, device=cuda)
    tok = torch.tensor([[3, 4, 5, 6], [7, 8, 0, 0]], device=cuda)
    want = model.forward_tree(tok, par, cache)
    odd = tok.clone()
    odd[1, 2:] = torch.tensor([-1, 1 << 40])
    got = model.forward_tree(odd, par, cache)
    assert flags(cuda) == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :2], want[1, :2])


def test_captured_tree_steps(cuda, K):
    """forward_tree, verify_tree and the commit in one graph, replayed as the
    sequences grow, against the same steps called."""
    torch.set_grad_enabled(False)
    try:
        model = tiny(cuda, BF)
        r = random.Random(8)
        B, N = 2, 6
        cache = model.make_cache(max_len=64, batch=B)
        cache.remap = True
        prefill(model, cache, [[r.randrange(512) for _ in range(n)] for n in (11, 4)])
        par = torch.tensor([[-1, 0, 0, 1, 1, 2], [-1, 0, 1, 2, -2, -2]], dtype=torch.int32, device=cuda)
        inputs = [(torch.randint(0, 512, (B, N), device=cuda), torch.rand(B, N, device=cuda)) for _ in range(3)]
        tok, u = torch.zeros_like(inputs[0][0]), torch.zeros_like(inputs[0][1])
        start = cache.snapshot()

        def step(kept=None):
            logits = model.forward_tree(tok, par, cache)
            out = K.verify_tree(logits, tok, par, u, temperature=1.0, top_p=0.95, top_k=20)
            cache.commit_tree(*out[:2], kept=kept)
            return (logits, *out)

        want = []
        for t, x in inputs:
            tok.copy_(t)
            u.copy_(x)
            want.append([y.clone() for y in step()] + [cache.seqlen.clone(), list(cache.seen)])
        rows = [t.clone() for t in cache.k + cache.v]
        cache.restore(start)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.forward_tree(tok, par, cache)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(kept=[0] * B)  # the host's counts follow each replay
        torch.cuda.current_stream().wait_stream(side)
        cache.restore(start)
        for (t, x), w in zip(inputs, want):
            tok.copy_(t)
            u.copy_(x)
            graph.replay()
            cache.seen = [a + b for a, b in zip(cache.seen, out[2].tolist())]
            for got, y in zip((*out, cache.seqlen), w):
                assert torch.equal(got, y)
            assert cache.seen == w[-1]
        for got, y in zip(cache.k + cache.v, rows):
            for b in range(B):
                assert torch.equal(got[b, :, :cache.seen[b]], y[b, :, :cache.seen[b]])
    finally:
        torch.set_grad_enabled(True)


def test_tree_steps_are_steps_of_one_node(cuda, K):
    """fp32: every node's logits and cache rows against its path taken one node
    at a time by trees of one, committed one by one, from the same cache.  All but
    the attention's order of sums is the same arithmetic.  fp32 sums of 64
    products with sum |q k| scale <= 8 are off by 64 half steps of it at worst
    (3e-5) and by sqrt(64) of them (4e-6) as they fall, for two routes, two
    layers and a gain of up to six through the norms and the experts: 1e-4 of the
    largest logit, where a wrong position or slot changes its second digit.  The
    first layer's K and V have no attention before them: the same bits, as plain
    decoding of the accepted tokens has."""
    torch.set_grad_enabled(False)
    try:
        model = tiny(cuda, F32)
        r = random.Random(9)
        texts = [[r.randrange(512) for _ in range(n)] for n in (25, 2, 14)]
        par = [[-1, 0, 0, 1, 1, 2, 5, 3], [-1, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 0, 0, 2, -2, -2, -2]]
        B, N = 3, 8
        cache = model.make_cache(max_len=64, batch=B)
        cache.remap = True
        prefill(model, cache, texts)
        cache.swap_slots(0, 1)
        texts[0], texts[1] = texts[1], texts[0]
        lens = list(cache.seen)
        tok = [[r.randrange(512) for _ in range(N)] for _ in range(B)]
        pt = torch.tensor(par, dtype=torch.int32, device=cuda)
        start = cache.snapshot()
        logits = model.forward_tree(torch.tensor(tok, device=cuda), pt, cache)
        tree = [t.clone() for t in cache.k + cache.v]
        top = float(logits.abs().max())
        one, root = torch.ones(1, dtype=torch.int32, device=cuda), torch.full((1, 1), -1, dtype=torch.int32, device=cuda)
        paths = []
        for b in range(B):
            longest = []
            for i in range(N):
                if par[b][i] < -1:
                    continue
                line, j = [], i
                while j >= 0:
                    line.append(j)
                    j = par[b][j]
                line = line[::-1]
                longest = max(longest, line, key=len)
                cache.restore(start)
                with cache.prefill_slot(b):
                    for d, j in enumerate(line):
                        got = model.forward_tree(torch.tensor([[tok[b][j]]], device=cuda), root, cache)
                        cache.commit_tree(torch.zeros_like(root), one)
                assert cache.seen[b] == int(cache.seqlen[b]) == lens[b] + len(line)
                err = float((got[0, 0] - logits[b, i]).abs().max())
                assert err <= 1e-4 * top, (b, i, err, top)
                row, at = cache.row_of[b], lens[b]
                for li, (x, y) in enumerate(zip(cache.k + cache.v, tree)):
                    x, y = x[row, :, at + len(line) - 1], y[row, :, at + i]
                    if li % len(cache.k) == 0:
                        assert torch.equal(x, y), (b, i)
                    else:
                        assert float((x - y).abs().max()) <= 1e-4 * float(y.abs().max()), (b, i, li)
            paths.append(longest)
        # the longest paths accepted, against plain decoding
        cache.restore(start)
        model.forward_tree(torch.tensor(tok, device=cuda), pt, cache)
        cache.commit_tree(torch.tensor([p + [-1] * (N - len(p)) for p in paths], device=cuda),
                          torch.tensor([len(p) for p in paths], dtype=torch.int32, device=cuda))
        for b, p in enumerate(paths):
            plain = model.make_cache(max_len=64)
            model.forward(torch.tensor(texts[b] + [tok[b][j] for j in p], device=cuda).reshape(1, -1), cache=plain)
            assert cache.seen[b] == plain.seen[0]
            for got, want in ((cache.k[0], plain.k[0]), (cache.v[0], plain.v[0])):
                assert torch.equal(got[cache.row_of[b], :, :cache.seen[b]], want[0, :, :cache.seen[b]])
    finally:
        torch.set_grad_enabled(True)
