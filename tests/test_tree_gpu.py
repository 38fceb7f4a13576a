"""Speculative-decoding operators on the GPU against their 64-bit restatements.

Tolerances count roundings (``eps / 2`` of a type, relative to the value).  The
attention's: the output's own rounding; the weights' rounding to the inputs'
type before the product with V (bf16: half a step of each p_t v_t, so at most
that of sum p |v|); the scores' fp32 sums of D products (D half steps of
sum |q k| at worst, which moves a weight by twice that, once in the sum it is
divided by); the exponential's 2^-20; and the fp32 sums over the keys.
"""

from __future__ import annotations

import random

import numpy as np
import pytest

from tests import tree_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def K():
    from maple_flash_dgx_spark_b200 import kernels

    return kernels


@pytest.fixture(autouse=True)
def clean_error_word(cuda):
    from maple_flash_dgx_spark_b200 import _lib

    _lib.take_device_errors(cuda)
    yield
    assert _lib.take_device_errors(cuda) == 0


def flags(cuda):
    from maple_flash_dgx_spark_b200 import _lib

    return _lib.take_device_errors(cuda)


def trees(seed, B, N, chain=False, ragged=False):
    r = random.Random(seed)
    rows = []
    for _ in range(B):
        n = r.randint(1, N) if ragged else N
        rows.append([-1] + [i - 1 if chain or r.random() < 0.3 else r.randrange(max(0, i - 9), i)
                            for i in range(1, n)] + [-2] * (N - n))
    return rows


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ------------------------------------------------------------------- plan --
@pytest.mark.parametrize("B,N,chain,ragged", [(1, 1, False, False), (3, 8, False, True), (5, 33, True, False),
                                              (130, 64, False, True), (2, 64, True, False)])
def test_plan(cuda, K, B, N, chain, ragged):
    par = trees(B + N, B, N, chain, ragged)
    got = K.tree_plan(torch.tensor(par, dtype=torch.int32, device=cuda))
    mask, depth, _ = ref.plan(par)
    np.testing.assert_array_equal(got.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(got.depth.cpu().numpy(), depth)


def test_plan_flags_bad_parents_and_takes_strides(cuda, K):
    par = [[-1, 0, 1, 3, 3, -2, 5, 7], [-2, -1, 1, 5, 2, 3, 0, 2]]
    mask, depth, bad = ref.plan(par)
    wide = torch.full((2, 16), 99, dtype=torch.int64, device=cuda)
    wide[:, ::2] = torch.tensor(par, device=cuda)
    got = K.tree_plan(wide[:, ::2])
    np.testing.assert_array_equal(got.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(got.depth.cpu().numpy(), depth)
    assert bad and flags(cuda) == 2
    with pytest.raises(ValueError):
        K.tree_plan(torch.zeros(1, 65, dtype=torch.int32, device=cuda))
    with pytest.raises(TypeError):
        K.tree_plan(torch.zeros(1, 5, device=cuda))


# -------------------------------------------------------------- attention --
def check_attention(got, want, mass, reach, dtype, n_keys):
    D = got.shape[-1]
    half = torch.finfo(dtype).eps / 2
    weights = 2 * (D * 2.0 ** -24 * reach + 2.0 ** -20) + 2 * n_keys * 2.0 ** -24
    inner = mass * (weights + (half if dtype == BF else 0.0))
    tol = inner + half * (want.abs() + inner)
    bad = ((got.double() - want).abs() > tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / (tol + 1e-30)).max()))


def attn_case(seed, B, N, H, Hkv, D, T, lens, dtype, *, chain=False, ragged=False, rows=None, mask=None):
    g = gen(seed)
    Bc = B if rows is None else max(rows) + 1
    q = normal(g, B, N, H, D, dtype=dtype, scale=2.0)
    k, v = normal(g, Bc, Hkv, T, D, dtype=dtype), normal(g, Bc, Hkv, T, D, dtype=dtype)
    if mask is None:
        mask = ref.plan(trees(seed, B, N, chain, ragged))[0]
    return dict(q=q, k=k, v=v, lens=lens, mask=np.asarray(mask, np.int64), rows=rows, scale=D ** -0.5)


def run_attn(K, c, window=0):
    dev = c["q"].device
    return K.tree_gqa_attn(c["q"], c["k"], c["v"], torch.tensor(c["lens"], device=dev),
                           torch.from_numpy(c["mask"]).to(dev),
                           row_map=None if c["rows"] is None else torch.tensor(c["rows"], dtype=torch.int32, device=dev),
                           scale=c["scale"], window=window or None)


def verify_attn(K, c, window=0):
    got = run_attn(K, c, window)
    want, mass, reach = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], c["rows"], c["scale"], window)
    check_attention(got, want, mass, reach, c["q"].dtype, max(c["lens"]) + c["q"].shape[1])
    return got


ATTN = [
    # B, N, H, Hkv, D, T, lens, window, chain, ragged, rows
    (1, 1, 4, 2, 64, 64, [0], 0, False, False, None),            # nothing cached
    (1, 1, 8, 1, 128, 64, [63], 0, False, False, None),          # the last slot of the cache
    (2, 2, 8, 8, 128, 160, [1, 127], 0, True, False, None),      # one query head per KV head
    (3, 5, 32, 4, 128, 640, [600, 0, 131], 0, True, False, None),
    (2, 13, 10, 2, 64, 400, [383, 384], 0, False, True, None),   # five heads per group, padding
    (4, 16, 32, 4, 128, 300, [128, 1, 255, 256], 0, False, False, [2, 0, 3, 5]),
    (2, 17, 32, 4, 128, 1100, [1050, 500], 0, False, False, None),  # more rows than one 128-row tile
    (1, 64, 32, 4, 128, 2100, [2000], 0, False, False, None),
    (2, 64, 6, 1, 64, 700, [600, 13], 0, False, True, None),
    (2, 33, 14, 2, 128, 512, [300, 2], 0, False, False, None),   # seven heads per group
    (3, 9, 16, 4, 128, 900, [800, 40, 5], 64, False, False, None),   # sliding windows
    (2, 40, 8, 2, 64, 900, [800, 300], 7, True, False, None),    # a window shorter than the tree
    (2, 8, 8, 2, 128, 900, [800, 300], 1, False, False, None),   # each node sees itself alone
    (2, 12, 8, 2, 128, 400, [200, 100], 5000, False, False, None),
    (1, 7, 48, 2, 64, 333, [300], 0, False, False, None),        # 24 query heads per KV head
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,N,H,Hkv,D,T,lens,window,chain,ragged,rows", ATTN)
def test_attention(cuda, K, B, N, H, Hkv, D, T, lens, window, chain, ragged, rows, dtype):
    c = attn_case(B * 100 + N, B, N, H, Hkv, D, T, lens, dtype, chain=chain, ragged=ragged, rows=rows)
    verify_attn(K, c, window)


@pytest.mark.parametrize("N,H,D", [(5, 8, 128), (40, 8, 128), (3, 4, 64), (64, 8, 64)])
@pytest.mark.parametrize("window", [0, 300])
def test_attention_splits_of_ragged_lengths(cuda, K, N, H, D, window):
    """Caches cut into up to eight splits (and more where 40 tiles allow), of which
    a sequence uses none, one, some or all."""
    lens = [0, 1, 127, 128, 129, 383, 700, 1060]
    verify_attn(K, attn_case(26, 8, N, H, 2, D, 1124, lens, BF, ragged=True), window)
    verify_attn(K, attn_case(27, 2, N, H, 2, D, 5100, [5000, 130], BF), window)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_heads_of_256(cuda, K, dtype):
    verify_attn(K, attn_case(5, 2, 6, 8, 2, 256, 300, [280, 31], dtype))


@pytest.mark.parametrize("L", list(range(0, 20)) + [60, 63, 64, 65, 119, 120, 121, 127, 128, 129, 250, 255, 256, 257])
def test_attention_every_length_near_a_tile(cuda, K, L):
    verify_attn(K, attn_case(L, 1, 8, 16, 2, 128, L + 8, [L], BF))


def test_attention_long_ragged_batch(cuda, K):
    r = random.Random(3)
    lens = [r.randrange(0, 4000) for _ in range(12)]
    verify_attn(K, attn_case(9, 12, 11, 16, 2, 128, 4096, lens, BF, ragged=True))


def test_attention_single_token_is_decode(cuda, K):
    c = attn_case(21, 3, 1, 16, 2, 128, 512, [500, 3, 77], F32)
    got = run_attn(K, c)
    want = K.decode_gqa_attn(c["q"].transpose(1, 2).contiguous(), c["k"], c["v"],
                             torch.tensor(c["lens"], device=cuda), scale=c["scale"], window=None)
    # decode_gqa_attn rounds its weights to bf16 (half a step, at most that of sum p |v|)
    _, mass, _ = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], None, c["scale"], 0)
    assert ((got[:, 0] - want[:, :, 0]).abs().double() <= mass[:, 0] * (2.0 ** -8 + 1e-4)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [0, 9])
def test_attention_any_mask_and_rows_that_see_nothing(cuda, K, dtype, window):
    """Masks that are no tree: bits of later nodes, without the node itself,
    padding between nodes, bits past the last node."""
    B, N = 3, 20
    r = np.random.RandomState(4)
    mask = r.randint(0, 1 << 62, (B, N)).astype(np.int64) | (r.randint(0, 2, (B, N)).astype(np.int64) << 63)
    mask[:, 3] = 0
    mask[1, ::2] = 0
    mask[2, :] = 0
    mask[0, 5] = -1 << 30  # only nodes that do not exist: as if 0
    c = attn_case(6, B, N, 8, 2, 128, 300, [200, 0, 150], dtype, mask=mask)
    got = verify_attn(K, c, window)
    assert (got[2] == 0).all() and (got[:, 3] == 0).all() and (got[0, 5] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_attention_garbage_where_nobody_looks(cuda, K, dtype, window, value):
    """NaN and infinities in K and V before the window, behind the tree and in
    the other branches' rows reach no node that does not see them."""
    B, N, L, T = 2, 12, 300, 400
    par = [[-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 7], [-1, 0, 1, 2, 3, 4, 5, -2, -2, -2, -2, -2]]
    mask, _, _ = ref.plan(par)
    c = attn_case(8, B, N, 16, 2, 128, T, [L, L - 37], dtype, mask=mask)
    clean = run_attn(K, c, window)
    k, v = c["k"].clone(), c["v"].clone()
    for b, n in enumerate(c["lens"]):
        used = N if b == 0 else 7
        for t in (k, v):
            t[b, :, n + used:] = value
            if window:
                t[b, :, : n - window] = value
    bad = 6  # sequence 0: node 6 and what hangs on it
    k[0, :, L + bad], v[0, :, L + bad, ::3] = value, value
    got = run_attn(K, {**c, "k": k, "v": v}, window)
    sees = np.array([[(int(m) >> bad) & 1 for m in mask[0]], [0] * N], bool)
    keep = torch.from_numpy(~sees).to(cuda)
    torch.testing.assert_close(got[keep], clean[keep], rtol=0, atol=0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_carries_what_a_row_sees(cuda, K, dtype):
    """A NaN or infinity in a V row reaches exactly the nodes and dimensions
    that see it, in a branch as in the cached part."""
    par = [[-1, 0, 0, 1, 2, 3]]
    c = attn_case(8, 1, 6, 8, 2, 128, 400, [300], dtype, mask=ref.plan(par)[0])
    clean = run_attn(K, c)
    v = c["v"].clone()
    v[0, 0, 300 + 2, 5] = float("inf")     # node 2, seen by 2 and 4
    v[0, 1, 300 + 1, 7] = float("nan")     # node 1, seen by 1, 3 and 5
    v[0, 1, 17, 9] = float("-inf")         # a cached position: every node
    got = run_attn(K, {**c, "v": v}).float()
    want = clean.float().clone()
    for i in (2, 4):
        want[0, i, :4, 5] = float("inf")
    for i in (1, 3, 5):
        want[0, i, 4:, 7] = float("nan")
    want[0, :, 4:, 9] = float("-inf")
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("L,T", [(300, 400), (3000, 8000)])  # one part, and several joined
def test_attention_nan_queries_and_keys(cuda, K, dtype, L, T):
    """A NaN in a query reaches its own row alone, though no score of it is a
    number; a NaN key every row that sees it, and no other."""
    par = [[-1, 0, 0, 1, 2, 3]]
    c = attn_case(18, 1, 6, 8, 2, 128, T, [L], dtype, mask=ref.plan(par)[0])
    clean = run_attn(K, c)
    q, k = c["q"].clone(), c["k"].clone()
    q[0, 4, 3, 17] = float("nan")
    k[0, 1, L + 1, 5] = float("nan")  # node 1 of KV head 1: nodes 1, 3 and 5, heads 4 to 7
    want = clean.float().clone()
    want[0, 4, 3] = float("nan")
    for i in (1, 3, 5):
        want[0, i, 4:] = float("nan")
    torch.testing.assert_close(run_attn(K, {**c, "q": q, "k": k}).float(), want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_infinite_keys(cuda, K, dtype):
    """A key with an infinity: a score of -inf weighs nothing, one of +inf leaves
    no number."""
    c = attn_case(19, 1, 4, 4, 2, 64, 200, [150], dtype, chain=True)
    q, k = c["q"].clone(), c["k"].clone()
    q[0, :, :, 3] = torch.tensor([1.0, -1.0, 1.0, -1.0], device=cuda, dtype=dtype)  # per head
    k[0, :, 20, 3] = float("inf")
    got = run_attn(K, {**c, "q": q, "k": k})
    assert torch.isnan(got[0, :, 0]).all() and torch.isnan(got[0, :, 2]).all()
    kz = k.clone()
    kz[0, :, 20] = 0
    v0 = c["v"].clone()
    want, mass, reach = ref.attention(q, torch.cat([kz[:, :, :20], kz[:, :, 21:]], 2), torch.cat([v0[:, :, :20], v0[:, :, 21:]], 2),
                                      [149], c["mask"], None, c["scale"], 0)
    check_attention(got[:, :, 1::2], want[:, :, 1::2], mass[:, :, 1::2], reach[:, :, 1::2], dtype, 154)


@pytest.mark.parametrize("D,dtype", [(64, F32), (128, F32), (256, F32), (128, BF), (256, BF)])
def test_attention_largest_keys_and_values(cuda, K, D, dtype):
    """The type's largest number in a key (scores near 1) and in a value, where
    rounding it up on the way would leave the type."""
    c = attn_case(24, 1, 6, 4, 2, D, 200, [150], dtype)
    big = torch.finfo(dtype).max
    c["q"] = c["q"].clone()
    c["q"][..., 3] = c["q"][..., 3] * (4.0 / big)
    c["k"][0, 0, [5, 77], 3] = big
    c["k"][0, 1, 151, 3] = -big
    c["v"][0, 0, 9, 1] = big
    verify_attn(K, c)


@pytest.mark.parametrize("D,L", [(64, 1500), (128, 1500), (256, 700)])
def test_attention_fp32_is_as_close_as_a_plain_one(cuda, K, D, L):
    """Not worse than fp32 products, softmax and sums one after the other, whose
    own error varies by less than twice from one order of summing to another."""
    c = attn_case(25, 2, 8, 8, 2, D, L + 20, [L, L - 9], F32)
    got = run_attn(K, c).double()
    want, _, _ = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], None, c["scale"], 0)
    k, v = (c[x].repeat_interleave(4, 1)[:, :, :L + 8] for x in "kv")
    s = (c["q"].transpose(1, 2) @ k.transpose(2, 3)) * c["scale"]
    for b, n in enumerate(c["lens"]):
        sees = torch.arange(L + 8, device=cuda) < n
        sees = sees.repeat(8, 1)
        for i in range(8):
            for j in range(8):
                sees[i, n + j] = bool(int(c["mask"][b, i]) >> j & 1)
        s[b].masked_fill_(~sees, float("-inf"))
    plain = (s.softmax(-1) @ v).transpose(1, 2).double()
    assert (got - want).norm() <= 2 * (plain - want).norm()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_expanded_caches(cuda, K, dtype):
    """One prefix for all sequences, one KV head for all groups: strides of 0."""
    c = attn_case(20, 3, 5, 8, 4, 128, 300, [250, 250, 100], dtype)
    k, v = c["k"][:1, :1].expand(3, 4, 300, 128), c["v"][:1, :1].expand(3, 4, 300, 128)
    want = run_attn(K, {**c, "k": k.contiguous(), "v": v.contiguous()})
    torch.testing.assert_close(run_attn(K, {**c, "k": k, "v": v}), want, rtol=0, atol=0)
    k, v = c["k"][:1].expand(3, 4, 300, 128), c["v"][:1].expand(3, 4, 300, 128)
    want = run_attn(K, {**c, "k": k.contiguous(), "v": v.contiguous()})
    torch.testing.assert_close(run_attn(K, {**c, "k": k, "v": v}), want, rtol=0, atol=0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_scale_zero_and_negative(cuda, K, dtype, scale):
    c = attn_case(23, 2, 6, 8, 2, 128, 400, [300, 17], dtype, ragged=True)
    c["scale"] = scale
    got = run_attn(K, c)
    want, mass, reach = ref.attention(c["q"], c["k"], c["v"], c["lens"], c["mask"], None, scale, 0)
    check_attention(got, want, mass, reach.abs(), dtype, 306)


def test_attention_huge_scores(cuda, K):
    """Scores far apart (weights underflow) and negative maxima."""
    for scale in (1.0, 8.0):
        c = attn_case(31, 2, 10, 8, 2, 128, 500, [450, 60], BF)
        c["scale"] = scale
        c["k"] = c["k"] - 3.0
        c["q"] = c["q"].abs()
        verify_attn(K, c)


def test_attention_strided_queries_and_unaligned(cuda, K):
    c = attn_case(12, 2, 7, 8, 2, 128, 300, [250, 9], BF)
    want = run_attn(K, c)
    wide = torch.zeros(2, 7, 24, 128, dtype=BF, device=cuda)
    wide[:, :, 8:16] = c["q"]
    torch.testing.assert_close(run_attn(K, {**c, "q": wide[:, :, 8:16]}), want, rtol=0, atol=0)
    flat = torch.zeros(2 * 7 * 8 * 128 + 3, dtype=BF, device=cuda)
    off = flat[3:].view(2, 7, 8, 128)
    off.copy_(c["q"])
    torch.testing.assert_close(run_attn(K, {**c, "q": off}), want, rtol=0, atol=0)
    heads_first = c["q"].transpose(1, 2).contiguous().transpose(1, 2)
    torch.testing.assert_close(run_attn(K, {**c, "q": heads_first}), want, rtol=0, atol=0)
    # caches inside a larger allocation: other batch and head strides
    big = torch.full((2, 3, 2, 300, 128), float("nan"), dtype=BF, device=cuda)
    big[:, 1] = c["k"]
    big[:, 2] = c["v"]
    torch.testing.assert_close(run_attn(K, {**c, "k": big[:, 1], "v": big[:, 2]}), want, rtol=0, atol=0)


def test_attention_row_depends_on_no_other_sequence(cuda, K):
    c = attn_case(14, 6, 9, 16, 2, 128, 2100, [2000, 1, 700, 1500, 64, 0], BF)
    want = run_attn(K, c)
    c2 = attn_case(15, 6, 9, 16, 2, 128, 2100, [3, 1200, 700, 2, 2090, 5], BF)
    for t in ("q", "k", "v"):
        c2[t][2] = c[t][2]
    c2["mask"][2] = c["mask"][2]
    torch.testing.assert_close(run_attn(K, c2)[2], want[2], rtol=0, atol=0)
    for _ in range(3):  # and the same call gives the same bits
        torch.testing.assert_close(run_attn(K, c), want, rtol=0, atol=0)


def test_attention_flags_lengths_and_rows_outside_the_cache(cuda, K):
    c = attn_case(16, 4, 6, 8, 2, 128, 200, [100, 195, 120, 50], BF, rows=[0, 1, 2, 3])
    want = run_attn(K, {**c, "lens": [100, 100, 120, 50]})
    got = run_attn(K, c)  # 195 + 6 > 200
    assert flags(cuda) == 2
    assert (got[1] == 0).all()
    torch.testing.assert_close(got[[0, 2, 3]], want[[0, 2, 3]], rtol=0, atol=0)
    for lens, rows in (([100, -1, 120, 50], [0, 1, 2, 3]), ([100, 1 << 62, 120, 50], [0, 1, 2, 3]),
                       ([100, (1 << 63) - 1, 120, 50], [0, 1, 2, 3]), ([100, 100, 120, 50], [0, 4, 2, 3]),
                       ([100, 100, 120, 50], [0, -1, 2, 3])):
        got = run_attn(K, {**c, "lens": lens, "rows": rows})
        assert flags(cuda) == 2, (lens, rows)
        assert (got[1] == 0).all()
        torch.testing.assert_close(got[[0, 2, 3]], want[[0, 2, 3]], rtol=0, atol=0)
    # padding only: nothing is looked at
    c["mask"][1] = 0
    got = run_attn(K, {**c, "lens": [100, -1, 120, 50]})
    assert flags(cuda) == 0 and (got[1] == 0).all()


def test_attention_offsets_past_32_bits(cuda, K):
    Bc, T = 66, 65536  # 2.2e9 elements in each cache
    g = gen(2)
    k = torch.empty(Bc, 4, T, 128, dtype=BF, device=cuda)
    v = torch.empty(Bc, 4, T, 128, dtype=BF, device=cuda)
    k[65], v[65] = normal(g, 4, T, 128, dtype=BF), normal(g, 4, T, 128, dtype=BF)
    c = dict(q=normal(g, 1, 4, 8, 128, dtype=BF, scale=2.0), k=k, v=v, lens=[T - 4], rows=[65], scale=128 ** -0.5,
             mask=ref.plan(trees(1, 1, 4))[0])
    verify_attn(K, c)


def test_attention_refusals(cuda, K):
    c = attn_case(1, 2, 3, 4, 2, 64, 40, [3, 4], BF)
    sl, m = torch.tensor([3, 4], device=cuda), torch.from_numpy(c["mask"]).to(cuda)

    def call(q=c["q"], k=c["k"], v=c["v"], s=sl, mask=m, rows=None, window=None):
        return K.tree_gqa_attn(q, k, v, s, mask, row_map=rows, scale=1.0, window=window)

    call()
    for bad in (dict(q=c["q"][:, :, :3]), dict(s=sl[:1]), dict(mask=m[:, :2]), dict(mask=m.int()), dict(window=-1),
                dict(k=c["k"][:1], v=c["v"][:1]), dict(k=c["k"][..., :32], v=c["v"][..., :32]),
                dict(k=c["k"].transpose(1, 2), v=c["v"].transpose(1, 2)), dict(rows=torch.zeros(3, dtype=torch.int32, device=cuda)),
                dict(q=c["q"][..., :16].contiguous(), k=c["k"][..., :16].contiguous(), v=c["v"][..., :16].contiguous())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(q=c["q"].float())
    with pytest.raises(TypeError):
        call(q=c["q"].half(), k=c["k"].half(), v=c["v"].half())
    with pytest.raises(RuntimeError):
        call(s=sl.cpu())


# ----------------------------------------------------------- verification --
def verify_inputs(seed, B, N, V, *, dtype=BF, chain=False, ragged=False, draft=None, twins=False):
    r = np.random.RandomState(seed)
    logits = torch.from_numpy((r.standard_normal((B, N, V)) * 2.5).astype(np.float32)).to("cuda", dtype)
    lg = logits.float().cpu().numpy()
    par = trees(seed, B, N, chain, ragged)
    tok = np.zeros((B, N), np.int64)
    q = None
    if draft is not None:
        z = lg + r.standard_normal(lg.shape) * 0.3
        z = np.where(z >= np.sort(z, -1)[..., -min(12, V)][..., None], z, -np.inf)
        e = np.exp(z - z.max(-1, keepdims=True))
        q = torch.from_numpy((e / e.sum(-1, keepdims=True)).astype(np.float32)).to("cuda", draft)
    for b in range(B):
        for i in range(1, N):
            p = max(par[b][i], 0)
            if q is not None:
                w = q[b, p].double().cpu().numpy()
                tok[b, i] = r.choice(V, p=w / w.sum())
            else:
                best = np.argsort(-lg[b, p])[: 2 if twins else 4]
                tok[b, i] = best[r.randint(len(best))]
    return logits, tok, par, r.random_sample((B, N)).astype(np.float32), q


def check_verify(K, logits, tok, par, u, q, **kw):
    dev = logits.device
    got = K.verify_tree(logits, torch.from_numpy(tok).to(dev), torch.tensor(par, dtype=torch.int32, device=dev),
                        torch.from_numpy(u).to(dev), draft_probs=q, **kw)
    want = ref.verify(logits.float().cpu().numpy(), tok, par, u, temperature=kw["temperature"], top_p=kw["top_p"],
                      top_k=kw["top_k"], draft=None if q is None else q.float().cpu().numpy(),
                      replacement=kw.get("replacement", False))
    for g, w, name in zip(got, want, ("path", "n_path", "ids")):
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
    return want


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("draft", [None, F32, BF])
@pytest.mark.parametrize("B,N,V,top_k,top_p,temperature,chain,ragged", [
    (1, 1, 1, 1, 1.0, 1.0, True, False),
    (2, 1, 37, 20, 0.9, 0.7, True, False),
    (9, 5, 1000, 1, 1.0, 1.0, True, False),
    (40, 8, 999, 20, 0.95, 1.0, True, True),
    (40, 33, 513, 64, 1.0, 1.5, False, True),
    (20, 64, 300, 7, 0.8, 0.5, False, False),
    (3, 16, 20001, 50, 0.9, 1.0, False, False),
    (2, 7, 50, 64, 1.0, 1.0, False, False),    # top_k above the vocabulary
])
def test_verify(cuda, K, B, N, V, top_k, top_p, temperature, chain, ragged, draft, dtype):
    x = verify_inputs(B * 7 + N + V, B, N, V, dtype=dtype, chain=chain, ragged=ragged, draft=draft)
    for replacement in ((False, True) if draft is not None else (False,)):
        check_verify(K, *x, temperature=temperature, top_p=top_p, top_k=top_k, replacement=replacement)


def test_verify_full_vocabulary(cuda, K):
    g = gen(3)
    B, N, V = 4, 6, 151936
    logits = normal(g, B, N, V, dtype=BF, scale=2.5)
    tok = np.zeros((B, N), np.int64)
    tok[:, 1:] = logits.argmax(-1)[:, :-1].cpu().numpy()
    u = np.random.RandomState(1).random_sample((B, N)).astype(np.float32) * 0.7
    want = check_verify(K, logits, tok, trees(2, B, N, chain=True), u, None, temperature=0.3, top_p=0.95, top_k=20)
    assert want[1].max() > 2


@pytest.mark.parametrize("order", ["rising", "falling", "one block"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_verify_logits_in_bad_orders(cuda, K, order, dtype):
    """Sorted logits and all the large ones side by side: the selection's worst
    cases."""
    V, N = 30011, 3
    x = np.linspace(-20, 20, V)
    if order == "falling":
        x = x[::-1]
    elif order == "one block":
        x = np.where((np.arange(V) >= 17000) & (np.arange(V) < 17300), 5.0 + np.arange(V) * 1e-3, -5.0)
    logits = torch.from_numpy(np.broadcast_to(x, (2, N, V)).astype(np.float32).copy()).to(cuda, dtype)
    tok = np.full((2, N), int(np.argmax(x)), np.int64)
    u = np.array([[0.99, 0.01, 0.5], [0.3, 0.6, 0.1]], np.float32)
    for k in (1, 5, 64):
        check_verify(K, logits, tok, [[-1, 0, 1]] * 2, u, None, temperature=1.0, top_p=1.0, top_k=k)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_verify_ties_and_special_logits(cuda, K, dtype):
    """Ties go to the lowest id; NaN ranks lowest, -0 is 0, infinities have
    weights; rows of one value are uniform over the lowest ids."""
    V, N, B = 4000, 2, 7
    lg = np.random.RandomState(0).standard_normal((B, N, V)).astype(np.float32)
    lg[0] = 1.5                                   # all equal
    lg[1] = -np.inf
    lg[2, :, ::2] = -np.inf
    lg[2, :, 1::2] = np.nan
    lg[2, :, 3999] = 0.25                         # one finite value, at the end
    lg[3] = np.where(np.arange(V) % 1000 == 7, 9.0, 0.0)   # four ties at the top, then thousands
    lg[4] = np.where(np.arange(V) % 2 == 0, 0.0, -0.0)
    lg[5, :, 100] = np.inf
    lg[5, :, 50] = np.inf
    lg[6] = np.round(lg[6])                       # many ties everywhere
    logits = torch.from_numpy(lg).to(cuda, dtype)
    tok = np.array([[0, 0], [0, 2], [0, 3999], [0, 1007], [0, 1], [0, 100], [0, 5]], np.int64)
    for k in (1, 2, 20, 64):
        for seed in range(4):
            u = np.random.RandomState(seed).random_sample((B, N)).astype(np.float32)
            check_verify(K, logits, tok, [[-1, 0]] * B, u, None, temperature=1.0, top_p=0.9, top_k=k)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,finite", [(600001, None), (100000, 30), (100000, 64), (40000, 500), (17000, 0)])
def test_verify_masked_and_long_vocabularies(cuda, K, V, finite, dtype):
    """Constrained decoding: all but a few logits -inf, none in the first tile;
    and a vocabulary of more tiles than one pass of the selection takes."""
    r = np.random.RandomState(V % 1000)
    lg = (r.standard_normal((2, 2, V)) * 2.5).astype(np.float32)
    tok = np.zeros((2, 2), np.int64)
    if finite is not None:
        keep = np.zeros((2, 2, V), bool)
        for b in range(2):
            for n in range(2):
                keep[b, n, 16400 + r.permutation(V - 16400)[:finite]] = True
        lg = np.where(keep, lg, -np.inf)
    tok[:, 1] = lg[:, 0].argmax(-1)
    logits = torch.from_numpy(lg).to(cuda, dtype)
    for k in (1, 20, 64):
        for seed in range(3):
            u = np.random.RandomState(seed).random_sample((2, 2)).astype(np.float32)
            check_verify(K, logits, tok, [[-1, 0]] * 2, u, None, temperature=0.9, top_p=0.97, top_k=k)


def test_verify_border_uniforms(cuda, K):
    """0 accepts whatever the target gives weight to, and draws the first token;
    the largest value below 1 draws the last kept one."""
    lg = torch.log(torch.tensor([0.5, 0.25, 0.125, 0.125], device=cuda)).expand(2, 3, 4).contiguous()
    top = np.float32(1) - np.float32(2.0 ** -24)
    for u0 in (0.0, 0.5, 0.75, top):
        for u1 in (0.0, 0.25, top):
            u = np.array([[u0, u1, u1]] * 2, np.float32)
            check_verify(K, lg, np.array([[0, 1, 1], [0, 3, 0]], np.int64), [[-1, 0, 0], [-1, 0, 1]], u, None,
                         temperature=1.0, top_p=1.0, top_k=4)


def test_verify_siblings_with_one_token(cuda, K):
    for draft in (None, F32):
        x = verify_inputs(77, 60, 10, 30, dtype=F32, draft=draft, twins=True)
        par = [[-1] + [0] * 9] * 60
        for replacement in (False, True):
            check_verify(K, x[0], x[1], par, x[3], x[4], temperature=1.0, top_p=1.0, top_k=30, replacement=replacement)


def test_verify_follows_the_target(cuda, K):
    """The first token's frequencies over 40000 sequences are the target's,
    whatever was drafted: within six standard deviations sqrt(p (1 - p) / n)."""
    n, V = 40000, 6
    p = torch.tensor([0.35, 0.25, 0.2, 0.1, 0.07, 0.03], device=cuda)
    lg = p.log().expand(n, 3, V).contiguous()
    r = np.random.RandomState(11)
    u = torch.from_numpy(r.random_sample((n, 3)).astype(np.float32)).to(cuda)
    par = torch.tensor([[-1, 0, 0]], dtype=torch.int32, device=cuda).expand(n, 3)
    q = np.array([0.1, 0.1, 0.1, 0.2, 0.2, 0.3])
    dq = torch.tensor(q, dtype=F32, device=cuda).expand(n, 3, V)
    for mode in ("certain", "without", "with"):
        if mode == "without":
            tok = np.stack([r.choice(V, 2, replace=False, p=q) for _ in range(n)])
        elif mode == "with":
            tok = r.choice(V, (n, 2), p=q)
        else:
            tok = np.tile([[4, 1]], (n, 1))
        tok = torch.from_numpy(np.concatenate([np.zeros((n, 1), np.int64), tok], 1)).to(cuda)
        _, _, ids = K.verify_tree(lg, tok, par, u, temperature=1.0, top_p=1.0, top_k=6,
                                  draft_probs=None if mode == "certain" else dq, replacement=mode == "with")
        freq = torch.bincount(ids[:, 0], minlength=V).double() / n
        want = p.double() / p.double().sum()
        assert ((freq - want).abs() <= 6 * (want * (1 - want) / n).sqrt()).all(), (mode, freq, want)


def test_verify_without_drafts_is_the_sampler(cuda, K):
    g = gen(8)
    logits = normal(g, 64, 1, 5000, dtype=BF, scale=2.5)
    u = torch.rand(64, 1, device=cuda, generator=g)
    par = torch.full((64, 1), -1, dtype=torch.int32, device=cuda)
    path, n, ids = K.verify_tree(logits, torch.zeros(64, 1, dtype=torch.int64, device=cuda), par, u, temperature=0.8,
                                 top_p=0.9, top_k=20)
    want = K.fused_sample_batched(logits[:, 0], u[:, 0], temperature=0.8, top_p=0.9, top_k=20)
    assert (path == 0).all() and (n == 1).all()
    assert torch.equal(ids[:, 0], want)


def test_verify_flags_bad_tokens_and_parents(cuda, K):
    logits, tok, par, u, q = verify_inputs(5, 3, 6, 100, draft=F32, chain=True)
    bad = tok.copy()
    bad[0, 1], bad[1, 1], bad[2, 1] = 100, -1, 1 << 40
    want = check_verify(K, logits, bad, par, u, q, temperature=1.0, top_p=1.0, top_k=20)
    assert (want[1] == 1).all() and flags(cuda) == 2
    check_verify(K, logits, bad, par, u, None, temperature=1.0, top_p=1.0, top_k=20)
    assert flags(cuda) == 2
    par = [list(p) for p in par]
    par[0][3] = 5
    check_verify(K, logits, tok, par, u, q, temperature=1.0, top_p=1.0, top_k=20)
    assert flags(cuda) == 2


def test_verify_strides_and_refusals(cuda, K):
    logits, tok, par, u, q = verify_inputs(6, 3, 6, 1001, draft=F32)  # rows of odd length: no 16-byte alignment
    kw = dict(temperature=1.0, top_p=0.9, top_k=20)
    check_verify(K, logits, tok, par, u, q, **kw)
    wide = torch.full((6, 3, 1100), 50.0, dtype=BF, device=cuda)
    wide[..., 50:1051] = logits.transpose(0, 1)
    check_verify(K, wide[..., 50:1051].transpose(0, 1), tok, par, u, q, **kw)
    check_verify(K, logits.transpose(1, 2).contiguous().transpose(1, 2), tok, par, u, q.transpose(1, 2).contiguous().transpose(1, 2), **kw)
    t, p, un = torch.from_numpy(tok).to(cuda), torch.tensor(par, device=cuda), torch.from_numpy(u).to(cuda)
    for bad in (dict(temperature=0.0), dict(top_p=0.0), dict(top_k=0), dict(top_k=65)):
        with pytest.raises(ValueError):
            K.verify_tree(logits, t, p, un, **{**kw, **bad})
    with pytest.raises(ValueError):
        K.verify_tree(logits, t[:, :5], p, un, **kw)
    with pytest.raises(ValueError):
        K.verify_tree(logits, t, p, un, draft_probs=q[..., :1000], **kw)
    with pytest.raises(TypeError):
        K.verify_tree(logits.half(), t, p, un, **kw)
    with pytest.raises(RuntimeError):
        K.verify_tree(logits, t.cpu(), p, un, **kw)


# ----------------------------------------------------------------- commit --
def paths(r, B, N, full=False):
    path, n = np.full((B, N), -1, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        m = N if full else r.randint(0, N + 1)
        n[b] = m
        if m:
            path[b, :m] = [0] + sorted(r.choice(np.arange(1, N), m - 1, replace=False)) if N > 1 else [0]
    return path, n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layers,B,N,Hkv,D,T,rows", [(1, 1, 1, 1, 64, 8, None), (3, 4, 9, 2, 64, 50, None),
                                                     (5, 3, 64, 4, 128, 200, [4, 0, 2]), (130, 2, 17, 1, 64, 40, None)])
def test_commit(cuda, K, layers, B, N, Hkv, D, T, rows, dtype):
    r = np.random.RandomState(layers * 10 + N)
    Bc = B if rows is None else 5
    caches = [torch.randn(Bc, Hkv, T, D, device=cuda).to(dtype) for _ in range(2 * layers)]
    before = [c.float().cpu().numpy() for c in caches]
    lens = r.randint(0, T - N + 1, B)
    path, n = paths(r, B, N)
    handle = K.CacheRows(caches[:layers], caches[layers:])
    K.commit_tree(handle, torch.from_numpy(lens).to(cuda), torch.from_numpy(path).to(cuda), torch.from_numpy(n).to(cuda),
                  row_map=None if rows is None else torch.tensor(rows, dtype=torch.int32, device=cuda))
    for c, old in zip(caches, before):
        np.testing.assert_array_equal(c.float().cpu().numpy(), ref.commit(old, lens, path, n, rows))


def test_commit_flags_bad_paths_and_moves_nothing(cuda, K):
    T, N = 30, 6
    c = [torch.randn(5, 2, T, 64, device=cuda).to(BF) for _ in range(4)]
    handle = K.CacheRows(c[:2], c[2:])
    good = [0, 2, 4, -1, -1, -1]
    path = torch.tensor([good, [0, 2, 2, -1, -1, -1], [0, 3, 1, -1, -1, -1], [0, 2, 6, -1, -1, -1], good],
                        dtype=torch.int32, device=cuda)
    n = torch.tensor([3, 3, 3, 3, 3], dtype=torch.int32, device=cuda)
    lens = torch.tensor([3, 3, 3, 3, 26], device=cuda)  # the last: slot 30 of 30
    before = [t.clone() for t in c]
    K.commit_tree(handle, lens, path, n)
    assert flags(cuda) == 2
    for t, old in zip(c, before):
        torch.testing.assert_close(t[1:], old[1:], rtol=0, atol=0)
        want = old[0].clone()
        want[:, 4], want[:, 5] = old[0][:, 5], old[0][:, 7]
        torch.testing.assert_close(t[0], want, rtol=0, atol=0)
    before = [t.clone() for t in c]
    huge = (1 << 63) - 1
    for lens, rows, n_ in (([-1] * 5, None, [3] * 5), ([huge] * 5, None, [3] * 5), ([3] * 5, [5, -1, 9, 5, 5], [3] * 5),
                           ([3] * 5, None, [7] * 5)):
        K.commit_tree(handle, torch.tensor(lens, device=cuda), path, torch.tensor(n_, dtype=torch.int32, device=cuda),
                      row_map=None if rows is None else torch.tensor(rows, dtype=torch.int32, device=cuda))
        assert flags(cuda) == 2
        for t, old in zip(c, before):
            torch.testing.assert_close(t, old, rtol=0, atol=0)


def test_commit_refusals(cuda, K):
    c = [torch.zeros(2, 2, 30, 64, dtype=BF, device=cuda) for _ in range(2)]
    with pytest.raises(ValueError):
        K.CacheRows([c[0], c[0][:1]], c)
    with pytest.raises(TypeError):
        K.CacheRows([c[0], c[1].half()], c)
    for k, v in (([c[0]], [c[0]]), ([c[0], c[0]], [c[1], c[1].clone()]),
                 ([c[0][:1].expand(2, 2, 30, 64)], [c[1][:1].expand(2, 2, 30, 64)]),
                 ([c[0][:, :1].expand(2, 2, 30, 64)], [c[1][:, :1].expand(2, 2, 30, 64)])):
        with pytest.raises(ValueError, match="overlap"):
            K.CacheRows(k, v)
    h = K.CacheRows(c[:1], c[1:])
    path, n, s = (torch.zeros(3, 4, dtype=torch.int32, device=cuda), torch.ones(3, dtype=torch.int32, device=cuda),
                  torch.zeros(3, dtype=torch.int64, device=cuda))
    with pytest.raises(ValueError):
        K.commit_tree(h, s, path, n)          # three sequences, two cache rows
    with pytest.raises(ValueError):
        K.commit_tree(h, s[:1], path[:2], n[:2])
    with pytest.raises(RuntimeError):
        K.commit_tree(h, s[:2].cpu(), path[:2], n[:2])


# ------------------------------------------------ streams, graphs, devices --
def one_step(K, s):
    plan = K.tree_plan(s["par"])
    o = K.tree_gqa_attn(s["q"], s["k"], s["v"], s["len"], plan.mask, scale=0.1)
    path, n, ids = K.verify_tree(s["logits"], s["tok"], s["par"], s["u"], temperature=1.0, top_p=0.9, top_k=20)
    K.commit_tree(s["rows"], s["len"], path, n)
    return o, path, n, ids


def step_state(K, cuda, seed, B=3, N=9, T=600):
    logits, tok, par, u, _ = verify_inputs(seed, B, N, 700)
    g = gen(seed)
    k, v = normal(g, B, 2, T, 128, dtype=BF), normal(g, B, 2, T, 128, dtype=BF)
    return dict(par=torch.tensor(par, dtype=torch.int32, device=cuda), q=normal(g, B, N, 16, 128, dtype=BF), k=k, v=v,
                rows=K.CacheRows([k], [v]), len=torch.tensor([500, 10, 130][:B], device=cuda), logits=logits,
                tok=torch.from_numpy(tok).to(cuda), u=torch.from_numpy(u).to(cuda))


def test_streams_and_graphs(cuda, K):
    """The four operators on a side stream, captured, replayed with new inputs,
    and two graphs replayed at the same time."""
    a, b = step_state(K, cuda, 1), step_state(K, cuda, 2)
    keep = [{n: t.clone() for n, t in s.items() if torch.is_tensor(t)} for s in (a, b)]

    def reset(s, old):
        for n, t in old.items():
            s[n].copy_(t)

    want = []
    for s, old in zip((a, b), keep):
        out = [t.clone() for t in one_step(K, s)] + [s["k"].clone(), s["v"].clone()]
        want.append(out)
        reset(s, old)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [*one_step(K, a), a["k"], a["v"]]
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want[0]):
        torch.testing.assert_close(x, y, rtol=0, atol=0)
    reset(a, keep[0])
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one_step(K, s)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, old in zip((a, b), keep):
            reset(s, old)
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, out), s, w in zip(graphs, (a, b), want):
            for x, y in zip([*out, s["k"], s["v"]], w):
                torch.testing.assert_close(x, y, rtol=0, atol=0)
    # the first graph with the second's inputs
    reset(a, keep[1])
    graphs[0][0].replay()
    for x, y in zip([*graphs[0][1], a["k"], a["v"]], want[1]):
        torch.testing.assert_close(x, y, rtol=0, atol=0)


def test_empty_batches(cuda, K):
    z = torch.zeros(0, 4, dtype=torch.int32, device=cuda)
    assert K.tree_plan(z).mask.shape == (0, 4)
    c = torch.zeros(0, 2, 8, 64, dtype=BF, device=cuda)
    s = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert K.tree_gqa_attn(torch.zeros(0, 4, 4, 64, dtype=BF, device=cuda), c, c, s, z.long(), scale=1.0).shape == (0, 4, 4, 64)
    out = K.verify_tree(torch.zeros(0, 4, 9, device=cuda), z.long(), z, z.float(), temperature=1.0, top_p=1.0, top_k=1)
    assert [t.shape[0] for t in out] == [0, 0, 0]


# -------------------------------------------------- together, in the model --
def tiny(cuda, dtype):
    from pathlib import Path

    from maple_flash_dgx_spark_b200.model import MapleForCausalLM

    return MapleForCausalLM.from_packed(str(Path(__file__).resolve().parent / "golden" / "tiny_packed"), device=cuda,
                                        dtype=dtype)


def prefill(model, cache, prompts):
    for b, p in enumerate(prompts):
        with cache.prefill_slot(b):
            model.forward(torch.tensor(p, device=model.device).reshape(1, -1), cache=cache)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_speculative_steps_in_the_model(cuda, K, dtype):
    """Three steps of draft, tree forward, verification and commit over a ragged
    batch of the converted checkpoint (sliding window of 16, NoPE layer, partial
    RoPE): each node's logits are plain decoding's over its path, to the
    attention's bound of 1e-2 of their scale; the verification follows them; the
    cache after the commit is that of a forward over the accepted tokens."""
    torch.set_grad_enabled(False)
    try:
        model = tiny(cuda, dtype)
        r = random.Random(5)
        texts = [[r.randrange(512) for _ in range(n)] for n in (14, 3, 23)]
        B, N = 3, 7
        cache = model.make_cache(max_len=64, batch=B)
        cache.remap = True
        prefill(model, cache, [t[:-1] for t in texts])
        cache.swap_slots(0, 2)
        texts[0], texts[2] = texts[2], texts[0]
        for step in range(3):
            par = [[-1, 0, 0, 1, 1, 2, 3], [-1, 0, 1, 2, 3, 4, 5], [-1, 0, 0, 0, 2, -2, -2]]
            tok = [[t[-1]] + [r.randrange(512) for _ in range(N - 1)] for t in texts]
            pt, tt = torch.tensor(par, dtype=torch.int32, device=cuda), torch.tensor(tok, device=cuda)
            first = model.forward_tree(tt, pt, cache).float()
            for b in range(B):  # draft what the model likes: the path along the first children stands
                likes = {0: first[b, 0].argmax().item()}
                tok[b][1] = likes[0]
            tt = torch.tensor(tok, device=cuda)
            lens = list(cache.seen)
            logits = model.forward_tree(tt, pt, cache)
            assert cache.seen == lens and cache.seqlen.tolist() == lens
            for b in range(B):  # every node against plain decoding of its path
                for i in range(N):
                    if par[b][i] < -1:
                        continue
                    line, j = [], i
                    while j >= 0:
                        line.append(tok[b][j])
                        j = par[b][j]
                    plain = model.make_cache(max_len=64)
                    want = model.forward(torch.tensor(texts[b][:-1] + line[::-1], device=cuda).reshape(1, -1),
                                         cache=plain)[0, -1].float()
                    err = (logits[b, i].float() - want).abs().max() / want.abs().max()
                    assert err <= 1e-2, (step, b, i, float(err))
            u = torch.tensor([[r.random() for _ in range(N)] for _ in range(B)], device=cuda)
            greedy = step < 2
            kw = dict(temperature=1.0, top_p=0.95, top_k=1 if greedy else 20)
            path, n, ids = K.verify_tree(logits, tt, pt, u, **kw)
            want = ref.verify(logits.float().cpu().numpy(), np.array(tok), par, u.cpu().numpy(), **kw)
            for x, y in zip((path, n, ids), want):
                np.testing.assert_array_equal(x.cpu().numpy(), y)
            if greedy:
                assert (n >= 2).all()
            cache.commit_tree(path, n)
            kept = n.tolist()
            assert cache.seen == [x + m for x, m in zip(lens, kept)] == cache.seqlen.tolist()
            for b in range(B):
                texts[b] = texts[b] + ids[b, : kept[b]].tolist()
                assert len(texts[b]) == cache.seen[b] + 1
        # what the caches hold now is what plain decoding of the same tokens holds, to the same bound
        for b in range(B):
            plain = model.make_cache(max_len=64)
            model.forward(torch.tensor(texts[b][:-1], device=cuda).reshape(1, -1), cache=plain)
            row = cache.row_of[b]
            for got, want in zip(cache.k + cache.v, plain.k + plain.v):
                x, y = got[row, :, : cache.seen[b]].float(), want[0, :, : cache.seen[b]].float()
                assert (x - y).abs().max() <= 1e-2 * y.abs().max()
    finally:
        torch.set_grad_enabled(True)


def test_forward_tree_refusals(cuda):
    model = tiny(cuda, BF)
    cache = model.make_cache(max_len=16, batch=2)
    par = torch.tensor([[-1, 0, 1]] * 2, dtype=torch.int32, device=cuda)
    tok = torch.zeros(2, 3, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError):
        model.forward_tree(tok[:, :2], par, cache)
    with pytest.raises(ValueError):
        model.forward_tree(tok[:0], par[:0], cache)
    with pytest.raises(ValueError):
        model.forward_tree(tok.repeat(2, 1), par.repeat(2, 1), cache)
    cache.seen[1] = 14
    with pytest.raises(RuntimeError):
        model.forward_tree(tok, par, cache)
    with cache.prefill_slot(0):
        assert model.forward_tree(tok[:1], par[:1], cache).shape == (1, 3, 512)
        with pytest.raises(ValueError):
            model.forward_tree(tok, par, cache)
