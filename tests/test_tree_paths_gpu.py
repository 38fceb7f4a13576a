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
