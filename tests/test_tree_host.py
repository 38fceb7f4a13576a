"""Speculative-decoding operators, host side (no GPU): the C entry points refuse
what they cannot run before any launch, the Python wrappers raise the types the
other operators raise, and the restatements the GPU tests compare with hold on
cases worked out by hand."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests import tree_reference as ref

torch = pytest.importorskip("torch")

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def L():
    from maple_flash_dgx_spark_b200 import _lib
    from maple_flash_dgx_spark_b200.build import build

    build()
    return _lib.lib()


def _attn(L, *, scale=0.1, q=P, dtype=1, B=2, N=8, H=32, Hkv=4, T=1024, D=128, k=P, out=P, ws=P, nbytes=1 << 40, err=P, sb=None,
          window=0, qsh=None, Bc=2):
    qsh = D if qsh is None else qsh
    sb = Hkv * T * D if sb is None else sb
    return L.maple_tree_gqa_attn(q, dtype, B, N, H, N * H * D, H * D, qsh, k, k, Bc, Hkv, sb, T * D, T, D, P, P, None,
                                 scale, window, out, ws, nbytes, err, None)


def test_tree_attention_refuses_before_any_launch(L):
    assert _attn(L, B=0) == 0                        # nothing to do
    for bad in (dict(B=-1), dict(N=0), dict(N=65), dict(H=0), dict(Hkv=0), dict(H=30), dict(D=96), dict(T=0),
                dict(window=-1), dict(B=1 << 17), dict(Bc=0), dict(T=1 << 31), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(scale=-3e38), dict(H=8192, Hkv=1)):
        assert _attn(L, **bad) == 1, bad
    for null in ("q", "k", "out", "err"):
        assert _attn(L, **{null: None}) == 1, null
    assert _attn(L, dtype=2) == 2
    assert _attn(L, q=ctypes.c_void_p(264)) == 7     # 8-byte aligned
    assert _attn(L, k=ctypes.c_void_p(264)) == 7
    assert _attn(L, sb=4 * 1024 * 128 + 4) == 7
    assert _attn(L, qsh=132) == 7
    need = L.maple_tree_gqa_workspace_bytes(2, 8, 32, 4, 128, 65536, 0, 1)
    assert need > 0
    assert _attn(L, T=65536, ws=None) == 6
    assert _attn(L, T=65536, nbytes=need - 1) == 6
    assert _attn(L, dtype=0, ws=None) == 6           # fp32: splits of its own
    assert L.maple_tree_gqa_workspace_bytes(2, 65, 32, 4, 128, 1024, 0, 1) == -1
    assert L.maple_tree_gqa_workspace_bytes(2, 8, 30, 4, 128, 1024, 0, 1) == -1
    assert L.maple_tree_gqa_workspace_bytes(1, 8, 8192, 1, 128, 1024, 0, 1) == -1


def test_tree_plan_refuses_before_any_launch(L):
    assert L.maple_tree_plan(P, 0, 8, 8, 1, P, P, P, None) == 0
    for B, N in ((-1, 8), (1, 0), (1, 65)):
        assert L.maple_tree_plan(P, B, N, 8, 1, P, P, P, None) == 1
    for k in (0, 5, 6, 7):
        args = [P, 1, 8, 8, 1, P, P, P, None]
        args[k] = None
        assert L.maple_tree_plan(*args) == 1


def _verify(L, *, dtype=1, B=2, N=8, V=1000, draft=None, d_dtype=0, T=1.0, top_p=0.9, top_k=20, ws=P, nbytes=1 << 40,
            null=None):
    a = {k: P for k in ("logits", "tokens", "parents", "uniform", "path", "n_path", "out", "err")}
    if null:
        a[null] = None
    return L.maple_verify_tree(a["logits"], dtype, B, N, V, N * V, V, a["tokens"], a["parents"], a["uniform"], draft,
                               d_dtype, N * V, V, T, top_p, top_k, 0, a["path"], a["n_path"], a["out"], ws, nbytes,
                               a["err"], None)


def test_verify_refuses_before_any_launch(L):
    assert _verify(L, B=0) == 0
    nan = float("nan")
    for bad in (dict(B=-1), dict(N=0), dict(N=65), dict(V=0), dict(V=1 << 31), dict(B=1 << 17), dict(T=0.0),
                dict(T=-1.0), dict(T=nan), dict(top_p=0.0), dict(top_p=nan), dict(top_k=0), dict(top_k=65)):
        assert _verify(L, **bad) == 1, bad
    for name in ("logits", "tokens", "parents", "uniform", "path", "n_path", "out", "err"):
        assert _verify(L, null=name) == 1, name
    assert _verify(L, dtype=5) == 2
    assert _verify(L, draft=P, d_dtype=5) == 2
    need = L.maple_verify_tree_workspace_bytes(2, 8, 1000, 20)
    assert need > 0
    assert _verify(L, ws=None) == 6
    assert _verify(L, nbytes=need - 1) == 6


def test_commit_refuses_before_any_launch(L):
    def call(layers=2, dtype=1, B=2, N=8, Hkv=4, T=64, D=128, ptrs=(256, 512), sb=4 * 64 * 128, null=None):
        table = (ctypes.c_void_p * max(len(ptrs), 1))(*ptrs)
        a = {k: P for k in ("seqlen", "path", "n_path", "err")}
        if null:
            a[null] = None
        return L.maple_commit_tree(table, table, layers, dtype, B, N, 2, Hkv, sb, T * D, T, D, a["seqlen"], a["path"],
                                   a["n_path"], None, a["err"], None)

    assert call(layers=0) == 0 and call(B=0) == 0
    for bad in (dict(layers=-1), dict(B=-1), dict(N=0), dict(N=65), dict(Hkv=0), dict(T=0), dict(D=0),
                dict(ptrs=(256, 0)), dict(sb=0)):
        assert call(**bad) == 1, bad
    for name in ("seqlen", "path", "n_path", "err"):
        assert call(null=name) == 1, name
    assert call(dtype=7) == 2
    assert call(ptrs=(256, 264)) == 7
    assert call(sb=4 * 64 * 128 + 4) == 7


def test_wrappers_refuse_cpu_tensors_and_shapes():
    from maple_flash_dgx_spark_b200 import kernels as K

    par = torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        K.tree_plan(par)
    q, c = torch.zeros(1, 3, 4, 64), torch.zeros(1, 2, 16, 64)
    with pytest.raises(RuntimeError):
        K.tree_gqa_attn(q, c, c, torch.zeros(1, dtype=torch.int64), torch.ones(1, 3, dtype=torch.int64), scale=0.1)
    with pytest.raises(ValueError):
        K.tree_gqa_attn(q[0], c, c, torch.zeros(1, dtype=torch.int64), torch.ones(1, 3, dtype=torch.int64), scale=0.1)
    with pytest.raises(RuntimeError):
        K.verify_tree(torch.zeros(1, 3, 9), torch.zeros(1, 3, dtype=torch.int64), par, torch.zeros(1, 3),
                      temperature=1.0, top_p=1.0, top_k=1)
    with pytest.raises(ValueError):
        K.verify_tree(torch.zeros(3, 9), torch.zeros(1, 3, dtype=torch.int64), par, torch.zeros(1, 3),
                      temperature=1.0, top_p=1.0, top_k=1)
    with pytest.raises(RuntimeError):
        K.CacheRows([c], [c])
    with pytest.raises(ValueError):
        K.CacheRows([c], [c, c])
    with pytest.raises(ValueError):
        K.CacheRows([c.transpose(2, 3)], [c.transpose(2, 3)])


def test_reference_plan_by_hand():
    mask, depth, bad = ref.plan([[-1, 0, 0, 1, 3, -2, 5], [-2, -1, 1, 5, 2, 3, 0]])
    assert mask[0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0, 0]
    assert depth[0].tolist() == [0, 1, 1, 2, 3, 0, 0]
    # node 3's parent is not before it: its branch (5) drops out; node 0 is padding, so is its child 6
    assert mask[1].tolist() == [0, 0b10, 0b110, 0, 0b10110, 0, 0] and bad


def test_reference_verify_by_hand():
    logits = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.8, 0.1], [0.2, 0.2, 0.6]]]))
    kw = dict(temperature=1.0, top_p=1.0, top_k=3)
    par, tok = [[-1, 0, 1]], [[9, 0, 1]]
    # 0.4 < 0.5 accepts token 0; 0.9 >= 0.8 refuses token 1; the rest is half token 0, half token 2
    path, n, ids = ref.verify(logits, tok, par, [[0.3, 0.4, 0.9]], **kw)
    assert (path.tolist(), n.tolist(), ids.tolist()) == ([[0, 1, -1]], [2], [[0, 0, -1]])
    path, n, ids = ref.verify(logits, tok, par, [[0.6, 0.4, 0.9]], **kw)
    assert ids.tolist() == [[0, 2, -1]]
    # both accepted: the last token comes from node 2
    path, n, ids = ref.verify(logits, tok, par, [[0.5, 0.4, 0.7]], **kw)
    assert n.tolist() == [3] and ids.tolist() == [[0, 1, 2]]
    # a draft that over-weights token 0: refused at u q >= p, then p - q leaves tokens 1 and 2
    q = np.array([[[0.8, 0.1, 0.1]] * 3])
    path, n, ids = ref.verify(logits, tok, par, [[0.5, 0.7, 0.0]], draft=q, **kw)
    assert n.tolist() == [1] and ids.tolist() == [[1, -1, -1]]      # rest 0.2 : 0.1, u 0.5 -> token 1
    path, n, ids = ref.verify(logits, tok, par, [[0.7, 0.7, 0.0]], draft=q, **kw)
    assert ids.tolist() == [[2, -1, -1]]
