"""The plain restatements of the gate, the gated activation and products on 4-bit weights, pinned on the CPU by hand-made
answers and finite differences; and what the library and the front end refuse."""

import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi, moe
from oracle import expert_ops_oracle as oracle


def test_gate_by_hand():
    row = np.log(np.array([[1.0, 4.0, 2.0, 1.0]]))
    ids, w = oracle.gate(row, 2)
    assert ids.tolist() == [[1, 2]] and np.allclose(w, [[4 / 6, 2 / 6]])
    ids, w = oracle.gate(row, 2, renormalize=False, scale=3.0)
    assert np.allclose(w, [[3 * 4 / 8, 3 * 2 / 8]])
    ids, w = oracle.gate(row, 3, bias=np.array([1.0, 0, 0, 0]), renormalize=False)  # the bias moves the choice alone
    assert ids.tolist() == [[0, 1, 2]] and np.allclose(w, [[1 / 8, 4 / 8, 2 / 8]])
    ids, _ = oracle.gate(np.zeros((1, 5)), 3)
    assert ids.tolist() == [[0, 1, 2]]  # ties
    ids, w = oracle.gate(np.array([[0.0, -np.inf, -np.inf]]), 2)
    assert ids.tolist() == [[0, -1]] and w.tolist() == [[1.0, 0.0]]
    ids, w = oracle.gate(np.full((1, 3), -np.inf), 2)
    assert ids.tolist() == [[-1, -1]] and w.tolist() == [[0.0, 0.0]]


def test_gate_clusters_by_hand():
    row = np.array([[5.0, 0, 0, 4, 4, 4, 3, 3, 0]])
    assert oracle.gate(row, 2, clusters=3, top_clusters=1)[0].tolist() == [[0, 1]]
    top2 = oracle.gate(row, 2, score="sigmoid", clusters=3, top_clusters=1, cluster_score="top2")[0]
    assert top2.tolist() == [[3, 4]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gate_gradient_against_differences(score, renormalize):
    rng = np.random.default_rng(0)
    l, dw = rng.standard_normal((3, 9)), rng.standard_normal((3, 4))
    l[1, 2] = -np.inf
    kw = dict(score=score, renormalize=renormalize, scale=2.5)
    ids, _ = oracle.gate(l, 4, **kw)
    grad = oracle.gate_grad(l, ids, dw, **kw)
    eps = 1e-6
    for t in range(3):
        for e in range(9):
            if l[t, e] == -np.inf:
                assert grad[t, e] == 0
                continue
            up, down = l.copy(), l.copy()
            up[t, e] += eps
            down[t, e] -= eps
            (iu, wu), (id_, wd) = oracle.gate(up, 4, **kw), oracle.gate(down, 4, **kw)
            assert np.array_equal(iu, ids) and np.array_equal(id_, ids)
            assert abs(((wu - wd) * dw).sum() / (2 * eps) - grad[t, e]) < 1e-8


def test_swiglu_gradient_against_differences():
    rng = np.random.default_rng(1)
    y, dout = 2 * rng.standard_normal((2, 10)), rng.standard_normal((2, 5))
    grad, eps = oracle.swiglu_grad(y, dout), 1e-6
    for i in range(2):
        for j in range(10):
            up, down = y.copy(), y.copy()
            up[i, j] += eps
            down[i, j] -= eps
            assert abs(((oracle.swiglu(up) - oracle.swiglu(down)) * dout).sum() / (2 * eps) - grad[i, j]) < 1e-8


def test_int4_by_hand():
    q = np.array([[[0], [8], [15]]], np.uint8)
    assert oracle.int4_dense(q, np.array([[[0.5]]]), None, 32)[0, :, 0].tolist() == [-4.0, 0.0, 3.5]
    assert oracle.int4_dense(q, np.array([[[0.5]]]), np.array([[[1]]], np.uint8), 32)[0, :, 0].tolist() == [-0.5, 3.5, 7.0]


# ---- refusals --------------------------------------------------------------------------------------------------------------
P = 4096  # a pointer that no refused call reads


def _gate(spec=(2, 1, 1, 0, 1.0), logits=P, ids=P, weights=P, tokens=4, experts=8, dtype=_capi.RD_DTYPE_BF16):
    s = None if spec is None else ctypes.byref(_capi.GateSpec(*spec))
    return _capi.lib.rd_moe_gate(None, logits, None, ids, weights, tokens, experts, s, dtype)


@pytest.mark.parametrize("kw", [
    dict(spec=None), dict(spec=(0, 1, 1, 0, 1.0)), dict(spec=(65, 1, 1, 0, 1.0), experts=128), dict(spec=(9, 1, 1, 0, 1.0)),
    dict(spec=(2, 0, 1, 0, 1.0)), dict(spec=(2, 3, 1, 0, 1.0)), dict(spec=(2, 65, 1, 0, 1.0), experts=130), dict(spec=(2, 2, 0, 0, 1.0)),
    dict(spec=(2, 2, 3, 0, 1.0)), dict(spec=(5, 2, 1, 0, 1.0)), dict(spec=(2, 1, 1, 8, 1.0)), dict(spec=(2, 1, 1, 0, 0.0)),
    dict(spec=(2, 1, 1, 0, float("inf"))), dict(spec=(2, 1, 1, 0, float("nan"))), dict(logits=None), dict(ids=None),
    dict(weights=None), dict(tokens=-1), dict(tokens=(1 << 25) + 1), dict(experts=0), dict(experts=1025), dict(dtype=_capi.RD_DTYPE_F8E4M3_BF16)],
    ids=lambda kw: ",".join(f"{k}={v}" for k, v in kw.items()))
def test_gate_refusals(kw):
    assert _gate(**kw) == -1 and _capi.lib.rd_last_error()


def test_gate_of_no_tokens_does_nothing():
    assert _gate(tokens=0, logits=None, ids=None, weights=None) == 0


def test_swiglu_refusals():
    lib = _capi.lib
    for rows, f, dtype, y, out in ((-1, 8, 0, P, P), (4, -1, 0, P, P), (4, 1 << 30, 0, P, P), (4, 8, 3, P, P), (4, 8, 0, None, P), (4, 8, 0, P, None)):
        assert lib.rd_moe_swiglu(None, y, out, rows, f, dtype) == -1
        assert lib.rd_moe_swiglu_grad(None, y, P, out, rows, f, dtype) == -1
    assert lib.rd_moe_swiglu_grad(None, P, None, P, 4, 8, 0) == -1
    assert lib.rd_moe_swiglu(None, None, None, 0, 8, 0) == 0 and lib.rd_moe_swiglu(None, None, None, 8, 0, 0) == 0


def _int4(x=P, codes=P, scales=P, gs=P, y=P, m=4, k=64, n=8, g=2, first=0, local=2, block=32, sdtype=0, dtype=0, ws=None, kernel=0):
    return _capi.lib.rd_gmm_int4(None, x, codes, scales, None, gs, y, m, k, n, g, first, local, block, sdtype, dtype, kernel, ws, 0)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(codes=None), dict(codes=P + 4), dict(scales=None), dict(gs=None), dict(y=None), dict(m=-1), dict(m=1 << 25),
    dict(k=-1), dict(n=-1), dict(g=0, local=0), dict(local=0), dict(first=1), dict(first=-1), dict(first=2 ** 31 - 1), dict(local=3),
    dict(block=16), dict(block=256), dict(sdtype=3), dict(sdtype=2), dict(sdtype=1), dict(kernel=3), dict(kernel=-1), dict(k=(1 << 24) + 1), dict(dtype=1), dict(dtype=3),
    dict(g=4096, local=4096, k=1 << 20, n=1 << 20)], ids=lambda kw: ",".join(f"{k}={v}" for k, v in kw.items()))
def test_int4_refusals(kw):
    assert _int4(**kw) == -1 and _capi.lib.rd_last_error()


def test_int4_sizes():
    lib = _capi.lib
    assert lib.rd_int4_codes_bytes(2, 128, 3) == 2 * 1024 and lib.rd_int4_codes_bytes(2, 129, 17) == 2 * 2 * 2 * 1024
    assert lib.rd_int4_codes_bytes(2, 0, 3) == 0 and lib.rd_int4_codes_bytes(-1, 8, 8) == 0
    assert _int4(m=0) == 0 and _int4(n=0) == 0
    assert lib.rd_int4_pack(None, None, P, 1, 32, 8, 0) == -1 and lib.rd_int4_pack(None, P, P + 2, 1, 32, 8, 0) == -1
    assert _int4(ws=P + 4) == -3 and lib.rd_gmm_int4_workspace_bytes(8, 64, 64, 2, 0) == 0
    for kernel in (0, 1, 2):  # more tiles than a launch has
        assert _int4(m=(1 << 25) - 1, n=1 << 24, g=2, kernel=kernel) == -2


def test_front_end_refusals():
    rand = torch.randn
    with pytest.raises(ValueError, match="score"):
        moe.gate(rand(4, 8), 2, score="relu")
    with pytest.raises(ValueError, match="cluster_score"):
        moe.gate(rand(4, 8), 2, cluster_score="sum")
    with pytest.raises(ValueError, match="tokens, experts"):
        moe.gate(rand(8), 2)
    for top_k in (0, -3, 9, 2 ** 40):
        with pytest.raises(ValueError, match="top_k"):
            moe.gate(rand(4, 8), top_k)
    with pytest.raises(TypeError):
        moe.gate(rand(4, 8).double(), 2)
    with pytest.raises(RuntimeError, match="ROCm"):
        moe.gate(rand(4, 8), 2)
    with pytest.raises(ValueError, match="gate and up"):
        moe.swiglu(rand(4, 7))
    with pytest.raises(TypeError):
        moe.swiglu(rand(4, 8).double())
    with pytest.raises(RuntimeError, match="ROCm"):
        moe.swiglu(rand(4, 8))
    q, scales = torch.zeros((2, 64, 8), dtype=torch.uint8), torch.ones((2, 2, 8)).half()
    with pytest.raises(RuntimeError, match="ROCm"):
        rd.pack_int4(q, scales, block=32)
    for bad in (dict(block=16), dict(block=48)):
        with pytest.raises(AssertionError, match="block"):
            rd.pack_int4(q, scales, **bad)
    with pytest.raises(ValueError, match="scales"):
        rd.pack_int4(q, scales, block=64)
    with pytest.raises(ValueError, match="zeros"):
        rd.pack_int4(q, scales, torch.zeros((2, 1, 8), dtype=torch.uint8), block=32)
    with pytest.raises(TypeError, match="zeros"):
        rd.pack_int4(q, scales, torch.zeros((2, 2, 8)), block=32)
    with pytest.raises(TypeError, match="scales"):
        rd.pack_int4(q, scales.float(), block=32)
    with pytest.raises(TypeError):
        rd.pack_int4(q.float(), scales, block=32)
    scales = torch.ones((2, 1, 8, 4)).half()
    w = rd.Int4Weights(torch.zeros((2, 1, 1, 64, 4), dtype=torch.int32), scales, None, 64, 8, 32)
    gs, x = torch.tensor([1, 3], dtype=torch.int32), rand(4, 64).bfloat16()
    with pytest.raises(RuntimeError, match="ROCm"):
        rd.ragged_dot_int4(x, w, gs)
    for case, error in ((dict(x=x.float()), TypeError), (dict(x=x[:, :32]), AssertionError), (dict(gs=gs[:1]), AssertionError),
                        (dict(w=w._replace(codes=w.codes[:, :, :, :8])), AssertionError), (dict(w=w._replace(block=64)), AssertionError),
                        (dict(w=w._replace(scales=scales.float())), TypeError), (dict(x=x.clone().requires_grad_()), NotImplementedError),
                        (dict(w=w._replace(zeros=torch.zeros((2, 1, 8, 4)))), TypeError), (dict(w=w._replace(codes=w.codes.float())), AssertionError)):
        with pytest.raises(error):
            rd.ragged_dot_int4(case.get("x", x), case.get("w", w), case.get("gs", gs))
    with pytest.raises(AssertionError):
        rd.ragged_dot_int4(x, w, gs, group_offset=1)


def test_tangents_are_refused():
    with fwAD.dual_level():
        dual = lambda *s: fwAD.make_dual(torch.randn(*s), torch.randn(*s))
        w = rd.Int4Weights(torch.zeros((1, 1, 1, 64, 4), dtype=torch.int32), torch.ones((1, 1, 8, 2)), None, 64, 8, 64)
        for call in (lambda: moe.gate(dual(4, 8), 2), lambda: moe.swiglu(dual(4, 8)),
                     lambda: rd.ragged_dot_int4(dual(4, 64).bfloat16(), w, torch.tensor([4]))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
