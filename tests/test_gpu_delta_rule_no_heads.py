"""Gated delta rule with queries and keys that no head of values reads: their gradients are
zeros, whatever the memory that they lie in held before."""
import ctypes

import pytest
import torch

import cpab
from cpab.pytorch import _native
from test_heads_capi import delta_rule

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def keys(cuda, dtype, B, T, K, dk):
    gen = torch.Generator().manual_seed(T + dk)
    return [torch.randn(B, T, K, dk, generator=gen).to(cuda, dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,K,dk", [(2, 5, 1, 16), (1, 1, 1, 1), (3, 71, 3, 33), (2, 700, 2, 128)])
@pytest.mark.parametrize("wanted", [(0, 1), (0,), (1,)])
def test_gradients(cuda, dtype, B, T, K, dk, wanted):
    given = keys(cuda, dtype, B, T, K, dk)
    v = torch.zeros(B, T, 0, 8, device=cuda, dtype=dtype, requires_grad=True)
    gates = torch.zeros(B, T, 0, device=cuda, dtype=dtype, requires_grad=True)
    for _ in range(3):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(given)]
        o, h = cpab.gated_delta_rule(*leaves, v, gates, gates)
        assert o.shape == (B, T, 0, 8) and h.shape == (B, 0, dk, 8)
        # what the allocator hands out next holds no zeros
        junk = [torch.full((B, T, K, dk), float("nan"), device=cuda, dtype=dtype) for _ in range(4)]
        del junk
        grads = torch.autograd.grad(o.sum() + h.sum(), [leaves[i] for i in wanted] + [v, gates])
        for g, t in zip(grads, [given[i] for i in wanted] + [v, gates]):
            assert g.shape == t.shape and g.dtype == t.dtype and (g == 0).all()


def test_graph_replays(cuda):
    q, k = keys(cuda, BF16, 2, 9, 3, 7)
    v, gates = torch.zeros(2, 9, 0, 8, device=cuda, dtype=BF16), torch.zeros(2, 9, 0, device=cuda, dtype=BF16)

    def passes():
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        o, h = cpab.gated_delta_rule(*leaves, v, gates, gates)
        return torch.autograd.grad(o.sum() + h.sum(), leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes()
    for _ in range(3):
        for g in captured:
            g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all((g == 0).all() for g in captured)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_c_entry(cuda, dtype):
    # exactly the gradients' values are written, and only those that are asked for
    lib, n = _native.load_library(), 2 * 5 * 3 * 7
    rule = delta_rule(dtype=int(dtype == BF16), gate_dtype=0, B=2, T=5, heads=0, key_heads=3, dk=7, dv=8, q=None, k=None,
                      v=None, decay=None, beta=None)
    room = torch.full((2, n + 2), 3.0, device=cuda, dtype=dtype)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(gq, gk):
        at = [ctypes.c_void_p(room[i].data_ptr() + room.element_size()) if on else None for i, on in enumerate((gq, gk))]
        return lib.cpab_delta_rule_backward(rule, None, None, None, *at, None, None, None, None, None, 0, stream)
    assert call(False, False) == 0
    torch.cuda.synchronize()
    assert (room == 3).all()
    assert call(False, True) == 0
    torch.cuda.synchronize()
    assert (room[0] == 3).all() and (room[1, 1:-1] == 0).all() and (room[1, [0, -1]] == 3).all()
    assert call(True, True) == 0
    torch.cuda.synchronize()
    assert (room[:, 1:-1] == 0).all() and (room[:, [0, -1]] == 3).all()
