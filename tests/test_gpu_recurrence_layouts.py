"""Inputs whose samples lie far apart: read where they lie as far as a tile's offsets reach,
copied beyond that, and never refused where the copy is not."""
import pytest
import torch

import cpab
from cpab.pytorch import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_time_major_inputs_are_not_copied(cuda, dtype):
    # [T, B, C] in memory: 60,000 values from sample to sample
    B, T, C = 60, 70, 1000
    gen = torch.Generator(device=cuda).manual_seed(1)
    x, f, g = (torch.randn(T, B, C, device=cuda, generator=gen).to(dtype).transpose(0, 1) for _ in range(3))
    plain = [t.contiguous() for t in (x, f, g)]
    y0, h0 = cpab.gated_recurrence(*plain)
    dy = torch.randn(B, T, C, device=cuda, generator=gen).to(dtype)

    def run(inputs):
        leaves = [t.detach().requires_grad_() for t in inputs]
        y, h = cpab.gated_recurrence(*leaves)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, torch.ones_like(h))))

    assert all(torch.equal(a, b) for a, b in zip(run((x, f, g)), run(plain)))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y, h = cpab.gated_recurrence(x, f, g)
    room = 1 << 21   # the allocator's rounding of the outputs and a workspace
    assert torch.cuda.max_memory_allocated() - before < y.numel() * y.element_size() + room
    assert torch.equal(y, y0) and torch.equal(h, h0)


def test_slices_too_far_apart_are_copied(cuda):
    # 2.16 million values from sample to sample, more than a tile's offsets reach in 32 bits
    T, C = 260, 720000
    whole = torch.empty(1, T, 3 * C, device=cuda)
    for t in range(0, T, 20):
        whole[:, t:t + 20].normal_()
    x, f, g = whole.split(C, -1)
    with torch.no_grad():
        y, h = cpab.gated_recurrence(x, f, g)
        for at in (0, C // 2, C - 64):
            part = slice(at, at + 64)
            a, b = cpab.gated_recurrence(*(t[..., part].contiguous() for t in (x, f, g)))
            assert torch.equal(y[..., part], a) and torch.equal(h[..., part], b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_single_samples_at_any_stride(cuda, dtype):
    # over one sample its stride says nothing
    B, C = 3, 40
    x, f, g = (torch.randn(B, C, device=cuda).to(dtype) for _ in range(3))
    want = cpab.gated_recurrence(x[:, None], f[:, None], g[:, None])
    for stride in (0, 1, 2 ** 28, 2 ** 40):
        far = [t.as_strided((B, 1, C), (C, stride, 1)).requires_grad_() for t in (x.clone(), f.clone(), g.clone())]
        got = cpab.gated_recurrence(*far)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        grads = torch.autograd.grad(got, far, (torch.ones_like(got[0]), torch.ones_like(got[1])))
        near = [t.detach().contiguous().view(B, 1, C).requires_grad_() for t in (x, f, g)]
        out = cpab.gated_recurrence(*near)
        for a, b in zip(grads, torch.autograd.grad(out, near, (torch.ones_like(out[0]), torch.ones_like(out[1])))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,C", [(2, 8), (16, 100), (40, 64), (300, 64), (1100, 8)])
@pytest.mark.parametrize("more", [0, 1])
def test_as_far_apart_as_the_kernels_reach(cuda, dtype, T, C, more):
    # samples over 2^31 bytes of a tile, read in place, and one value further, copied
    kind = 0 if dtype == torch.float32 else 1
    stride = _native.load_library().cpab_recurrence_max_stride(kind, 1, T, C) + more
    near = [torch.randn(1, T, C, device=cuda).to(dtype) for _ in range(3)]
    room = torch.empty((T - 1) * stride + C, device=cuda, dtype=dtype)
    far = room.as_strided((1, T, C), (0, stride, 1))
    far.copy_(near[0])
    dy = torch.randn(1, T, C, device=cuda).to(dtype)

    def run(x, f, g):
        leaves = [t.detach().requires_grad_() for t in (x, f, g)]
        y, h = cpab.gated_recurrence(*leaves)
        return (y, h, *torch.autograd.grad((y, h), leaves, (dy, torch.ones_like(h))))

    want = run(*near)
    assert all(torch.equal(a, b) for a, b in zip(run(far, *near[1:]), want))
    far.copy_(near[1])
    assert all(torch.equal(a, b) for a, b in zip(run(near[0], far, near[2]), want))
    far.copy_(near[2])
    assert all(torch.equal(a, b) for a, b in zip(run(*near[:2], far), want))
