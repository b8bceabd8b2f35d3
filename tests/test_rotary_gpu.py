"""Rotary positions on the GPU: both layouts, part of the head, types, strides, far positions, gradients."""

from __future__ import annotations

import pytest
import torch

import paged_oracle as oracle
from conftest import announce

pytestmark = pytest.mark.gpu

SHAPES = [  # tokens, heads, head_dim, rotated
    (1, 1, 2, 2), (3, 5, 64, 64), (17, 2, 128, 32), (200, 12, 64, 64), (33, 3, 80, 20), (5, 1, 512, 512), (2050, 4, 128, 128),
    (64, 40, 128, 128), (7, 2, 6, 4),
]


def _inputs(pe, tokens, heads, d, rot, dtype, seed=0, span=5000):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, d, generator=gen).to(dtype)
    positions = torch.randint(0, span, (tokens,), generator=gen)
    inv, _ = pe.rotary_frequencies(rot, 10000.0)
    return x, positions, inv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation(pe, shape, interleaved, dtype):
    x, positions, inv = _inputs(pe, *shape, dtype)
    announce(f"rotary {shape} {dtype} interleaved {interleaved}")
    got = pe.rotary(x.cuda(), positions.cuda(), inv.cuda(), interleaved=interleaved, scale=1.5)
    oracle.assert_within(got, *oracle.rotate(x, positions, inv, interleaved=interleaved, scale=1.5))
    assert got.is_contiguous() and got.dtype == dtype
    assert torch.equal(got[..., 2 * inv.numel():].cpu(), x[..., 2 * inv.numel():])


@pytest.mark.parametrize("base", [0, 1 << 20, (1 << 31) - 5000, -100000])
def test_far_positions_keep_their_angles(pe, base):
    """Positions whose fp32 product with a frequency is off by many turns; negative ones too."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(300, 2, 64, generator=gen)
    positions = base + torch.randint(0, 4000, (300,), generator=gen)
    inv, _ = pe.rotary_frequencies(64, 10000.0)
    for index in (torch.int64, torch.int32):
        got = pe.rotary(x.cuda(), positions.to(index).cuda(), inv.cuda())
        oracle.assert_within(got, *oracle.rotate(x, positions, inv), f"{base} {index}")


def test_more_tokens_than_a_grid_holds(pe):
    """A grid's axis has fewer than 2^32 threads, 256 for four tokens: the rest is another launch's."""
    edge = (2 ** 32 - 1) // 256 * 4
    n = edge + 700
    x = torch.randn(n, 1, 2, device="cuda", dtype=torch.bfloat16)
    positions = torch.arange(n, device="cuda", dtype=torch.int32)
    inv = torch.ones(1)
    got = pe.rotary(x, positions, inv.cuda())
    for at in (0, edge - 300, n - 500):
        part = slice(at, at + 500)
        want = oracle.rotate(x[part].cpu(), positions[part].cpu(), inv)
        oracle.assert_within(got[part], *want, f"tokens from {at}")


def test_strides_and_leading_axes(pe):
    gen = torch.Generator().manual_seed(2)
    rows = torch.randn(4, 30, 9, 64, generator=gen).bfloat16()
    positions = torch.randint(0, 900, (4, 30), generator=gen)
    inv = pe.rotary_frequencies(64, 10000.0)[0]
    want, bound = oracle.rotate(rows.reshape(120, 9, 64), positions.reshape(-1), inv)
    got = pe.rotary(rows.cuda(), positions.cuda(), inv.cuda())
    assert got.shape == rows.shape
    oracle.assert_within(got.reshape(120, 9, 64), want, bound)
    dev = rows.cuda()
    for view, pick in ((dev[:, :, 2:7], (slice(None), slice(2, 7))), (dev[:, :, 1:2], (slice(None), slice(1, 2)))):
        got = pe.rotary(view, positions.cuda(), inv.cuda())
        oracle.assert_within(got.reshape(120, -1, 64), want[pick], bound[pick])
    heads_first = dev.transpose(1, 2).contiguous().transpose(1, 2)  # [B, H, S, D] seen as [B, S, H, D]
    oracle.assert_within(pe.rotary(heads_first, positions.cuda(), inv.cuda()).reshape(120, 9, 64), want, bound)
    last = dev.transpose(2, 3).contiguous().transpose(2, 3)  # no unit stride
    oracle.assert_within(pe.rotary(last, positions.cuda(), inv.cuda()).reshape(120, 9, 64), want, bound)
    # positions that broadcast over the batch, and one for all
    shared = positions[0]
    want, bound = oracle.rotate(rows.reshape(120, 9, 64), shared.repeat(4), inv)
    oracle.assert_within(pe.rotary(dev, shared.cuda(), inv.cuda()).reshape(120, 9, 64), want, bound)
    want, bound = oracle.rotate(rows[0], torch.full((30,), 7), inv)
    oracle.assert_within(pe.rotary(dev[0], torch.tensor(7).cuda(), inv.cuda()), want, bound)
    one = dev[0, 3]  # [heads, head_dim], one position
    want, bound = oracle.rotate(rows[0, 3:4], torch.tensor([41]), inv)
    oracle.assert_within(pe.rotary(one, torch.tensor(41).cuda(), inv.cuda())[None], want, bound)
    # a broadcast row, and bases off 16 bytes
    one = dev[0, :1].expand(30, 9, 64)
    want, bound = oracle.rotate(rows[0, :1].expand(30, 9, 64), positions[0], inv)
    oracle.assert_within(pe.rotary(one, positions[0].cuda(), inv.cuda()), want, bound)
    odd = torch.zeros(30, 9, 65, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(dev[0])
    want, bound = oracle.rotate(rows[0], positions[0], inv)
    oracle.assert_within(pe.rotary(odd, positions[0].cuda(), inv.cuda()), want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [(3, 5, 64, 64), (33, 3, 80, 20), (2050, 2, 64, 32)])
def test_gradient_is_the_opposite_rotation(pe, shape, interleaved, dtype):
    x, positions, inv = _inputs(pe, *shape, dtype)
    grad = torch.randn(x.shape, generator=torch.Generator().manual_seed(7)).to(dtype)
    leaf = x.cuda().requires_grad_()
    y = pe.rotary(leaf, positions.cuda(), inv.cuda(), interleaved=interleaved, scale=1.25)
    oracle.assert_within(y.detach(), *oracle.rotate(x, positions, inv, interleaved=interleaved, scale=1.25))
    y.backward(grad.cuda())
    want, bound = oracle.rotate(grad, positions, inv, interleaved=interleaved, scale=1.25, inverse=True)
    oracle.assert_within(leaf.grad, want, bound)


def test_gradient_against_differences(pe):
    """The rotation is linear, so a difference has no error but fp32 rounding: f(x + e) - f(x) of a sum
    weighted by g, against the gradient along e. Each of the 2 * 640 products rounds by 2^-24 of itself."""
    x, positions, inv = _inputs(pe, 10, 2, 32, 16, torch.float32, seed=3)
    gen = torch.Generator().manual_seed(8)
    e, g = torch.randn(x.shape, generator=gen), torch.randn(x.shape, generator=gen)
    leaf = x.cuda().requires_grad_()
    y = pe.rotary(leaf, positions.cuda(), inv.cuda(), interleaved=True)
    (y * g.cuda()).sum().backward()
    moved = pe.rotary((x + e).cuda(), positions.cuda(), inv.cuda(), interleaved=True)
    change = float(((moved - y.detach()).double().cpu() * g.double()).sum())
    along = float((leaf.grad.double().cpu() * e.double()).sum())
    size = float((g.double().abs() * (x.double().abs() + e.double().abs()) * 2).sum())
    assert abs(change - along) <= 1e-6 * size


def test_gradients_of_views_shared_heads_and_twice(pe):
    """A broadcast input gathers its rows' gradients; a non-contiguous output gradient; second derivatives."""
    inv = pe.rotary_frequencies(64, 10000.0)[0].cuda()
    positions = torch.arange(6, device="cuda")
    one = torch.randn(1, 2, 64, device="cuda", requires_grad=True)
    pe.rotary(one.expand(6, 2, 64), positions, inv).sum().backward()  # the gradient of sum is a broadcast one
    want, bound = oracle.rotate(torch.ones(6, 2, 64), positions.cpu(), inv.cpu(), inverse=True)
    oracle.assert_within(one.grad, want.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 6 * 2.0 ** -24 * 2)
    x = torch.randn(6, 2, 64, device="cuda", requires_grad=True)
    g = torch.randn(6, 2, 64, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(pe.rotary(x, positions, inv), x, g, create_graph=True)
    (dg,) = torch.autograd.grad(dx, g, torch.ones_like(dx))
    want, bound = oracle.rotate(torch.ones(6, 2, 64), positions.cpu(), inv.cpu())
    oracle.assert_within(dg.detach(), want, bound)


def test_training_step_in_a_graph(pe):
    """Forward and backward captured and replayed with new inputs; eager steps of other leaves between."""
    inv = pe.rotary_frequencies(64, 10000.0)[0].cuda()
    positions = torch.arange(40, device="cuda")
    x = torch.randn(40, 3, 64, device="cuda").bfloat16().requires_grad_()
    g = torch.randn(40, 3, 64, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pe.rotary(x, positions, inv), x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pe.rotary(x, positions, inv)
        (dx,) = torch.autograd.grad(y, x, g)
    for n in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(40, 3, 64, device="cuda"))
            g.copy_(torch.randn(40, 3, 64, device="cuda"))
            positions.add_(1000)
        graph.replay()
        got, grad = y.detach().clone(), dx.clone()
        torch.cuda.synchronize()
        leaf = x.detach().clone().requires_grad_()
        want = pe.rotary(leaf, positions, inv)
        want.backward(g)
        assert torch.equal(got, want.detach()) and torch.equal(grad, leaf.grad), n


def test_rotary_agrees_with_the_packed_layers(pe):
    """Split-half pairs over the whole head: the packed encoder's rope_qkv within its tables' rounding, each
    of cos and sin off by half a bf16 step (2^-9 of at most 1) before the products."""
    from packed_encoders_amd import ops
    from packed_encoders_amd.hip_attention import rope_qkv

    tokens, heads, d, theta = 50, 4, 64, 10000.0
    qkv = torch.randn(1, tokens, 3 * heads * d, device="cuda").bfloat16()
    positions = torch.randint(0, 800, (tokens,), device="cuda")
    with torch.inference_mode():
        cos, sin = ops.rope_rows(positions, 800, d, theta, torch.bfloat16)
        q, _ = rope_qkv(qkv, heads, d, cos, sin)
    got = pe.rotary(qkv.view(tokens, 3, heads, d)[:, 0], positions, pe.rotary_frequencies(d, theta, device="cuda")[0])
    x = qkv.view(tokens, 3, heads, d)[:, 0].float().abs()
    pair = x + torch.cat((x[..., d // 2:], x[..., :d // 2]), -1)
    limit = pair * (2.0 ** -8 + 1e-4) + 2 * 2.0 ** -8 * got.float().abs() + 1e-6  # tables' step and angle, both outputs' steps
    assert ((got.float() - q[0].float()).abs() <= limit).all()


def test_refusals(pe):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos, inv = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(32, device="cuda")
    for args in ((x.double(), pos, inv), (x[0, 0], pos, inv), (x, pos.float(), inv), (x, pos[:3], inv), (x, pos.cpu(), inv),
                 (x, pos, inv.double()), (x, pos, inv.cpu()), (x, pos, inv[None]), (x, pos, torch.ones(33, device="cuda")),
                 (x, pos, inv[:0]), (x, pos[:, None], inv), (x, pos, inv.clone().requires_grad_()), (x.int(), pos, inv)):
        with pytest.raises(ValueError):
            pe.rotary(*args)
        if args[0].is_floating_point():
            with pytest.raises(ValueError):
                pe.rotary(args[0].clone().requires_grad_(), *args[1:])
    assert pe.rotary(x[:0], pos[:0], inv).shape == (0, 2, 64)
    assert pe.rotary(x[:, :0], pos, inv).shape == (4, 0, 64)
