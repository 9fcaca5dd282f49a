"""Rotary positions with several axes on the GPU: the rotation against its float64 definition for every dtype,
pairing, section layout, stride and position type, and its gradient against the formula and differences."""

import pytest
import torch

import gguf_train_amd as g
from gguf_train_amd.nn import functional as F

import _kv_ref as ref
from _util import randn

pytestmark = pytest.mark.gpu


def positions(B, S, far, seed=0, axes=3):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, far, (axes, B, S), generator=gen)


def check(got, want, slack, what):
    got = got.double().cpu()
    assert got.shape == want.shape
    over = (got - want).abs() - slack
    assert not torch.isnan(got).any() and over.max().item() <= 0.0, (what, over.max().item())


def bound(want, slack, dtype):
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0, torch.float64: 0.0}[dtype]
    if dtype == torch.float64:
        slack = slack * 2.0 ** -26  # float64 sine, cosine and rotation; the angle's own part is below 2^-46
    return slack + ref.HALF_STEP[dtype] * want.abs() + tiny


SHAPES = [  # B, H, S, D, n_dims, sections
    (1, 1, 1, 2, None, (1,)),
    (4, 32, 1, 128, None, (16, 24, 24)),
    (2, 3, 17, 64, None, (10, 11, 11)),
    (1, 5, 300, 80, None, (14, 13, 13)),
    (2, 2, 33, 96, 64, (12, 10, 10)),
    (1, 2, 9, 10, 6, (1, 1, 1)),
    (3, 1, 40, 72, 40, (20, 0, 0)),
    (1, 2, 3, 1024, None, (200, 156, 156)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("B,H,S,D,n_dims,sections", SHAPES)
def test_rotation(dev, B, H, S, D, n_dims, sections, mode, dtype):
    x = randn((B, H, S, D), 1, dtype)
    pos = positions(B, S, 70000, axes=len(sections))
    got = F.rope_axes(x.to(dev), pos.to(dev), sections, n_dims=n_dims, mode=mode)
    assert got.dtype == dtype and got.is_contiguous()
    want, slack = ref.rope_axes(x, pos, sections, n_dims, mode)
    check(got, want, bound(want, slack, dtype), (B, H, S, D))


@pytest.mark.parametrize("sections", [(24, 20, 20), (22, 21, 21), (64, 0, 0), (0, 0, 0, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_section_layouts(dev, sections, interleaved):
    if interleaved and sections == (0, 0, 0, 64):
        pytest.skip("does not fit: every fourth pair")
    x, pos = randn((2, 4, 50, 128), 2), positions(2, 50, 5000, axes=len(sections))
    got = F.rope_axes(x.to(dev), pos.to(dev), sections, interleaved=interleaved, freq_base=500000.0, freq_scale=0.25)
    want, slack = ref.rope_axes(x, pos, sections, interleaved=interleaved, freq_base=500000.0, freq_scale=0.25)
    check(got, want, bound(want, slack, torch.float32), sections)


def test_float64_stays_float64(dev):
    x, pos = randn((1, 3, 20, 64), 3, torch.float64), positions(1, 20, 60000)
    got = F.rope_axes(x.to(dev), pos.to(dev), (12, 10, 10))
    want, slack = ref.rope_axes(x, pos, (12, 10, 10))
    angle_part = 60000 * 2.0 ** -50 * 8  # (the angle's float64 rounding, of both sides)
    check(got, want, bound(want, slack, torch.float64) + angle_part * 6, "float64")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64, torch.int16, torch.uint8, torch.float16])
def test_position_types_and_strides(dev, kind):
    B, S = 2, 30
    pos = positions(B, S, 200).to(kind)
    x = randn((B, 4, S, 64), 4)
    want, slack = ref.rope_axes(x, pos, (12, 10, 10))
    tol = bound(want, slack, torch.float32)
    check(F.rope_axes(x.to(dev), pos.to(dev), (12, 10, 10)), want, tol, "dense")
    apart = torch.zeros((B, 3, 2 * S), dtype=kind)
    apart[:, :, ::2] = pos.permute(1, 0, 2)
    check(F.rope_axes(x.to(dev), apart.to(dev)[:, :, ::2].permute(1, 0, 2), (12, 10, 10)), want, tol, "strided")
    check(F.rope_axes(x.to(dev), pos, (12, 10, 10)), want, tol, "host positions")
    check(F.rope_axes(x, pos.to(dev), (12, 10, 10)), want, tol, "host input")


def test_fractions_and_far_positions(dev):
    x = randn((1, 2, 4, 64), 5)
    pos = torch.tensor([[0.5, 1.25, 1e6, -3.75], [2.0 ** 31, 1.0, 0.0, 7.5], [0.1, 0.2, 0.3, 2.0 ** 40]], dtype=torch.float64)[:, None]
    want, slack = ref.rope_axes(x, pos, (12, 10, 10))
    # (the reference's own float64 angles of 2^40 are off by 2^-13: compare the others' bound)
    got = F.rope_axes(x.to(dev), pos.to(dev), (12, 10, 10))
    check(got[:, :, :3], want[:, :, :3], bound(want, slack, torch.float32)[:, :, :3] + 1e-6, "fractions")


def test_shared_batch_and_three_dimensional_input(dev):
    x, pos = randn((3, 4, 12, 64), 6), positions(1, 12, 900)
    want, slack = ref.rope_axes(x, pos.expand(3, 3, 12), (12, 10, 10))
    tol = bound(want, slack, torch.float32)
    for p in (pos, pos[:, 0], torch.cat([pos[:, 0], pos[:, 0]], 1)):  # (more positions than tokens: the first)
        check(F.rope_axes(x.to(dev), p.to(dev), (12, 10, 10)), want, tol, "shared")
    check(F.rope_axes(x[0].to(dev), pos.to(dev), (12, 10, 10)), want[0], tol[0], "3-D")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 34])
def test_strided_and_misaligned_input(dev, dtype, D):
    B, H, S, sec = 2, 3, 21, (D // 2 - 10, 5, 5)
    x, pos = randn((B, H, S, D), 7, dtype), positions(B, S, 4000)
    want, slack = ref.rope_axes(x, pos, sec)
    tol = bound(want, slack, dtype)
    xd, pd = x.to(dev), pos.to(dev)
    views = {"(B,S,H,D) memory": xd.transpose(1, 2).contiguous().transpose(1, 2),
             "dims apart": torch.stack([xd, xd], -1)[..., 0],
             "one element in": torch.cat([xd.new_zeros(1), xd.reshape(-1)])[1:].reshape(x.shape),
             "rows apart": torch.cat([xd, xd], -1)[..., :D]}
    for name, view in views.items():
        check(F.rope_axes(view, pd, sec), want, tol, name)
    expanded = xd[:, :1].expand(B, H, S, D)
    check(F.rope_axes(expanded, pd, sec), want[:, :1].expand(B, H, S, D), tol[:, :1].expand(B, H, S, D), "expanded")


def test_same_positions_on_every_axis_are_one_axis(dev):
    x, p = randn((2, 4, 60, 128), 8), torch.arange(60)
    got = F.rope_axes(x.to(dev), p.expand(3, 60).to(dev), (24, 20, 20))
    one = F.rope(x.to(dev), p.to(dev), mode=2)
    # rope's float32 angles: 64 products, each off by 2^-24 of an angle up to 59
    assert (got - one).abs().max().item() <= 59 * 64 * 2.0 ** -24 * 2 * x.abs().max().item()


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_inverse_rotation(dev, mode, interleaved):
    B, H, S, D, sec = 2, 3, 19, 64, (12, 10, 10)
    x, dy, pos = randn((B, H, S, D), 9), randn((B, H, S, D), 10), positions(B, S, 3000)
    xd = x.to(dev).requires_grad_()
    y = F.rope_axes(xd, pos.to(dev), sec, mode=mode, interleaved=interleaved)
    (gx,) = torch.autograd.grad(y, xd, dy.to(dev))
    want, slack = ref.rope_axes(dy, pos, sec, mode=mode, interleaved=interleaved, inverse=True)
    check(gx, want, bound(want, slack, torch.float32), "gradient")


def test_gradient_against_differences_and_twice(dev):
    pos = positions(1, 3, 50).to(dev)
    x = randn((1, 2, 3, 8), 11, torch.float64).to(dev).requires_grad_()
    fn = lambda t: F.rope_axes(t, pos, (2, 1, 1), interleaved=True)
    assert torch.autograd.gradcheck(fn, (x,))
    assert torch.autograd.gradgradcheck(fn, (x,))


def test_gradient_of_a_broadcast_input(dev):
    pos, sec = positions(2, 5, 100).to(dev), (12, 10, 10)
    x = randn((1, 1, 1, 64), 12, torch.float64).to(dev).requires_grad_()
    y = F.rope_axes(x.expand(2, 3, 5, 64), pos, sec)
    dy = randn((2, 3, 5, 64), 13, torch.float64).to(dev)
    (gx,) = torch.autograd.grad(y, x, dy)
    want, _ = ref.rope_axes(dy.cpu(), pos.cpu(), sec, inverse=True)
    assert torch.allclose(gx.cpu(), want.sum((0, 1, 2), keepdim=True), atol=1e-10, rtol=0)


def test_empty(dev):
    for shape in ((0, 2, 3, 64), (1, 0, 3, 64), (1, 2, 0, 64)):
        y = F.rope_axes(torch.ones(shape, device=dev), torch.zeros((3, shape[0], shape[2]), dtype=torch.int64, device=dev), (12, 10, 10))
        assert tuple(y.shape) == shape


def test_nan_positions_and_values_stay_in_their_rows(dev):
    x, pos = randn((1, 2, 4, 64), 14), positions(1, 4, 100).double()
    want, slack = ref.rope_axes(x, pos, (12, 10, 10))
    x[:, :, 1] = float("inf")
    pos[1, 0, 2] = float("nan")
    got = F.rope_axes(x.to(dev), pos.to(dev), (12, 10, 10)).cpu()
    for s in (0, 3):
        check(got[:, :, s], want[:, :, s], bound(want, slack, torch.float32)[:, :, s], s)
    assert torch.isnan(got[0, 0, 2, 12]) and torch.isfinite(got[0, 0, 2, 0])


def test_other_stream(dev):
    x, pos, sec = randn((2, 4, 40, 64), 15, torch.bfloat16).to(dev), positions(2, 40, 900).to(dev), (12, 10, 10)
    want = F.rope_axes(x, pos, sec)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.rope_axes(x, pos, sec)
    s.synchronize()
    assert torch.equal(got, want)


def test_ops_name(dev):
    x, pos = randn((1, 2, 4, 64), 16).to(dev), positions(1, 4, 100).to(dev)
    assert torch.equal(g.rope_axes(x, pos, (12, 10, 10), 64), F.rope_axes(x, pos, (12, 10, 10)))
