"""Rotary positions with several axes: what is refused, before any device work, and empty inputs."""

import ctypes

import pytest
import torch

from gguf_train_amd import _C, _bridge
from gguf_train_amd.nn import functional as F

X = torch.ones(2, 3, 4, 8)
P = torch.zeros(3, 2, 4, dtype=torch.int64)


@pytest.mark.parametrize("pos", [P[0, 0], P[:2], P[..., :3], torch.zeros(3, 3, 4), torch.zeros(1, 3, 2, 4), P[:, :, None]])
def test_position_shapes(pos):
    with pytest.raises(RuntimeError, match="pos must be of shape"):
        F.rope_axes(X, pos, (2, 1, 1))


@pytest.mark.parametrize("sections", [(2, 1), (4,)])
def test_sections_without_positions(sections):
    with pytest.raises(RuntimeError, match="must be pairs of each axis|pos must be of shape"):
        F.rope_axes(X, P, sections)


@pytest.mark.parametrize("sections", [(1, 1, 1), (2, 2, 2), (6, -1, -1), (2 ** 31 - 1, 1, 1)])
def test_sections_that_do_not_add_up(sections):
    with pytest.raises(RuntimeError, match="must be pairs of each axis, n_dims / 2 = 4 in all"):
        F.rope_axes(X, P, sections)


@pytest.mark.parametrize("sections", [(), (1, 1, 1, 1, 0)])
def test_number_of_axes(sections):
    with pytest.raises(RuntimeError, match="1 to 4 axes"):
        F.rope_axes(X, P, sections)


def test_interleaved_sections_that_do_not_fit():
    with pytest.raises(RuntimeError, match="axis 1 does not fit"):
        F.rope_axes(X, P, (0, 3, 1), interleaved=True)


@pytest.mark.parametrize("n_dims", [3, 10, 0, -2])
def test_n_dims(n_dims):
    with pytest.raises(RuntimeError, match="n_dims must be an even number between 2 and the head dimension 8"):
        F.rope_axes(X, P, (2, 1, 1), n_dims=n_dims)


@pytest.mark.parametrize("kw", [{"mode": 1}, {"mode": 8}])
def test_mode(kw):
    with pytest.raises(RuntimeError, match="mode must be 0 \\(normal\\) or 2 \\(NeoX\\)"):
        F.rope_axes(X, P, (2, 1, 1), **kw)


@pytest.mark.parametrize("kw", [{"freq_base": 0.0}, {"freq_base": -1.0}, {"freq_base": float("nan")}, {"freq_base": float("inf")},
                                {"freq_scale": float("inf")}, {"freq_scale": float("nan")}])
def test_frequencies(kw):
    with pytest.raises(RuntimeError, match="freq_base must be positive and finite"):
        F.rope_axes(X, P, (2, 1, 1), **kw)


def test_types_and_shapes():
    with pytest.raises(RuntimeError, match="floating point"):
        F.rope_axes(X.long(), P, (2, 1, 1))
    with pytest.raises(RuntimeError, match="expected x of shape"):
        F.rope_axes(X[0, 0], P, (2, 1, 1))
    with pytest.raises(RuntimeError, match="integer or float positions"):
        F.rope_axes(X, P.bool(), (2, 1, 1))
    with pytest.raises(RuntimeError, match="above 4096"):
        F.rope_axes(torch.ones(1, 1, 1, 4098), torch.zeros(1, 1), (2049,))


def test_null_arguments():
    h, sec = _bridge.borrow(X), (ctypes.c_int * 1)(4)
    for args in ((None, h.ptr, sec), (h.ptr, None, sec), (h.ptr, h.ptr, None)):
        assert not _C.lib.gt_rope_axes(args[0], args[1], 1, args[2], 0, 8, 2, 10000.0, 1.0)
        assert "required" in _C.last_error()
        assert not _C.lib.gt_rope_axes_backward(args[0], args[1], 1, args[2], 0, 8, 2, 10000.0, 1.0)


def test_empty_input():
    y = F.rope_axes(torch.ones(2, 3, 0, 8, dtype=torch.float64), torch.zeros(3, 2, 0), (2, 1, 1))
    assert tuple(y.shape) == (2, 3, 0, 8) and y.dtype == torch.float64
