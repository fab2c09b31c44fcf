"""Which strided tensors share memory, as clipping asks before it writes any of them, against counting their bytes."""
from __future__ import annotations

import itertools
import random

import pytest
import torch

from latent_bounded_interfaces_amd.hip.gradients import _check_apart, _column, _folded, _meet


def _addresses(t):
    return [t.data_ptr() + t.element_size() * sum(x * s for x, s in zip(index, t.stride())) for index in itertools.product(*map(range, t.shape))]


def _view(rng, base):
    sizes, strides = [], []
    for _ in range(rng.randint(0, 3)):
        sizes.append(rng.randint(1, 4))
        strides.append(rng.choice((0, 1, 1, 2, 3, 4, 5, 7, 12, 20)))
    return base.as_strided(sizes, strides, rng.randint(0, 60))


def _columns(rng, base):
    pitch = rng.choice((6, 10))
    return base.as_strided((rng.randint(1, 5), rng.randint(1, 4)), (pitch, rng.choice((1, 2))), rng.randint(0, 30))


@pytest.mark.parametrize("view", [_view, _columns])
def test_against_counting(view):
    rng = random.Random(5)
    base = {torch.float32: torch.zeros(256)}
    base[torch.bfloat16] = base[torch.float32].view(torch.bfloat16)  # the same bytes
    seen, folds, skipped = {True: 0, False: 0}, {True: 0, False: 0}, 0
    for _ in range(4000):
        a, b = (view(rng, base[rng.choice(list(base))]) for _ in range(2))
        at, bt = _addresses(a), _addresses(b)
        bytes_of = [{p + i for p in places for i in range(t.element_size())} for places, t in ((at, a), (bt, b))]
        want = bool(bytes_of[0] & bytes_of[1])
        assert _meet(a, b) is want and _meet(b, a) is want, (a.shape, a.stride(), b.shape, b.stride(), a.data_ptr() - b.data_ptr())
        seen[want] += 1
        for t, places in ((a, at), (b, bt)):
            pitch, begin, end = _column(t)
            assert not pitch or all(begin <= p % pitch and p % pitch + t.element_size() <= end for p in places)
        (pitch, begin, end), other = _column(a), _column(b)
        apart = pitch > 0 and other[0] == pitch and (other[2] <= begin or end <= other[1])
        assert not (want and apart)
        skipped += apart
        want = len(set(at)) < len(at)
        assert _folded(a) is want, (a.shape, a.stride())
        folds[want] += 1
    assert min(seen.values()) > 500 and (folds[True] > 500 if view is _view else skipped > 100)


def test_parts_of_one_matrix_are_apart():
    """Columns, rows and interleaved columns of one tensor, each result in its place or in a twin."""
    base = torch.zeros(40, 48, 3)
    parts = [base[:, :16], base[:, 16:31], base[:, 31:47:2], base[:, 32:47:2], base[:, 47:]]
    _check_apart(parts, parts, set(range(5)))
    twin = torch.zeros_like(base)
    twins = [twin[:, :16], twin[:, 16:31], twin[:, 31:47:2], twin[:, 32:47:2], twin[:, 47:]]
    _check_apart(parts, twins, set(range(5)))
    _check_apart([p.detach() for p in parts], parts, set(range(5)))  # the same views in other objects
    for outs in ([*twins[:4], twin[:, 46:47]], [*twins[:4], base[:, 0:1]], [twin[:, :16], twin[:, 15:30], *twins[2:]],
                 [base[:, 1:17], *twins[1:]], [*twins[:4], torch.zeros(40, 1, 1).expand(40, 1, 3)]):
        try:
            _check_apart(parts, outs, set(range(5)))
        except ValueError as bad:
            assert "overlaps" in str(bad) or "share" in str(bad)
        else:
            raise AssertionError([o.stride() for o in outs])


def test_columns_side_by_side_are_told_apart_without_a_search(monkeypatch):
    """180 thousand pairs of 600 columns: 0.02 s, and a second by searching each."""
    from latent_bounded_interfaces_amd.hip import gradients

    base = torch.zeros(64, 1200)
    parts = [base[:, i:i + 2] for i in range(0, 1200, 2)]
    searched = []
    monkeypatch.setattr(gradients, "_meet", lambda a, b: searched.append((a, b)))
    _check_apart(parts, parts, set(range(600)))
    assert not searched
    _check_apart([*parts, base[3, 7:9]], [*parts, base[3, 7:9]], set(range(601)))
    assert len(searched) == 600  # a row's part, against each column
