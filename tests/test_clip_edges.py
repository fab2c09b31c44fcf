"""Which strided tensors share memory, as clipping asks before it writes any of them, against counting their bytes."""
from __future__ import annotations

import itertools
import random

import torch

from latent_bounded_interfaces_amd.hip.gradients import _check_apart, _folded, _meet


def _addresses(t):
    return [t.data_ptr() + t.element_size() * sum(x * s for x, s in zip(index, t.stride())) for index in itertools.product(*map(range, t.shape))]


def _view(rng, base):
    sizes, strides = [], []
    for _ in range(rng.randint(0, 3)):
        sizes.append(rng.randint(1, 4))
        strides.append(rng.choice((0, 1, 1, 2, 3, 4, 5, 7, 12, 20)))
    return base.as_strided(sizes, strides, rng.randint(0, 60))


def test_against_counting():
    rng = random.Random(5)
    base = {torch.float32: torch.zeros(256), torch.bfloat16: torch.zeros(512, dtype=torch.bfloat16)}
    base[torch.bfloat16] = base[torch.float32].view(torch.bfloat16)  # the same bytes
    seen = {True: 0, False: 0}
    folds = {True: 0, False: 0}
    for _ in range(4000):
        a, b = (_view(rng, base[rng.choice(list(base))]) for _ in range(2))
        at, bt = _addresses(a), _addresses(b)
        bytes_of = [{p + i for p in places for i in range(t.element_size())} for places, t in ((at, a), (bt, b))]
        want = bool(bytes_of[0] & bytes_of[1])
        assert _meet(a, b) is want and _meet(b, a) is want, (a.shape, a.stride(), b.shape, b.stride(), a.data_ptr() - b.data_ptr())
        seen[want] += 1
        want = len(set(at)) < len(at)
        assert _folded(a) is want, (a.shape, a.stride())
        folds[want] += 1
    assert min(*seen.values(), *folds.values()) > 500


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
