"""Which sizes Categorical over linear class logits takes in pieces: those that
are no slower so, or too large to write out, and that the entry point takes.  (The
tensors here have shapes only.)"""
import pytest
import torch

from zhusuan_amd.distributions import univariate
from zhusuan_amd.distributions.univariate import LinearClassLogits


@pytest.fixture(autouse=True)
def shapes_only(monkeypatch):
    monkeypatch.setattr(univariate, 'as_tensor', lambda t: t)


def logits(N, D, V, *lead):
    return LinearClassLogits(torch.empty(*lead, V, D, device='meta'),
                             torch.empty(N, D, device='meta'))


@pytest.mark.parametrize('sizes,many', [
    ((3000, 40, 1500), True), ((3000, 40, 1500, 2), True),
    ((2000, 300, 20000), True), ((1024, 784, 4096), True),
    ((1024, 1024, 4096), False),         # few classes a feature
    ((300, 4096, 14000), False),
    ((1000, 40, 1500), False),           # few logits
    ((1 << 20, 4, 1000), False),         # few classes
    ((3000, 40, 1500, 0), False),        # no chains
    ((3000, 40, 1500, 2, 0), False),
    ((8192, 4096, 16384, 15), False),    # 2^31 logits of all chains
    ((8192, 4096, 16384, 16), True),
    ((100, 4096, 16384, 2000), False),   # ... of chains too small
    ((1 << 27, 1 << 20, 1024), True),
    ((1 << 27, (1 << 20) + 1, 1024), False),
    ((1 << 28, 4, 1024), False),
    ((0, 40, 1500), False)])
def test_sizes(sizes, many):
    assert logits(*sizes).many_classes() is many


def test_a_program_sets_its_own():
    l = logits(3000, 40, 1500)
    l.MANY_LOGITS = 1 << 62
    assert not l.many_classes() and logits(3000, 40, 1500).many_classes()
    l = logits(100, 40, 30)
    l.MANY_LOGITS = l.MANY_CLASSES = l.CLASSES_A_FEATURE = 0
    assert l.many_classes()
