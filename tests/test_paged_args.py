"""CPU checks of what PagedDecoder.step refuses, before anything changes on the GPU."""
import pytest

from spindle_b200.paged import PagedDecoder


class Stop(Exception):
    pass


class Reached(PagedDecoder):
    """Without weights: a step that is not refused gets as far as its plan."""

    def __init__(self):
        self.cfg, self.n_req, self.n_blocks, self.page, self.max_tokens = dict(vocab=100, max_seq=64), 3, 12, 16, 40
        self.held = [0] * 3

    @property
    def plan(self):
        raise Stop


@pytest.mark.parametrize("tokens,kw", [
    ({0: [100]}, {}), ({0: [5, -1]}, {}), ({1: [5], 2: [1 << 40]}, {}), ({3: [1]}, {}), ({-1: [1]}, {}), ({0: [1]}, dict(end=[3])),
    ({0: [1]}, dict(end=[-1])), ({0: [1]}, dict(end=[0])), ({0: [1]}, dict(end=iter([0]))), ({0: [1]}, dict(top=65)), ({0: [1]}, dict(top=-1)),
    ({0: [1] * 65}, {}), ({0: [1] * 30, 1: [1] * 30}, {})])
def test_step_refuses(tokens, kw):
    d = Reached()
    with pytest.raises(ValueError):
        d.step(tokens, **kw)
    assert d.held == [0] * 3


def test_step_goes_on():
    for tokens, kw in (({0: [0, 99], 2: [1]}, dict(end=iter([1]), top=64)), ({}, dict(end=[0])), ({1: range(3)}, {})):
        with pytest.raises(Stop):
            Reached().step(tokens, **kw)
