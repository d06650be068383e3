"""The front of training from a teacher, without a GPU."""
import numpy as np
import pytest


class _Lib:
    """Stands in for the library: takes down what set_teacher is called with."""

    def __init__(self):
        self.calls = []

    def tgbm_booster_set_teacher(self, handle, top, ids, logits, lse, temperature, alpha):
        self.calls.append((top, ids is not None, logits is not None, lse is not None, temperature, alpha))
        return 0 if top >= 1 else 1


def _booster(n):
    from thundergbm_b200.booster import Booster
    b = Booster.__new__(Booster)
    b._lib, b.handle = _Lib(), 1
    Info = type('Info', (), dict(n_rows=n))
    return type('B', (Booster,), dict(info=property(lambda self: Info), close=lambda self: None, __del__=lambda self: None)), b


@pytest.mark.parametrize('bad', [dict(ids=np.zeros((4, 2))), dict(logits=np.zeros((5, 3))), dict(ids=np.zeros(5)), dict(ids=[['a'] * 2] * 5), dict(lse=np.zeros(4)),
                                 dict(temperature='hot'), dict(alpha=None)])
def test_a_rank_that_refuses_its_arguments_tells_the_others(bad):
    """What is refused in Python reaches the library all the same, as a call that it refuses: with a communicator the ranks meet there."""
    kind, b = _booster(5)
    b.__class__ = kind
    args = dict(ids=np.zeros((5, 2), np.int32), logits=np.zeros((5, 2), np.float32), lse=np.zeros(5, np.float32), temperature=2.0, alpha=0.5)
    with pytest.raises((ValueError, TypeError)):
        b.set_teacher(**{**args, **bad})
    assert [c[0] for c in b._lib.calls] == [0]
    b._lib.calls.clear()
    b.set_teacher(**args)
    assert b._lib.calls == [(2, True, True, True, 2.0, 0.5)]
