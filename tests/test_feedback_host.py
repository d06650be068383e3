"""The front of training from drawn classes, without a GPU."""
import numpy as np
import pytest

from test_teacher_host import _booster


class _Lib:
    """Stands in for the library: takes down what set_feedback is called with."""

    def __init__(self):
        self.calls = []

    def tgbm_booster_set_feedback(self, handle, draws, classes, gains, old, weights, temperature, low, high, entropy):
        self.calls.append((draws, old is not None, weights is not None, temperature, low, high, entropy))
        return 0 if draws >= 1 else 1


@pytest.mark.parametrize('bad', [dict(classes=np.zeros((4, 2))), dict(gains=np.zeros((5, 3))), dict(classes=[['a'] * 2] * 5), dict(classes=np.full((5, 2), 0.5)), dict(old=np.zeros(5)),
                                 dict(weights=np.zeros((5, 2))), dict(temperature='hot'), dict(entropy=None), dict(clip=(1, 2, 3)), dict(clip='tight'), dict(classes=np.zeros((5, 2, 1)))])
def test_a_rank_that_refuses_its_arguments_tells_the_others(bad):
    """What is refused in Python reaches the library all the same, as a call that it refuses: with a communicator the ranks meet there."""
    kind, b = _booster(5)
    b.__class__ = kind
    b._lib = _Lib()
    args = dict(classes=np.zeros((5, 2), np.int32), gains=np.zeros((5, 2), np.float32), old=np.zeros((5, 2)), weights=np.ones(5), temperature=2.0, clip=0.25, entropy=0.5)
    with pytest.raises((ValueError, TypeError)):
        b.set_feedback(**{**args, **bad})
    assert [c[0] for c in b._lib.calls] == [0]
    b._lib.calls.clear()
    b.set_feedback(**args)
    b.set_feedback(args['classes'][:, 0], args['gains'][:, 0])
    assert b._lib.calls == [(2, True, True, 2.0, 0.25, 0.25, 0.5), (1, False, False, 1.0, 1.0, float('inf'), 0.0)]


def test_class_numbers_that_int32_does_not_hold_are_no_class():
    kind, b = _booster(2)
    b.__class__ = kind
    seen = []

    def take(handle, draws, classes, *rest):
        import ctypes as C
        if draws:
            seen.append(np.ctypeslib.as_array(C.cast(classes, C.POINTER(C.c_int)), (2, draws)).copy())
        return 0 if draws else 1
    b._lib = type('L', (), dict(tgbm_booster_set_feedback=staticmethod(take)))
    b.set_feedback(np.array([[1, 2 ** 32 + 1], [2 ** 31, -5]], np.int64), np.zeros((2, 2)))
    assert seen.pop().tolist() == [[1, -1], [-1, -1]]
