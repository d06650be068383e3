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


BIG = [2 ** 32 + 1, 2 ** 31, -2 ** 40]


def test_class_numbers_that_int32_does_not_hold_are_no_class():
    """They are passed over, as all numbers are that are no class; a cast would have made some other class of them."""
    kind, b = _booster(2)
    b.__class__ = kind
    seen = []

    def take(handle, top, ids, logits, lse, temperature, alpha):
        import ctypes as C
        if top:
            seen.append(np.ctypeslib.as_array(C.cast(ids, C.POINTER(C.c_int)), (2, top)).copy())
        return 0 if top else 1
    b._lib.tgbm_booster_set_teacher = take
    for ids in (np.array([[1] + BIG, [0, 2, -1, 3]], np.int64), np.array([[1] + BIG, [0, 2, -1, 3]], np.float64)):
        b.set_teacher(ids, np.zeros((2, 4)))
        assert seen.pop().tolist() == [[1, -1, -1, -1], [0, 2, -1, 3]]
    b.set_teacher(np.array([[1, 2 ** 64 - 1], [0, 2]], np.uint64), np.zeros((2, 2)))
    assert seen.pop().tolist() == [[1, -1], [0, 2]]
    for ids in (np.array([[0.5, 1], [0, 2]]), np.array([[np.nan, 1], [0, 2]])):
        with pytest.raises(ValueError, match='whole'):
            b.set_teacher(ids, np.zeros((2, 2)))
    assert not seen


def test_histories_and_rows_masks_of_predict_top():
    import ctypes as C
    from thundergbm_b200.thundergbm import TGBMClassifier
    got = {}

    class Lib:
        def tgbm_predict_top_dense(self, n, f, x, is_f64, model, trees, per_iter, rate, rules, k, T, values, ids, lse):
            r = rules._obj
            ptr = np.ctypeslib.as_array(C.cast(r.history_ptr, C.POINTER(C.c_longlong)), (n + 1,)).copy()
            got.update(ptr=ptr.tolist(), row=np.ctypeslib.as_array(C.cast(r.allowed_row, C.POINTER(C.c_int)), (n,)).tolist(),
                       past=np.ctypeslib.as_array(C.cast(r.history, C.POINTER(C.c_int)), (int(ptr[-1]),)).tolist())
            return 0
    m = TGBMClassifier.__new__(TGBMClassifier)
    m._lib, m.model, m.tree_per_iter, m.n_trees, m.learning_rate = Lib(), C.c_void_p(None), 5, 1, 1.0
    past = [[], [2 ** 32 + 1, 3], np.array([2 ** 33, 4, 2 ** 31 + 2]), (1, 1)]
    m.predict_top(np.ones((4, 2), np.float32), 2, allowed=np.ones((2, 5)), allowed_row=np.array([0, 1, 2 ** 32, -1]), history=past)
    assert got == dict(ptr=[0, 0, 2, 5, 7], past=[-1, 3, -1, 4, -1, 1, 1], row=[0, 1, -1, -1])
    with pytest.raises(ValueError, match='whole'):
        m.predict_top(np.ones((4, 2), np.float32), 2, history=[[], [1.5], [], []])
