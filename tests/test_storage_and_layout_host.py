"""CPU-only: what a DeviceStorage asks the library, and when; layouts that are changed, copied or pickled after they were used."""
import copy
import pickle

import pytest

from weta_b200.backend import DeviceStorage
from weta_b200.core import DType, Layout


class CountingLib:
    def __init__(self):
        self.asked = []

    def __getattr__(self, name):
        answers = {"wb_storage_data": 4096, "wb_storage_len": 12, "wb_storage_dtype": DType.F64, "wb_free": 0}
        if name not in answers:
            raise AttributeError(name)

        def call(*args):
            self.asked.append(name)
            return answers[name]

        return call


class Backend:
    def __init__(self):
        self.lib, self.handle = CountingLib(), 1


def test_making_a_storage_asks_the_library_nothing():
    be = Backend()
    s = DeviceStorage(7, be)
    assert be.lib.asked == []
    assert (s.ptr, s.ptr, s.length, s.nbytes, s.nbytes) == (4096, 4096, 12, 96, 96)
    assert sorted(be.lib.asked) == ["wb_storage_data", "wb_storage_dtype", "wb_storage_len"]
    with pytest.raises(AttributeError):
        s.no_such_name
    del s
    assert be.lib.asked[-1] == "wb_free"


def of(l):
    v = l.view(0, DType.F32)
    return list(v.shape)[:v.ndim], list(v.stride)[:v.ndim], v.offset


def test_a_changed_layout_gives_its_new_view():
    l = Layout.contiguous([2, 3])
    assert of(l) == ([2, 3], [3, 1], 0) and l.rows_cols(1) == (2, 3)
    l.offset = 5
    assert of(l) == ([2, 3], [3, 1], 5)
    l.shape, l.strides = (3, 2), (1, 3)
    assert of(l) == ([3, 2], [1, 3], 5) and l.rows_cols(1) == (3, 2)
    l.shape, l.strides = [4], [2]
    assert of(l) == ([4], [2], 5) and l.rows_cols(1) == (1, 4)
    l.shape[0] = 6
    assert of(l) == ([6], [2], 5) and l.rows_cols(1) == (1, 6)


@pytest.mark.parametrize("clone", [copy.copy, copy.deepcopy, lambda l: pickle.loads(pickle.dumps(l))])
def test_a_layout_that_was_used_can_be_copied(clone):
    l = Layout([2, 3], [1, 2], 4)
    before = of(l), l.rows_cols(1)
    c = clone(l)
    assert (of(c), c.rows_cols(1)) == before
    c.offset = 0
    assert of(c)[2] == 0 and of(l)[2] == 4
