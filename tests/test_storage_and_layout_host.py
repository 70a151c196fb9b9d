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
