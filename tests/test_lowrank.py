"""Refusals of the shared projection's entry points that are decided before any device is touched, and the grouping of rows by site (run
without a GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from cnn_cort import _hip
from cnn_cort.adapters import Projection, group_rows


class NoDevice:
    device, h = 0, None


def test_c_entries_refuse_null():
    lib = _hip.load_library()
    n = ctypes.c_size_t(0)
    assert lib.scs_lowrank_workspace(None, None, 0, None, 0, ctypes.byref(n)) == -1
    assert lib.scs_lowrank_forward(None, None, None, 0, None, 0, None, None, 0, None) == -1
    assert lib.scs_lowrank_backward(None, None, None, 0, None, 0, None, None, 0, None, None, None, 0, None) == -1
    assert lib.scs_forward_features(None, None, None, None, None, 0, None, None) == -1
    assert b'null' in lib.scs_last_error()


def test_arguments_are_checked_before_the_device():
    w, a, b = torch.zeros(4, 6), torch.zeros(2, 3, 4), torch.zeros(2, 3, 6)
    for args, match in (((w[0], a, b), '2-D'), ((w.double(), a, b), 'float32, bfloat16'), ((w, a[:, :, :3], b), 'a must be'), ((w, a, b[:1]), 'a must be'),
                        ((w, torch.zeros(2, 129, 4), torch.zeros(2, 129, 6)), 'rank 1 to 128'), ((w, a, b), 'is on cpu'), ((w, a.half(), b), 'torch.float32 tensor')):
        with pytest.raises(ValueError, match=match):
            Projection(NoDevice, *args)


def test_group_rows():
    sites = np.array([2, 0, -1, 2, 0, 0])
    order, offsets, ids = group_rows(sites)
    assert order.tolist() == [2, 1, 4, 5, 0, 3] and offsets.tolist() == [0, 1, 4, 6] and ids.tolist() == [-1, 0, 2]
    order, offsets, ids = group_rows(np.zeros((0,), np.int64))
    assert order.size == 0 and offsets.tolist() == [0] and ids.size == 0


def test_rows_beyond_a_launch_are_refused():
    """2^26 rows are the most of one call: the limit is checked before anything else happens."""
    from cnn_cort.adapters import _Call
    lib, n = _hip.load_library(), ctypes.c_size_t(0)
    some = ctypes.c_void_p(16)
    call = _Call(4, 8, 2, 1, (1 << 26) + 1, 64, 64, 64, some, None, some, some, None, some, some)
    assert lib.scs_lowrank_workspace(some, ctypes.byref(call), 0, None, 64, ctypes.byref(n)) == -1
    assert b'rows lies in' in lib.scs_last_error()
    call.rows = 1 << 26
    assert lib.scs_lowrank_workspace(some, ctypes.byref(call), 1, None, 64, ctypes.byref(n)) == 0 and n.value > 0
