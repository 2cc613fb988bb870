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


@pytest.fixture
def on_host(monkeypatch):
    """Projections over host tensors: what is decided before a launch."""
    monkeypatch.setattr(Projection, '_own', lambda self, t, what, dtype: None)


@pytest.mark.parametrize('which', ['w', 'a', 'b', 'bias', 'scale'])
def test_a_tensor_that_has_moved_is_refused(on_host, which):
    """Every tensor whose address the projection holds: its memory replaced, or the attribute itself."""
    d = {'w': torch.zeros(4, 6), 'a': torch.zeros(2, 3, 4), 'b': torch.zeros(2, 3, 6), 'bias': torch.zeros(6), 'scale': torch.ones(2)}
    p = Projection(NoDevice, **d)
    x, off, ids = torch.zeros(5, 4), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    p._call(x, 5, off, ids)
    old = d[which].data
    d[which].data = d[which].clone()
    with pytest.raises(RuntimeError, match='has moved'):
        p._call(x, 5, off, ids)
    d[which].data = old
    p._call(x, 5, off, ids)
    with pytest.raises(AttributeError):
        setattr(p, which, d[which].clone())
    assert getattr(p, which) is d[which]


def test_the_memory_of_a_moved_tensor_is_kept(on_host):
    """A captured call goes on reading where its tensors lay: that memory stays the projection's."""
    d = {'w': torch.zeros(4, 6), 'a': torch.zeros(2, 3, 4), 'b': torch.zeros(2, 3, 6), 'bias': torch.zeros(6), 'scale': torch.ones(2)}
    p = Projection(NoDevice, **d)
    at = [t.data_ptr() for t in d.values()]
    for t in d.values():
        t.data = t.clone()
    assert sorted(t.data_ptr() for t in p._held) == sorted(at)


def test_inline_assembly_names_the_register_that_it_overwrites():
    """m0 is the compiler's: a statement that writes it says so, or a value kept there would be lost without a word."""
    import glob
    import os
    import re
    from conftest import PKG
    found = 0
    for path in glob.glob(os.path.join(PKG, 'csrc', '*.h')) + glob.glob(os.path.join(PKG, 'csrc', '*.hip')):
        with open(path) as f:
            for statement in re.findall(r'asm volatile\((.*?)\);', f.read(), re.S):
                if re.search(r's_mov_b32 m0\b', statement):
                    found += 1
                    assert statement.rstrip().endswith('"m0"'), (path, statement)
    assert found == 2


@pytest.mark.parametrize('t', ['f32', 'bf16', 'f16'])
def test_the_device_tests_reach_every_form(t, tmp_path):
    """Every variant that the rules on sizes can choose is one that a test compares with float64; a rule that is changed shows here."""
    import lowrank_forms
    from test_gpu_lowrank import CASES
    calls = [(t,) + c[:5] + (len(c[6]),) for c in CASES.values()] + [(t,) + s + (3, 5) for s in lowrank_forms.sizes(t)]
    reached = set().union(*lowrank_forms.forms(calls, tmp_path))
    assert reached == lowrank_forms.every_form(t)


@pytest.mark.parametrize('requests,most', [(10, 1.5), (100, 1.7), (900, 1.2), (8192, 1.2)])
def test_partial_sums_of_short_requests_do_not_outweigh_the_rows(requests, most):
    """Workspace of the gradients of 8192 rows of 4096 + 4096 columns in bf16 (128 MB), in their bytes."""
    from cnn_cort.adapters import _Call
    lib, n = _hip.load_library(), ctypes.c_size_t(0)
    some = ctypes.c_void_p(16)
    call = _Call(6, 16, 8, requests, 8192, 4096, 4096, 4096, some, None, some, some, None, some, some)
    assert lib.scs_lowrank_workspace(some, ctypes.byref(call), 1, some, 4096, ctypes.byref(n)) == 0
    assert n.value <= most * 8192 * 8192 * 2
