"""Refusals of the AdamW entry points that are decided before any device is touched (run without a GPU)."""
import ctypes

import pytest
import torch

from cnn_cort import _hip
from cnn_cort.optim import AdamW, blocks_of


class NoDevice:
    device, h = 0, None


def test_arguments_are_checked_before_the_device():
    p = torch.zeros(4)
    with pytest.raises(ValueError, match='at least one'):
        AdamW(NoDevice, [])
    with pytest.raises(ValueError, match='state_bits'):
        AdamW(NoDevice, [p], state_bits=16)
    with pytest.raises(ValueError, match='max_norm'):
        AdamW(NoDevice, [p], max_norm=0.0)
    with pytest.raises(ValueError, match='weight decays'):
        AdamW(NoDevice, [p], weight_decay=[0.1, 0.2])
    with pytest.raises(ValueError, match='is on cpu'):
        AdamW(NoDevice, [p])
    with pytest.raises(ValueError, match='float32, bfloat16 or float16'):
        AdamW(NoDevice, [p.double()])


def test_c_entries_refuse_null():
    lib = _hip.load_library()
    out = ctypes.c_void_p()
    assert lib.scs_adamw_create(None, None, 1, 32, None, None, None, None, 0, ctypes.byref(out)) == -1 and not out.value
    assert lib.scs_adamw_create(None, None, 1, 32, None, None, None, None, 0, None) == -1
    assert lib.scs_adamw_step(None, None, None, 1e-3, 0.9, 0.999, 1e-8, 1.0, 0.0, None, None) == -1
    assert lib.scs_adamw_states(None, None, None, None) == -1
    assert lib.scs_adamw_get_step(None, None, None) == -1 and lib.scs_adamw_set_step(None, 0, None) == -1
    assert lib.scs_adamw_destroy(None) == 0
    assert b'null' in lib.scs_last_error()


def test_blocks():
    assert [blocks_of(n) for n in (0, 1, 256, 257)] == [0, 1, 1, 2]
