"""Refusals of the AdamW entry points that are decided before any device is touched (run without a GPU)."""
import ctypes

import pytest
import torch

from cnn_cort import _hip
from cnn_cort.optim import BLOCK, AdamW, blocks_of


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


class OnHost:
    device, h = -1, None                               # (what a host tensor says of its device)


@pytest.fixture
def on_host(monkeypatch):
    """Optimisers over host tensors, their library a list of the steps it was asked for: what is decided before a launch."""
    steps = []

    class Library:
        scs_adamw_create = staticmethod(lambda *a: 0)
        scs_adamw_destroy = staticmethod(lambda *a: 0)
        scs_adamw_step = staticmethod(lambda *a: steps.append(a) or 0)
        scs_adamw_states = staticmethod(lambda *a: steps.append(a) or 0)

    cpu = torch.device('cpu')
    monkeypatch.setattr(torch, 'device', lambda *a: cpu)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: type('Stream', (), {'synchronize': lambda self: None})())
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda device: 0, raising=False)
    monkeypatch.setattr(_hip, 'load_library', lambda: Library)
    return steps


def tensors():
    return [torch.zeros(300, dtype=torch.bfloat16), torch.zeros(5, 7), torch.zeros(0)]


def exchange(t):
    """The tensor's memory replaced; the way back."""
    old = t.data
    t.data = t.clone()

    def back():
        t.data = old
    return back


@pytest.mark.parametrize('what', ['m', 'v', 'm_scale', 'v_scale', 'master', 'parameter', 'grad_norm'])
def test_what_has_moved_is_refused(on_host, what):
    """Every tensor whose address the optimiser holds."""
    params, grads = tensors(), tensors()
    opt = AdamW(OnHost, params, state_bits=8, master=True, max_norm=1.0).bind(grads)
    opt.step()
    back = exchange({'master': opt.masters[0], 'parameter': params[1]}[what] if what in ('master', 'parameter') else getattr(opt, what))
    reads = opt.states if what in ('m', 'v', 'm_scale', 'v_scale') else opt.step              # (the read-out looks at no parameter)
    for call in (opt.step, lambda: opt.step(grads), reads):
        with pytest.raises(RuntimeError, match='moved'):
            call()
    assert len(on_host) == 1
    back()
    opt.step()
    assert len(on_host) == 2


def test_bound_gradients_are_memory(on_host):
    """step() reads the memory that was bound: tensors of the optimiser's own hold it, whatever becomes of the caller's."""
    params, grads = tensors(), tensors()
    opt = AdamW(OnHost, params).bind(grads)
    at = [g.data_ptr() for g in grads]
    for g in grads:
        g.data = g.clone()
    opt.step()
    assert [g.data_ptr() for g in opt.grads] == at and [p or 0 for p in on_host[0][1]] == at
    opt.bind(grads).step()
    assert [p or 0 for p in on_host[1][1]] == [g.data_ptr() for g in grads] != at
    with pytest.raises(AttributeError):
        opt.grads = grads


def test_the_tensors_of_an_optimiser_cannot_be_exchanged(on_host):
    """A replaced arena would be read by nobody and its predecessor freed under the next step."""
    opt = AdamW(OnHost, tensors(), state_bits=8, master=True, max_norm=1.0)
    for name in ('params', 'masters', 'm', 'v', 'm_scale', 'v_scale', 'grad_norm'):
        with pytest.raises(AttributeError):
            setattr(opt, name, getattr(opt, name))
    for name in ('params', 'masters'):
        with pytest.raises(TypeError):
            getattr(opt, name)[0] = None


def test_the_memory_of_what_has_moved_is_kept(on_host):
    """A captured step goes on using the memory that it was captured with."""
    params, grads = tensors()[:2], tensors()[:2]
    opt = AdamW(OnHost, params, state_bits=8, master=True, max_norm=1.0).bind(grads)
    held = params + grads + [opt.masters[0], opt.m, opt.v, opt.m_scale, opt.v_scale, opt.grad_norm]
    at = {t.data_ptr() for t in held}
    for t in held:
        t.data = t.clone()
    assert at <= {t.data_ptr() for t in opt._held + list(opt.grads)}


@pytest.mark.parametrize('bits,case', [(32, 'm and v'), (32, 'm in a parameter'), (32, 'v in a master'), (8, 'm and v'), (8, 'the scales'), (8, 'a scale in v'),
                                       (8, 'v in a master'), (8, 'a scale in a parameter')])
def test_moments_that_share_memory_are_refused(bits, case):
    """The entry looks at sizes and addresses alone before it asks for a device: 1000 and 600 bf16 parameters with masters own 7 blocks."""
    from cnn_cort.optim import _Tensor
    lib = _hip.load_library()
    handle = ctypes.create_string_buffer(1 << 16)                     # (read for its device number alone)
    table = (_Tensor * 2)(_Tensor(0x100000, 0x200000, 1000, 0.0, 6, 0), _Tensor(0x110000, 0x210000, 600, 0.0, 6, 0))
    at = {'m': 0x300000, 'v': 0x400000, 'm_scale': 0x500000, 'v_scale': 0x600000}
    size = 7 * BLOCK * (4 if bits == 32 else 1)
    at.update({'m and v': {'v': at['m'] + size - 16}, 'm in a parameter': {'m': 0x110000 + 1200 - 16}, 'v in a master': {'v': 0x210000 - size + 16},
               'the scales': {'v_scale': at['m_scale'] + 24}, 'a scale in v': {'m_scale': at['v'] + size - 4},
               'a scale in a parameter': {'v_scale': 0x100000 + 1996}}[case])
    out = ctypes.c_void_p()
    scales = [at['m_scale'], at['v_scale']] if bits == 8 else [None, None]
    assert lib.scs_adamw_create(handle, table, 2, bits, at['m'], at['v'], *scales, 0, ctypes.byref(out)) == -1 and not out.value
    assert b'overlap' in lib.scs_last_error()


def test_read_out_into_memory_in_use_is_refused(on_host):
    opt = AdamW(OnHost, tensors(), state_bits=8, master=True)
    free = [torch.zeros(opt.blocks * BLOCK) for _ in range(2)]
    opt.states(out=free)
    arena = torch.zeros(opt.blocks * BLOCK + 4)
    other = AdamW(OnHost, [torch.zeros(opt.blocks * BLOCK)], state_bits=8)
    for bad in ([free[0], free[0]], [arena[:-4], arena[4:]]):
        with pytest.raises(ValueError, match='shares memory'):
            opt.states(out=bad)
    with pytest.raises(ValueError, match='shares memory'):
        other.states(out=[other.params[0], free[1]])
    assert len(on_host) == 1


def test_gradients_of_another_shape_are_refused(on_host):
    """As many elements in another order are another gradient; flat ones (slices of a gradient arena) are the parameter's own order."""
    p = torch.zeros(5, 7)
    opt = AdamW(OnHost, [p])
    for bad in (torch.zeros(7, 5), torch.zeros(35, 1), torch.zeros(1, 5, 7)):
        with pytest.raises(ValueError, match='shape'):
            opt.step([bad])
        with pytest.raises(ValueError, match='shape'):
            opt.bind([bad])
    opt.step([torch.zeros(5, 7)])
    opt.step([torch.zeros(35)])
    AdamW(OnHost, [p.view(-1)]).step([torch.zeros(5, 7)])
    assert len(on_host) == 3


def test_masters_are_handed_back(on_host):
    """A resumed optimiser goes on from the masters it is given, not from their rounded copies."""
    params = tensors()
    first = AdamW(OnHost, params, master=True)
    first.masters[0].add_(2.0 ** -20)
    again = AdamW(OnHost, params, master=first.masters)
    assert again.masters[0] is first.masters[0] and again.masters[1:] == (None, None)
    kept = first.masters[0]
    for bad, match in (([kept], '1 masters'), ([None] * 3, 'master 0'), ([kept[:-1], None, None], 'master 0'), ([kept.bfloat16(), None, None], 'master 0'),
                       ([kept, torch.zeros(5, 7), None], 'master 1'), ([torch.zeros(600)[::2], None, None], 'master 0')):
        with pytest.raises(ValueError, match=match):
            AdamW(OnHost, params, master=bad)


def test_a_nets_optimiser_options_are_checked_when_it_is_made():
    from cnn_cort.nets import Net
    for bad, match in (({'optimizer_bits': 16}, 'optimizer_bits'), ({'max_norm': 0.0}, 'max_norm'), ({'max_norm': -1.0}, 'max_norm'),
                       ({'max_norm': float('nan')}, 'max_norm'), ({'weight_decay': float('nan')}, 'weight_decay'), ({'weight_decay': float('inf')}, 'weight_decay')):
        with pytest.raises(ValueError, match=match):
            Net(optimizer='adamw', **bad)
    Net(optimizer='adamw', optimizer_bits=8, max_norm=1.0, weight_decay=0.0)


def test_what_an_optimiser_fills_is_filled_before_it_returns(on_host, monkeypatch):
    """Steps may run on another stream than the one it was made on: nothing is written there behind the wait (a late fill would wipe out a norm)."""
    order = []
    zeros = torch.zeros
    monkeypatch.setattr(torch, 'zeros', lambda *a, **k: order.append('fill') or zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: type('Stream', (), {'synchronize': lambda self: order.append('wait')})())
    for bits in (32, 8):
        del order[:]
        AdamW(OnHost, [torch.ones(300, dtype=torch.bfloat16)], state_bits=bits, master=True, max_norm=1.0)
        assert 'fill' in order and order[-1] == 'wait' and order.count('wait') == 1
