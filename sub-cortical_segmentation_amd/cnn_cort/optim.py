"""
AdamW over many tensors at once, on libscs (scs_adamw_*, include/scs.h): one launch updates every tensor of a list, with the moments in
32 bits or in 8 bits (one scale per 256 elements), decoupled weight decay per tensor and clipping by the norm over all gradients.

The reference trains with lasagne.updates.adam (nets.py:236-237); that update stays the default of Net.fit, this one is what
Net.fit(optimizer='adamw') and Net.fit_adapters use.
"""
import bisect
import ctypes
import math

from . import _hip

__all__ = ['AdamW', 'BLOCK', 'blocks_of']

BLOCK = 256                     # elements that share a scale of 8-bit moments


def blocks_of(n):
    """Blocks that a tensor of n elements owns in the moment arenas."""
    return (int(n) + BLOCK - 1) // BLOCK


class _Tensor(ctypes.Structure):
    _fields_ = [('param', ctypes.c_void_p), ('master', ctypes.c_void_p), ('n', ctypes.c_int64), ('weight_decay', ctypes.c_double),
                ('type', ctypes.c_int32), ('reserved', ctypes.c_int32)]


class AdamW:
    """AdamW on a list of contiguous device tensors (float32, bfloat16, float16; a zero-element tensor is passed over).

      handle        _hip.Handle of the tensors' device
      weight_decay  one number, or one per tensor
      state_bits    32: moments m, v as float32 arenas; 8: int8 / uint8 codes with a float32 scale per 256 elements
      max_norm      None, or the norm over all gradients to clip at; a step whose norm is not finite changes nothing
      master        True: 16-bit parameters are rounded copies of float32 values that the optimiser keeps (self.masters; made from the parameters
                    as they are), or the masters of another AdamW over the same parameters, to go on from (used where they lie, as `states` are)
      states        None (zeros), or (m, v, m_scale, v_scale) of another AdamW over tensors of the same sizes; `step`: steps they have seen

    self.m, self.v, self.m_scale, self.v_scale are the arenas: tensor i owns blocks [self.first[i], self.first[i] + blocks_of(n_i)) of 256
    elements.  The optimiser's tensors stay the ones it was made with (none of these attributes can be set): step() is refused when the memory of one of
    them has been replaced since, and their old memory stays allocated as long as the optimiser does.  step() runs on the current torch stream of the device; it may be captured into a graph, whose replays count as steps."""

    def __init__(self, handle, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, max_norm=None, master=False,
                 states=None, step=0):
        import torch
        self._torch = torch
        self._o = None
        self.handle = handle
        params = tuple(params)
        if not params:
            raise ValueError('AdamW needs at least one tensor')
        if state_bits not in (8, 32):
            raise ValueError('state_bits must be 32 or 8, got %r' % (state_bits,))
        self.state_bits = state_bits
        self.lr, self.eps = float(lr), float(eps)
        self.betas = (float(betas[0]), float(betas[1]))
        self.max_norm = None if max_norm is None else float(max_norm)
        if self.max_norm is not None and not self.max_norm > 0:
            raise ValueError('max_norm must be positive, got %r' % (max_norm,))
        decays = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(params)
        if len(decays) != len(params):
            raise ValueError('%d weight decays for %d tensors' % (len(decays), len(params)))
        self._types = {torch.float32: 4, torch.bfloat16: 6, torch.float16: 7}          # SCS_F32, SCS_BF16, SCS_F16
        dev = torch.device('cuda', handle.device)
        for i, p in enumerate(params):
            self._check(p, i, 'parameter', dev)
        self.device = dev
        self.first, at = [], 0
        for p in params:
            self.first.append(at)
            at += blocks_of(p.numel())
        self.blocks = at
        if states is None:
            dt = (torch.float32, torch.float32) if state_bits == 32 else (torch.int8, torch.uint8)
            m, v = (torch.zeros((at * BLOCK,), dtype=d, device=dev) for d in dt)
            m_scale, v_scale = (torch.zeros((at,), device=dev) if state_bits == 8 else None for _ in range(2))
        else:
            m, v, m_scale, v_scale = (tuple(states) + (None, None))[:4]
        want = [(m, at * BLOCK, torch.float32 if state_bits == 32 else torch.int8, 'm'),
                (v, at * BLOCK, torch.float32 if state_bits == 32 else torch.uint8, 'v')]
        if state_bits == 8:
            want += [(m_scale, at, torch.float32, 'm_scale'), (v_scale, at, torch.float32, 'v_scale')]
        for t, n, dt, what in want:
            if not torch.is_tensor(t) or t.dtype != dt or t.device != dev or t.numel() != n or not t.is_contiguous():
                raise ValueError('state %s must be a contiguous %s tensor of %d elements on %s' % (what, dt, n, dev))
        if not isinstance(master, int):                        # (True and False are)
            masters = tuple(master)
            if len(masters) != len(params):
                raise ValueError('%d masters for %d tensors' % (len(masters), len(params)))
            for i, (w, p) in enumerate(zip(masters, params)):
                if p.dtype == torch.float32:
                    if w is not None:
                        raise ValueError('master %d: a float32 parameter takes none' % i)
                elif not torch.is_tensor(w) or w.dtype != torch.float32 or w.device != dev or w.shape != p.shape or not w.is_contiguous():
                    raise ValueError('master %d must be a contiguous float32 %r on %s' % (i, tuple(p.shape), dev))
        else:
            masters = tuple(p.detach().float() if master and p.dtype != torch.float32 else None for p in params)
        table = (_Tensor * len(params))()
        for t, p, w, d in zip(table, params, masters, decays):
            t.param, t.master, t.n = p.data_ptr(), None if w is None else w.data_ptr(), p.numel()
            t.weight_decay, t.type = float(d), self._types[p.dtype]
        grad_norm = torch.zeros((1,), device=dev) if self.max_norm is not None else None           # of the last step, before clipping
        o = ctypes.c_void_p()
        lib = _hip.load_library()
        torch.cuda.current_stream(dev).synchronize()           # masters, zeros and the norm are written on this stream; steps may run on another
        _hip._check(lib.scs_adamw_create(handle.h, table, len(params), state_bits, m.data_ptr(), v.data_ptr(),
                                         _hip._ptr(m_scale), _hip._ptr(v_scale), int(step), ctypes.byref(o)), 'scs_adamw_create')
        self._lib, self._o = lib, o
        self._address, self._index, self._stream = torch.Tensor.data_ptr, handle.device, torch._C._cuda_getCurrentRawStream
        self._grads = self._bound = None
        self._given = {'params': params, 'masters': masters, 'm': m, 'v': v, 'm_scale': m_scale, 'v_scale': v_scale, 'grad_norm': grad_norm}
        self._watched = list(params) + [t for t in masters + (m, v, m_scale, v_scale, grad_norm) if t is not None]
        self._held = [t.detach() for t in self._watched]               # (of the same memory, whatever becomes of the caller's)
        self._where = [t.data_ptr() for t in self._watched]
        self._arenas = [t.data_ptr for t in (m, v, m_scale, v_scale) if t is not None]
        self._arenas_where = [f() for f in self._arenas]
        self._norm_at = None if grad_norm is None else grad_norm.data_ptr()
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self._watched if t.numel())
        self._starts, self._ends = [a for a, _ in spans] + [math.inf], [b for _, b in spans]             # (they share no memory: both ascend)

    params, masters, m, v, m_scale, v_scale, grad_norm = (
        property(lambda self, k=k: self._given[k]) for k in ('params', 'masters', 'm', 'v', 'm_scale', 'v_scale', 'grad_norm'))

    grads = property(lambda self: self._grads)

    def _check(self, t, i, what, dev):
        torch = self._torch
        if not torch.is_tensor(t) or t.dtype not in self._types:
            raise ValueError('%s %d must be a float32, bfloat16 or float16 tensor' % (what, i))
        if t.device != dev:
            raise ValueError('%s %d is on %s, the optimiser on %s' % (what, i, t.device, dev))
        if not t.is_contiguous():
            raise ValueError('%s %d must be contiguous' % (what, i))

    def _shares(self, at, end):
        """Whether memory from `at` to `end` holds some of what the optimiser holds."""
        return self._starts[bisect.bisect_right(self._ends, at)] < end and at < end

    def _gradients(self, grads):
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError('%d gradients for %d tensors' % (len(grads), len(self.params)))
        n = len(grads)
        ptrs, types = (ctypes.c_void_p * n)(), (ctypes.c_int32 * n)()
        for i, (g, p) in enumerate(zip(grads, self.params)):
            self._check(g, i, 'gradient', self.device)
            if g.numel() != p.numel():
                raise ValueError('gradient %d has %d elements, its parameter %d' % (i, g.numel(), p.numel()))
            if g.shape != p.shape and g.dim() != 1 and p.dim() != 1:
                raise ValueError('gradient %d has the shape %r, its parameter %r' % (i, tuple(g.shape), tuple(p.shape)))
            at = ptrs[i] = g.data_ptr()
            types[i] = self._types[g.dtype]
            if self._shares(at, at + g.numel() * g.element_size()):
                raise ValueError('gradient %d shares memory with a parameter or a moment' % i)
        return grads, ptrs, types

    def _moved(self):
        if list(map(self._address, self._watched)) != self._where:
            raise RuntimeError('a parameter, a master or a moment has moved since the optimiser was made')

    def bind(self, grads):
        """The gradient buffers that step() reads when it is given none, checked here, once.  What is bound is their MEMORY: self.grads are tensors of
        the optimiser's own over it, and they keep it allocated.  A program that gives a gradient other memory binds again (looking at 77 gradients
        in every step took 3 us of the host, 20 where they had left its caches)."""
        grads, *self._bound = self._gradients(grads)
        self._grads = tuple(g.detach() for g in grads)
        return self

    def step(self, grads=None, grad_scale=1.0, lr=None):
        """One update from `grads` (one tensor per parameter, of its shape or flat, float32 / bfloat16 / float16; default: the bound ones), each
        multiplied by grad_scale first.  `lr` replaces self.lr for this step."""
        if self._o is None:
            raise RuntimeError('the optimiser is closed')
        if grads is None:
            if self._bound is None:
                raise ValueError('step() needs gradients: pass them or bind() them')
            ptrs, types = self._bound
        else:
            _, ptrs, types = self._gradients(grads)
        self._moved()
        rc = self._lib.scs_adamw_step(self._o, ptrs, types, self.lr if lr is None else float(lr), *self.betas, self.eps, float(grad_scale),
                                      self.max_norm or 0.0, self._norm_at, self._stream(self._index) or None)
        if rc:
            _hip._check(rc, 'scs_adamw_step')

    def states(self, out=None):
        """(m, v) as float32 arenas [blocks * 256]: the values that 8-bit moments stand for (into `out`, a pair of such tensors, when it is
        given); with state_bits 32 the arenas themselves."""
        torch = self._torch
        if self.state_bits == 32:
            return self.m, self.v
        n = self.blocks * BLOCK
        if out is None:
            out = tuple(torch.empty((n,), device=self.device) for _ in range(2))
        m, v = out
        for t in (m, v):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != self._index or t.numel() != n or not t.is_contiguous():
                raise ValueError('out must be two contiguous float32 tensors of %d elements on %s' % (n, self.device))
        at, to = m.data_ptr(), v.data_ptr()
        if n and (abs(at - to) < 4 * n or self._shares(at, at + 4 * n) or self._shares(to, to + 4 * n)):
            raise ValueError('out shares memory with what the optimiser holds, or the two with each other')
        if [f() for f in self._arenas] != self._arenas_where:
            raise RuntimeError('a moment or its scales have moved since the optimiser was made')
        rc = self._lib.scs_adamw_states(self._o, at, to, self._stream(self._index) or None)
        if rc:
            _hip._check(rc, 'scs_adamw_states')
        return m, v

    def _of(self, arena, i):
        p = self.params[i]
        return arena[self.first[i] * BLOCK:self.first[i] * BLOCK + p.numel()].view(p.shape)

    def state_of(self, i):
        """(m, v) of tensor i as float32 tensors of its shape."""
        m, v = self.states()
        return self._of(m, i), self._of(v, i)

    @property
    def step_count(self):
        """Steps taken (waits for the current stream)."""
        n = ctypes.c_int64(0)
        _hip._check(self._lib.scs_adamw_get_step(self._o, ctypes.byref(n), self._torch.cuda.current_stream(self.device).cuda_stream or None), 'scs_adamw_get_step')
        return int(n.value)

    @step_count.setter
    def step_count(self, n):
        _hip._check(self._lib.scs_adamw_set_step(self._o, int(n), self._torch.cuda.current_stream(self.device).cuda_stream or None), 'scs_adamw_set_step')

    def bytes_per_element(self):
        """Memory of the moments per parameter element."""
        n = sum(p.numel() for p in self.params)
        return math.inf if not n else self.blocks * (BLOCK * 8 if self.state_bits == 32 else BLOCK * 2 + 8) / n

    def close(self):
        if getattr(self, '_o', None):
            self._lib.scs_adamw_destroy(self._o)
            self._o = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
