"""
Site adapters: low-rank adapters of the dense layers, one set per site (scanner, protocol), beside the shared weights - on libscs
(scs_lowrank_*, include/scs.h).

`Projection` is one dense layer x W + bias with a bank of adapters; the rows of a call belong to requests (a subject, a site's share of a
mini-batch, one new token), each with its own adapter or none.  The layers it stands beside are the reference's DenseLayer nodes
(nets.py:179, 217, 227); W keeps their (in, out) order.
"""
import ctypes
import threading

import numpy as np

from . import _hip

__all__ = ['Projection', 'SiteAdapters', 'group_rows']


class _Call(ctypes.Structure):
    _fields_ = [('dtype', ctypes.c_int32), ('rank', ctypes.c_int32), ('n_adapters', ctypes.c_int32), ('n_requests', ctypes.c_int32),
                ('rows', ctypes.c_int64), ('in_features', ctypes.c_int64), ('out_features', ctypes.c_int64), ('ldw', ctypes.c_int64),
                ('w', ctypes.c_void_p), ('bias', ctypes.c_void_p), ('a', ctypes.c_void_p), ('b', ctypes.c_void_p), ('scale', ctypes.c_void_p),
                ('offsets', ctypes.c_void_p), ('adapters', ctypes.c_void_p)]


class Projection:
    """y_i = x_i W + bias + scale_s (x_i A_s^T) B_s, s the adapter of row i's request.

      handle  _hip.Handle of the tensors' device
      w       [in, out], rows of any stride            bias  [out] or None
      a       [adapters, rank, in], contiguous         b     [adapters, rank, out], contiguous       rank 1..128
      scale   float32 [adapters] or None (1)
    w, bias, a and b share one type: float32, bfloat16 or float16.  The tensors are used where they lie: updating a and b in place
    (an optimiser's step) is seen by the next call.  The five stay the ones that were given, and a call is refused when the memory of any of them has
    been replaced since (its old memory stays allocated as long as the projection does).

    Calls run on the current torch stream of the device and may be captured into a graph.  They record nothing for autograd: gradients are
    backward()'s.  An output may not lie inside the span of memory that an input's rows cover, not even between the rows."""

    def __init__(self, handle, w, a, b, bias=None, scale=None):
        import torch
        self._torch = torch
        self._types = {torch.float32: 4, torch.bfloat16: 6, torch.float16: 7}          # SCS_F32, SCS_BF16, SCS_F16
        self.handle, self.device = handle, torch.device('cuda', handle.device)
        self._given = {'w': w, 'a': a, 'b': b, 'bias': bias, 'scale': scale}
        if not torch.is_tensor(w) or w.dtype not in self._types or w.dim() != 2:
            raise ValueError('w must be a 2-D float32, bfloat16 or float16 tensor')
        self.dtype = w.dtype
        self.n_in, self.n_out = (int(n) for n in w.shape)
        if not torch.is_tensor(a) or not torch.is_tensor(b) or a.dim() != 3 or b.dim() != 3 or a.shape[:2] != b.shape[:2] or \
                int(a.shape[2]) != self.n_in or int(b.shape[2]) != self.n_out:
            raise ValueError('a must be [adapters, rank, %d] and b [adapters, rank, %d]' % (self.n_in, self.n_out))
        self.n_adapters, self.rank = int(a.shape[0]), int(a.shape[1])
        if not 1 <= self.rank <= 128 or not 1 <= self.n_adapters <= 65535:
            raise ValueError('between 1 and 65535 adapters of rank 1 to 128, got %d of rank %d' % (self.n_adapters, self.rank))
        if not (1 <= self.n_in <= 1 << 20 and 1 <= self.n_out <= 1 << 20):
            raise ValueError('between 1 and 2^20 features, got %d and %d' % (self.n_in, self.n_out))
        for t, what in ((a, 'a'), (b, 'b')):
            self._own(t, what, self.dtype)
            if not t.is_contiguous():
                raise ValueError('%s must be contiguous' % what)
        self._own(w, 'w', self.dtype)
        ldw = self._stride(w, 'w')
        if bias is not None:
            self._own(bias, 'bias', self.dtype)
            if tuple(bias.shape) != (self.n_out,) or not bias.is_contiguous():
                raise ValueError('bias must be a contiguous [%d]' % self.n_out)
        if scale is not None:
            self._own(scale, 'scale', torch.float32)
            if tuple(scale.shape) != (self.n_adapters,) or not scale.is_contiguous():
                raise ValueError('scale must be a contiguous [%d]' % self.n_adapters)
        self._lib = _hip.load_library()
        given = [t for t in self._given.values() if t is not None]
        self._held = [t.detach() for t in given]                                        # (of the same memory, whatever becomes of the caller's)
        self._where = [t.data_ptr() for t in given]
        self._at = [t.data_ptr for t in given]
        self._tensor, self._int32, self._bytes, self._index = torch.Tensor, torch.int32, torch.uint8, handle.device
        self._empty, self._stream = torch.empty, torch._C._cuda_getCurrentRawStream             # (of a device's current stream, without an object for it)
        self._item = w.element_size()
        self._plan = (self._types[self.dtype], self.rank, self.n_adapters, 0, 0, self.n_in, self.n_out, ldw, w.data_ptr(), _hip._ptr(bias), a.data_ptr(),
                      b.data_ptr(), _hip._ptr(scale), None, None)
        self._reads = [(t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * ldw + self.n_out if t is w else t.numel()) * t.element_size())
                       for t in (w, a, b, bias, scale) if t is not None]
        self._sizes, self._tls = {}, threading.local()

    w, a, b, bias, scale = (property(lambda self, k=k: self._given[k]) for k in ('w', 'a', 'b', 'bias', 'scale'))

    def _own(self, t, what, dtype):
        if not self._torch.is_tensor(t) or t.dtype != dtype:
            raise ValueError('%s must be a %s tensor' % (what, dtype))
        if t.device != self.device:
            raise ValueError('%s is on %s, the projection on %s' % (what, t.device, self.device))

    @staticmethod
    def _stride(t, what):
        """Row stride of a 2-D tensor whose rows are contiguous."""
        (rows, cols), (d0, d1) = t.shape, t.stride()
        if (cols > 1 and d1 != 1) or (rows > 1 and d0 < cols):
            raise ValueError('the rows of %s must be contiguous and apart' % what)
        return d0 if rows > 1 and d0 > cols else cols

    def _rows(self, t, rows, cols, what):
        """(address, row stride, end address) of a [rows, cols] tensor of the projection's type."""
        if not isinstance(t, self._tensor) or t.dtype is not self.dtype or t.get_device() != self._index:
            self._own(t, what, self.dtype)
        if t.shape != (rows, cols):
            raise ValueError('%s must be [%d, %d], got %r' % (what, rows, cols, tuple(t.shape)))
        ld, step = t.stride()
        if rows <= 1 or step != 1 or ld < cols:
            ld = self._stride(t, what)
        at = t.data_ptr()
        return at, ld, at + (((rows - 1) * ld + cols) * self._item if rows else 0)

    def _flat(self, t, shape, what):
        """(address, 0, end address) of a contiguous float32 tensor of a shape."""
        self._own(t, what, self._torch.float32)
        if tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError('%s must be a contiguous float32 %r' % (what, shape))
        at = t.data_ptr()
        return at, 0, at + 4 * t.numel()

    @staticmethod
    def _apart(outs, reads):
        """No output shares memory with what the call reads or with another output."""
        for i, (what, (at, _, end)) in enumerate(outs):
            for a, b in reads:
                if at < b and a < end:
                    raise ValueError('%s shares memory with a tensor that the call reads' % what)
            for _, (a, _, b) in outs[:i]:
                if at < b and a < end:
                    raise ValueError('%s shares memory with another output' % what)

    def _call(self, x, rows, offsets, adapters):
        """The call's description on this thread (one per thread: two threads may call at once)."""
        if [f() for f in self._at] != self._where:
            raise RuntimeError('w, a, b, bias or scale has moved since the projection was made')
        if x.dim() != 2:
            raise ValueError('x must be [rows, %d], got %r' % (self.n_in, tuple(x.shape)))
        for t, what in ((offsets, 'offsets'), (adapters, 'adapters')):
            if not isinstance(t, self._tensor) or t.dtype is not self._int32 or t.get_device() != self._index:
                self._own(t, what, self._int32)
            if t.dim() != 1 or not t.is_contiguous():
                raise ValueError('%s must be 1-D and contiguous' % what)
        n = adapters.numel()
        if offsets.numel() != n + 1:
            raise ValueError('%d offsets for %d requests (one more than requests)' % (offsets.numel(), n))
        call = getattr(self._tls, 'call', None)
        if call is None:
            call = self._tls.call = _Call(*self._plan)
            self._tls.ref = ctypes.byref(call)
        call.rows, call.n_requests, call.offsets, call.adapters = rows, n, offsets.data_ptr(), adapters.data_ptr()
        return self._tls.ref

    def _workspace(self, call, back, rows, requests, at, ld):
        """Workspace of a call; its size hangs on the numbers of rows and requests and on whether the rows lie at multiples of 16 bytes."""
        key = (back, rows, requests, at % 16, ld)
        n = self._sizes.get(key)
        if n is None:
            size = ctypes.c_size_t(0)
            _hip._check(self._lib.scs_lowrank_workspace(self.handle.h, call, back, at, ld, ctypes.byref(size)), 'scs_lowrank_workspace')
            if len(self._sizes) > 4096:
                self._sizes.clear()
            n = self._sizes[key] = size.value
        return self._empty(n + 16, dtype=self._bytes, device=self.device), n

    def forward(self, x, offsets, adapters, out=None, hidden=None):
        """y [rows, out] for x [rows, in].  Request q owns rows [offsets[q], offsets[q + 1]) (int32 on the device, ascending) and uses adapter
        adapters[q] (int32; -1, or a number outside the bank: none).  Rows outside [offsets[0], offsets[-1]) of `out` are left as they were;
        without `out` they are zeros.  `hidden` (float32 [rows, rank]) receives x_i A_s^T for backward()."""
        torch = self._torch
        rows = x.shape[0]
        call = self._call(x, rows, offsets, adapters)
        px = self._rows(x, rows, self.n_in, 'x')
        if out is None:
            out = torch.zeros((rows, self.n_out), dtype=self.dtype, device=self.device)
        py = self._rows(out, rows, self.n_out, 'out')
        outs = [('out', py)]
        if hidden is not None:
            outs.append(('hidden', self._flat(hidden, (rows, self.rank), 'hidden')))
        self._apart(outs, [(px[0], px[2])] + self._reads)
        ws, n = self._workspace(call, 0, rows, adapters.numel(), px[0], px[1])
        rc = self._lib.scs_lowrank_forward(self.handle.h, call, px[0], px[1], py[0], py[1], outs[1][1][0] if hidden is not None else None,
                                           ws.data_ptr(), n, self._stream(self._index) or None)
        if rc:
            _hip._check(rc, 'scs_lowrank_forward')
        return out

    def backward(self, x, dy, offsets, adapters, hidden=None, dx=None, da=None, db=None, want=('dx', 'da', 'db')):
        """(dx, da, db) for dy [rows, out]: da [adapters, rank, in] and db [adapters, rank, out] in float32, summed over the rows of each
        adapter's requests (zeros where there are none); None for what `want` does not name.  `hidden`: what forward() left, or None (formed
        again).  Rows of `dx` outside the requests are left as they were, without `dx` they are zeros."""
        torch = self._torch
        rows = x.shape[0]
        call = self._call(x, rows, offsets, adapters)
        px, pdy = self._rows(x, rows, self.n_in, 'x'), self._rows(dy, rows, self.n_out, 'dy')
        if not want or any(k not in ('dx', 'da', 'db') for k in want):
            raise ValueError("want names some of 'dx', 'da' and 'db', got %r" % (want,))
        outs = []
        if 'dx' in want:
            if dx is None:
                dx = torch.zeros((rows, self.n_in), dtype=self.dtype, device=self.device)
            pdx = self._rows(dx, rows, self.n_in, 'dx')
            outs.append(('dx', pdx))
        else:
            dx, pdx = None, (None, 0)
        pg = []
        for k, t, cols in (('da', da, self.n_in), ('db', db, self.n_out)):
            if k not in want:
                pg.append((None, None))
                continue
            shape = (self.n_adapters, self.rank, cols)
            if t is None:
                t = torch.empty(shape, dtype=torch.float32, device=self.device)
            outs.append((k, self._flat(t, shape, k)))
            pg.append((t, outs[-1][1][0]))
        reads = [(px[0], px[2]), (pdy[0], pdy[2])] + self._reads
        ph = None
        if hidden is not None:
            ph = self._flat(hidden, (rows, self.rank), 'hidden')
            reads.append((ph[0], ph[2]))
        self._apart(outs, reads)
        ws, n = self._workspace(call, 1, rows, adapters.numel(), pdy[0], pdy[1])
        rc = self._lib.scs_lowrank_backward(self.handle.h, call, px[0], px[1], pdy[0], pdy[1], ph and ph[0], pdx[0], pdx[1], pg[0][1], pg[1][1],
                                            ws.data_ptr(), n, self._stream(self._index) or None)
        if rc:
            _hip._check(rc, 'scs_lowrank_backward')
        return dx, pg[0][0], pg[1][0]


def group_rows(sites):
    """(order, offsets, adapters) of rows by site: `order` sorts them (stable), request q of the sorted rows is
    [offsets[q], offsets[q + 1]) and uses adapters[q]."""
    sites = np.asarray(sites, dtype=np.int64).ravel()
    order = np.argsort(sites, kind='stable')
    s = sites[order]
    starts = np.flatnonzero(np.concatenate([[True], s[1:] != s[:-1]])) if s.size else np.zeros((0,), np.int64)
    return order, np.concatenate([starts, [s.size]]).astype(np.int32), s[starts].astype(np.int32)


class SiteAdapters:
    """Low-rank adapters of the dense head (FC1, fc_2, out_layer: nets.py:217, 227, 231) for a number of sites, beside the weights of a Net.

      params  parameter dict of the Net (the shared weights are copied to the device)
      state   None - A ~ N(0, 1 / in), B = 0: every site predicts what the shared weights predict - or the arrays of state_dict()

    The head's rectifiers sit between the layers as in the net (PReLU behind ReLU is the identity); dropout is off."""

    LAYERS = ('FC1', 'fc_2', 'out_layer')

    def __init__(self, handle, params, sites, rank=8, scale=1.0, seed=0, state=None):
        import torch
        self._torch = torch
        self.device = torch.device('cuda', handle.device)
        self.sites, self.rank = int(sites), int(rank)
        up = lambda a: torch.from_numpy(np.array(a, dtype=np.float32, order='C')).to(self.device)
        rng = np.random.default_rng(seed)
        self.layers, self.tensors, self.names = [], [], []
        self.scale = up(np.full((self.sites,), scale, np.float32) if state is None else state['scale'])
        for name in self.LAYERS:
            w, b = params[name]
            n_in, n_out = w.shape
            shapes = {'a': (self.sites, self.rank, n_in), 'b': (self.sites, self.rank, n_out)}
            if state is None:
                first = {'a': rng.normal(0.0, n_in ** -0.5, shapes['a']), 'b': np.zeros(shapes['b'])}
            else:
                first = {k: state['%s.%s' % (name, k)] for k in shapes}
                for k, sh in shapes.items():
                    if tuple(first[k].shape) != sh:
                        raise ValueError('adapter array %s.%s has shape %r, expected %r' % (name, k, first[k].shape, sh))
            a, d = up(first['a']), up(first['b'])
            self.layers.append(Projection(handle, up(w), a, d, bias=up(b), scale=self.scale))
            self.tensors += [a, d]
            self.names += [name + '.a', name + '.b']

    def set_weights(self, params):
        """The shared weights of another parameter dict, into the layers' own tensors."""
        for name, layer in zip(self.LAYERS, self.layers):
            for t, a in zip((layer.w, layer.bias), params[name]):
                t.copy_(self._torch.from_numpy(np.array(a, dtype=np.float32, order='C')))

    def state_dict(self):
        """Host arrays: scale, <layer>.a, <layer>.b."""
        d = {n: t.cpu().numpy() for n, t in zip(self.names, self.tensors)}
        d['scale'] = self.scale.cpu().numpy()
        return d

    def _forward(self, features, atlas, offsets, sites, keep):
        torch = self._torch
        rows = features.shape[0]
        hidden = [torch.zeros((rows, self.rank), device=self.device) for _ in self.layers] if keep else [None] * 3
        x1 = features
        y1 = torch.relu_(self.layers[0].forward(x1, offsets, sites, hidden=hidden[0]))
        x2 = torch.cat([y1, atlas], 1)
        y2 = torch.relu_(self.layers[1].forward(x2, offsets, sites, hidden=hidden[1]))
        z = self.layers[2].forward(y2, offsets, sites, hidden=hidden[2])
        return z, (x1, y1, x2, y2, hidden)

    def logits(self, features, atlas, offsets, sites):
        """[rows, 15] for features [rows, 540] (Net.features) and prior rows [rows, 15]; requests as in Projection.forward."""
        return self._forward(features, atlas, offsets, sites, False)[0]

    def loss_and_gradients(self, features, atlas, y, offsets, sites, grads=None):
        """(mean cross-entropy as a device scalar, gradients in the order of self.tensors) for labels y int64 [rows]."""
        torch = self._torch
        z, (x1, y1, x2, y2, hidden) = self._forward(features, atlas, offsets, sites, True)
        logp = torch.log_softmax(z, 1)
        loss = -logp.gather(1, y[:, None]).mean()
        dz = logp.exp()
        dz.scatter_add_(1, y[:, None], torch.full_like(y, -1, dtype=torch.float32)[:, None])
        dz /= max(1, z.shape[0])
        g = grads if grads is not None else [torch.empty_like(t) for t in self.tensors]
        dy2 = self.layers[2].backward(y2, dz, offsets, sites, hidden=hidden[2], da=g[4], db=g[5])[0].mul_(y2 > 0)
        dx2 = self.layers[1].backward(x2, dy2, offsets, sites, hidden=hidden[1], da=g[2], db=g[3])[0]
        dy1 = dx2[:, :y1.shape[1]] * (y1 > 0)
        self.layers[0].backward(x1, dy1, offsets, sites, hidden=hidden[0], da=g[0], db=g[1], want=('da', 'db'))
        return loss, g
