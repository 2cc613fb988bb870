"""
Site adapters: low-rank adapters of the dense layers, one set per site (scanner, protocol), beside the shared weights - on libscs
(scs_lowrank_*, include/scs.h).

`Projection` is one dense layer x W + bias with a bank of adapters; the rows of a call belong to requests (a subject, a site's share of a
mini-batch, one new token), each with its own adapter or none.  The layers it stands beside are the reference's DenseLayer nodes
(nets.py:179, 217, 227); W keeps their (in, out) order.
"""
import ctypes

from . import _hip

__all__ = ['Projection']


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
    (an optimiser's step) is seen by the next call.

    Calls run on the current torch stream of the device and may be captured into a graph."""

    def __init__(self, handle, w, a, b, bias=None, scale=None):
        import torch
        self._torch = torch
        self._types = {torch.float32: 4, torch.bfloat16: 6, torch.float16: 7}          # SCS_F32, SCS_BF16, SCS_F16
        self.handle, self.device = handle, torch.device('cuda', handle.device)
        self.w, self.a, self.b, self.bias, self.scale = w, a, b, bias, scale
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
        self._plan = (self._types[self.dtype], ldw, w.data_ptr(), _hip._ptr(bias), a.data_ptr(), b.data_ptr(), _hip._ptr(scale))

    def _own(self, t, what, dtype):
        if not self._torch.is_tensor(t) or t.dtype != dtype:
            raise ValueError('%s must be a %s tensor' % (what, dtype))
        if t.device != self.device:
            raise ValueError('%s is on %s, the projection on %s' % (what, t.device, self.device))

    @staticmethod
    def _stride(t, what):
        """Row stride of a 2-D tensor whose rows are contiguous."""
        rows, cols = t.shape
        if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
            raise ValueError('the rows of %s must be contiguous and apart' % what)
        return max(int(t.stride(0)), int(cols)) if rows > 1 else int(cols)

    def _rows(self, t, cols, what, rows=None):
        self._own(t, what, self.dtype)
        if t.dim() != 2 or int(t.shape[1]) != cols or (rows is not None and int(t.shape[0]) != rows):
            raise ValueError('%s must be [%s, %d], got %r' % (what, 'rows' if rows is None else rows, cols, tuple(t.shape)))
        return self._stride(t, what)

    def _call(self, rows, offsets, adapters):
        torch = self._torch
        for t, what in ((offsets, 'offsets'), (adapters, 'adapters')):
            self._own(t, what, torch.int32)
            if t.dim() != 1 or not t.is_contiguous():
                raise ValueError('%s must be 1-D and contiguous' % what)
        if offsets.numel() != adapters.numel() + 1:
            raise ValueError('%d offsets for %d requests (one more than requests)' % (offsets.numel(), adapters.numel()))
        dt, ldw, w, bias, a, b, scale = self._plan
        return _Call(dt, self.rank, self.n_adapters, adapters.numel(), rows, self.n_in, self.n_out, ldw, w, bias, a, b, scale,
                     offsets.data_ptr(), adapters.data_ptr() if adapters.numel() else None)

    def _workspace(self, call, back):
        n = ctypes.c_size_t(0)
        _hip._check(self._lib.scs_lowrank_workspace(self.handle.h, ctypes.byref(call), back, ctypes.byref(n)), 'scs_lowrank_workspace')
        return self._torch.empty((max(16, n.value),), dtype=self._torch.uint8, device=self.device), n.value

    def _hidden(self, hidden, rows):
        self._own(hidden, 'hidden', self._torch.float32)
        if tuple(hidden.shape) != (rows, self.rank) or not hidden.is_contiguous():
            raise ValueError('hidden must be a contiguous float32 [%d, %d]' % (rows, self.rank))
        return hidden.data_ptr()

    def _apart(self, out, what, *others):
        """An output must not share memory with what the call reads."""
        lo, hi = self._extent(out)
        for t in others:
            if t is not None:
                a, b = self._extent(t)
                if lo < b and a < hi:
                    raise ValueError('%s shares memory with a tensor that the call reads or writes' % what)

    @staticmethod
    def _extent(t):
        n = t.numel() and sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1
        return t.data_ptr(), t.data_ptr() + n * t.element_size()

    def forward(self, x, offsets, adapters, out=None, hidden=None):
        """y [rows, out] for x [rows, in].  Request q owns rows [offsets[q], offsets[q + 1]) (int32 on the device, ascending) and uses adapter
        adapters[q] (int32; -1, or a number outside the bank: none).  Rows outside [offsets[0], offsets[-1]) of `out` are left as they were;
        without `out` they are zeros.  `hidden` (float32 [rows, rank]) receives x_i A_s^T for backward()."""
        torch = self._torch
        ldx = self._rows(x, self.n_in, 'x')
        rows = int(x.shape[0])
        call = self._call(rows, offsets, adapters)
        if out is None:
            out = torch.zeros((rows, self.n_out), dtype=self.dtype, device=self.device)
        ldy = self._rows(out, self.n_out, 'out', rows)
        self._apart(out, 'out', x, self.w, self.a, self.b, self.bias, hidden)
        hp = None if hidden is None else self._hidden(hidden, rows)
        ws, n = self._workspace(call, 0)
        _hip._check(self._lib.scs_lowrank_forward(self.handle.h, ctypes.byref(call), x.data_ptr(), ldx, out.data_ptr(), ldy, hp, ws.data_ptr(), n,
                                                  torch.cuda.current_stream(self.device).cuda_stream or None), 'scs_lowrank_forward')
        return out

    def backward(self, x, dy, offsets, adapters, hidden=None, dx=None, da=None, db=None, want=('dx', 'da', 'db')):
        """(dx, da, db) for dy [rows, out]: da [adapters, rank, in] and db [adapters, rank, out] in float32, summed over the rows of each
        adapter's requests (zeros where there are none); None for what `want` does not name.  `hidden`: what forward() left, or None (formed
        again).  Rows of `dx` outside the requests are left as they were, without `dx` they are zeros."""
        torch = self._torch
        ldx = self._rows(x, self.n_in, 'x')
        rows = int(x.shape[0])
        lddy = self._rows(dy, self.n_out, 'dy', rows)
        call = self._call(rows, offsets, adapters)
        for k in want:
            if k not in ('dx', 'da', 'db'):
                raise ValueError("want names 'dx', 'da' and 'db', got %r" % (k,))
        if not want:
            raise ValueError('want names nothing')
        lddx = 0
        if 'dx' in want:
            if dx is None:
                dx = torch.zeros((rows, self.n_in), dtype=self.dtype, device=self.device)
            lddx = self._rows(dx, self.n_in, 'dx', rows)
        else:
            dx = None
        shapes = {'da': (self.n_adapters, self.rank, self.n_in), 'db': (self.n_adapters, self.rank, self.n_out)}
        grads = {}
        for k, t in (('da', da), ('db', db)):
            if k not in want:
                grads[k] = None
                continue
            if t is None:
                t = torch.empty(shapes[k], dtype=torch.float32, device=self.device)
            self._own(t, k, torch.float32)
            if tuple(t.shape) != shapes[k] or not t.is_contiguous():
                raise ValueError('%s must be a contiguous float32 %r' % (k, shapes[k]))
            grads[k] = t
        da, db = grads['da'], grads['db']
        for t, what, more in ((dx, 'dx', (da, db)), (da, 'da', (db,)), (db, 'db', ())):
            if t is not None:
                self._apart(t, what, x, dy, self.w, self.a, self.b, hidden, *more)
        hp = None if hidden is None else self._hidden(hidden, rows)
        ws, n = self._workspace(call, 1)
        _hip._check(self._lib.scs_lowrank_backward(self.handle.h, ctypes.byref(call), x.data_ptr(), ldx, dy.data_ptr(), lddy, hp, _hip._ptr(dx), lddx,
                                                   _hip._ptr(da), _hip._ptr(db), ws.data_ptr(), n,
                                                   torch.cuda.current_stream(self.device).cuda_stream or None), 'scs_lowrank_backward')
        return dx, da, db
