"""
ctypes binding of libscs.so (include/scs.h) - the only route from the Python surface to the HIP kernels.

There is deliberately no CPU fallback: if the library is missing, or no MI355X-class device is visible,
every compute entry point raises.  (The oracle under /oracle is test infrastructure and is never imported
from here.)
"""
import ctypes
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get('SCS_LIB_PATH') or os.path.join(os.path.dirname(_HERE), 'lib', 'libscs.so')   # override: A/B runs of two builds
N_PARAMS = 883455

_lib = None

# name -> (restype, argtypes); mirrors include/scs.h one to one
_c = ctypes
_f32p = _c.POINTER(_c.c_float)
_vp = _c.c_void_p
SIGNATURES = {
    'scs_last_error': (_c.c_char_p, []),
    'scs_abi_version': (_c.c_int, []),
    'scs_target_arch': (_c.c_char_p, []),
    'scs_create': (_c.c_int, [_c.c_int, _c.POINTER(_vp)]),
    'scs_destroy': (_c.c_int, [_vp]),
    'scs_set_params': (_c.c_int, [_vp, _vp, _c.c_size_t]),
    'scs_get_params': (_c.c_int, [_vp, _vp, _c.c_size_t]),
    'scs_set_chunk': (_c.c_int, [_vp, _c.c_int]),
    'scs_set_option': (_c.c_int, [_vp, _c.c_char_p, _c.c_int64]),
    'scs_get_option': (_c.c_int, [_vp, _c.c_char_p, _c.POINTER(_c.c_int64)]),
    'scs_probe_f32_mfma': (_c.c_int, [_vp, _c.POINTER(_c.c_double)]),
    'scs_probe_f32_mfma_clock': (_c.c_int, [_vp, _c.POINTER(_c.c_double), _c.POINTER(_c.c_double)]),
    'scs_forward': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _c.c_int64, _vp, _vp, _vp]),
    'scs_forward_features': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _c.c_int64, _vp, _vp]),
    'scs_forward_host': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _c.c_int64, _vp, _vp]),
    'scs_forward_volume': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _c.c_int64, _vp, _vp, _vp]),
    'scs_forward_volume_rows': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _c.c_int64, _vp, _vp, _vp]),
    'scs_forward_volume_shared': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _c.c_int64, _vp, _vp, _vp, _vp]),
    'scs_forward_profiled': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _c.c_int64, _vp, _vp, _vp, _vp, _c.POINTER(_c.c_int)]),
    'scs_get_activation': (_c.c_int, [_vp, _c.c_int, _vp, _c.c_size_t]),
    'scs_dilate_mask': (_c.c_int, [_vp, _vp, _vp, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _vp]),
    'scs_zscore_volume': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _vp]),
    'scs_roi_prepare': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _vp, _c.POINTER(_c.c_int64), _vp]),
    'scs_roi_centers': (_c.c_int, [_vp, _vp, _c.c_int, _c.c_int, _c.c_int, _vp, _vp, _c.c_int64, _vp]),
    'scs_train_step': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _c.c_int64, _c.c_uint64, _vp, _vp, _vp]),
    'scs_train_step_volume': (_c.c_int, [_vp, _vp, _vp, _c.c_int32, _vp, _c.c_int64, _vp, _vp, _vp, _vp, _c.c_int64, _c.c_uint64, _vp, _vp, _vp]),
    'scs_gather_labels': (_c.c_int, [_vp, _vp, _vp, _c.c_int32, _vp, _c.c_int64, _vp, _vp]),
    'scs_eval_batch_volume': (_c.c_int, [_vp, _vp, _vp, _c.c_int32, _vp, _c.c_int64, _vp, _vp, _vp, _c.c_int64, _c.POINTER(_c.c_double),
                                         _c.POINTER(_c.c_int64), _vp]),
    'scs_train_stage_count': (_c.c_int, []),
    'scs_train_stage_name': (_c.c_char_p, [_c.c_int]),
    'scs_train_step_profiled': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _c.c_int64, _c.c_uint64, _vp, _vp]),
    'scs_get_train_buffer': (_c.c_int, [_vp, _c.c_int, _vp, _c.c_size_t]),
    'scs_param_arena': (_c.c_int, [_vp, _c.POINTER(_vp), _c.POINTER(_c.c_size_t)]),
    'scs_train_loss': (_c.c_int, [_vp, _c.POINTER(_c.c_void_p)]),
    'scs_grad_arena': (_c.c_int, [_vp, _c.POINTER(_vp), _c.POINTER(_c.c_size_t)]),
    'scs_wait_head_grads': (_c.c_int, [_vp, _vp, _c.POINTER(_c.c_size_t), _c.POINTER(_c.c_size_t)]),
    'scs_adam_apply': (_c.c_int, [_vp, _c.c_float, _c.c_float, _c.c_float, _c.c_float, _c.c_float, _vp]),
    'scs_set_fused_adam': (_c.c_int, [_vp, _c.c_int, _c.c_float, _c.c_float, _c.c_float, _c.c_float]),
    'scs_eval_batch': (_c.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _c.c_int64, _c.POINTER(_c.c_double),
                                  _c.POINTER(_c.c_int64), _vp]),
    'scs_lowrank_workspace': (_c.c_int, [_vp, _vp, _c.c_int, _vp, _c.c_int64, _c.POINTER(_c.c_size_t)]),
    'scs_lowrank_forward': (_c.c_int, [_vp, _vp, _vp, _c.c_int64, _vp, _c.c_int64, _vp, _vp, _c.c_size_t, _vp]),
    'scs_lowrank_backward': (_c.c_int, [_vp, _vp, _vp, _c.c_int64, _vp, _c.c_int64, _vp, _vp, _c.c_int64, _vp, _vp, _vp, _c.c_size_t, _vp]),
    'scs_adamw_create': (_c.c_int, [_vp, _vp, _c.c_int32, _c.c_int, _vp, _vp, _vp, _vp, _c.c_int64, _c.POINTER(_vp)]),
    'scs_adamw_destroy': (_c.c_int, [_vp]),
    'scs_adamw_step': (_c.c_int, [_vp, _vp, _vp, _c.c_double, _c.c_double, _c.c_double, _c.c_double, _c.c_double, _c.c_double, _vp, _vp]),
    'scs_adamw_states': (_c.c_int, [_vp, _vp, _vp, _vp]),
    'scs_adamw_get_step': (_c.c_int, [_vp, _c.POINTER(_c.c_int64), _vp]),
    'scs_adamw_set_step': (_c.c_int, [_vp, _c.c_int64, _vp]),
}


class ScsError(RuntimeError):
    pass


def load_library():
    """dlopen libscs.so and attach the prototypes.  Raises ScsError when the library has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ScsError('HIP extension missing: %s (build it with __graft_entry__.build() or '
                       '`make -C sub-cortical_segmentation_amd/csrc`)' % LIB_PATH)
    try:
        import torch  # noqa: F401  - FIRST: torch brings its own HIP runtime; libscs.so then binds to that one.  Loaded the other
    except ImportError:            # way round, /opt/rocm's runtime comes in ahead of torch's and the process has two (the second
        pass                       # one finds "no ROCm-capable device")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in SIGNATURES.items():
        if os.environ.get('SCS_LIB_PATH') and not hasattr(lib, name):
            continue                      # an older build under test
        fn = getattr(lib, name)           # AttributeError here = header/library mismatch
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _check(rc, what):
    if rc != 0:
        msg = load_library().scs_last_error()
        raise ScsError('%s failed (%d): %s' % (what, rc, msg.decode() if msg else ''))


def _ptr(x):
    """Device/host pointer of a torch tensor, numpy array or None as an integer."""
    if x is None:
        return None
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    return x.data_ptr()


_ITEM = {'f32': 4, 'i32': 4, 'u8': 1}


def _dtype_name(x):
    return str(x.dtype).replace('torch.', '')


def _need(x, count, what, dtype='f32'):
    """A buffer handed to the library must be C-contiguous, of the element type the kernels read, and hold at least `count`
    elements: the kernels trust their sizes, and a short buffer (or a float64 view that happens to have enough elements) is
    a GPU memory fault (which can take the whole node down), not an exception."""
    if x is None:
        return
    names = {'f32': ('float32',), 'i32': ('int32',), 'u8': ('uint8', 'bool')}[dtype]
    if _dtype_name(x) not in names:
        raise ValueError('%s must be %s, got %s' % (what, names[0], _dtype_name(x)))
    contiguous = x.flags['C_CONTIGUOUS'] if isinstance(x, np.ndarray) else x.is_contiguous()
    if not contiguous:
        raise ValueError('%s must be C-contiguous' % what)
    have = x.size if isinstance(x, np.ndarray) else x.numel()
    if have < count:
        raise ValueError('%s holds %d elements, the call needs %d' % (what, have, count))


def _table(x, cols, what, dtype):
    """A 2-D table [rows, cols] of `dtype` (sample rows, volume descriptors): returns rows.  The row count the kernels clamp
    against is taken from the shape, so the shape has to be the real one."""
    if x is None or len(x.shape) != 2 or int(x.shape[1]) != cols:
        raise ValueError('%s must be a 2-D [N, %d] array, got shape %r' % (what, cols, None if x is None else tuple(x.shape)))
    _need(x, int(x.shape[0]) * cols, what, dtype)
    return int(x.shape[0])


# ---- libscs_io.so: host-side file helpers (include/scs_io.h).  No HIP dependency: safe to load before torch has brought its own
# HIP runtime into the process (libscs.so must NOT be: it would pull /opt/rocm's ahead of torch's and leave the process with two).
IO_LIB_PATH = os.environ.get('SCS_IO_LIB_PATH') or os.path.join(os.path.dirname(LIB_PATH), 'libscs_io.so')   # (override: sanitizer builds)
IO_SIGNATURES = {
    'scs_io_last_error': (_c.c_char_p, []),
    'scs_gz_gather': (_c.c_int, [_c.c_char_p, _vp, _c.c_int64, _c.c_int, _vp, _c.POINTER(_c.c_int64)]),
    'scs_gz_read': (_c.c_int, [_c.c_char_p, _c.c_int64, _c.c_int64, _vp]),
    'scs_gz_member': (_c.c_int, [_vp, _c.c_int64, _vp, _c.c_int64, _c.POINTER(_c.c_int64)]),
    'scs_gz_member_scatter': (_c.c_int, [_c.c_int64, _vp, _c.c_int, _vp, _vp, _c.c_int64, _vp, _c.c_int64, _c.POINTER(_c.c_int64)]),
}
_io_lib = None


def load_io_library():
    global _io_lib
    if _io_lib is None:
        if not os.path.exists(IO_LIB_PATH):
            raise ScsError('host IO library missing: %s (build it with __graft_entry__.build())' % IO_LIB_PATH)
        lib = ctypes.CDLL(IO_LIB_PATH)
        for name, (res, args) in IO_SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _io_lib = lib
    return _io_lib


def _io_error(lib, what, rc):
    msg = lib.scs_io_last_error()
    return IOError(msg.decode() if msg else '%s failed (%d)' % (what, rc))


def gz_gather(path, byte_offsets, elem_bytes, total=False):
    """Elements of a gzip file at ascending byte offsets of its inflated content (scs_gz_gather: host code of the library, no
    GPU needed) -> uint8 array [n, elem_bytes] (and the inflated length when `total`)."""
    lib = load_io_library()
    off = np.ascontiguousarray(byte_offsets, dtype=np.int64)
    out = np.empty((off.size, int(elem_bytes)), np.uint8)
    n_out = ctypes.c_int64(0)
    rc = lib.scs_gz_gather(os.fsencode(path), off.ctypes.data, off.size, int(elem_bytes), out.ctypes.data, ctypes.byref(n_out) if total else None)
    if rc != 0:
        raise _io_error(lib, 'scs_gz_gather', rc)
    return (out, int(n_out.value)) if total else out


def gz_read(path, offset, out):
    """Bytes [offset, offset + out.nbytes) of the inflated content of a gzip file into the uint8 array `out` (scs_gz_read)."""
    lib = load_io_library()
    rc = lib.scs_gz_read(os.fsencode(path), int(offset), int(out.nbytes), out.ctypes.data)
    if rc != 0:
        raise _io_error(lib, 'scs_gz_read', rc)
    return out


def gz_member(buf):
    """One gzip member holding the bytes of `buf` (any C-contiguous buffer), by the library's encoder for sparse volumes
    (scs_gz_member): zero runs and 8-byte repeats are matches, the rest literals."""
    lib = load_io_library()
    src = np.frombuffer(buf, dtype=np.uint8)
    out = np.empty(src.size + src.size // 8 + 64, dtype=np.uint8)
    n = ctypes.c_int64(0)
    rc = lib.scs_gz_member(src.ctypes.data, int(src.size), out.ctypes.data, int(out.size), ctypes.byref(n))
    if rc != 0:
        raise _io_error(lib, 'scs_gz_member', rc)
    return out[:n.value].tobytes()


def gz_member_scatter(n_elements, fill, index, values):
    """One gzip member holding n_elements copies of the scalar `fill` (its dtype is the element type) with values[k] at element
    index[k] (scs_gz_member_scatter: the buffer is built and deflated inside the library, no interpreter lock held)."""
    lib = load_io_library()
    values = np.ascontiguousarray(values)
    fill = np.asarray(fill, dtype=values.dtype).reshape(1)
    index = np.ascontiguousarray(index, dtype=np.int64)
    if index.shape != values.shape or values.ndim != 1:
        raise ValueError('index and values must be 1-D arrays of the same length')
    item = values.dtype.itemsize
    nbytes = int(n_elements) * item
    n = ctypes.c_int64(0)
    for cap in (nbytes // 32 + values.nbytes * 9 // 8 + 1024, nbytes + nbytes // 8 + 64):     # sparse rows deflate to a few per cent
        out = np.empty(cap, dtype=np.uint8)
        rc = lib.scs_gz_member_scatter(nbytes, fill.ctypes.data, item, index.ctypes.data, values.ctypes.data, int(values.size),
                                       out.ctypes.data, int(cap), ctypes.byref(n))
        if rc == 0:
            return out[:n.value].tobytes()
        if b'too small' not in (lib.scs_io_last_error() or b''):
            break
    raise _io_error(lib, 'scs_gz_member_scatter', rc)


class Handle:
    """Owns one scs_handle on one device."""

    def __init__(self, device=0):
        self.lib = load_library()
        h = ctypes.c_void_p()
        _check(self.lib.scs_create(int(device), ctypes.byref(h)), 'scs_create')
        self.h = h
        self.device = int(device)

    def close(self):
        if getattr(self, 'h', None):
            self.lib.scs_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- parameters
    def set_params(self, flat):
        flat = np.ascontiguousarray(flat, dtype=np.float32)
        if flat.size != N_PARAMS:
            raise ValueError('parameter arena has %d floats, expected %d' % (flat.size, N_PARAMS))
        _check(self.lib.scs_set_params(self.h, flat.ctypes.data, flat.size), 'scs_set_params')

    def get_params(self):
        out = np.empty(N_PARAMS, np.float32)
        _check(self.lib.scs_get_params(self.h, out.ctypes.data, out.size), 'scs_get_params')
        return out

    def set_chunk(self, n):
        return self.lib.scs_set_chunk(self.h, int(n))

    def set_option(self, name, value):
        """Behaviour switch of the training step on THIS handle (include/scs.h: scs_set_option); -1 restores the default."""
        _check(self.lib.scs_set_option(self.h, name.encode(), int(value)), 'scs_set_option(%s)' % name)

    def get_option(self, name):
        v = ctypes.c_int64(0)
        _check(self.lib.scs_get_option(self.h, name.encode(), ctypes.byref(v)), 'scs_get_option(%s)' % name)
        return int(v.value)

    def probe_f32_mfma(self):
        """TFLOP/s at which this device issues back-to-back v_mfma_f32_16x16x4_f32 (include/scs.h: scs_probe_f32_mfma)."""
        v = ctypes.c_double(0.0)
        _check(self.lib.scs_probe_f32_mfma(self.h, ctypes.byref(v)), 'scs_probe_f32_mfma')
        return float(v.value)

    def probe_f32_mfma_clock(self):
        """(TFLOP/s of the same probe, shader clock in GHz held while it ran) - include/scs.h: scs_probe_f32_mfma_clock."""
        v, g = ctypes.c_double(0.0), ctypes.c_double(0.0)
        _check(self.lib.scs_probe_f32_mfma_clock(self.h, ctypes.byref(v), ctypes.byref(g)), 'scs_probe_f32_mfma_clock')
        return float(v.value), float(g.value)

    # ---- inference
    def _check_inputs(self, ax, co, sa, atlas, n, y=None, probs=None, labels=None):
        for name, x in (('axial view', ax), ('coronal view', co), ('sagittal view', sa)):
            _need(x, 1024 * n, name)
        _need(atlas, 15 * n, 'atlas rows')
        _need(y, n, 'labels', 'u8')
        _need(probs, 15 * n, 'probs')
        _need(labels, n, 'labels out', 'i32')

    def forward(self, ax, co, sa, atlas, n, probs=None, labels=None, stream=0):
        self._check_inputs(ax, co, sa, atlas, n, probs=probs, labels=labels)
        _check(self.lib.scs_forward(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), int(n), _ptr(probs),
                                    _ptr(labels), stream or None), 'scs_forward')

    def forward_features(self, ax, co, sa, atlas, n, features, stream=0):
        """features float32 [n, 540]: the dense head's input of the forward pass (scs_forward_features)."""
        self._check_inputs(ax, co, sa, atlas, n)
        _need(features, 540 * n, 'features')
        _check(self.lib.scs_forward_features(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), int(n), _ptr(features), stream or None),
               'scs_forward_features')

    def forward_host(self, ax, co, sa, atlas, n, probs=None, labels=None):
        self._check_inputs(ax, co, sa, atlas, n, probs=probs, labels=labels)
        _check(self.lib.scs_forward_host(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), int(n), _ptr(probs),
                                         _ptr(labels)), 'scs_forward_host')

    def _check_volume(self, vol, dims, centers, n, probs, labels):
        nvox = int(dims[0]) * int(dims[1]) * int(dims[2])
        if min(int(d) for d in dims) < 1:
            raise ValueError('volume dimensions must be positive, got %r' % (tuple(dims),))
        _need(vol, nvox, 'volume')
        _need(centers, 3 * n, 'centre list', 'i32')
        _need(probs, 15 * n, 'probs')
        _need(labels, n, 'labels out', 'i32')
        return nvox

    def forward_volume(self, vol, dims, centers, atlas4d, n, probs=None, labels=None, stream=0):
        _need(atlas4d, 15 * self._check_volume(vol, dims, centers, n, probs, labels), 'atlas volume')
        _check(self.lib.scs_forward_volume(self.h, _ptr(vol), int(dims[0]), int(dims[1]), int(dims[2]), _ptr(centers),
                                           _ptr(atlas4d), int(n), _ptr(probs), _ptr(labels), stream or None),
               'scs_forward_volume')

    def forward_volume_rows(self, vol, dims, centers, atlas_rows, n, probs=None, labels=None, stream=0):
        self._check_volume(vol, dims, centers, n, probs, labels)
        _need(atlas_rows, 15 * n, 'atlas rows')
        _check(self.lib.scs_forward_volume_rows(self.h, _ptr(vol), int(dims[0]), int(dims[1]), int(dims[2]),
                                                _ptr(centers), _ptr(atlas_rows), int(n), _ptr(probs), _ptr(labels),
                                                stream or None), 'scs_forward_volume_rows')

    def forward_volume_shared(self, vol, dims, centers, atlas_rows, n, box, probs=None, labels=None, stream=0):
        """forward_volume_rows with the tower work shared between neighbouring voxels (include/scs.h: scs_forward_volume_shared).
        box: (xmin, xmax, ymin, ymax, zmin, zmax) of the centres, host integers."""
        self._check_volume(vol, dims, centers, n, probs, labels)
        _need(atlas_rows, 15 * n, 'atlas rows')
        b = np.ascontiguousarray(np.asarray(box, dtype=np.int64).reshape(6))
        if (b[0::2] > b[1::2]).any() or (b[0::2] < -4096).any() or (b[1::2] - b[0::2] >= 4096).any():
            raise ValueError('box %r is not (xmin, xmax, ymin, ymax, zmin, zmax) of a centre list' % (b.tolist(),))
        b32 = b.astype(np.int32)
        _check(self.lib.scs_forward_volume_shared(self.h, _ptr(vol), int(dims[0]), int(dims[1]), int(dims[2]), _ptr(centers),
                                                  _ptr(atlas_rows), int(n), b32.ctypes.data, _ptr(probs), _ptr(labels),
                                                  stream or None), 'scs_forward_volume_shared')

    def forward_profiled(self, ax, co, sa, atlas, n, probs=None, labels=None, stream=0):
        """-> (stage_ms float32[8], launches) measured with HIP events on `stream`."""
        self._check_inputs(ax, co, sa, atlas, n, probs=probs, labels=labels)
        ms = np.zeros(8, np.float32)
        k = ctypes.c_int(0)
        _check(self.lib.scs_forward_profiled(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), int(n), _ptr(probs),
                                             _ptr(labels), stream or None, ms.ctypes.data, ctypes.byref(k)),
               'scs_forward_profiled')
        return ms, int(k.value)

    def dilate_mask(self, mask_dev, scratch_dev, dims, iterations, stream=0):
        nvox = int(dims[0]) * int(dims[1]) * int(dims[2])
        _need(mask_dev, nvox, 'mask', 'u8')
        _need(scratch_dev, nvox, 'dilation scratch', 'u8')
        _check(self.lib.scs_dilate_mask(self.h, _ptr(mask_dev), _ptr(scratch_dev), int(dims[0]), int(dims[1]), int(dims[2]),
                                        int(iterations), stream or None), 'scs_dilate_mask')

    # raw volumes as they lie in a NIfTI file: element type -> SCS_U8 .. SCS_F64 (include/scs.h)
    RAW_DTYPES = {'uint8': 0, 'int16': 1, 'uint16': 2, 'int32': 3, 'float32': 4, 'float64': 5}
    STAT_DOUBLES = 3 * 1024 + 3

    def _raw(self, raw_dev, dims, what):
        code = self.RAW_DTYPES.get(_dtype_name(raw_dev))
        if code is None:
            raise ValueError('%s: element type %s is not one of %s' % (what, _dtype_name(raw_dev), ', '.join(self.RAW_DTYPES)))
        nvox = int(dims[0]) * int(dims[1]) * int(dims[2])
        if min(int(d) for d in dims) < 1 or raw_dev.numel() < nvox or not raw_dev.is_contiguous():
            raise ValueError('%s must be a contiguous buffer of %d voxels' % (what, nvox))
        return code, nvox

    def zscore_volume(self, raw_dev, dims, fortran_order, out_dev, scratch_dev, stream=0):
        code, nvox = self._raw(raw_dev, dims, 'raw volume')
        _need(out_dev, nvox, 'normalised volume')
        if _dtype_name(scratch_dev) != 'float64' or scratch_dev.numel() < self.STAT_DOUBLES:
            raise ValueError('z-score scratch must hold %d float64' % self.STAT_DOUBLES)
        _check(self.lib.scs_zscore_volume(self.h, _ptr(raw_dev), code, int(dims[0]), int(dims[1]), int(dims[2]), 1 if fortran_order else 0,
                                          _ptr(out_dev), _ptr(scratch_dev), stream or None), 'scs_zscore_volume')

    def roi_prepare(self, mask_raw_dev, dims, fortran_order, iterations, mask_dev, scratch_dev, run_offsets_dev, stream=0):
        code, nvox = self._raw(mask_raw_dev, dims, 'raw mask')
        _need(mask_dev, nvox, 'mask', 'u8')
        _need(scratch_dev, nvox, 'dilation scratch', 'u8')
        _need(run_offsets_dev, (nvox + 1023) // 1024 + 1, 'run offsets', 'i32')
        total = ctypes.c_int64(0)
        _check(self.lib.scs_roi_prepare(self.h, _ptr(mask_raw_dev), code, int(dims[0]), int(dims[1]), int(dims[2]), 1 if fortran_order else 0,
                                        int(iterations), _ptr(mask_dev), _ptr(scratch_dev), _ptr(run_offsets_dev), ctypes.byref(total),
                                        stream or None), 'scs_roi_prepare')
        return int(total.value)

    def roi_centers(self, mask_dev, dims, run_offsets_dev, centers_dev, n, stream=0):
        nvox = int(dims[0]) * int(dims[1]) * int(dims[2])
        _need(mask_dev, nvox, 'mask', 'u8')
        _need(run_offsets_dev, (nvox + 1023) // 1024 + 1, 'run offsets', 'i32')
        _need(centers_dev, 3 * n, 'centre list', 'i32')
        _check(self.lib.scs_roi_centers(self.h, _ptr(mask_dev), int(dims[0]), int(dims[1]), int(dims[2]), _ptr(run_offsets_dev),
                                        _ptr(centers_dev), int(n), stream or None), 'scs_roi_centers')

    def get_activation(self, which, count):
        out = np.empty(count, np.float32)
        _check(self.lib.scs_get_activation(self.h, int(which), out.ctypes.data, out.size), 'scs_get_activation')
        return out

    # ---- training
    @staticmethod
    def _desc_count(descs):
        """Number of scs_volume records (24 bytes each: int64 offset, int32 x, y, z, reserved) in a descriptor table given as
        int64 [V, 3] or int32 [V, 6]."""
        name = _dtype_name(descs)
        if name == 'int64':
            cols = 3
        elif name == 'int32':
            cols = 6
        else:
            raise ValueError('volume descriptors must be int64 [V,3] or int32 [V,6] (scs_volume records), got %s' % name)
        if len(descs.shape) != 2 or int(descs.shape[1]) != cols or int(descs.shape[0]) < 1:
            raise ValueError('volume descriptors must have shape [V,%d], got %r' % (cols, tuple(descs.shape)))
        contiguous = descs.flags['C_CONTIGUOUS'] if isinstance(descs, np.ndarray) else descs.is_contiguous()
        if not contiguous:
            raise ValueError('volume descriptors must be C-contiguous')
        return int(descs.shape[0])

    def _check_tables(self, samples, descs, atlas_rows, y, index, n):
        """Shapes and types of the compact training-set tables: the device clamps row and volume numbers against the counts
        passed here, so they must be the real counts (a flat int32 view would report 4x the rows)."""
        n_samples = _table(samples, 4, 'sample rows', 'i32')
        n_vols = self._desc_count(descs)
        _need(atlas_rows, 15 * n_samples, 'atlas rows')
        _need(y, n_samples, 'labels', 'u8')
        _need(index, n, 'batch index', 'i32')
        if index is None and n > n_samples:
            raise ValueError('more samples asked for (%d) than the table holds (%d)' % (n, n_samples))
        return n_samples, n_vols

    def train_step(self, ax, co, sa, atlas, y, n, seed=0, masks=None, want_loss=True, stream=0):
        self._check_inputs(ax, co, sa, atlas, n, y=y)
        _need(masks, 5 * 540 * n, 'dropout masks', 'u8')
        loss = ctypes.c_float(0.0)
        _check(self.lib.scs_train_step(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), _ptr(y), int(n),
                                       ctypes.c_uint64(int(seed) & (2 ** 64 - 1)), _ptr(masks),
                                       ctypes.addressof(loss) if want_loss else None, stream or None),
               'scs_train_step')
        return float(loss.value) if want_loss else None

    def train_step_volume(self, vols, descs, samples, atlas_rows, y, index, n, seed=0, masks=None, want_loss=True, stream=0, flips=None):
        """Gather-fused step: patches are cut inside the kernels from `vols` (concatenated volumes on the device) around
        the voxels of `samples[index]` (include/scs.h: scs_train_step_volume)."""
        n_samples, n_vols = self._check_tables(samples, descs, atlas_rows, y, index, n)
        _need(flips, n, 'flip flags', 'u8')
        _need(masks, 5 * 540 * n, 'dropout masks', 'u8')
        loss = ctypes.c_float(0.0)
        _check(self.lib.scs_train_step_volume(self.h, _ptr(vols), _ptr(descs), n_vols, _ptr(samples), n_samples,
                                              _ptr(atlas_rows), _ptr(y), _ptr(index), _ptr(flips), int(n), ctypes.c_uint64(int(seed) & (2 ** 64 - 1)), _ptr(masks),
                                              ctypes.addressof(loss) if want_loss else None, stream or None),
               'scs_train_step_volume')
        return float(loss.value) if want_loss else None

    def gather_labels(self, label_vols, descs, samples, n, y_out, stream=0):
        if _table(samples, 4, 'sample rows', 'i32') < n:
            raise ValueError('sample table holds fewer than %d rows' % n)
        n_vols = self._desc_count(descs)
        _need(label_vols, 1, 'label volumes', 'u8')
        _need(y_out, n, 'labels out', 'u8')
        _check(self.lib.scs_gather_labels(self.h, _ptr(label_vols), _ptr(descs), n_vols, _ptr(samples), int(n), _ptr(y_out),
                                          stream or None),
               'scs_gather_labels')

    def eval_batch_volume(self, vols, descs, samples, atlas_rows, y, index, n, stream=0):
        n_samples, n_vols = self._check_tables(samples, descs, atlas_rows, y, index, n)
        ls, nc = ctypes.c_double(0.0), ctypes.c_int64(0)
        _check(self.lib.scs_eval_batch_volume(self.h, _ptr(vols), _ptr(descs), n_vols, _ptr(samples), n_samples,
                                              _ptr(atlas_rows), _ptr(y), _ptr(index), int(n), ctypes.byref(ls), ctypes.byref(nc), stream or None), 'scs_eval_batch_volume')
        return float(ls.value), int(nc.value)

    def train_step_profiled(self, ax, co, sa, atlas, y, n, seed=0, stream=0):
        """-> {stage name: ms}: one training step with HIP events around every launch (scs_train_step_profiled)."""
        self._check_inputs(ax, co, sa, atlas, n, y=y)
        k = self.lib.scs_train_stage_count()
        ms = np.zeros(k, np.float32)
        _check(self.lib.scs_train_step_profiled(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), _ptr(y), int(n),
                                                ctypes.c_uint64(int(seed) & (2 ** 64 - 1)), ms.ctypes.data, stream or None),
               'scs_train_step_profiled')
        return {self.lib.scs_train_stage_name(i).decode(): float(ms[i]) for i in range(k)}

    def get_train_buffer(self, which, count):
        out = np.empty(count, np.float32)
        _check(self.lib.scs_get_train_buffer(self.h, int(which), out.ctypes.data, out.size), 'scs_get_train_buffer')
        return out

    def train_loss_ptr(self):
        """Device address of the last train step's mean loss (float32)."""
        p = ctypes.c_void_p()
        _check(self.lib.scs_train_loss(self.h, ctypes.byref(p)), 'scs_train_loss')
        return p.value

    def set_fused_adam(self, enable, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8):
        """Single-rank training: every following train_step applies the Adam update itself (scs_set_fused_adam); adam_apply must
        not be called while this is on."""
        _check(self.lib.scs_set_fused_adam(self.h, 1 if enable else 0, lr, b1, b2, eps), 'scs_set_fused_adam')
        self.fused_adam = bool(enable)

    def adam_apply(self, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, grad_scale=1.0, stream=0):
        _check(self.lib.scs_adam_apply(self.h, lr, b1, b2, eps, grad_scale, stream or None), 'scs_adam_apply')

    def eval_batch(self, ax, co, sa, atlas, y, n, stream=0):
        self._check_inputs(ax, co, sa, atlas, n, y=y)
        ls, nc = ctypes.c_double(0.0), ctypes.c_int64(0)
        _check(self.lib.scs_eval_batch(self.h, _ptr(ax), _ptr(co), _ptr(sa), _ptr(atlas), _ptr(y), int(n),
                                       ctypes.byref(ls), ctypes.byref(nc), stream or None), 'scs_eval_batch')
        return float(ls.value), int(nc.value)

    def _arena(self, fn):
        p, n = ctypes.c_void_p(), ctypes.c_size_t()
        _check(fn(self.h, ctypes.byref(p), ctypes.byref(n)), 'arena query')
        return p.value, n.value

    def grad_arena(self):
        return self._arena(self.lib.scs_grad_arena)

    def wait_head_grads(self, stream):
        """Make `stream` wait for the dense head's gradients of the last train_step (scs_wait_head_grads) -> (first float, count) of
        that bucket in the gradient arena."""
        a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
        _check(self.lib.scs_wait_head_grads(self.h, stream, ctypes.byref(a), ctypes.byref(b)), 'scs_wait_head_grads')
        return int(a.value), int(b.value)

    def param_arena(self):
        return self._arena(self.lib.scs_param_arena)
