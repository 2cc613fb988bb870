"""The shared projection with a low-rank adapter per request (cnn_cort.adapters.Projection, scs_lowrank_*) against the same formulas in
float64.  Needs an MI355X.

Tolerances, in units of u = 2^-24 (float32) and r = eps / 2 of the outputs' type.  A sum of n products of exact operands, formed in float32
in any order, is off by at most n u sum |products|; the bounds below use |x| |W| sums formed in float64 ("big"), the inner value
h = x A^T has n_in u big_h, and its way through scale (1 u), the two 16-bit pieces (2 r^2: below u for bf16's r = 2^-9 only up to
2^-17, which is counted), B and the sum adds the rest.  The output's own rounding is r |y| (on the value with its error)."""
import numpy as np
import pytest
import torch

import lowrank_forms
from cnn_cort import _hip
from cnn_cort.adapters import Projection

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
HALF = {'f32': 2.0 ** -24, 'bf16': 2.0 ** -8, 'f16': 2.0 ** -11}                      # half a step, relative
PIECES = {'f32': 0.0, 'bf16': 2.0 ** -16, 'f16': 2.0 ** -22}                          # what two 16-bit pieces leave of a float32


def data(t, rows, n_in, n_out, rank, adapters, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(TYPES[t]).to('cuda:0')
    return {'x': mk(rows, n_in), 'dy': mk(rows, n_out), 'w': mk(n_in, n_out, std=n_in ** -0.5), 'a': mk(adapters, rank, n_in, std=n_in ** -0.5),
            'b': mk(adapters, rank, n_out, std=0.3), 'bias': mk(n_out) if bias else None,
            'scale': (0.5 + torch.rand((adapters,), generator=g)).to('cuda:0')}


def requests(off, ids):
    return torch.tensor(off, dtype=torch.int32, device='cuda:0'), torch.tensor(ids, dtype=torch.int32, device='cuda:0')


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def reference(d, off, ids, t, hidden=None):
    """Values and bounds of the forward and backward results on the live rows."""
    x, dy, w, a, b = (f64(d[k]) for k in ('x', 'dy', 'w', 'a', 'b'))
    sc = f64(d['scale']) if d['scale'] is not None else np.ones(a.shape[0])
    bias = f64(d['bias']) if d['bias'] is not None else np.zeros(w.shape[1])
    rows, n_in, n_out, rank = x.shape[0], x.shape[1], w.shape[1], a.shape[1]
    half, pc = HALF[t], PIECES[t]
    y, by = x @ w + bias, (n_in + 2) * U * (np.abs(x) @ np.abs(w) + np.abs(bias))
    dx, bdx = dy @ w.T, (n_out + 2) * U * (np.abs(dy) @ np.abs(w).T)
    h = np.zeros((rows, rank))
    bh = np.zeros((rows, rank))
    da, db = np.zeros_like(a), np.zeros_like(b)
    bda, bdb = np.zeros_like(a), np.zeros_like(b)
    live = np.zeros(rows, bool)
    for q, s in enumerate(ids):
        lo, hi = off[q], off[q + 1]
        live[lo:hi] = True
        if s < 0 or s >= a.shape[0] or hi <= lo:
            continue
        X, D = x[lo:hi], dy[lo:hi]
        h[lo:hi] = X @ a[s].T
        bh[lo:hi] = n_in * U * (np.abs(X) @ np.abs(a[s]).T)
        H, BH = h[lo:hi], bh[lo:hi]
        k = (rank + 4) * U + pc
        y[lo:hi] += sc[s] * H @ b[s]
        by[lo:hi] += abs(sc[s]) * (BH + k * np.abs(H)) @ np.abs(b[s]) + 2 * U * abs(sc[s]) * np.abs(H) @ np.abs(b[s])
        G, BG = D @ b[s].T, n_out * U * (np.abs(D) @ np.abs(b[s]).T)
        dx[lo:hi] += sc[s] * G @ a[s]
        bdx[lo:hi] += abs(sc[s]) * (BG + (k + 2 * U) * np.abs(G)) @ np.abs(a[s])
        da[s] += sc[s] * G.T @ X
        db[s] += sc[s] * H.T @ D
        bda[s] += abs(sc[s]) * (BG + (rows + 4) * U * np.abs(G)).T @ np.abs(X)
        bdb[s] += abs(sc[s]) * (BH + (rows + 4) * U * np.abs(H)).T @ np.abs(D)
    by += half * (np.abs(y) + by) + 1e-30
    bdx += half * (np.abs(dx) + bdx) + 1e-30
    if t == 'f16':                                                       # f16's smallest steps
        by, bdx = by + 2.0 ** -25, bdx + 2.0 ** -25
    return {'y': (y, by), 'dx': (dx, bdx), 'h': (h, bh + 1e-30), 'da': (da, bda + 1e-30), 'db': (db, bdb + 1e-30), 'live': live}


def within(got, ref, bound, what):
    got = f64(got)
    bad = ~(np.abs(got - ref) <= bound)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - ref) / bound, 0)), got.shape)
        raise AssertionError('%s: %d of %d beyond their bound; worst at %r: %r for %r (bound %.3g)' % (what, bad.sum(), bad.size, i, got[i], ref[i], bound[i]))


def check_all(handle, d, off, ids, t, with_hidden=True):
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    o, i = requests(off, ids)
    rows = d['x'].shape[0]
    ref = reference(d, off, ids, t)
    live = ref['live']
    out = torch.full((rows, p.n_out), 3.0, dtype=TYPES[t], device='cuda:0')
    hidden = torch.full((rows, p.rank), 5.0, device='cuda:0')
    y = p.forward(d['x'], o, i, out=out, hidden=hidden)
    assert y is out
    within(y[torch.from_numpy(live).cuda()], ref['y'][0][live], ref['y'][1][live], 'y')
    within(hidden[torch.from_numpy(live).cuda()], ref['h'][0][live], ref['h'][1][live], 'hidden')
    assert (f64(out)[~live] == 3.0).all() and (f64(hidden)[~live] == 5.0).all()
    dx0 = torch.full((rows, p.n_in), 3.0, dtype=TYPES[t], device='cuda:0')
    dx, da, db = p.backward(d['x'], d['dy'], o, i, hidden=hidden if with_hidden else None, dx=dx0)
    within(dx[torch.from_numpy(live).cuda()], ref['dx'][0][live], ref['dx'][1][live], 'dx')
    assert (f64(dx)[~live] == 3.0).all()
    within(da, ref['da'][0], ref['da'][1], 'da')
    within(db, ref['db'][0], ref['db'][1], 'db')
    again = p.backward(d['x'], d['dy'], o, i, hidden=hidden if with_hidden else None)
    assert torch.equal(again[1], da) and torch.equal(again[2], db)                # the same bits every time
    assert torch.equal(p.forward(d['x'], o, i)[torch.from_numpy(live).cuda()], y[torch.from_numpy(live).cuda()])


# rows, in, out, rank, adapters, offsets, adapters of the requests
CASES = {
    'one row': (1, 64, 64, 16, 2, [0, 1], [1]),
    'one of everything': (1, 1, 1, 1, 1, [0, 1], [0]),
    'the second dense layer': (128, 555, 270, 8, 4, [0, 40, 41, 90, 128], [2, 0, 3, 1]),
    'the first dense layer': (300, 540, 540, 8, 4, [0, 100, 200, 290], [0, 1, 0]),
    'one token each': (33, 128, 192, 4, 5, list(range(34)), [i % 6 - 1 for i in range(33)]),
    'odd': (70, 77, 131, 5, 3, [0, 3, 3, 64, 70], [2, 1, -1, 0]),
    'requests end inside tiles': (700, 96, 200, 16, 3, [0, 15, 17, 127, 129, 600, 700], [0, 1, 2, 0, -1, 1]),
    'rank above a slab': (530, 160, 96, 40, 2, [0, 200, 530], [1, 0]),
    'largest rank': (40, 136, 72, 128, 2, [0, 20, 40], [1, 0]),
    'rank of many rows': (600, 256, 128, 100, 2, [0, 333, 600], [1, 0]),
    'rows behind and before the requests': (600, 64, 80, 8, 2, [20, 300, 577], [0, 1]),
    'no request': (20, 32, 32, 4, 2, [0], []),
    'only empty requests': (20, 32, 32, 4, 2, [7, 7, 7], [0, 1]),
    'no adapter at all': (600, 64, 64, 4, 2, [0, 600], [-1]),
    'numbers outside the bank': (64, 64, 64, 4, 2, [0, 20, 64], [2, -7]),
    'more requests than a wave is wide': (1500, 72, 88, 8, 7, [15 * i for i in range(101)], [i % 8 - 1 for i in range(100)]),
    'aligned': (1100, 512, 768, 16, 4, [0, 1, 256, 512, 1000, 1100], [0, 1, 2, 3, -1]),
    'wide': (260, 64, 1000, 16, 2, [0, 130, 260], [0, 1]),
    'one row, long contractions': (1, 4096, 1040, 16, 3, [0, 1], [2]),
    'few rows, long contractions': (13, 2056, 1500, 33, 3, [0, 1, 5, 5, 12], [2, 0, 1, -1]),
    'tokens, long contractions': (48, 2000, 1111, 20, 5, list(range(49)), [i % 7 - 1 for i in range(48)]),
    'few rows above a tile': (61, 1033, 640, 8, 2, [0, 30, 60], [1, 0]),
    'many tiles': (3100, 264, 4104, 16, 3, [0, 100, 1500, 1501, 3000, 3090], [0, 1, 2, -1, 0]),
    'low tiles': (2200, 132, 648, 8, 3, [0, 100, 900, 2200], [0, 1, 2]),
    'low tiles, odd': (3000, 131, 517, 8, 3, [0, 100, 900, 3000], [0, 1, 2]),
    'rows in between': (700, 2052, 1033, 8, 3, [0, 100, 300, 699], [0, 1, 2]),
    'medium tiles': (1500, 192, 2056, 16, 3, [0, 100, 900, 1500], [0, 1, 2]),
    'medium tiles, odd': (1600, 197, 2051, 9, 3, [0, 100, 900, 1600], [0, 1, 2]),
    'many tiles, odd': (3333, 131, 4099, 17, 3, [0, 1000, 2222, 3333], [2, 1, 0]),
    'many tiles the other way': (2100, 4096, 328, 24, 3, [0, 700, 1500, 2100], [0, 1, 2]),
}


@pytest.mark.parametrize('t', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('case', list(CASES))
def test_against_float64(handle, case, t):
    rows, n_in, n_out, rank, adapters, off, ids = CASES[case]
    check_all(handle, data(t, rows, n_in, n_out, rank, adapters, len(case) + rows, bias=rows % 2 == 0), off, ids, t, with_hidden=rows % 3 != 0)


def some(t, rows=700, n_in=96, n_out=200, rank=8, adapters=3, seed=3):
    d = data(t, rows, n_in, n_out, rank, adapters, seed)
    return d, [0, 15, rows // 2, rows], [2, -1, 0]


@pytest.mark.parametrize('t', ['f32', 'bf16'])
@pytest.mark.parametrize('rows', [20, 700])
@pytest.mark.parametrize('shift', [0, 1, 8])
def test_strides_and_alignments(handle, t, rows, shift):
    """Every matrix as a view inside a larger one, `shift` elements off its start; what lies around the outputs stays."""
    d, off, ids = some(t, rows)
    o, i = requests(off, ids)

    def inside(m, fill):
        r, c = m.shape
        big = torch.full((r + 2, c + 24), fill, dtype=m.dtype, device='cuda:0')
        big[1:r + 1, shift:shift + c] = m
        return big, big[1:r + 1, shift:shift + c]

    w = inside(d['w'], 9.0)[1]
    x, dy = inside(d['x'], float('nan'))[1], inside(d['dy'], float('nan'))[1]
    p = Projection(handle, w, d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    q = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    yb, y = inside(torch.zeros((rows, 200), dtype=TYPES[t], device='cuda:0'), 4.0)
    db_, dx = inside(torch.zeros((rows, 96), dtype=TYPES[t], device='cuda:0'), 4.0)
    p.forward(x, o, i, out=y)
    assert torch.equal(y, q.forward(d['x'], o, i))
    _, da, db = p.backward(x, dy, o, i, dx=dx)
    ref = q.backward(d['x'], d['dy'], o, i)
    assert torch.equal(dx, ref[0]) and torch.equal(da, ref[1]) and torch.equal(db, ref[2])
    for big, part in ((yb, y), (db_, dx)):
        part.fill_(4.0)
        assert (big == 4.0).all()


@pytest.mark.parametrize('t', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows', [40, 700])
def test_what_is_not_finite_stays_with_its_own(handle, t, rows):
    """An adapter of infinities, a row of NaN and NaN behind the last request touch their own rows (and gradients) alone."""
    d, off, ids = some(t, rows)
    clean = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    o, i = requests(off[:-1] + [rows - 5], ids)
    y0 = clean.forward(d['x'], o, i)
    g0 = clean.backward(d['x'], d['dy'], o, i)
    a = d['a'].clone()
    b = d['b'].clone()
    a[2], b[2] = float('inf'), float('nan')                  # the first request's: rows 0..14
    x, dy = d['x'].clone(), d['dy'].clone()
    x[20], dy[20] = float('nan'), float('nan')                # a row of the request without an adapter (there is none at 20 rows of 40)
    x[rows - 5:], dy[rows - 5:] = float('nan'), float('nan')
    p = Projection(handle, d['w'], a, b, bias=d['bias'], scale=d['scale'])
    y = p.forward(x, o, i)
    g = p.backward(x, dy, o, i)
    keep = torch.ones(rows, dtype=torch.bool, device='cuda:0')
    keep[:15] = False
    keep[20] = False
    assert torch.equal(y[keep], y0[keep]) and torch.equal(g[0][keep], g0[0][keep])
    if rows == 700:                                          # row 20 has no adapter: adapter 0's gradients do not see it
        assert torch.equal(g[1][0], g0[1][0]) and torch.equal(g[2][0], g0[2][0])
    assert torch.equal(g[1][1], torch.zeros_like(g[1][1]))
    assert not torch.isfinite(y[:15].float()).any() and (y[rows - 5:] == 0).all()


@pytest.mark.parametrize('t', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,n_in', [(9, 1024), (33, 2048), (700, 96), (2048, 128)])
def test_captured_calls_replay(handle, t, rows, n_in):
    """Forward and backward in one graph, replayed with new inputs between eager work, against eager calls."""
    d, off, ids = some(t, rows, n_in)
    off[1] = min(off[1], rows // 2)
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    y, hid = torch.zeros((rows, 200), dtype=TYPES[t], device='cuda:0'), torch.zeros((rows, 8), device='cuda:0')
    dx, da, db = torch.zeros_like(d['x']), torch.zeros(d['a'].shape, device='cuda:0'), torch.zeros(d['b'].shape, device='cuda:0')
    p.forward(d['x'], o, i, out=y, hidden=hid)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.forward(d['x'], o, i, out=y, hidden=hid)
        p.backward(d['x'], d['dy'], o, i, hidden=hid, dx=dx, da=da, db=db)
    for k in range(4):
        fresh = data(t, rows, n_in, 200, 8, 3, 50 + k)
        for key in ('x', 'dy', 'w', 'a', 'b'):
            d[key].copy_(fresh[key])
        graph.replay()
        e = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
        hid2 = torch.zeros_like(hid)
        y2 = e.forward(d['x'], o, i, hidden=hid2)
        dx2, da2, db2 = e.backward(d['x'], d['dy'], o, i, hidden=hid2)
        torch.cuda.synchronize()
        for a_, b_ in ((y, y2), (hid, hid2), (dx, dx2), (da, da2), (db, db2)):
            assert torch.equal(a_, b_), 'replay %d' % k


def test_two_streams_and_two_threads_at_once(handle):
    import threading
    d, off, ids = some('bf16', 48, 2048)
    off[1] = 15
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'], scale=d['scale'])
    want = p.forward(d['x'], o, i)
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [p.forward(d['x'], o, i) for _ in range(20)]
                torch.cuda.current_stream().synchronize()
                got[k] = outs
        except Exception as e:          # surfaced below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    assert all(torch.equal(y, want) for outs in got.values() for y in outs)


def test_hidden_may_be_formed_again(handle):
    for rows in (60, 700):
        d, off, ids = some('bf16', rows)
        o, i = requests(off, ids)
        p = Projection(handle, d['w'], d['a'], d['b'], scale=d['scale'])
        hid = torch.empty((rows, 8), device='cuda:0')
        p.forward(d['x'], o, i, hidden=hid)
        a, b = p.backward(d['x'], d['dy'], o, i, hidden=hid), p.backward(d['x'], d['dy'], o, i)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        for want in (('dx',), ('da',), ('db',), ('da', 'db')):
            c = p.backward(d['x'], d['dy'], o, i, want=want)
            for k, s, t in zip(('dx', 'da', 'db'), a, c):
                assert (t is None) if k not in want else torch.equal(s, t)


def test_offsets_out_of_order_stay_inside(handle):
    """Offsets are read on the device and clamped to the rows: wrong ones give wrong rows, and nothing around the outputs changes."""
    for t in ('f32', 'bf16'):
        for rows in (50, 700):
            d, _, _ = some(t, rows)
            p = Projection(handle, d['w'], d['a'], d['b'])
            for off in ([rows, 5, 0, 3], [-7, 20, 2 * rows, 10 ** 9], [0, -2 ** 31, 2 ** 31 - 1, 9]):
                o, i = requests(off, [0, 1, 2])
                big = torch.full((rows + 4, 200), 2.0, dtype=TYPES[t], device='cuda:0')
                bdx = torch.full((rows + 4, 96), 2.0, dtype=TYPES[t], device='cuda:0')
                p.forward(d['x'], o, i, out=big[2:rows + 2])
                p.backward(d['x'], d['dy'], o, i, dx=bdx[2:rows + 2])
                torch.cuda.synchronize()
                for b in (big, bdx):
                    assert (b[:2] == 2.0).all() and (b[rows + 2:] == 2.0).all()


@pytest.mark.parametrize('ld', [2097152, 2100000])
def test_row_offsets_beyond_32_bits(handle, ld):
    rows, n_in, n_out = 1100, 64, 72
    d, off, ids = some('bf16', rows, n_in, n_out)
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    store = torch.empty((rows * ld,), dtype=torch.bfloat16, device='cuda:0')           # 4.6 GB
    x = torch.as_strided(store, (rows, n_in), (ld, 1))
    y = torch.as_strided(store, (rows, n_out), (ld, 1), 1024)
    x.copy_(d['x'])
    xin = x.clone()
    with pytest.raises(ValueError, match='shares memory'):
        p.forward(x, o, i, out=y)                                                          # (interleaved views count as shared)
    other = torch.empty((rows * ld,), dtype=torch.bfloat16, device='cuda:0')
    y = torch.as_strided(other, (rows, n_out), (ld, 1), 1024)
    p.forward(x, o, i, out=y)
    assert torch.equal(y, p.forward(xin, o, i))
    dy = y
    dx = torch.as_strided(store, (rows, n_in), (ld, 1), 512)
    g = p.backward(xin, dy, o, i, dx=dx)
    ref = p.backward(xin, dy.contiguous(), o, i)
    assert all(torch.equal(a, b) for a, b in zip(g, ref))


@pytest.mark.parametrize('t', ['f32', 'bf16'])
def test_no_rows(handle, t):
    d, _, _ = some(t, 8)
    p = Projection(handle, d['w'], d['a'], d['b'])
    for off, ids in (([0], []), ([0, 0, 0], [1, -1])):
        o, i = requests(off, ids)
        x, dy = d['x'][:0], d['dy'][:0]
        assert p.forward(x, o, i).shape == (0, 200)
        dx, da, db = p.backward(x, dy, o, i, da=torch.ones((3, 8, 96), device='cuda:0'), db=torch.ones((3, 8, 200), device='cuda:0'))
        assert dx.shape == (0, 96) and not da.any() and not db.any()


def test_refusals(handle):
    d, off, ids = some('bf16')
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    x = d['x']
    bad = [lambda: p.forward(x.float(), o, i), lambda: p.forward(x[:, :95], o, i), lambda: p.forward(x.t(), o, i), lambda: p.forward(x.cpu(), o, i),
           lambda: p.forward(x, o[:-1], i), lambda: p.forward(x, o.long(), i), lambda: p.forward(x, o, i, out=x), lambda: p.forward(x[0], o, i),
           lambda: p.forward(x, o, i, hidden=torch.empty((3, 8), device='cuda:0')), lambda: p.backward(x, d['dy'], o, i, want=()),
           lambda: p.backward(x, d['dy'], o, i, want=('dw',)), lambda: p.backward(x, d['dy'], o, i, da=torch.empty((3, 8, 95), device='cuda:0')),
           lambda: p.backward(x, d['dy'][:9], o, i), lambda: p.backward(x, d['dy'], o, i, dx=x),
           lambda: Projection(handle, d['w'].double(), d['a'], d['b']), lambda: Projection(handle, d['w'], d['a'], d['b'][:2]),
           lambda: Projection(handle, d['w'], d['a'].transpose(0, 1), d['b'].transpose(0, 1)), lambda: Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'][:-1]),
           lambda: Projection(handle, d['w'], d['a'], d['b'], scale=d['scale'].half()),
           lambda: Projection(handle, d['w'], d['a'].new_zeros((3, 129, 96)), d['b'].new_zeros((3, 129, 200)))]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError('call %d was accepted' % k)


@pytest.mark.parametrize('rows,n_in,n_out', [(40, 96, 200), (700, 96, 200), (1500, 96, 2056), (3100, 96, 4104)])
def test_f16_inner_values_outside_its_range(handle, rows, n_in, n_out):
    """x A^T beyond f16's largest number (and, backward, among its smallest steps) where y and dx are ordinary."""
    d = data('f16', rows, n_in, n_out, 20, 3, rows)
    d['x'] *= 512
    d['a'] *= 256
    d['b'] *= 2.0 ** -13
    d['dy'] *= 2.0 ** -6
    off, ids = [0, 15, rows // 2, rows], [2, 1, 0]
    h = f64(d['x'][rows // 2:]) @ f64(d['a'][0]).T
    assert np.abs(h).max() > 2 * 65504
    check_all(handle, d, off, ids, 'f16')


@pytest.mark.parametrize('t', ['f32', 'bf16'])
@pytest.mark.parametrize('rank', [8, 40])
def test_gradients_of_many_short_requests(handle, t, rank):
    """Requests of no row to a few rows: the gradients' waves take them in turn."""
    rng = np.random.default_rng(rank)
    off = np.concatenate([[0], np.cumsum(rng.integers(0, 5, 300))]).tolist()
    ids = rng.integers(-1, 3, 300).tolist()
    check_all(handle, data(t, off[-1], 72, 200, rank, 3, 5), off, ids, t)


def test_a_moved_tensor_is_refused(handle):
    """The projection reads its tensors where they lay: one whose memory was replaced is refused, not read behind the owner's back."""
    d, off, ids = some('f32')
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'])
    y = p.forward(d['x'], o, i)
    old = d['b'].data
    d['b'].data = d['b'].clone()
    with pytest.raises(RuntimeError):
        p.forward(d['x'], o, i)
    d['b'].data = old
    assert torch.equal(p.forward(d['x'], o, i), y)


@pytest.mark.parametrize('t', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('n_in,n_out,rank', [(1, 32, 1), (7, 33, 5), (8, 47, 16), (540, 270, 8), (2049, 100, 17), (4100, 64, 32), (9001, 5000, 16), (8193, 48, 8), (555, 31, 8), (300, 64, 33)])
def test_one_row(handle, t, n_in, n_out, rank):
    """One new token: every adapter, none, and a row that no request owns; rows at any element."""
    d = data(t, 1, n_in, n_out, rank, 3, n_in + n_out, bias=n_out % 2 == 0)
    for off, ids in (([0, 1], [2]), ([0, 0, 1, 1], [1, 0, 2]), ([0, 1], [-1]), ([1, 1], [0]), ([0, 0], [0])):
        check_all(handle, d, off, ids, t)
    wide = torch.zeros((n_in, n_out + 3), dtype=TYPES[t], device='cuda:0')
    wide[:, 1:n_out + 1] = d['w']
    wide[:, 0], wide[:, n_out + 1:] = float('nan'), float('inf')
    flat = torch.full((n_in + 2,), float('nan'), dtype=TYPES[t], device='cuda:0')
    flat[1:n_in + 1] = d['x'][0]
    d['w'], d['x'] = wide[:, 1:n_out + 1], flat[1:n_in + 1].view(1, n_in)
    check_all(handle, d, [0, 1], [1], t)


@pytest.mark.parametrize('t', ['f32', 'bf16'])
def test_one_row_in_a_graph(handle, t):
    d = data(t, 1, 1000, 520, 12, 3, 4)
    o, i = requests([0, 1], [2])
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    out, hidden = torch.zeros((1, 520), dtype=TYPES[t], device='cuda:0'), torch.zeros((1, 12), device='cuda:0')
    p.forward(d['x'], o, i, out=out, hidden=hidden)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.forward(d['x'], o, i, out=out, hidden=hidden)
    for k in range(4):
        d['x'].normal_()
        i.fill_(k - 1)
        graph.replay()
        h2 = torch.empty_like(hidden)
        y = p.forward(d['x'], o, i, hidden=h2)
        torch.cuda.synchronize()
        assert torch.equal(out, y) and torch.equal(hidden, h2), 'replay %d' % k


@pytest.mark.parametrize('t', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows', [0, 20, 300, 700, 2000])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_an_unused_adapters_gradients_are_zeros_whatever_its_scale(handle, t, rows, bad):
    """An adapter that no row uses has zero gradients: its scale (an unfinished site's, say) takes no part."""
    d = data(t, rows, 96, 200, 8, 4, 7)
    d['scale'][1], d['scale'][3] = bad, bad
    p = Projection(handle, d['w'], d['a'], d['b'], scale=d['scale'])
    q = Projection(handle, d['w'], d['a'], d['b'], scale=torch.where(torch.isfinite(d['scale']), d['scale'], torch.ones_like(d['scale'])))
    # adapter 1: a request without rows, adapter 3: no request; the last rows use none
    o, i = requests([0, rows // 2, rows // 2, rows - rows // 8, rows], [0, 1, 2, -1])
    for n in (4, 0):
        got, want = (x.backward(d['x'], d['dy'], o[:n + 1], i[:n], da=torch.ones(d['a'].shape, device='cuda:0'), db=torch.ones(d['b'].shape, device='cuda:0')) for x in (p, q))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for g in got[1:]:
            assert not g[1].any() and not g[3].any() and (rows < 8 or n == 0 or g[0].any())


@pytest.mark.parametrize('t,rows,n_in,n_out,rank', [(t,) + s for t in TYPES for s in lowrank_forms.sizes(t)])
def test_every_form_against_float64(handle, t, rows, n_in, n_out, rank):
    """The kernels that the other sizes do not reach (test_lowrank.py sees to it that none is left)."""
    off, ids = lowrank_forms.requests(rows)
    check_all(handle, data(t, rows, n_in, n_out, rank, 3, rows + n_in + rank, bias=rank % 2 == 0), off, ids, t)


@pytest.mark.parametrize('which', ['w', 'a', 'b', 'bias', 'scale'])
def test_each_moved_tensor_is_refused_and_captured_calls_keep_theirs(handle, which):
    """forward() and backward() refuse; a graph captured before reads the memory that it was captured with, which is still the projection's."""
    d, off, ids = some('bf16', 40)
    o, i = requests(off, ids)
    p = Projection(handle, d['w'], d['a'], d['b'], bias=d['bias'], scale=d['scale'])
    y = torch.zeros((40, 200), dtype=torch.bfloat16, device='cuda:0')
    want = p.forward(d['x'], o, i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.forward(d['x'], o, i, out=y)
    d[which].data = torch.full_like(d[which], float('nan'))
    for call in (lambda: p.forward(d['x'], o, i), lambda: p.backward(d['x'], d['dy'], o, i)):
        with pytest.raises(RuntimeError, match='moved'):
            call()
    junk = [torch.full_like(t, 3.0) for t in d.values() for _ in range(4)]             # (would land in memory that had been freed)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del junk
