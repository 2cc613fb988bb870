"""AdamW over many tensors (cnn_cort.optim, scs_adamw_*): against the same formulas in NumPy float32 - every operation rounded once, so
the results are the same BITS, 8-bit codes included - and against float64 with bounds counted in roundings.  Needs an MI355X."""
import numpy as np
import pytest
import torch

from cnn_cort import _hip
from cnn_cort.optim import BLOCK, AdamW, blocks_of

pytestmark = pytest.mark.gpu
F32 = np.float32
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZES = [1, 255, 256, 257, 4096, 4097, 0, 10007, 3, 64]
U = 2.0 ** -24                       # half a step of float32, relative


# ------------------------------------------------------------------------------------------- the formulas, in NumPy float32
def encode(x, levels, at_least_one):
    s = (x.max(1, keepdims=True) * F32(1.0 / levels ** 2)).astype(F32)
    s = np.where(s < F32(2.0 ** -126), F32(0), s)
    with np.errstate(divide='ignore', invalid='ignore'):
        inv = np.where(s > 0, F32(1) / s, F32(0))
        t = (x * inv).astype(np.float64)
        q = np.floor(np.sqrt(np.maximum(t - 0.25, 0)) + 0.5)
    if at_least_one:
        q = np.where(x > 0, np.maximum(q, 1), q)
    return np.minimum(q, levels).astype(F32), s.astype(F32)


class Ref:
    """One tensor in NumPy float32; p as float32 values (rounded to the parameter's type after every step unless a master is kept)."""

    def __init__(self, p, dtype, bits, wd, master):
        self.shape, self.n = p.shape, p.size
        self.p, self.dtype, self.bits, self.wd, self.master = p.astype(F32).ravel(), dtype, bits, wd, master
        nb = blocks_of(self.n)
        self.m, self.v = np.zeros((nb, BLOCK), F32), np.zeros((nb, BLOCK), F32)
        self.qm, self.qv = np.zeros((nb, BLOCK), F32), np.zeros((nb, BLOCK), F32)

    def step(self, g, t, lr, b1, b2, eps, gscale):
        n, nb = self.n, blocks_of(self.n)
        pad = nb * BLOCK - n
        g = (np.concatenate([g.astype(F32).ravel(), np.zeros(pad, F32)]) * F32(gscale)).reshape(nb, BLOCK)
        p = np.concatenate([self.p, np.zeros(pad, F32)]).reshape(nb, BLOCK)
        m = self.m * F32(b1) + g * F32(1.0 - b1)
        v = self.v * F32(b2) + (g * g) * F32(1.0 - b2)
        u = np.sqrt(v)
        size, root = F32(lr / (1.0 - b1 ** t)), F32(1.0 / np.sqrt(1.0 - b2 ** t))
        p = p * F32(1.0 - lr * self.wd) - m / (u * root + F32(eps)) * size
        self.p = p.ravel()[:n]
        if not self.master:
            self.p = torch.from_numpy(self.p).to(self.dtype).float().numpy()
        if self.bits == 32:
            self.m, self.v = m, v
        else:
            q, self.sm = encode(np.abs(m), 127, False)
            self.qm = (q * np.sign(m)).astype(F32)
            self.m = self.qm * np.abs(self.qm) * self.sm
            self.qv, self.sv = encode(u, 255, True)
            u = self.qv * self.qv * self.sv
            self.v = u * u
        assert self.m.dtype == F32 and self.v.dtype == F32 and p.dtype == F32


def make(sizes, dtype, seed, offset=0):
    """Tensors as views of one arena, each `offset` elements behind the end of the one before."""
    rng = np.random.default_rng(seed)
    arena = torch.zeros((sum(sizes) + offset * (len(sizes) + 1) + 1,), dtype=dtype, device='cuda:0')
    out, at = [], offset
    for n in sizes:
        t = arena[at:at + n]
        t.copy_(torch.from_numpy(rng.normal(size=n).astype(F32)).to(dtype))
        out.append(t)
        at += n + offset
    return out


def gradients(sizes, dtype, seed, spread=True):
    rng = np.random.default_rng(seed)
    out = []
    for i, n in enumerate(sizes):
        g = rng.normal(size=n) * (10.0 ** -(i % 4) if spread else 1.0)
        g[rng.random(n) < 0.2] = 0.0
        out.append(torch.from_numpy(g.astype(F32)).to(dtype).to('cuda:0'))
    return out


def gscale_of(grads, grad_scale, max_norm):
    if max_norm is None:
        return F32(grad_scale), None
    sq = sum(float((g.double() ** 2).sum()) for g in grads if g.numel())
    norm = abs(grad_scale) * np.sqrt(sq)
    return F32(grad_scale * min(1.0, max_norm / (norm + 1e-6))), norm


def check_same(opt, refs, params):
    mo, vo = opt.states()
    for i, r in enumerate(refs):
        lo = opt.first[i] * BLOCK
        hi = lo + blocks_of(r.n) * BLOCK
        assert np.array_equal(params[i].float().cpu().numpy(), torch.from_numpy(r.p).to(r.dtype).float().numpy()), 'parameter %d' % i
        assert np.array_equal(mo[lo:hi].cpu().numpy(), r.m.ravel()), 'm of tensor %d' % i
        assert np.array_equal(vo[lo:hi].cpu().numpy(), r.v.ravel()), 'v of tensor %d' % i
        if r.master and opt.masters[i] is not None:
            assert np.array_equal(opt.masters[i].cpu().numpy(), r.p)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('pt,gt,offset,clip,master', [
    ('f32', 'f32', 0, None, False), ('f32', 'f32', 1, 0.5, False), ('f32', 'bf16', 3, None, False), ('f32', 'f16', 0, 100.0, False),
    ('bf16', 'bf16', 1, 1.0, False), ('bf16', 'f32', 0, None, True), ('f16', 'f16', 0, None, False), ('f16', 'f32', 5, 2.0, True)])
def test_same_bits_as_the_formulas(handle, bits, pt, gt, offset, clip, master):
    params = make(SIZES, TYPES[pt], 1, offset)
    wds = [0.0 if i % 3 == 0 else 0.05 for i in range(len(SIZES))]
    opt = AdamW(handle, params, lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=wds, state_bits=bits, max_norm=clip, master=master)
    refs = [Ref(p.float().cpu().numpy(), TYPES[pt], bits, w, master and pt != 'f32') for p, w in zip(params, wds)]
    for t in range(1, 5):
        grads = gradients(SIZES, TYPES[gt], 10 + t)
        gs, norm = gscale_of(grads, 0.5, clip)
        opt.step(grads, grad_scale=0.5)
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
        for r, g in zip(refs, grads):
            r.step(g.float().cpu().numpy(), t, 3e-3, 0.8, 0.95, 1e-7, gs)
        check_same(opt, refs, params)
    assert opt.step_count == 4
    opt.close()


@pytest.mark.parametrize('bits,pt,gt', [(32, 'f32', 'f32'), (8, 'bf16', 'bf16'), (8, 'f32', 'f16')])
def test_many_chunks_give_the_same_bits(handle, bits, pt, gt):
    """Enough elements for the larger chunks, with tensors that end inside them."""
    sizes = [8400000, 4097, 1, 300001]
    params = make(sizes, TYPES[pt], 2, 1)
    opt = AdamW(handle, params, state_bits=bits, max_norm=1.0)
    refs = [Ref(p.float().cpu().numpy(), TYPES[pt], bits, 0.01, False) for p in params]
    for t in (1, 2):
        grads = gradients(sizes, TYPES[gt], 40 + t)
        gs, _ = gscale_of(grads, 1.0, 1.0)
        opt.step(grads)
        for r, g in zip(refs, grads):
            r.step(g.float().cpu().numpy(), t, 1e-3, 0.9, 0.999, 1e-8, gs)
    check_same(opt, refs, params)


def test_against_float64(handle):
    """One step in 32 bits.  In units of 2^-24, counted along the formula (each constant and each operation one): m 5 (b1 |m| + c1 |g|) =: 5 M,
    v 8 relative, the denominator 8 relative, p 3 |p| + 18 size M / denominator."""
    rng = np.random.default_rng(3)
    n = 5000
    p, g, m = rng.normal(size=n), rng.normal(size=n), rng.normal(size=n) * 0.1
    v = rng.random(n) * 0.1
    dev = lambda a: torch.from_numpy(a.astype(F32)).to('cuda:0')
    pad = lambda a: np.concatenate([a, np.zeros(blocks_of(n) * BLOCK - n)])
    P, M, V = dev(p), dev(pad(m)), dev(pad(v))
    p, g, m, v = (a.astype(F32).astype(np.float64) for a in (p, g, m, v))
    opt = AdamW(handle, [P], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1, states=(M, V, None, None), step=6)
    opt.step([dev(g)])
    m2, v2 = 0.9 * m + (1 - 0.9) * g, 0.99 * v + (1 - 0.99) * g * g
    size, den = 1e-2 / (1 - 0.9 ** 7), np.sqrt(v2 / (1 - 0.99 ** 7)) + 1e-8
    p2 = p * (1 - 1e-2 * 0.1) - size * m2 / den
    big = 0.9 * np.abs(m) + (1 - 0.9) * np.abs(g)
    assert (np.abs(M.cpu().numpy()[:n] - m2) <= 5 * U * big).all()
    assert (np.abs(V.cpu().numpy()[:n] - v2) <= 8 * U * v2).all()
    assert (np.abs(P.cpu().numpy() - p2) <= U * (3 * np.abs(p) + 18 * size * big / den)).all()


def test_eight_bit_codes_are_the_nearest_values(handle):
    """A value between codes q and q + 1 is off by at most half their distance, (q + 1/2) s <= (sqrt(value / s) + 1/2) s; the largest of a block
    is off by its scale's and its reciprocal's roundings alone."""
    rng = np.random.default_rng(4)
    n = 4096
    g = rng.normal(size=n) * 10.0 ** -rng.uniform(0, 6, n)
    P = torch.zeros((n,), device='cuda:0')
    opt = AdamW(handle, [P], state_bits=8, betas=(0.9, 0.999))
    G = torch.from_numpy(g.astype(F32)).to('cuda:0')
    opt.step([G])
    m, v = (a.cpu().numpy().astype(np.float64) for a in opt.states())
    wm, wu = np.abs(G.cpu().numpy().astype(np.float64)) * (1 - 0.9), np.abs(G.cpu().numpy().astype(np.float64)) * np.sqrt(1 - 0.999)
    sm = np.repeat(opt.m_scale.cpu().numpy().astype(np.float64), BLOCK)
    su = np.repeat(opt.v_scale.cpu().numpy().astype(np.float64), BLOCK)
    assert (np.abs(np.abs(m) - wm) <= (np.sqrt(wm / sm) + 0.5) * sm * (1 + 1e-5)).all()
    u = np.sqrt(v)
    near = (np.sqrt(wu / su) + 0.5) * su * (1 + 1e-5)
    assert (np.abs(u - wu) <= np.where(wu < 0.5 * su, su, near)).all()               # (a root that is not zero never takes code 0)
    assert (u[wu > 0] > 0).all() and (u[wu == 0] == 0).all()
    for b in range(n // BLOCK):
        i = b * BLOCK + int(np.argmax(wm[b * BLOCK:(b + 1) * BLOCK]))
        assert abs(abs(m[i]) - wm[i]) <= 8 * U * wm[i]


def test_gradients_of_several_types_in_one_step(handle):
    sizes = [5000, 300, 70000]
    params = make(sizes, torch.float32, 21)
    opt = AdamW(handle, params, max_norm=0.5)
    refs = [Ref(p.cpu().numpy(), torch.float32, 32, 0.01, False) for p in params]
    grads = [g.to(t) for g, t in zip(gradients(sizes, torch.float32, 22), (torch.float32, torch.bfloat16, torch.float16))]
    gs, norm = gscale_of(grads, 1.0, 0.5)
    opt.step(grads)
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm
    for r, g in zip(refs, grads):
        r.step(g.float().cpu().numpy(), 1, 1e-3, 0.9, 0.999, 1e-8, gs)
    check_same(opt, refs, params)


def test_zero_and_tiny_blocks(handle):
    sizes = [512, 300]
    params = [torch.ones((n,), device='cuda:0') for n in sizes]
    for bits in (32, 8):
        opt = AdamW(handle, params, weight_decay=0.0, state_bits=bits)
        before = [p.clone() for p in params]
        opt.step([torch.zeros((n,), device='cuda:0') for n in sizes])
        assert all(torch.equal(a, b) for a, b in zip(params, before))               # nothing moved, nothing was divided by zero
        opt.step([torch.full((n,), 1e-38, device='cuda:0') for n in sizes])
        for t in list(params) + list(opt.states()):
            assert torch.isfinite(t).all()


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_a_norm_that_is_not_finite_changes_nothing(handle, bits, bad):
    params = make([700, 300], torch.float32, 5)
    opt = AdamW(handle, params, state_bits=bits, max_norm=1.0)
    good = gradients([700, 300], torch.float32, 6)
    opt.step(good)
    keep = [t.clone() for t in params + [opt.m, opt.v]]
    g = [t.clone() for t in good]
    g[1][299] = bad
    opt.step(g)
    assert all(torch.equal(a, b) for a, b in zip(keep, params + [opt.m, opt.v])) and opt.step_count == 1
    assert not np.isfinite(float(opt.grad_norm))
    opt.step(good)
    assert opt.step_count == 2 and not torch.equal(keep[0], params[0])


@pytest.mark.parametrize('bits', [32, 8])
def test_without_clipping_a_nan_stays_where_it_is(handle, bits):
    params = make([1024], torch.float32, 7)
    opt = AdamW(handle, params, state_bits=bits)
    g = gradients([1024], torch.float32, 8)
    g[0][300] = float('nan')
    opt.step(g)
    m, v = opt.states()
    nan = torch.zeros(1024, dtype=torch.bool, device='cuda:0')
    nan[300] = True
    assert torch.equal(torch.isnan(params[0]), nan)
    if bits == 8:
        nan[256:512] = True                                                        # its block's moments
    assert torch.equal(torch.isnan(m), nan) and torch.equal(torch.isnan(v), nan)


@pytest.mark.parametrize('clip', [None, 0.3])
def test_more_tensors_than_one_launch_takes(handle, clip):
    sizes = [(i * 37) % 600 for i in range(1000)]
    params = make(sizes, torch.float32, 9, 1)
    opt = AdamW(handle, params, max_norm=clip)
    refs = [Ref(p.cpu().numpy(), torch.float32, 32, 0.01, False) for p in params]
    for t in (1, 2):
        grads = gradients(sizes, torch.float32, 20 + t)
        gs, _ = gscale_of(grads, 1.0, clip)
        opt.step(grads)
        for r, g in zip(refs, grads):
            r.step(g.cpu().numpy(), t, 1e-3, 0.9, 0.999, 1e-8, gs)
    check_same(opt, refs, params)
    assert opt.step_count == 2


@pytest.mark.parametrize('bits', [32, 8])
def test_captured_steps_count_and_equal_eager_ones(handle, bits):
    sizes = [5000, 77, 256]
    params, twin = make(sizes, torch.float32, 11), make(sizes, torch.float32, 11)
    grads = gradients(sizes, torch.float32, 12)
    opt = AdamW(handle, params, state_bits=bits, max_norm=0.7)
    eager = AdamW(handle, twin, state_bits=bits, max_norm=0.7)
    opt.bind(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(4):
        fresh = gradients(sizes, torch.float32, 30 + i)
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        eager.step(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params + [opt.m, opt.v], twin + [eager.m, eager.v])), 'replay %d' % i
        assert opt.step_count == i + 1


def test_on_another_stream_and_two_optimisers_at_once(handle):
    sizes = [100000, 333]
    a, b, want = (make(sizes, torch.float32, 13) for _ in range(3))
    grads = gradients(sizes, torch.float32, 14)
    ref = AdamW(handle, want, max_norm=1.0)
    for _ in range(5):
        ref.step(grads)
    oa, ob = AdamW(handle, a, max_norm=1.0), AdamW(handle, b, max_norm=1.0)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            oa.step(grads)
        with torch.cuda.stream(sb):
            ob.step(grads)
    torch.cuda.synchronize()
    for x in (a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, want))


def test_refusals(handle):
    p = torch.zeros((10,), device='cuda:0')
    g = torch.zeros((10,), device='cuda:0')
    with pytest.raises(_hip.ScsError, match='overlap'):
        AdamW(handle, [p, p])
    base = torch.zeros((20,), device='cuda:0')
    with pytest.raises(_hip.ScsError, match='overlap'):
        AdamW(handle, [base[:11], base[10:]])
    with pytest.raises(ValueError, match='contiguous'):
        AdamW(handle, [torch.zeros((4, 4), device='cuda:0').t()[1:]])
    opt = AdamW(handle, [p])
    for bad in ([], [g, g], [g[:9]], [g.double()], [g.cpu()], [torch.zeros((20,), device='cuda:0')[::2]]):
        with pytest.raises(ValueError):
            opt.step(bad)
    with pytest.raises(ValueError, match='bind'):
        opt.step()
    with pytest.raises(_hip.ScsError, match='betas'):
        opt.betas = (0.9, 1.0)
        opt.step([g])
    opt.betas = (0.9, 0.999)
    with pytest.raises(_hip.ScsError, match='finite'):
        opt.step([g], lr=float('nan'))
    with pytest.raises(ValueError):
        AdamW(handle, [p], states=(torch.zeros((10,), device='cuda:0'), torch.zeros((256,), device='cuda:0'), None, None))
    opt.step([g])
    p.data = torch.zeros((10,), device='cuda:0')
    with pytest.raises(RuntimeError, match='moved'):
        opt.step([g])
    opt.close()
    with pytest.raises(RuntimeError, match='closed'):
        opt.step([g])


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_in_the_optimisers_memory_are_refused(handle, bits):
    """A gradient that shares memory with a parameter, a master or a moment would be read while it is written."""
    flat = torch.zeros((4096,), dtype=torch.bfloat16, device='cuda:0')
    params = [flat[:1000], flat[2000:2600]]
    opt = AdamW(handle, params, state_bits=bits, master=True)
    free = [torch.zeros((1000,), device='cuda:0'), torch.zeros((600,), device='cuda:0')]
    opt.step([flat[1000:2000], flat[2600:3200]])                       # (beside them is fine)
    taken = [params[0], flat[1999:2999], opt.masters[0]]
    if bits == 32:
        taken.append(opt.m[24:1024])
    for t in taken:
        with pytest.raises(ValueError, match='shares memory'):
            opt.step([t, free[1]])
    opt.step(free)
    assert opt.step_count == 2


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('pt', ['bf16', 'f16'])
def test_a_resumed_run_with_masters_is_the_uninterrupted_one(handle, bits, pt):
    """Steps far below a 16-bit step of the parameters add up in the masters alone: everything an optimiser holds, through host copies, into another one."""
    kw = dict(lr=1e-5, weight_decay=0.01, state_bits=bits, max_norm=1.0)
    whole, part = make(SIZES, TYPES[pt], 61), make(SIZES, TYPES[pt], 61)
    start = [p.clone() for p in whole]
    one = AdamW(handle, whole, master=True, **kw)
    two = AdamW(handle, part, master=True, **kw)
    for t in range(3):
        g = gradients(SIZES, TYPES[pt], 70 + t)
        one.step(g)
        two.step(g)
    back = lambda t: None if t is None else t.cpu().clone().to('cuda:0')
    fresh = [back(p) for p in part]
    three = AdamW(handle, fresh, master=[back(t) for t in two.masters], states=[back(t) for t in (two.m, two.v, two.m_scale, two.v_scale)],
                  step=two.step_count, **kw)
    two.close()
    for t in range(3, 40):
        g = gradients(SIZES, TYPES[pt], 70 + t % 5)
        one.step(g)
        three.step(g)
    assert one.step_count == three.step_count == 40
    for a, b in zip(list(whole) + list(one.masters) + [one.m, one.v], list(fresh) + list(three.masters) + [three.m, three.v]):
        assert torch.equal(a, b)
    assert any(not torch.equal(a, b) for a, b in zip(start, whole))


@pytest.mark.parametrize('clip', [None, 1.0])
def test_steps_over_nothing_are_counted(handle, clip):
    """Tensors of no element are passed over; the step is one all the same."""
    opt = AdamW(handle, [torch.zeros((0,), device='cuda:0'), torch.zeros((4, 0), device='cuda:0')], max_norm=clip)
    grads = [torch.zeros((0,), device='cuda:0'), torch.zeros((4, 0), device='cuda:0')]
    opt.step(grads)
    opt.step(grads)
    assert opt.step_count == 2
    if clip:
        assert float(opt.grad_norm) == 0.0
    opt.step_count = 7
    opt.step(grads)
    assert opt.step_count == 8


@pytest.mark.parametrize('bits', [32, 8])
def test_states_by_tensor_and_their_memory(handle, bits):
    params = [p.view(s) for p, s in zip(make([35, 600, 0, 1], torch.float32, 81), ((5, 7), (600,), (0, 3), ()))]
    opt = AdamW(handle, params, state_bits=bits)
    grads = [torch.randn(p.shape, device='cuda:0') for p in params]
    opt.step(grads)
    m, v = opt.states()
    for i, (p, g) in enumerate(zip(params, grads)):
        mi, vi = opt.state_of(i)
        at = opt.first[i] * BLOCK
        assert mi.shape == vi.shape == p.shape
        assert torch.equal(mi.reshape(-1), m[at:at + p.numel()]) and torch.equal(vi.reshape(-1), v[at:at + p.numel()])
        assert ((mi != 0) | (g == 0)).all() or bits == 8
    assert opt.blocks == 1 + 3 + 0 + 1
    assert opt.bytes_per_element() == 5 * (BLOCK * 8 if bits == 32 else BLOCK * 2 + 8) / 636


@pytest.mark.parametrize('bits', [32, 8])
def test_a_moved_arena_or_master_is_refused(handle, bits):
    """Their old memory stays allocated, so that a graph that was captured before goes on with what it had."""
    params = make([1000, 300], torch.bfloat16, 82)
    opt = AdamW(handle, params, state_bits=bits, master=True, max_norm=1.0)
    g = gradients([1000, 300], torch.bfloat16, 83)
    opt.step(g)
    for t in [opt.masters[1], opt.m, opt.v, opt.grad_norm] + ([opt.m_scale, opt.v_scale] if bits == 8 else []):
        old = t.data
        t.data = t.clone()
        with pytest.raises(RuntimeError, match='moved'):
            opt.step(g)
        t.data = old
    opt.step(g)
    assert opt.step_count == 2
    with pytest.raises(_hip.ScsError, match='overlap'):
        both = torch.zeros((6 * BLOCK,), device='cuda:0')
        AdamW(handle, params, states=(both, both, None, None))
