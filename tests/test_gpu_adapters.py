"""Site adapters of the dense head through Net (fit_adapters, predict with sites) and fit with AdamW: the operators as a user has them.
Needs an MI355X."""
import numpy as np
import pytest
import torch

from cnn_cort import params as P
from cnn_cort.adapters import SiteAdapters, group_rows
from cnn_cort.nets import Net
from cnn_cort.optim import AdamW
from conftest import gold

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def batch():
    g = gold('g2_volume.npz')
    n = 256
    X = {'in1': g['ax'][:n], 'in2': g['co'][:n], 'in3': g['sa'][:n], 'in4': g['atlas'][:n]}
    n = X['in1'].shape[0]
    rng = np.random.default_rng(0)
    return X, rng.integers(0, 15, n), rng.integers(-1, 3, n)


def make_net(weights, **kw):
    net = Net(device=0, **kw)
    net.load_params_from(weights)
    return net


def test_features_are_the_dense_heads_input(handle, weights, batch):
    X = batch[0]
    net = make_net(weights)
    n = X['in1'].shape[0]
    f = net.features(X).cpu().numpy()
    h = net._ensure_handle()
    h.set_option('fwd_split', 0)
    dev = [torch.from_numpy(np.ascontiguousarray(X[k])).cuda() for k in ('in1', 'in2', 'in3', 'in4')]
    h.forward(*dev, n, torch.empty((n, 15), device='cuda:0'), None, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(f, h.get_activation(4, n * 540).reshape(n, 540))


def test_untrained_adapters_predict_what_the_net_predicts(weights, batch):
    X, _, sites = batch
    net = make_net(weights)
    h = net._ensure_handle()
    h.set_option('fwd_split', 0)
    net.adapters = SiteAdapters(h, net.get_all_params_values(), 3, rank=4)
    base = net.predict_proba(X)
    for s in (sites, 0, -1):
        assert np.abs(net.predict_proba(X, sites=s) - base).max() < 1e-4           # (the same sums in another order)
    # a site's adapter moves its own samples alone
    net.adapters.tensors[5][1].normal_()
    moved = np.abs(net.predict_proba(X, sites=sites) - base).max(1) > 1e-4
    assert moved[sites == 1].any() and not moved[sites != 1].any()


def test_gradients_of_the_adapted_head(weights, batch):
    """Against autograd in float64, and against differences of the float64 loss."""
    X, y, sites = batch
    net = make_net(weights)
    h = net._ensure_handle()
    params = net.get_all_params_values()
    ad = SiteAdapters(h, params, 3, rank=5, scale=0.5, seed=1)
    gen = torch.Generator().manual_seed(2)
    for t in ad.tensors:
        t.copy_(torch.randn(t.shape, generator=gen) * 0.05)
    order, offsets, ids = group_rows(sites)
    feat = net.features(X)[torch.from_numpy(order).cuda()].contiguous()
    atlas = net._atlas_rows(X)[torch.from_numpy(order).cuda()].contiguous()
    labels = torch.from_numpy(y[order]).cuda()
    loss, grads = ad.loss_and_gradients(feat, atlas, labels, torch.from_numpy(offsets).cuda(), torch.from_numpy(ids).cuda())

    site = torch.from_numpy(sites[order])
    W = [[torch.from_numpy(np.asarray(a, np.float64)) for a in params[n]] for n in SiteAdapters.LAYERS]
    leaves = [t.double().cpu().requires_grad_() for t in ad.tensors]

    def head(leaves):
        x = feat.double().cpu()
        for l in range(3):
            w, b = W[l]
            low = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64)
            for s in range(3):
                m = (site == s).double()[:, None]
                low = low + 0.5 * m * ((x * m) @ leaves[2 * l][s].t() @ leaves[2 * l + 1][s])
            x = x @ w + b + low
            if l < 2:
                x = torch.relu(x)
            if l == 0:
                x = torch.cat([x, atlas.double().cpu()], 1)
        return torch.nn.functional.cross_entropy(x, labels.cpu())

    ref = head(leaves)
    ref.backward()
    assert abs(float(loss) - float(ref)) <= 1e-5 * max(1.0, abs(float(ref)))
    for name, g, leaf in zip(ad.names, grads, leaves):
        want = leaf.grad.numpy()
        err = np.abs(g.cpu().numpy() - want).max()
        # three layers of at most 555 float32 products: 3 x 555 x 2^-24 = 1e-4 of the largest entry, and rectifiers at zero that may flip
        assert err <= 1e-4 * np.abs(want).max(), '%s: %g of %g' % (name, err, np.abs(want).max())
    with torch.no_grad():
        for k in (1, 5):
            at = np.unravel_index(np.argmax(np.abs(leaves[k].grad.numpy())), leaves[k].shape)
            step, values = 1e-5, []
            for sign in (1, -1):
                moved = [t.clone() for t in leaves]
                moved[k][at] += sign * step
                values.append(float(head(moved)))
            diff = (values[0] - values[1]) / (2 * step)
            assert abs(diff - float(grads[k][at])) <= 1e-3 * abs(diff)


def test_fit_adapters_save_and_load(weights, batch, tmp_path):
    X, y, sites = batch
    net = make_net(weights, batch_size=64, patience=3, eval_size=0.25, optimizer_bits=8, max_norm=1.0)
    before = net.get_all_params_values()
    base = net.predict_proba(X)
    history = net.fit_adapters(X, y, sites, rank=4, epochs=3, learning_rate=1e-2)
    assert [h['epoch'] for h in history] == [1, 2, 3] and all(np.isfinite(list(h.values())).all() for h in history)
    after = net.get_all_params_values()
    assert all(np.array_equal(a, b) for k in before for a, b in zip(before[k], after[k]))       # the shared weights stay
    adapted = net.predict_proba(X, sites=sites)
    assert np.abs(adapted - base)[sites >= 0].max() > 1e-4
    assert np.abs(net.predict_proba(X, sites=-1) - base).max() < 1e-4
    assert np.array_equal(net.predict(X, sites=sites), adapted.argmax(1))
    path = net.save_adapters_to(str(tmp_path / 'sites.npz'))
    other = make_net(weights)
    other.load_adapters_from(path)
    assert np.array_equal(other.predict_proba(X, sites=sites), adapted)
    with pytest.raises(ValueError):
        net.predict(X, sites=3)
    with pytest.raises(ValueError):
        net.predict(X, sites=sites[:-1])
    with pytest.raises(RuntimeError):
        make_net(weights).predict(X, sites=0)


def test_a_training_step_in_a_graph(weights, batch):
    """Forward, loss, gradients and the optimiser's step captured together, replayed with eager steps beside them."""
    X, y, sites = batch
    net = make_net(weights)
    h = net._ensure_handle()
    order, offsets, ids = group_rows(sites)
    o, i = torch.from_numpy(offsets).cuda(), torch.from_numpy(ids).cuda()
    feat, atlas = net.features(X), net._atlas_rows(X)
    labels = torch.from_numpy(y).cuda()
    both = []
    for _ in range(2):
        ad = SiteAdapters(h, net.get_all_params_values(), 3, rank=4)
        opt = AdamW(h, ad.tensors, lr=1e-2, state_bits=8, max_norm=1.0)
        grads = [torch.empty_like(t) for t in ad.tensors]
        both.append((ad, opt.bind(grads), grads))
    args = (feat[torch.from_numpy(order).cuda()].contiguous(), atlas[torch.from_numpy(order).cuda()].contiguous(), labels[torch.from_numpy(order).cuda()].contiguous(), o, i)
    ad, opt, grads = both[0]
    ad.loss_and_gradients(*args, grads)                        # (warms up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = ad.loss_and_gradients(*args, grads)
        opt.step()
    for k in range(4):
        graph.replay()
        l2, _ = both[1][0].loss_and_gradients(*args, both[1][2])
        both[1][1].step()
        torch.cuda.synchronize()
        assert torch.equal(loss, l2), 'replay %d' % k
        assert all(torch.equal(a, b) for a, b in zip(ad.tensors, both[1][0].tensors)), 'replay %d' % k
    assert opt.step_count == 4


@pytest.mark.parametrize('bits,clip', [(32, None), (8, 1.0)])
def test_fit_with_adamw_is_the_two_calls(weights, bits, clip):
    """Net(optimizer='adamw').fit takes the steps that train_step and AdamW.step take by hand; running statistics and vectors do not decay."""
    t = gold('g5_train.npz')
    X = {'in1': t['ax'], 'in2': t['co'], 'in3': t['sa'], 'in4': t['atlas']}
    n = X['in1'].shape[0]
    kw = dict(batch_size=n, eval_size=0.0, optimizer='adamw', optimizer_bits=bits, max_norm=clip, weight_decay=0.1, update_learning_rate=1e-3, seed=3)
    net = make_net(weights, **kw)
    net.fit(X, t['y'], epochs=3)
    got = net.get_all_params_values()
    assert all(np.isfinite(a).all() for v in got.values() for a in v)

    twin = make_net(weights, **kw)
    h = twin._ensure_handle()
    opt = twin._adamw(h)
    dev = [torch.from_numpy(np.ascontiguousarray(X[k])).cuda() for k in ('in1', 'in2', 'in3', 'in4')]
    y = torch.from_numpy(t['y'].astype(np.uint8)).cuda()
    for step in range(1, 4):
        h.train_step(*dev, y, n, seed=(3 << 32) + step * 131, want_loss=False, stream=torch.cuda.current_stream().cuda_stream)
        opt.step()
    torch.cuda.synchronize()
    want = P.flat_to_params(h.get_params())
    for k in want:
        for a, b in zip(got[k], want[k]):
            assert np.array_equal(a, b), k
    assert opt.step_count == 3 and len(opt.params) == sum(P.is_trainable(k, i) for k, s in P.LAYER_SPEC for i in range(len(s)))
    moved = [np.abs(a - b).max() for k in want for a, b in zip(got[k], weights[k])]
    assert max(moved) > 0
    # after fit the forward pass sees the trained weights
    assert np.isfinite(net.predict_proba(X)).all()


def test_optimizer_options():
    with pytest.raises(ValueError, match='optimizer'):
        Net(optimizer='sgd')


def test_new_weights_reach_the_adapted_head(weights, batch):
    """load_params_from and fit change the shared weights: predict with sites takes the new ones."""
    X, y, sites = batch
    net = make_net(weights)
    h = net._ensure_handle()
    h.set_option('fwd_split', 0)
    net.adapters = SiteAdapters(h, net.get_all_params_values(), 3, rank=4)
    other = {k: [a * np.float32(0.5) for a in v] if k in SiteAdapters.LAYERS else v for k, v in net.get_all_params_values().items()}
    net.load_params_from(other)
    net._ensure_handle().set_option('fwd_split', 0)
    base = net.predict_proba(X)
    assert np.abs(net.predict_proba(X, sites=-1) - base).max() < 1e-4
    net.max_epochs, net.eval_size, net.batch_size = 1, 0.0, 64
    net.fit(X, y)
    fitted = net.predict_proba(X)
    assert np.abs(fitted - base).max() > 1e-3
    assert np.abs(net.predict_proba(X, sites=sites) - fitted).max() < 1e-4


@pytest.mark.parametrize('bits,clip', [(32, None), (8, 1.0)])
def test_a_second_fit_goes_on_with_adamw(weights, bits, clip):
    """fit(epochs=1) three times is fit(epochs=3): moments and step count go on until weights are loaded, as Adam's do."""
    t = gold('g5_train.npz')
    X = {'in1': t['ax'], 'in2': t['co'], 'in3': t['sa'], 'in4': t['atlas']}
    kw = dict(batch_size=X['in1'].shape[0], eval_size=0.0, optimizer='adamw', optimizer_bits=bits, max_norm=clip, weight_decay=0.1, update_learning_rate=1e-3, seed=3)
    same = lambda a, b: all(np.array_equal(x, y) for k in a for x, y in zip(a[k], b[k]))
    whole, parts = make_net(weights, **kw), make_net(weights, **kw)
    whole.fit(X, t['y'], epochs=3)
    once = None
    for i in range(3):
        parts.fit(X, t['y'], epochs=1)
        once = once or parts.get_all_params_values()
    assert same(whole.get_all_params_values(), parts.get_all_params_values())
    # another rate or decay between the calls applies to the steps behind it; moments of other bits start anew
    assert parts._optimiser.step_count == 3
    parts.weight_decay, parts.optimizer_bits = 0.0, 40 - bits
    parts.fit(X, t['y'], epochs=1)
    assert parts._optimiser.step_count == 1 and parts._optimiser.state_bits == 40 - bits
    # new weights: the optimiser starts anew with them
    whole.load_params_from(weights)
    whole._step = 0
    whole.fit(X, t['y'], epochs=1)
    assert same(whole.get_all_params_values(), once)
