"""The layernorm, dropout and classifier layers through the `_ConvNet` boundary: one training step against a float64 formula of the
whole net, the classifier against the fc + softmax layers it stands for, gradient checks, streams, step graphs and refusals.

Tolerances: gradients of one step as in test_net_layers_gpu.py (1e-4 of a matrix's largest entry), three steps as in
test_net_gpu.py (costs 2e-4, increments 2e-3)."""
import copy
import os

import numpy as np
import pytest

import ccn_loader

ccn_loader.load()
from test_head_gpu import kept, norm_ref, undo_ref  # noqa: E402
from test_net_gpu import Native, build, check_costs, check_weights, preset  # noqa: E402

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
CFG, PARAMS = (os.path.join(HERE, 'cfg', n) for n in ('head.cfg', 'head_params.cfg'))


def net(cases, path=CFG, params=PARAMS, minibatch=32):
    return build(path, params, 'dummy', (4, 4, 3), cases, minibatch=minibatch, num_classes=10)


def randomise(L):
    rng = np.random.default_rng(8)
    for l in L:
        if l['name'] == 'norm1':
            l['weights'][0][:] = 1 + 0.3 * rng.standard_normal(l['weights'][0].shape)
            l['biases'][:] = 0.3 * rng.standard_normal(l['biases'].shape)


def run(L, data, env=None, minibatch=32, batches=1, dp=False):
    old = {k: os.environ.get(k) for k in env or {}}
    os.environ.update(env or {})
    try:
        with Native(L, minibatch) as lib:
            if dp:
                lib.initDataParallel(0, 1, lib.commUniqueId(), 1)
            for _ in range(batches):
                lib.startBatch(data, 0)
                got = lib.finishBatch()
            lib.syncWithHost()
    finally:
        for k, v in old.items():
            os.environ.pop(k, None) if v is None else os.environ.__setitem__(k, v)
    return got


@pytest.mark.parametrize('cases', [32, 7])
def test_one_step_matches_the_formula(cases):
    dp, L = net(cases)
    randomise(L)
    data = dp.get_next_batch()[2]
    want = copy.deepcopy(L)
    by = {l['name']: l for l in want}
    x, labels = data[0].astype(np.float64), data[1].ravel().astype(int)
    fc, norm, cls = by['fc1'], by['norm1'], by['id']
    w1, b1 = fc['weights'][0].astype(np.float64), fc['biases'].astype(np.float64).reshape(-1, 1)
    gain, shift = norm['weights'][0].astype(np.float64).ravel(), norm['biases'].astype(np.float64).ravel()
    w2, b2 = cls['weights'][0].astype(np.float64), cls['biases'].astype(np.float64).reshape(-1, 1)
    h = np.maximum(w1.T @ x + b1, 0)
    mean, var = h.mean(0), h.var(0)
    r = 1 / np.sqrt(var + norm['eps'])
    y = gain[:, None] * (h - mean) * r + shift[:, None]
    scale = kept(40 * cases, 0.4, 77, 1).reshape(40, cases) / (1 - float(np.float32(0.4)))
    d = y * scale
    z = w2.T @ d + b2
    p = np.exp(z - z.max(0)) / np.exp(z - z.max(0)).sum(0)
    logp = np.log(p[labels, np.arange(cases)])
    dz = -p
    dz[labels, np.arange(cases)] += 1
    dd = (w2 @ dz) * scale
    dh, dgain, dshift = undo_ref(dd, h, gain, mean, r)
    dh = dh * (h > 0)
    grads = {'fc1': (x @ dh.T, dh.sum(1)), 'norm1': (dgain[:, None], dshift), 'id': (d @ dz.T, dz.sum(1))}
    cost, n = run(L, data)
    assert n == cases
    assert cost['logprob'][0] == pytest.approx(-logp.sum(), rel=1e-4)
    assert cost['logprob'][1] == (z.argmax(0) != labels).sum()
    for l in L:
        if 'weights' in l:
            gw, gb = grads[l['name']]
            before = by[l['name']]
            iw = l['epsW'][0] / cases * gw - l['wc'][0] * l['epsW'][0] * before['weights'][0]
            for got, exp in ((l['weightsInc'][0], iw), (l['biasesInc'].ravel(), l['epsB'] / cases * gb)):
                assert np.abs(got - exp).max() <= 1e-4 * np.abs(exp).max() + 1e-9, l['name']
            assert np.array_equal(l['weights'][0], before['weights'][0] + l['weightsInc'][0])


def fc_softmax_cfg(tmp_path, src=CFG, params=PARAMS):
    """The same net with the classifier written as the layers it stands for."""
    s = open(src).read()
    a, b = s.index('[id]') if '[id]' in s else s.index('[identity]'), s.index('[logprob]')
    name = s[a + 1:s.index(']', a)]
    s = s[:a] + s[a:b].replace('type=classifier', 'type=fc') + '[probs]\ntype=softmax\ninputs=%s\n\n' % name + s[b:].replace('labels,' + name, 'labels,probs')
    p = tmp_path / 'fc.cfg'
    p.write_text(s)
    return str(p)


@pytest.mark.parametrize('env', [{}, {'MCN_NO_GRAD_STREAM': '1'}, {'MCN_NO_FUSION': '1'}])
def test_classifier_is_fc_and_softmax(tmp_path, env):
    """Three minibatches, the last one short; masks are the same (same seed), so costs, error counts and weights agree."""
    dp, La = net(80)
    _, Lb = net(80, fc_softmax_cfg(tmp_path))
    data = dp.get_next_batch()[2]
    a, b = run(La, data, env), run(Lb, data, env)
    check_costs(a, b)
    check_weights(La, [l for l in Lb if l['type'] != 'softmax'])


def test_head_preset_is_fc_and_softmax(tmp_path):
    from cuda_convnet_amd import CFG_DIR
    dp, La = preset('deepid-head', 256)
    _, Lb = build(fc_softmax_cfg(tmp_path, os.path.join(CFG_DIR, 'deepid_4213_head.cfg')), os.path.join(CFG_DIR, 'deepid_head_params.cfg'), 'deepid',
                  (55, 55, 3), 256)
    data = dp.get_next_batch()[2]
    a, b = run(La, data, minibatch=128), run(Lb, data, minibatch=128)
    check_costs(a, b)
    check_weights(La, [l for l in Lb if l['type'] != 'softmax'])


def test_streams_and_step_graphs_give_the_same_bits():
    """Two streams or one, eager or replayed graphs (whose masks come from the step in device memory): bit-identical weights."""
    results = []
    for env in ({}, {'MCN_NO_GRAD_STREAM': '1'}, {'MCN_STEP_GRAPH': '1'}):
        dp, L = net(96)
        data = dp.get_next_batch()[2]
        old = {k: os.environ.get(k) for k in env}
        os.environ.update(env)
        try:
            with Native(L, 32) as lib:
                lib.loadBatch(data)
                lib.startSteps(9, 0, 0)
                cost = lib.finishBatch()
                lib.syncWithHost()
        finally:
            for k, v in old.items():
                os.environ.pop(k, None) if v is None else os.environ.__setitem__(k, v)
        results.append((L, cost))
    for L, cost in results[1:]:
        assert cost == results[0][1]
        for a, b in zip(results[0][0], L):
            if 'weights' in a:
                assert np.array_equal(a['weights'][0], b['weights'][0]) and np.array_equal(a['biases'], b['biases']), a['name']


def test_forced_data_parallel_step_is_the_plain_step():
    dp, La = net(96)
    Lb = copy.deepcopy(La)
    data = dp.get_next_batch()[2]
    a, b = run(La, data), run(Lb, data, dp=True)
    check_costs(a, b)
    check_weights(La, Lb)


def test_masks_change_from_step_to_step_and_test_passes_have_none():
    dp, L = net(32)
    idx = {l['name']: i for i, l in enumerate(L)}
    data = dp.get_next_batch()[2]
    for l in L:
        for k in ('epsW', 'wc'):
            if k in l:
                l[k] = [0.0]
        if 'epsB' in l:
            l['epsB'] = 0.0
    with Native(L, 32) as lib:
        costs = []
        for _ in range(3):
            lib.startBatch(data, 0)
            costs.append(lib.finishBatch()[0]['logprob'][0])
        assert len(set(costs)) == 3  # (nothing was learned: only the masks differ)
        lib.startBatch(data, 1)
        test = lib.finishBatch()[0]['logprob'][0]
        lib.startBatch(data, 1)
        assert lib.finishBatch()[0]['logprob'][0] == test
        out = {}
        for name in ('norm1', 'drop1'):
            ftrs = np.full((32, 40), np.nan, np.float32)
            lib.startFeatureWriter(list(data) + [ftrs], idx[name])
            lib.finishBatch()
            out[name] = ftrs
        assert np.array_equal(out['norm1'], out['drop1']) and np.isfinite(out['norm1']).all()


def test_a_resumed_run_goes_on_with_the_masks():
    """Four minibatches at once, or two, a checkpoint's layers, and two: the same bits."""
    dp, L = net(32)
    randomise(L)
    data = dp.get_next_batch()[2]

    def train(layers, batches):
        with Native(layers, 32) as lib:
            for _ in range(batches):
                lib.startBatch(data, 0)
                lib.finishBatch()
            lib.syncWithHost()

    whole, parts = copy.deepcopy(L), copy.deepcopy(L)
    train(whole, 4)
    train(parts, 2)
    drop = [l for l in parts if l['type'] == 'dropout'][0]
    assert drop['steps'].tolist() == [[2, 0, 0]]
    drop['steps'][:] = 1048575, 7, 1  # (digits carry)
    train(parts, 0)
    assert drop['steps'].tolist() == [[1048575, 7, 1]]
    more = copy.deepcopy(parts)
    train(more, 1)
    assert [l['steps'].tolist() for l in more if l['type'] == 'dropout'] == [[[0, 8, 1]]]
    drop['steps'][:] = 2, 0, 0
    parts = copy.deepcopy(parts)
    train(parts, 2)
    for a, b in zip(whole, parts):
        for k in ('weights', 'weightsInc'):
            for p, q in zip(a.get(k, []), b.get(k, [])):
                assert np.array_equal(p, q), (a['name'], k)
        for k in ('biases', 'biasesInc', 'steps'):
            if k in a:
                assert np.array_equal(a[k], b[k]), (a['name'], k)


def cost64(q, x, labels, scale, eps):
    """-sum(log p[label]) of the net, float64; q: the six weight and bias matrices."""
    h = np.maximum(q[0].T @ x + q[1], 0)
    d = (q[2] * (h - h.mean(0)) / np.sqrt(h.var(0) + eps) + q[3]) * scale
    z = q[4].T @ d + q[5]
    top = z.max(0)
    return (top + np.log(np.exp(z - top).sum(0)) - z[labels, np.arange(z.shape[1])]).sum()


def test_gradient_check_reports_what_its_steps_allow():
    """The net's own gradient check (every element, central differences, the reference's steps: 0.1 and 0.01 for fully connected
    matrices, 0.001 and 0.002 else).  Steps that large are far off the derivative here -- the relative error that the check reports is
    that of the same differences of the float64 formula, whose gradient is a difference with a step of 1e-6.  What the float32 cost
    adds: 32 log probabilities of at most 6 with errors of some 16 u each, 3e-5 in all, over 2 x 32 x step per element."""
    dp, L = net(32)
    randomise(L)
    data = dp.get_next_batch()[2]
    x, labels = data[0].astype(np.float64), data[1].ravel().astype(int)
    by = {l['name']: l for l in L}
    col = lambda a: a.astype(np.float64).reshape(-1, 1)  # noqa: E731
    q = [by['fc1']['weights'][0].astype(np.float64), col(by['fc1']['biases']), col(by['norm1']['weights'][0]), col(by['norm1']['biases']),
         by['id']['weights'][0].astype(np.float64), col(by['id']['biases'])]
    scale = kept(40 * 32, 0.4, 77, 0).reshape(40, 32) / (1 - float(np.float32(0.4)))  # (no training step yet: the mask of step 0)
    with Native(L, 32) as lib:
        res = lib.checkGradients(data, 0, 1)
    assert [r[0].split()[0] for r in res] == ['fc1', 'fc1', 'norm1', 'norm1', 'id', 'id']
    for k, (step, r) in enumerate(zip((0.1, 0.01, 0.001, 0.002, 0.1, 0.01), res)):
        num, grad = np.zeros_like(q[k]), np.zeros_like(q[k])
        for out, h in ((num, step), (grad, 1e-6)):
            for i in np.ndindex(*q[k].shape):
                keep = q[k][i]
                q[k][i] = keep + h
                up = cost64(q, x, labels, scale, 0.001)
                q[k][i] = keep - h
                out[i] = (up - cost64(q, x, labels, scale, 0.001)) / (2 * 32 * h)
                q[k][i] = keep
        want = np.linalg.norm(num - grad) / np.linalg.norm(grad)
        noise = 3e-5 / (2 * 32 * step) / (np.linalg.norm(grad) / np.sqrt(grad.size))
        assert abs(r[1] - np.linalg.norm(grad)) <= 1e-3 * np.linalg.norm(grad), r
        assert abs(r[3] - want) <= 0.01 + noise, (r, want, noise)


def test_norm_with_a_neuron_in_a_residual_sum(tmp_path):
    """fc1 + dropout(relu(norm(fc1))): every layer's gradient arrives added onto another's; norms of the gradients against differences of
    the float64 formula (steps of 1e-6; a kink that lies within them is met by a negligible share of the entries)."""
    text = open(CFG).read().replace('eps=0.001', 'eps=0.001\nneuron=relu').replace('[id]', '[sum]\ntype=eltsum\ninputs=drop1,fc1\ncoeffs=1,1\n\n[id]')
    text = text.replace('type=classifier\noutputs=10\ninputs=drop1', 'type=classifier\noutputs=10\ninputs=sum')
    path = tmp_path / 'sum.cfg'
    path.write_text(text)
    dp, L = net(32, str(path))
    randomise(L)
    data = dp.get_next_batch()[2]
    x, labels = data[0].astype(np.float64), data[1].ravel().astype(int)
    by = {l['name']: l for l in L}
    col = lambda a: a.astype(np.float64).reshape(-1, 1)  # noqa: E731
    q = [by['fc1']['weights'][0].astype(np.float64), col(by['fc1']['biases']), col(by['norm1']['weights'][0]), col(by['norm1']['biases']),
         by['id']['weights'][0].astype(np.float64), col(by['id']['biases'])]
    scale = kept(40 * 32, 0.4, 77, 0).reshape(40, 32) / (1 - float(np.float32(0.4)))

    def cost():
        h = np.maximum(q[0].T @ x + q[1], 0)
        d = np.maximum(q[2] * (h - h.mean(0)) / np.sqrt(h.var(0) + 0.001) + q[3], 0) * scale + h
        z = q[4].T @ d + q[5]
        top = z.max(0)
        return (top + np.log(np.exp(z - top).sum(0)) - z[labels, np.arange(32)]).sum()

    with Native(L, 32) as lib:
        res = lib.checkGradients(data, 0, 1)
    assert [r[0].split()[0] for r in res] == ['fc1', 'fc1', 'norm1', 'norm1', 'id', 'id']
    for k, r in enumerate(res):
        grad, h = np.zeros_like(q[k]), 1e-6
        for i in np.ndindex(*q[k].shape):
            keep = q[k][i]
            q[k][i] = keep + h
            up = cost()
            q[k][i] = keep - h
            grad[i] = (up - cost()) / (2 * 32 * h)
            q[k][i] = keep
        assert abs(r[1] - np.linalg.norm(grad)) <= 1e-3 * np.linalg.norm(grad), r


def test_classifier_refusals():
    dp, L = net(32)
    idx = {l['name']: i for i, l in enumerate(L)}
    data = dp.get_next_batch()[2]
    with Native(L, 32) as lib:
        with pytest.raises(RuntimeError, match='keeps no outputs'):
            lib.startFeatureWriter(list(data) + [np.zeros((32, 10), np.float32)], idx['id'])
            lib.finishBatch()
        with pytest.raises(RuntimeError, match='keeps no probabilities'):
            lib.startMultiviewTest(data, 2, idx['logprob'])
            lib.finishBatch()
        lib.startBatch(data, 0)  # the model goes on
        assert lib.finishBatch()[1] == 32
    bad = copy.deepcopy(L)
    bad[idx['logprob']]['inputs'] = [idx['labels'], idx['labels']]
    with pytest.raises(RuntimeError, match='classifier layer'):
        with Native(bad, 32):
            pass


def test_dropout_layers_with_one_seed_are_refused(tmp_path):
    src = open(CFG).read().replace('inputs=drop1', 'inputs=drop2').replace('[id]', '[drop2]\ntype=dropout\ninputs=drop1\ndropout=0.2\nseed=78\n\n[id]')
    p = tmp_path / 'a.cfg'
    p.write_text(src)
    _, L = net(32, str(p))
    with Native(copy.deepcopy(L), 32):
        pass
    [l for l in L if l['name'] == 'drop2'][0]['seed'] = 77
    with pytest.raises(RuntimeError, match="its seed is layer 'drop1's"):
        with Native(L, 32):
            pass


@pytest.mark.parametrize('env', [{}, {'MCN_NO_GRAD_STREAM': '1'}, {'MCN_NO_FUSION': '1'}, 'data parallel'])
def test_classifier_beside_a_verification_cost(tmp_path, env):
    """DeepID2's own net with its fc6 and softmax as a classifier layer: the features get the identification's and the verification's
    gradients, the latter from another stream.  Three minibatches against the layers it stands for."""
    from cuda_convnet_amd import CFG_DIR
    text = open(os.path.join(CFG_DIR, 'deepid2_10575.cfg')).read()
    a, b = text.index('[fc6]'), text.index('[logprob]')
    text = text[:a] + '[fc6]\ntype=classifier\noutputs=10575\ninputs=fc5\ninitW=0.01\n\n' + text[b:].replace('labels,probs', 'labels,fc6')
    p = tmp_path / 'joint.cfg'
    p.write_text(text)
    dp, La = build(str(p), os.path.join(CFG_DIR, 'deepid_params.cfg'), 'deepid2', (55, 55, 3), 384)
    _, Lb = preset('deepid2', 384)
    data = dp.get_next_batch()[2]
    forced = env == 'data parallel'
    a, b = (run(L, data, {} if forced else env, minibatch=128, dp=forced) for L in (La, Lb))
    check_costs(a, b)
    check_weights(La, [l for l in Lb if l['type'] != 'softmax'])
