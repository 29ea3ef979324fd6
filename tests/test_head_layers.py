"""The layernorm, dropout and classifier layer types of the .cfg grammar: what the parser makes of them, and what it refuses."""
import os

import numpy as np
import pytest

import ccn_loader

ccn_loader.load()
from cuda_convnet_amd import CFG_DIR, layer  # noqa: E402
from cuda_convnet_amd.convnet import PRESETS  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
CFG, PARAMS = (os.path.join(HERE, 'cfg', n) for n in ('head.cfg', 'head_params.cfg'))


def parse(path=CFG, seed=3):
    return layer.parse_layers(path, PARAMS, {0: 48, 1: 1}, 10, seed=seed)


def test_head_layers_parse():
    by = {l['name']: l for l in parse()}
    n, d, c = by['norm1'], by['drop1'], by['id']
    assert n['outputs'] == 40 and n['eps'] == 0.001 and n['weights'][0].shape == (40, 1) and np.all(n['weights'][0] == 1)
    assert n['biases'].shape == (40, 1) and not n['biases'].any() and n['gradConsumer'] and n['epsW'] == [0.01]
    assert n['actsTarget'] == -1 and n['actsGradTarget'] == -1  # matrices of its own
    assert d['dropout'] == 0.4 and d['seed'] == 77 and d['outputs'] == 40 and 'weights' not in d
    assert d['actsTarget'] == 0 and d['actsGradTarget'] == 0  # in place: neither its input nor its output is read again as such
    assert c['outputs'] == 10 and c['weights'][0].shape == (40, 10) and c['weights'][0].flags['F_CONTIGUOUS'] and c['biases'].shape == (1, 10)
    assert c['actsTarget'] == -1 and c['actsGradTarget'] == -1
    assert by['logprob']['inputs'] == [[l['name'] for l in parse()].index(x) for x in ('labels', 'id')]


def test_dropout_seed_is_drawn_where_none_is_given(tmp_path):
    p = tmp_path / 'a.cfg'
    p.write_text(open(CFG).read().replace('seed=77\n', ''))
    seeds = [next(l['seed'] for l in parse(str(p), s) if l['name'] == 'drop1') for s in (3, 3, 4)]
    assert seeds[0] == seeds[1] != seeds[2] and 0 <= min(seeds)


def test_dropout_key_of_other_layers_stays_without_effect(tmp_path):
    """The DeepID definitions carry dropout=0.4 on fc5, which no parser of the reference reads."""
    p = tmp_path / 'a.cfg'
    p.write_text(open(CFG).read().replace('neuron=relu', 'neuron=relu\ndropout=0.4'))
    assert [(l['name'], l['type']) for l in parse(str(p))] == [(l['name'], l['type']) for l in parse()]


def test_dropout_layers_differ_in_their_seed(tmp_path):
    """The mask follows from (seed, step, element) alone: the same seed twice would drop the same elements in both layers."""
    src = open(CFG).read().replace('inputs=drop1', 'inputs=drop2').replace('[id]', '[drop2]\ntype=dropout\ninputs=drop1\ndropout=0.2\nseed=%d\n\n[id]')
    p = tmp_path / 'a.cfg'
    p.write_text(src % 77)
    with pytest.raises(layer.LayerParsingError, match="'drop2': seed 77 is layer 'drop1's"):
        parse(str(p))
    p.write_text(src % 78)
    assert [l['seed'] for l in parse(str(p)) if l['type'] == 'dropout'] == [77, 78]
    p.write_text(src % (1 << 63))
    with pytest.raises(layer.LayerParsingError, match='below 2'):
        parse(str(p))


@pytest.mark.parametrize('edit,msg', [
    (('dropout=0.4', 'dropout=1.0'), 'must be in'),
    (('dropout=0.4', 'dropout=-0.1'), 'must be in'),
    (('dropout=0.4\n', ''), 'dropout'),
    (('eps=0.001', 'eps=0'), 'must be positive'),
    (('eps=0.001', 'weightSource=fc1'), 'type'),
    (('outputs=10\n', 'outputs=0\n'), 'out of range'),
    (('outputs=10\n', 'outputs=11\n'), 'number of classes'),
    (('outputs=10\ninputs=drop1', 'outputs=10\nneuron=relu\ninputs=drop1'), 'no neuron'),
    (('inputs=drop1', 'inputs=drop1,fc1'), 'number of inputs'),
    (('inputs=labels,id', 'inputs=labels,drop1'), 'softmax'),
    (('[logprob]', '[more]\ntype=fc\noutputs=3\ninputs=id\ninitW=0.1\n\n[logprob]'), 'feeds one cost.logreg'),
])
def test_head_parser_errors(tmp_path, edit, msg):
    src = open(CFG).read()
    assert edit[0] in src
    p = tmp_path / 'bad.cfg'
    p.write_text(src.replace(edit[0], edit[1], 1))
    with pytest.raises(layer.LayerParsingError, match=msg):
        parse(str(p))


def test_head_preset_parses():
    ldef, lpar, _, _ = PRESETS['deepid-head']
    L = layer.parse_layers(os.path.join(CFG_DIR, ldef), os.path.join(CFG_DIR, lpar), {0: 9075, 1: 1}, 4213)
    assert [l['type'] for l in L[-4:]] == ['layernorm', 'dropout', 'classifier', 'cost.logreg'] and L[-2]['outputs'] == 4213
