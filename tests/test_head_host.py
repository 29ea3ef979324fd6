"""What the layer norm, dropout and classifier-cost entry points refuse, on the CPU: every call below ends at the host's checks.

The pointers are numbers that nothing may look at; a call that got past the checks would fail at the launch (no GPU) with another code."""
import ctypes as C
import glob
import math
import os
import re

import pytest

import ccn_loader

ccn_loader.load()
from cuda_convnet_amd import capi  # noqa: E402

EINVAL, EWORKSPACE = -1, -3
P = [(i + 1) << 32 for i in range(10)]
BIG = 1 << 40


def rc(name, *args):
    L = capi.lib()
    fn = L.raw(name)
    return fn(*args), L.dll.mcn_last_error().decode()


def norm(**k):
    a = dict(x=P[0], gain=P[1], bias=P[2], y=P[3], stats=P[4], f=8, n=4, eps=1e-5, ws=P[5], size=BIG)
    a.update(k)
    return rc('mcn_layer_norm', a['x'], a['gain'], a['bias'], a['y'], a['stats'], a['f'], a['n'], a['eps'], a['ws'], a['size'], None)


@pytest.mark.parametrize('k', [dict(x=None), dict(y=None), dict(f=0), dict(n=0), dict(f=-3), dict(n=-1), dict(f=(1 << 26) + 1), dict(n=(1 << 26) + 1), dict(y=P[0] + 4),
                               dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan), dict(ws=P[5] + 4)])
def test_layer_norm_refuses(k):
    code, msg = norm(**k)
    assert code == EINVAL and 'layerNorm' in msg


def test_layer_norm_workspace():
    need = capi.lib().raw('mcn_layer_norm_workspace_bytes')(9075, 128)
    for k in (dict(size=need - 1), dict(ws=None), dict(size=0)):
        code, msg = norm(f=9075, n=128, **k)
        assert code == EWORKSPACE and 'workspace' in msg
    assert capi.lib().raw('mcn_layer_norm_workspace_bytes')(0, 4) == 0


def undo(**k):
    a = dict(g=P[0], x=P[1], gain=P[2], stats=P[3], dx=P[4], dg=P[5], db=P[6], f=8, n=4, ws=P[7], size=BIG)
    a.update(k)
    return rc('mcn_layer_norm_undo', a['g'], a['x'], a['gain'], a['stats'], a['dx'], a['dg'], a['db'], a['f'], a['n'],
              0.0, 1.0, 0.0, 1.0, 0.0, 1.0, a['ws'], a['size'], None)


@pytest.mark.parametrize('k', [dict(g=None), dict(x=None), dict(stats=None), dict(dx=None, dg=None, db=None), dict(f=0), dict(n=0),
                               dict(dx=P[0]), dict(dx=P[1]), dict(dx=P[0] - 8), dict(dx=P[1] + 124), dict(ws=P[7] + 8)])
def test_layer_norm_undo_refuses(k):
    code, msg = undo(**k)
    assert code == EINVAL and 'layerNormUndo' in msg


def test_layer_norm_undo_workspace():
    need = capi.lib().raw('mcn_layer_norm_undo_workspace_bytes')(160, 128)
    code, _ = undo(f=160, n=128, size=need - 1)
    assert code == EWORKSPACE


@pytest.mark.parametrize('p', [1.0, -0.1, 2.0, math.nan, math.inf])
def test_dropout_refuses_probability(p):
    code, msg = rc('mcn_dropout', P[0], P[1], 16, p, 1, 2, None, 0.0, 1.0, None)
    assert code == EINVAL and 'probability' in msg


def test_dropout_refuses_pointers():
    assert rc('mcn_dropout', None, P[1], 16, 0.5, 1, 2, None, 0.0, 1.0, None)[0] == EINVAL
    assert rc('mcn_dropout', P[0], None, 16, 0.5, 1, 2, None, 0.0, 1.0, None)[0] == EINVAL
    assert rc('mcn_dropout', P[0], P[0] + 16, 16, 0.5, 1, 2, None, 0.0, 1.0, None)[0] == EINVAL  # overlaps in part
    assert rc('mcn_dropout', P[0], P[1], (1 << 62) + 5, 0.5, 1, 2, None, 0.0, 1.0, None)[0] == EINVAL  # more than there is memory for
    assert rc('mcn_dropout', P[0], P[1], 0, 0.5, 1, 2, None, 0.0, 1.0, None)[0] == 0  # nothing to do
    assert rc('mcn_counter_add', None, 1, None)[0] == EINVAL


def cost(**k):
    a = dict(w=P[0], x=P[1], b=P[2], l=P[3], st=P[4], lp=P[5], ok=P[6], d=16, v=100, n=8, ws=P[7], size=BIG)
    a.update(k)
    return rc('mcn_fc_logreg_cost', a['w'], a['x'], a['b'], a['l'], a['st'], a['lp'], a['ok'], a['d'], a['v'], a['n'], None, a['ws'], a['size'], None)


def grad(**k):
    a = dict(w=P[0], x=P[1], b=P[2], l=P[3], st=P[4], dx=P[5], dw=P[6], db=P[8], d=16, v=100, n=8, ws=P[7], size=BIG)
    a.update(k)
    return rc('mcn_fc_logreg_grad', a['w'], a['x'], a['b'], a['l'], a['st'], a['dx'], a['dw'], a['db'], a['d'], a['v'], a['n'],
              1.0, 0.0, 0.0, 1.0, 0.0, 1.0, a['ws'], a['size'], None)


SIZES = [dict(d=0), dict(v=0), dict(n=0), dict(n=-5), dict(v=(1 << 24) + 1), dict(d=(1 << 20) + 1), dict(n=(1 << 20) + 1),
         dict(d=1 << 18, n=(1 << 16) + 1), dict(ws=P[7] + 4)]


@pytest.mark.parametrize('k', SIZES + [dict(w=None), dict(x=None), dict(l=None), dict(st=None), dict(lp=None), dict(ok=None)])
def test_fc_logreg_cost_refuses(k):
    code, msg = cost(**k)
    assert code == EINVAL and 'fcLogregCost' in msg


@pytest.mark.parametrize('k', SIZES + [dict(w=None), dict(x=None), dict(l=None), dict(st=None), dict(dx=None, dw=None, db=None),
                                       dict(dx=P[1]), dict(dx=P[1] + 8), dict(dx=P[4] - 4), dict(dw=P[0]), dict(dw=P[0] - 64), dict(dw=P[3] - 4),
                                       dict(db=P[2]), dict(db=P[2] + 396), dict(db=P[4] + 60)])
def test_fc_logreg_grad_refuses(k):
    code, msg = grad(**k)
    assert code == EINVAL and 'fcLogregGrad' in msg


def test_fc_logreg_workspace():
    size = capi.lib().raw('mcn_fc_logreg_workspace_bytes')
    one, both = size(160, 4213, 128, 0), size(160, 4213, 128, 1)
    assert 0 < one <= both
    assert size(160, 4213, 0, 1) == 0
    assert cost(d=160, v=4213, n=128, size=one - 1)[0] == EWORKSPACE
    assert cost(d=160, v=4213, n=128, ws=None)[0] == EWORKSPACE
    assert grad(d=160, v=4213, n=128, size=0)[0] == EWORKSPACE
    # the workspace stays far below the matrix of logits where that is large
    assert size(512, 1 << 22, 1024, 1) < 4 * (1 << 22) * 1024 / 16


def test_dropout_plain_generator_known_answers():
    """The plain generator that the GPU tests compare with, against the published vectors of Philox-4x32-10."""
    from test_head_gpu import philox_words
    got = [int(v) for v in philox_words(4, 0, 0)]
    assert got == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = (1 << 64) - 1
    got = [int(v) for v in philox_words(4, ones, ones, first_quad=ones)]
    assert got == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


NORM = dict(x=32, gain=8, bias=8, y=32, stats=8)  # floats of each operand of norm()
UNDO = dict(g=32, x=32, gain=8, stats=8, dx=32, dg=8, db=8)


def overlaps(sizes, outs, ins):
    """(pointer to move, the one it is moved over): every output against every operand and every other output."""
    return [(o, i) for o in outs for i in list(ins) + [q for q in outs if q < o]]


@pytest.mark.parametrize('end', [False, True])
@pytest.mark.parametrize('o,i', [p for p in overlaps(NORM, ('y', 'stats'), ('x', 'gain', 'bias')) if p != ('y', 'x')])
def test_layer_norm_refuses_outputs_over_operands(o, i, end):
    """A block that is ahead of the others would write what they have still to read."""
    at = dict(x=P[0], gain=P[1], bias=P[2], y=P[3], stats=P[4])
    code, msg = norm(**{o: at[i] + (NORM[i] - 1 if end else 1 - NORM[o]) * 4})
    assert code == EINVAL and 'layerNorm' in msg and 'overlap' in msg


@pytest.mark.parametrize('end', [False, True])
@pytest.mark.parametrize('o,i', overlaps(UNDO, ('dx', 'dg', 'db'), ('g', 'x', 'gain', 'stats')))
def test_layer_norm_undo_refuses_outputs_over_operands(o, i, end):
    at = dict(g=P[0], x=P[1], gain=P[2], stats=P[3], dx=P[4], dg=P[5], db=P[6])
    code, msg = undo(**{o: at[i] + (UNDO[i] - 1 if end else 1 - UNDO[o]) * 4})
    assert code == EINVAL and 'layerNormUndo' in msg and 'overlap' in msg
    assert undo(**{o: at[i]})[0] == EINVAL  # in place of one another


COST = dict(w=1600, x=128, b=100, l=8, st=16, lp=8, ok=8, out=4)
GRAD = dict(w=1600, x=128, b=100, l=8, st=16, dx=128, dw=1600, db=100)


@pytest.mark.parametrize('end', [False, True])
@pytest.mark.parametrize('o,i', overlaps(COST, ('st', 'lp', 'ok', 'out'), ('w', 'x', 'b', 'l')))
def test_fc_logreg_cost_refuses_outputs_over_operands(o, i, end):
    """The labels are read again after the log probabilities are written."""
    at = dict(w=P[0], x=P[1], b=P[2], l=P[3], st=P[4], lp=P[5], ok=P[6], out=P[8])
    at[o] = at[i] + (COST[i] - 1 if end else 1 - COST[o]) * 4
    code, msg = rc('mcn_fc_logreg_cost', at['w'], at['x'], at['b'], at['l'], at['st'], at['lp'], at['ok'], 16, 100, 8, at['out'], P[7], BIG, None)
    assert code == EINVAL and 'fcLogregCost' in msg and 'overlap' in msg


@pytest.mark.parametrize('end', [False, True])
@pytest.mark.parametrize('o,i', overlaps(GRAD, ('dx', 'dw', 'db'), ('w', 'x', 'b', 'l', 'st')))
def test_fc_logreg_grad_refuses_outputs_over_operands(o, i, end):
    at = dict(w=P[0], x=P[1], b=P[2], l=P[3], st=P[4], dx=P[5], dw=P[6], db=P[8])
    code, msg = grad(**{o: at[i] + (GRAD[i] - 1 if end else 1 - GRAD[o]) * 4})
    assert code == EINVAL and 'fcLogregGrad' in msg and 'overlap' in msg


def test_inline_assembly_names_m0_where_it_writes_it():
    """The compiler keeps values of its own in m0 (LDS copies, indexed moves): a block that writes it has to say so."""
    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'cuda-convnet_amd', 'csrc', 'kernels')
    seen = 0
    for path in glob.glob(os.path.join(kernels, '*.h*')):
        for block in re.findall(r'\basm\b[^;]*;', open(path).read()):
            if re.search(r'\bm0\s*,', block):  # (as a destination)
                seen += 1
                assert re.search(r':[^:]*"m0"[^:]*\)\s*;$', block), (os.path.basename(path), block)
    assert seen
